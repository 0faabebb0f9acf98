"""policy.attention against the formulas in 64 bits: outputs, gradients, one step over a cache, and what it refuses.

Tolerances are element by element, from the roundings that the kernels state: with u the inputs' unit roundoff, probabilities P and
their gradients dS are rounded to the inputs' type before the second products and results once more, everything else is
float32. So |out - ref| <= u |ref| + (u + e) sum P |v|, with e for float32 (exponents of at most a few hundred: 2^-14); dS is off
by u |dS| + P (what delta is off by) + e P (|dP| + |delta| + sums of absolute products), and dq, dk, dv and dbias by the sums of
these with the other operand's absolute values. float16 adds half its smallest subnormal per rounded P and dS.
"""
import ctypes
import importlib
import math

import pytest

from util import b2

torch = pytest.importorskip("torch")
policy = b2.policy
abi = importlib.import_module(b2.__name__ + "._abi")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}  # half the smallest subnormal, where sums reach it
E32 = 2.0 ** -14
gpu = pytest.mark.gpu


def reference(q, k, v, bias=None, buckets=None, first=None, lengths=None, causal=True, scale=None, dout=None):
    """(values, tolerances) by name, float64 on the CPU, from the definition."""
    kind, bias_kind = q.dtype, None if bias is None else bias.dtype
    u, tiny = UNIT[kind], TINY[kind]
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    n, tq, h, d = q.shape
    tk, g = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    length = torch.full((n,), tk) if lengths is None else lengths.cpu().long().clamp(0, tk)
    pos = length[:, None] - tq + torch.arange(tq)
    j = torch.arange(tk)
    hi = torch.minimum(pos + 1, length[:, None]) if causal else length[:, None].expand(n, tq)
    lo = torch.zeros(n, tq, dtype=torch.long) if first is None else first.cpu().long().clamp_min(0)
    sees = (j >= lo[..., None]) & (j < hi[..., None])  # (n, tq, tk)
    seen = sees.any(1)
    zero = lambda x, keep: torch.where(keep, x, torch.zeros_like(x))  # noqa: E731
    k, v = (zero(x, seen[:, :, None, None]) for x in (k, v))  # what no query sees does not count, whatever it holds
    awake = sees.any(2)
    q = zero(q, awake[:, :, None, None])
    kk, vv = (x.repeat_interleave(h // g, 2).permute(0, 2, 1, 3) for x in (k, v))
    qq = q.permute(0, 2, 1, 3)
    s = scale * qq @ kk.mT
    if bias is not None:
        origin = 0 if causal else (buckets.numel() - 1) // 2
        at = (pos[:, :, None] - j + origin).clamp(0, buckets.numel() - 1)
        bucket = buckets.cpu().long()[at].clamp(0, bias.shape[1] - 1)  # (n, tq, tk)
        s = s + bias.detach().cpu().double()[:, bucket].transpose(0, 1)
    s = torch.where(sees[:, None], s, -math.inf)
    top = s.amax(3, keepdim=True) if tk else s.new_full((n, h, tq, 1), -math.inf)
    p = (s - top.nan_to_num(neginf=0.0)).exp()
    total = p.sum(3, keepdim=True)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    p = torch.where(total > 0, p / total, 0.0)
    out = p @ vv
    e_out = u * out.abs() + (u + E32) * (p @ vv.abs()) + tiny * vv.abs().sum(2, keepdim=True) + tiny
    back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    val, tol = {"out": back(out), "lse": lse}, {"out": back(e_out), "lse": E32 + 2.0 ** -20 * lse.abs().nan_to_num(posinf=0)}
    if dout is None:
        return val, tol
    go = zero(dout.detach().cpu().double(), awake[:, :, None, None]).permute(0, 2, 1, 3)
    dp = go @ vv.mT
    delta = (p * dp).sum(3, keepdim=True)
    ds = p * (dp - delta)
    e_delta = (go.abs() * e_out).sum(3, keepdim=True)
    size = go.abs() @ vv.abs().mT  # absolute products behind dP
    e_ds32 = p * e_delta + E32 * p * (size + (p * size).sum(3, keepdim=True))
    e_ds = (1 + u) * e_ds32 + u * ds.abs() + tiny
    group = lambda x: x.unflatten(1, (g, h // g)).sum(2)  # noqa: E731
    val["dq"], tol["dq"] = scale * ds @ kk, scale * e_ds @ kk.abs()
    val["dk"], tol["dk"] = group(scale * ds.mT @ qq), group(scale * e_ds.mT @ qq.abs())
    val["dv"], tol["dv"] = group(p.mT @ go), group(((u + E32) * p.mT + tiny) @ go.abs())
    for x in ("dq", "dk", "dv"):
        tol[x] = tol[x] * (1 + u) + u * val[x].abs() + tiny
        val[x], tol[x] = back(val[x]), back(tol[x])
    if bias is not None:
        by = [(bucket == b)[:, None] for b in range(bias.shape[1])]
        val["dbias"] = torch.stack([zero(ds, b.expand_as(ds)).sum((0, 2, 3)) for b in by], 1)
        tol["dbias"] = torch.stack([zero(e_ds32 + E32 * ds.abs(), b.expand_as(ds)).sum((0, 2, 3)) for b in by], 1) \
            + UNIT[bias_kind] * val["dbias"].abs() + TINY[bias_kind]
    return val, tol


def check(got, val, tol):
    for name, x in got.items():
        if x is None:
            continue
        x, y, e = x.detach().cpu().double(), val[name], tol[name]
        assert x.shape == y.shape, name
        fine = torch.isfinite(y)
        assert torch.equal(torch.isfinite(x), fine) and torch.equal(x[~fine], y[~fine]), name
        if not fine.any():
            continue
        over = ((x - y).abs() - 1.02 * e)[fine]
        assert over.max() <= 0, f"{name}: off by {(x - y).abs()[fine].max():.3g}, {int((over > 0).sum())} of {over.numel()} over"


def lse_of(stats):
    return (stats[..., 0].double() + stats[..., 1].double().log2()) * math.log(2.0)


def run_both(q, k, v, dout, **args):
    out, stats = policy.attention_forward(q, k, v, **args)
    dq, dk, dv, dbias = policy.attention_backward(dout, q, k, v, out, stats, **args)
    return {"out": out, "lse": lse_of(stats), "dq": dq, "dk": dk, "dv": dv, "dbias": dbias}


def tensors(n, tq, tk, h, g, d, dtype=BF16, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    make = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(dtype)  # noqa: E731
    return make(n, tq, h, d), make(n, tk, g, d), make(n, tk, g, d), make(n, tq, h, d)


def table(h, buckets=32, reach=128, dtype=BF16, seed=1, two_sided=False):
    gen = torch.Generator("cuda").manual_seed(seed)
    return dict(bias=torch.randn(h, buckets, generator=gen, device="cuda").to(dtype),
                buckets=policy.distance_buckets(buckets, reach, two_sided=two_sided))


def episodes(n, t, chance, seed=2):
    gen = torch.Generator("cuda").manual_seed(seed)
    begins = torch.rand(n, t, generator=gen, device="cuda") < chance
    at = torch.arange(t, device="cuda", dtype=torch.int32)
    return torch.where(begins, at, torch.zeros_like(at)).cummax(1).values.contiguous()


SIZES = [  # worlds, steps, heads, key heads, dim
    (1, 1, 1, 1, 8), (3, 2, 2, 1, 16), (2, 31, 4, 4, 32), (5, 32, 4, 2, 40), (2, 33, 3, 1, 64), (1, 64, 8, 1, 64),
    (2, 65, 6, 2, 72), (2, 127, 2, 2, 96), (1, 130, 5, 1, 128), (1, 257, 4, 2, 128), (1, 300, 16, 1, 32),
]


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,t,h,g,d", SIZES)
def test_windows(n, t, h, g, d, dtype):
    """Windows with episodes and a bias: odd lengths, shared heads, dims that fill no tile."""
    q, k, v, dout = tensors(n, t, t, h, g, d, dtype)
    args = dict(first=episodes(n, t, 0.05), **table(h, dtype=dtype))
    check(run_both(q, k, v, dout, **args), *reference(q, k, v, dout=dout, **args))


@gpu
@pytest.mark.parametrize("n,t,h,g,d", SIZES[1::2])
def test_windows_without_a_bias(n, t, h, g, d):
    q, k, v, dout = tensors(n, t, t, h, g, d)
    check(run_both(q, k, v, dout, scale=0.3), *reference(q, k, v, dout=dout, scale=0.3))


@gpu
@pytest.mark.parametrize("tq,tk", [(1, 1), (1, 77), (7, 50), (50, 7), (64, 200), (100, 31), (3, 0), (0, 5), (150, 140)])
@pytest.mark.parametrize("causal", [True, False])
def test_both_orders_and_lengths(tq, tk, causal):
    """More queries than keys, none of either, ragged lengths past both ends, a two-sided bias, a float32 bias."""
    n, h, g, d = 6, 6, 3, 48
    q, k, v, dout = tensors(n, tq, tk, h, g, d)
    lengths = torch.tensor([0, 1, tk // 2, tk - 1, tk, tk + 9], dtype=torch.int32, device="cuda")
    args = dict(lengths=lengths, causal=causal, **table(h, 20, 24, F32, two_sided=not causal))
    check(run_both(q, k, v, dout, **args), *reference(q, k, v, dout=dout, **args))


@gpu
@pytest.mark.parametrize("waves", [1, 2, 4])
def test_rows_without_keys(waves):
    """Rows whose mask leaves nothing, whole worlds of them, and NaN and infinities wherever nobody looks."""
    n, t, h, g, d = 4, 32 * waves - 5, 2, 2, 64
    q, k, v, dout = tensors(n, t, t, h, g, d)
    first = episodes(n, t, 0.1)
    first[1] = t           # a world that is over
    first[2, t // 2:] = t  # one that ends inside the window
    first[3] = torch.arange(t, device="cuda") + 1  # every step starts after itself
    first[0] = -5
    args = dict(first=first, **table(h))
    val, tol = reference(q, k, v, dout=dout, **args)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=BF16).repeat(64)[:d]
    for x in (q, dout):
        x[1], x[3] = bad, bad
        x[2, t // 2:] = bad
    for x in (k, v):
        x[1], x[3] = bad, bad
        x[2, t // 2:] = bad
    got = run_both(q, k, v, dout, **args)
    check(got, val, tol)
    for name in ("out", "dq", "dk", "dv"):
        assert not got[name][1].any() and not got[name][3].any(), name


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("t", [30, 100])
def test_values_that_only_some_rows_see(t, d, bad):
    """A broken episode (values that are not finite) shares tiles with a sound one: it reaches the rows and keys of its own
    episode only."""
    n, h, g = 2, 4, 2
    q, k, v, dout = tensors(n, t, t, h, g, d)
    cut = t // 2 + 3
    first = torch.zeros(n, t, dtype=torch.int32, device="cuda")
    first[0, cut:] = cut
    args = dict(first=first, **table(h))
    clean = [x.clone() for x in (q, k, v, dout)]
    for x in clean:
        x[0, :cut] = 0
    val, tol = reference(*clean[:3], dout=clean[3], **args)
    q[0, 5, :, 3] = bad
    k[0, 9, :, 1] = bad
    v[0, 7, :, 2] = bad
    dout[0, 11, :, 4] = bad
    got = run_both(q, k, v, dout, **args)
    assert not torch.isfinite(got["out"][0, 5]).any() and not torch.isfinite(got["out"][0, 7:cut, :, 2]).any()
    for name in ("out", "dq", "dk", "dv"):
        check({name: got[name][0, cut:]}, {name: val[name][0, cut:]}, {name: tol[name][0, cut:]})
        check({name: got[name][1]}, {name: val[name][1]}, {name: tol[name][1]})
        if name != "out":
            assert not torch.isfinite(got[name][0, :cut].float()).all(), name
    one_step = policy.attention(q[:, -1:], k, v, first=first[:, -1:].contiguous(), **table(h))
    check({"out": one_step}, {"out": val["out"][:, -1:]}, {"out": tol["out"][:, -1:]})


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,tk,h,g,d", [(1, 1, 4, 1, 64), (3, 60, 8, 2, 64), (40, 130, 4, 4, 32), (2, 5000, 8, 1, 128),
                                        (1, 40000, 16, 2, 64), (5, 700, 12, 4, 80)])
def test_one_step_over_a_cache(n, tk, h, g, d, dtype):
    """Acting: one query a world, ragged histories, the key axis split where worlds are few; the cache past a world's history
    is never looked at."""
    q, k, v, _ = tensors(n, 1, tk, h, g, d, dtype)
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, tk + 1, (n,), generator=gen, dtype=torch.int32)
    lengths[-1] = tk
    for w in range(n):
        k[w, lengths[w]:] = math.nan
        v[w, lengths[w]:] = math.inf
    args = dict(lengths=lengths.cuda(), **table(h, dtype=dtype))
    val, tol = reference(q, k, v, **args)
    out, stats = policy.attention_forward(q, k, v, **args)
    check({"out": out, "lse": lse_of(stats)}, val, tol)
    assert torch.equal(out, policy.attention(q, k, v, **args))


@gpu
def test_strides_and_alignment():
    """Views of one projection, a cache with its heads outside its steps, expanded worlds, rows off 16-byte alignment."""
    n, t, h, g, d = 3, 45, 4, 2, 64
    gen = torch.Generator("cuda").manual_seed(5)
    joint = torch.randn(n, t, (h + 2 * g) * d, generator=gen, device="cuda").to(BF16)
    q, k, v = joint.split([h * d, g * d, g * d], 2)
    q, k, v = q.unflatten(2, (h, d)), k.unflatten(2, (g, d)), v.unflatten(2, (g, d))
    dout = torch.randn(t, n, h, d, generator=gen, device="cuda").to(BF16).transpose(0, 1)
    by_head = torch.randn(n, g, t, d, generator=gen, device="cuda").to(BF16).transpose(1, 2)
    shared = torch.randn(1, t, g, d, generator=gen, device="cuda").to(BF16).expand(n, t, g, d)
    off = torch.randn(n * t * g * d + 1, generator=gen, device="cuda").to(BF16)[1:].view(n, t, g, d)
    strided = torch.randn(n, t, g, 2 * d, generator=gen, device="cuda").to(BF16)[..., ::2]
    args = table(h)
    for kk, vv in ((k, v), (by_head, v), (shared, by_head), (off, shared), (strided, off)):
        check(run_both(q, kk, vv, dout, **args), *reference(q, kk, vv, dout=dout, **args))


@gpu
@pytest.mark.parametrize("low", [torch.finfo(BF16).min, -math.inf])
def test_bias_as_a_mask(low):
    """Buckets of the type's lowest value or minus infinity: alone in a row the lowest value is a row of equal scores, minus
    infinity a row that sees nothing."""
    n, t, h, g, d = 2, 70, 2, 1, 64
    q, k, v, dout = tensors(n, t, t, h, g, d)
    args = table(h, 16, 40)
    args["bias"][0, :8] = low
    args["bias"][1, 8:] = low
    first = torch.zeros(n, t, dtype=torch.int32, device="cuda")
    first[1] = torch.arange(t, device="cuda")
    val, tol = reference(q, k, v, dout=dout, first=first, **args)
    got = run_both(q, k, v, dout, first=first, **args)
    if low != -math.inf:  # lse of a row of lowest values alone: that value, which float32 holds in powers of two to 1.7e38
        keep = val["lse"] > -1e30
        got["lse"], val["lse"], tol["lse"] = got["lse"].cpu()[keep], val["lse"][keep], tol["lse"][keep]
    check(got, val, tol)


@gpu
def test_gradients_against_differences():
    """The slope of sum(dout * out) along random directions, from the definition in 64 bits, against the kernels' gradients."""
    n, t, h, g, d = 2, 40, 4, 2, 32
    q, k, v, dout = tensors(n, t, t, h, g, d, F16)
    args = dict(first=episodes(n, t, 0.1), **table(h, dtype=F16))
    got = run_both(q, k, v, dout, **args)
    _, tol = reference(q, k, v, dout=dout, **args)
    gen = torch.Generator().manual_seed(9)
    at = {"dq": q, "dk": k, "dv": v, "dbias": args["bias"]}

    def loss(name, direction, step):
        moved = {x: (y.cpu().double() + (step * direction if x == name else 0.0)) for x, y in at.items()}
        rest = dict(first=args["first"], buckets=args["buckets"], bias=_Exact(moved["dbias"]))
        value, _ = reference(_Exact(moved["dq"]), _Exact(moved["dk"]), _Exact(moved["dv"]), **rest)
        return float((value["out"] * dout.cpu().double()).sum())

    for name, x in at.items():
        direction = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        slope = (loss(name, direction, 1e-4) - loss(name, direction, -1e-4)) / 2e-4
        along = float((got[name].cpu().double() * direction).sum())
        assert abs(along - slope) <= float((tol[name] * direction.abs()).sum()) + 1e-5 * abs(slope), name


class _Exact:
    """A float64 tensor with what reference() asks of an input of the operators."""

    def __init__(self, x):
        self.x, self.dtype, self.shape = x, F16, x.shape

    def detach(self):
        return self

    def cpu(self):
        return self

    def double(self):
        return self.x


@gpu
def test_autograd():
    """attention() under autograd gives attention_backward's gradients, and no gradient where none is asked."""
    n, t, h, g, d = 2, 50, 4, 2, 32
    q, k, v, dout = tensors(n, t, t, h, g, d)
    args = dict(first=episodes(n, t, 0.1), **table(h))
    want = run_both(q, k, v, dout, **args)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, args["bias"])]
    out = policy.attention(*leaves, buckets=args["buckets"], first=args["first"])
    out.backward(dout)
    assert torch.equal(out, want["out"])
    for x, name in zip(leaves, ("dq", "dk", "dv", "dbias")):
        assert torch.equal(x.grad, want[name]), name
    assert policy.attention(q, k, v).grad_fn is None


@gpu
def test_same_bits_every_time_and_on_another_stream():
    n, t, h, g, d = 8, 200, 8, 2, 64
    q, k, v, dout = tensors(n, t, t, h, g, d)
    args = dict(first=episodes(n, t, 0.02), **table(h))
    want = run_both(q, k, v, dout, **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            again = run_both(q, k, v, dout, **args)
        stream.synchronize()
        for name in want:
            assert torch.equal(want[name], again[name]), name


@gpu
def test_captured_in_a_graph():
    """Forward, backward and a split step replayed from a graph, with eager work between, give the eager results."""
    n, t, h, g, d = 3, 90, 4, 2, 64
    q, k, v, dout = tensors(n, t, t, h, g, d)
    step, cache_k, cache_v, _ = tensors(1, 1, 3000, h, g, d, seed=7)
    args = dict(first=episodes(n, t, 0.05), **table(h))

    def work():
        return [*run_both(q, k, v, dout, **args).values(), policy.attention(step, cache_k, cache_v)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for seed in range(3):
        fresh = tensors(n, t, t, h, g, d, seed=20 + seed)
        for x, y in zip((q, k, v, dout), fresh):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, work()):
            assert torch.equal(x, y)


def test_distance_buckets():
    """Whole and monotone: one bucket each below half, geometric ranges, the last from the reach on; both directions."""
    m = policy.distance_buckets(32, 128, device="cpu").tolist()
    assert len(m) == 129 and m[:16] == list(range(16)) and m[127] == 31 and m[128] == 31
    assert all(0 <= b - a <= 1 for a, b in zip(m, m[1:])) and set(m) == set(range(32))
    assert policy.distance_buckets(8, 4, device="cpu").tolist() == [0, 1, 2, 3, 7]
    two = policy.distance_buckets(8, 6, two_sided=True, device="cpu")
    one = policy.distance_buckets(4, 6, device="cpu")
    assert two.tolist() == [int(b) + 4 for b in one.flip(0)[:-1]] + one.tolist()
    for bad in ((1, 5), (16, 4)):
        with pytest.raises(ValueError):
            policy.distance_buckets(*bad, device="cpu")


def _call(name, **fields):
    a = abi.GoiAttention()
    a.n_worlds, a.q_steps, a.k_steps, a.heads, a.kv_heads, a.dim, a.type, a.causal, a.scale = 2, 8, 8, 4, 2, 64, abi.BF16, 1, 0.1
    for key in ("q", "k", "v", "out", "dout", "dq", "dk", "dv", "stats"):
        setattr(a, key, 4096)  # never reached: every call below is refused on the host
    for key, value in fields.items():
        setattr(a, key, value)
    L = abi.lib()
    return getattr(L, name)(ctypes.byref(a), None, 0, None), L.goi_last_error().decode()


@pytest.mark.parametrize("fields,code,text", [
    (dict(dim=12), abi.GOI_E_UNSUPPORTED, "dim 12"), (dict(dim=136), abi.GOI_E_UNSUPPORTED, "dim 136"),
    (dict(dim=0), abi.GOI_E_UNSUPPORTED, "dim 0"), (dict(type=abi.F32), abi.GOI_E_UNSUPPORTED, "bf16"),
    (dict(heads=3), abi.GOI_E_SHAPE, "multiple"), (dict(n_worlds=-1), abi.GOI_E_ARG, "negative"),
    (dict(kv_heads=0), abi.GOI_E_ARG, "no heads"), (dict(q=None), abi.GOI_E_ARG, "null"), (dict(v=4104), abi.GOI_E_ARG, "misaligned"),
    (dict(k_strides=(4, 8, 8)), abi.GOI_E_ARG, "misaligned"), (dict(bias=4096), abi.GOI_E_ARG, "buckets"),
    (dict(bias=4096, buckets=4096, n_buckets=65, n_distances=9, bias_type=abi.BF16), abi.GOI_E_UNSUPPORTED, "65|buckets"),
    (dict(bias=4096, buckets=4096, n_buckets=9, n_distances=4000, bias_type=abi.BF16), abi.GOI_E_UNSUPPORTED, "6144"),
    (dict(bias=4096, buckets=4096, n_buckets=9, n_distances=9, bias_type=abi.F16), abi.GOI_E_UNSUPPORTED, "16-bit"),
    (dict(bias=4096, buckets=4096, n_buckets=9, n_distances=8, causal=0), abi.GOI_E_SHAPE, "both directions"),
    (dict(q_steps=1 << 30, heads=8), abi.GOI_E_UNSUPPORTED, "31 bits"),
    (dict(q_steps=1, k_steps=1 << 20), abi.GOI_E_ARG, "workspace"),
])
def test_refusals_of_the_library(fields, code, text):
    import re
    if fields.get("bias") and "bias_type" not in fields:
        fields = dict(fields, bias_type=abi.BF16)
    got, message = _call("goi_attention_forward", **{k: abi._I64x3(*v) if isinstance(v, tuple) else v for k, v in fields.items()})
    assert got == code and re.search(text, message), (got, message)


def test_refusals_of_the_backward_call():
    assert _call("goi_attention_backward", dout=None)[0] == abi.GOI_E_ARG
    assert _call("goi_attention_backward", stats=None)[0] == abi.GOI_E_ARG
    code, message = _call("goi_attention_backward")
    assert code == abi.GOI_E_ARG and "workspace" in message
    L = abi.lib()
    assert L.goi_attention_workspace(None, 0, ctypes.byref(ctypes.c_uint64())) == abi.GOI_E_ARG
    assert L.goi_attention_workspace(ctypes.byref(abi.GoiAttention()), 0, None) == abi.GOI_E_ARG


def test_refusals_without_a_gpu_tensor():
    x = torch.zeros(1, 2, 2, 8, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        policy.attention(x, x, x)


@gpu
def test_refusals_of_the_package():
    q, k, v, dout = tensors(2, 8, 8, 4, 2, 64)
    t = table(4)
    bad = [dict(v=v[:, :4]), dict(k=k[:1], v=v[:1]), dict(q=q.float()), dict(q=q.half()), dict(q=q[0]),
           dict(first=torch.zeros(2, 7, dtype=torch.int32, device="cuda")), dict(first=torch.zeros(2, 8, device="cuda")),
           dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(bias=t["bias"]),
           dict(bias=t["bias"][:2], buckets=t["buckets"]), dict(bias=t["bias"].half(), buckets=t["buckets"]),
           dict(bias=t["bias"], buckets=t["buckets"].long()), dict(k=k.cpu(), v=v.cpu())]
    for change in bad:
        with pytest.raises(ValueError):
            policy.attention(**{**dict(q=q, k=k, v=v), **change})
    out, stats = policy.attention_forward(q, k, v)
    for o, l, g in ((out[:1], stats, dout), (out, stats.half(), dout), (out, stats[:1], dout), (out, stats, dout.float())):
        with pytest.raises(ValueError):
            policy.attention_backward(g, q, k, v, o, l)
    with pytest.raises(abi.GoiError) as e:
        policy.attention(torch.zeros(1, 2, 2, 12, dtype=BF16, device="cuda"), *[torch.zeros(1, 2, 2, 12, dtype=BF16, device="cuda")] * 2)
    assert e.value.code == abi.GOI_E_UNSUPPORTED


def test_library_exports_the_policy_operators():
    """Every function that include/goi_policy.h declares is in the library and bound."""
    import re
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "goi_policy.h"
    names = re.findall(r"^\S.*?\b(goi_[a-z0-9_]+)\s*\(", header.read_text(), re.M)
    assert set(names) == set(abi.POLICY_EXPORTS)
    for name in names:
        assert hasattr(abi.lib(), name), name
