"""policy.clip_gradients against the formula in 64 bits. The sum of squares is taken in float64, so the norm is the exact one
rounded to float32 (2^-23 with the sum's own error) and a clipped value is off by its factor's roundings (norm, addition, division:
2^-22) and its own."""
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
gpu = pytest.mark.gpu


def make(seed, *shape, dtype=F32, std=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def formula(grads, max_norm):
    norm = math.sqrt(sum(float(g.cpu().double().pow(2).sum()) for g in grads))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def check(grads, before, outs, norm, max_norm):
    ref, factor = formula(before, max_norm)
    assert norm.dtype == F32 and norm.dim() == 0 and abs(float(norm) - ref) <= 2.0 ** -23 * ref
    for b, o in zip(before, outs):
        want = b.cpu().double() * factor
        tol = (UNIT[o.dtype] + 2.0 ** -21) * want.abs() + (2.0 ** -25 if o.dtype == F16 else 0)
        assert bool(((o.cpu().double() - want).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("sizes", [[1], [0], [5, 0, 3], [16384], [16383, 16385, 7], [1000003, 2, 70000], [33] * 300])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_in_place(sizes, dtype):
    grads = [make(i, n, dtype=dtype) for i, n in enumerate(sizes)]
    before = [g.clone() for g in grads]
    for max_norm in (0.37, 1e9, 0.0):
        norm = policy.clip_gradients(grads, max_norm)
        check(grads, before, grads, norm, max_norm)
        if max_norm > 1:
            assert all(torch.equal(g, b) for g, b in zip(grads, before))
        for g, b in zip(grads, before):
            g.copy_(b)


@gpu
def test_mixed_types_into_other_tensors():
    """Types side by side, gradients left alone, None passed over, tensors off 16-byte alignment, more than one launch's tensors."""
    kinds = [F32, BF16, F16]
    grads, outs = [], []
    for i in range(260):
        n = (i * 37) % 400 + 1
        grads.append(make(i, n + 1, dtype=kinds[i % 3])[i % 2:][:n].contiguous() if i % 5 else make(i, n + 1, dtype=kinds[i % 3])[1:])
        outs.append(torch.full((grads[-1].numel() + 3,), 7.0, device="cuda", dtype=kinds[(i // 3) % 3])[3:])
    before = [g.clone() for g in grads]
    norm = policy.clip_gradients(grads[:100] + [None] + grads[100:], 2.5, out=outs[:100] + [None] + outs[100:])
    check(grads, before, outs, norm, 2.5)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    assert torch.equal(norm, policy.clip_gradients(grads, 2.5, out=outs))


@gpu
def test_values_whose_squares_leave_float32():
    for std in (1e30, 1e-30):
        grads = [make(1, 5000, std=std), make(2, 77, std=std)]
        before = [g.clone() for g in grads]
        check(grads, before, grads, policy.clip_gradients(grads, 1.0), 1.0)


@gpu
def test_norms_that_are_not_finite():
    """What the formula gives: an infinite norm a factor of 0 (and NaN where the value is infinite), a NaN norm NaN."""
    g, h = make(1, 100), make(2, 50)
    g[3] = math.inf
    assert float(policy.clip_gradients([g, h], 1.0)) == math.inf
    assert not h.any() and torch.isnan(g[3]) and not g[:3].any()
    h[1] = math.nan
    assert math.isnan(float(policy.clip_gradients([h], 1.0))) and torch.isnan(h).all()


@gpu
def test_nothing_to_clip():
    assert float(policy.clip_gradients([], 1.0)) == 0.0 and float(policy.clip_gradients([None], 1.0)) == 0.0
    assert float(policy.clip_gradients([torch.empty(0, device="cuda")], 1.0)) == 0.0


@gpu
def test_against_torch():
    params = [torch.nn.Parameter(make(i, 100 + i)) for i in range(9)]
    for i, p in enumerate(params):
        p.grad = make(50 + i, 100 + i)
    mine = [p.grad.clone() for p in params]
    ref = torch.nn.utils.clip_grad_norm_(params, 1.5)
    norm = policy.clip_gradients(mine, 1.5)
    assert abs(float(norm) - float(ref)) <= 1e-6 * float(ref)
    for p, m in zip(params, mine):
        assert torch.allclose(p.grad, m, rtol=1e-6, atol=0)


@gpu
def test_captured_in_a_graph():
    grads, out = [make(1, 40000, dtype=BF16), make(2, 33)], [torch.empty(40000, device="cuda"), torch.empty(33, device="cuda")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        policy.clip_gradients(grads, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = policy.clip_gradients(grads, 1.0, out=out)
    for seed in range(3):
        grads[0].copy_(make(seed + 5, 40000, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        want = [o.clone() for o in out]
        assert torch.equal(policy.clip_gradients(grads, 1.0, out=out), held)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    L = abi.lib()
    one = (ctypes.c_void_p * 1)(4096)
    args = dict(count=1, grads=one, outs=one, sizes=(ctypes.c_int64 * 1)(8), types=(ctypes.c_int32 * 1)(0), out_types=(ctypes.c_int32 * 1)(0),
                max_norm=1.0, norm=4096, workspace=4096, bytes=1 << 20, stream=None)
    bad = [dict(count=-1), dict(norm=None), dict(grads=None), dict(sizes=None), dict(types=None), dict(out_types=None),
           dict(max_norm=-1.0), dict(max_norm=math.nan), dict(workspace=None), dict(workspace=4104), dict(bytes=64),
           dict(grads=(ctypes.c_void_p * 1)(None)), dict(grads=(ctypes.c_void_p * 1)(4098)), dict(sizes=(ctypes.c_int64 * 1)(-1)),
           dict(out_types=(ctypes.c_int32 * 1)(2))]
    for change in bad:
        assert L.goi_clip_gradients(*{**args, **change}.values()) == abi.GOI_E_ARG, change
    for key in ("types", "out_types"):
        assert L.goi_clip_gradients(*{**args, key: (ctypes.c_int32 * 1)(5)}.values()) == abi.GOI_E_UNSUPPORTED
    assert L.goi_clip_workspace(-1, ctypes.byref(ctypes.c_uint64())) == abi.GOI_E_ARG
    with pytest.raises(ValueError):
        policy.clip_gradients([torch.zeros(3)], 1.0)


@gpu
def test_refusals_of_the_package():
    g = make(1, 6, 4)
    for grads, out in (([g.T], None), ([g.double()], None), ([g], [g[:3]]), ([g], [g, g]), ([g], [g.cpu()])):
        with pytest.raises(ValueError):
            policy.clip_gradients(grads, 1.0, out=out)
    with pytest.raises(abi.GoiError):
        policy.clip_gradients([g], -1.0)
