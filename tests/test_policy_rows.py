"""policy.rms_norm (with the residual, its gradient, and in 8 bits) and policy.linear_int8 against the formulas in 64 bits.

Tolerances, with u the unit roundoff of the type a result is rounded to: a row's sum is taken in float32, 32 elements a
thread and then pairwise, so 1 / sqrt(mean) is off by less than (32 + 16) 2^-24 < 2^-18 of itself and everything computed from it by
2^-17 of the absolute values that enter; sums over rows by (rows + 100) 2^-24 more. Integer sums are exact.
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
TINY = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}
E = 2.0 ** -17
gpu = pytest.mark.gpu

WIDTHS = [1, 2, 7, 8, 65, 200, 256, 257, 512, 1000, 1533, 2048, 2052, 4100, 32768]


def near(x, y, tol, name=""):
    x, tol = x.detach().cpu().double(), tol + 0 * y
    assert x.shape == y.shape, name
    fine = torch.isfinite(y)
    assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(torch.isfinite(x), fine), name
    over = ((x - y).abs() - tol)[fine]
    assert not over.numel() or over.max() <= 0, f"{name}: off by {(x - y).abs()[fine].max():.3g}, {int((over > 0).sum())} over"


def make(seed, *shape, dtype=F32, std=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def formula(x, weight, residual, eps=1e-6):
    r = x if residual is None else (x.float() + residual.float()).to(x.dtype)  # the stream is held in its type
    rd = r.cpu().double()
    inv = 1 / (rd.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return r, rd, inv, rd * inv * weight.cpu().double()


@gpu
@pytest.mark.parametrize("dtype,weight_dtype", [(BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 37])
def test_norm_and_gradient(rows, width, dtype, weight_dtype):
    x, res, dy, dres = (make(i, rows, width, dtype=dtype) for i in range(4))
    res = (res.float() * 3).to(dtype)
    weight = make(9, width, dtype=weight_dtype)
    y, r, inv = policy.rms_norm_forward(x, weight, res)
    r_ref, rd, inv_ref, y_ref = formula(x, weight, res)
    assert torch.equal(r, r_ref)
    near(inv, inv_ref[:, 0], E * inv_ref[:, 0], "inv")
    u, tiny = UNIT[dtype], TINY[dtype]
    near(y, y_ref, (u + E) * y_ref.abs() + tiny, "y")
    dx, dw = policy.rms_norm_backward(dy, r, weight, inv, dres)
    g = dy.cpu().double() * weight.cpu().double()
    dx_ref = inv_ref * g - rd * inv_ref ** 3 * (g * rd).mean(1, keepdim=True) + dres.cpu().double()
    size = inv_ref * g.abs() + rd.abs() * inv_ref ** 3 * (g * rd).abs().mean(1, keepdim=True) + dres.cpu().double().abs()
    near(dx, dx_ref, u * dx_ref.abs() + 4 * E * size + tiny, "dx")
    each = dy.cpu().double() * rd * inv_ref
    near(dw, each.sum(0), UNIT[weight_dtype] * each.sum(0).abs() + (E + (rows + 100) * 2.0 ** -24) * each.abs().sum(0)
         + TINY[weight_dtype], "dweight")


@gpu
def test_norm_without_a_residual_and_many_rows():
    x, weight, dy = make(1, 5000, 96, dtype=BF16), make(2, 96, dtype=BF16), make(3, 5000, 96, dtype=BF16)
    y, r, inv = policy.rms_norm_forward(x, weight, eps=1e-3)
    _, rd, inv_ref, y_ref = formula(x, weight, None, 1e-3)
    assert r is x
    near(y, y_ref, (UNIT[BF16] + E) * y_ref.abs())
    dx, dw = policy.rms_norm_backward(dy, r, weight, inv)
    each = dy.cpu().double() * rd * inv_ref
    near(dw, each.sum(0), UNIT[BF16] * each.sum(0).abs() + (E + 5100 * 2.0 ** -24) * each.abs().sum(0))
    again = policy.rms_norm_backward(dy, r, weight, inv)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@gpu
def test_norm_gradient_against_differences():
    """The slope of a random functional of y and r along random directions, from the definition in 64 bits."""
    x, weight, res = make(1, 5, 33), make(2, 33), make(3, 5, 33)
    cy, cr = make(4, 5, 33).cpu().double(), make(5, 5, 33).cpu().double()
    leaves = [t.clone().requires_grad_() for t in (x, weight, res)]
    y, r = policy.rms_norm(leaves[0], leaves[1], leaves[2])
    ((y * cy.cuda().float()).sum() + (r * cr.cuda().float()).sum()).backward()

    def loss(x, weight, res):
        s = x + res
        return float((s / (s.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * weight * cy).sum() + (s * cr).sum())

    at = [t.cpu().double() for t in (x, weight, res)]
    gen = torch.Generator().manual_seed(6)
    for i in range(3):
        d = torch.randn(at[i].shape, generator=gen, dtype=torch.float64)
        up, down = (loss(*[t + (h * d if j == i else 0) for j, t in enumerate(at)]) for h in (1e-5, -1e-5))
        slope, along = (up - down) / 2e-5, float((leaves[i].grad.cpu().double() * d).sum())
        assert abs(slope - along) <= 1e-4 * float((leaves[i].grad.cpu().double().abs() * d.abs()).sum()), i


@gpu
def test_norm_autograd_uses():
    """Only r used, only y used, no graph asked for, and no residual."""
    x, weight, res = make(1, 4, 40), make(2, 40), make(3, 4, 40)
    a, b = x.clone().requires_grad_(), res.clone().requires_grad_()
    _, r = policy.rms_norm(a, weight, b)
    r.sum().backward()
    assert torch.equal(a.grad, torch.ones_like(x)) and torch.equal(b.grad, torch.ones_like(x))
    c = x.clone().requires_grad_()
    policy.rms_norm(c, weight).sum().backward()
    y, r, inv = policy.rms_norm_forward(x, weight)
    assert torch.equal(c.grad, policy.rms_norm_backward(torch.ones_like(y), r, weight, inv)[0])
    assert policy.rms_norm(x, weight).grad_fn is None


@gpu
def test_norm_strides_and_shapes():
    """Rows of a wider buffer, rows off alignment, columns that are not contiguous, leading axes, nothing at all."""
    wide, weight = make(1, 12, 200, dtype=BF16), make(2, 64, dtype=BF16)
    for x in (wide[:, 8:72], wide[:, 3:67], wide[:, 1:129:2], wide[::2, 10:74], wide[:1, 4:68]):
        y, r, _ = policy.rms_norm_forward(x, weight, x)
        r_ref, _, _, y_ref = formula(x, weight, x)
        assert torch.equal(r, r_ref)
        near(y, y_ref, (UNIT[BF16] + E) * y_ref.abs())
    x = make(3, 2, 3, 5, 64, dtype=BF16)
    y, r = policy.rms_norm(x, weight, x)
    assert y.shape == x.shape and torch.equal(y.flatten(0, 2), policy.rms_norm(x.flatten(0, 2), weight, x.flatten(0, 2))[0])
    assert torch.equal(policy.rms_norm(x[0, 0, 0], weight), policy.rms_norm(x, weight)[0, 0, 0])
    none = x[:0]
    y, r, inv = policy.rms_norm_forward(none, weight)
    dx, dw = policy.rms_norm_backward(none, r, weight, inv)
    assert y.shape == none.shape and dx.shape == none.shape and not dw.any()
    assert policy.rms_norm_int8(none, weight)[0].shape == none.shape


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_in_8_bits(width, dtype):
    """Values within half a step of the norm, the largest of each row at 127, scales as defined; zeros, and rows so small that
    the scale has no inverse in float32."""
    x, res, weight = make(1, 19, width, dtype=dtype), make(2, 19, width, dtype=dtype), make(3, width, dtype=F32)
    x[4], res[4] = 0, 0
    if dtype != F16:
        x[5], res[5] = (x[5].float() * 1e-38).to(dtype), 0
    values, scales, r = policy.rms_norm_int8(x, weight, res)
    r_ref, _, _, y = formula(x, weight, res)
    assert torch.equal(r, r_ref) and values.dtype == torch.int8
    top = y.abs().amax(1)
    near(scales, torch.where(top > 0, top / 127, 1.0), E * top + 2.0 ** -149)
    v, s = values.cpu().double(), scales.cpu().double()[:, None]
    near(v * s, y, s * (0.5 + 127 * E) + E * y.abs())
    assert bool(((v.abs().amax(1) == 127) | (top < 2.0 ** -130)).all())


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_that_are_not_finite(bad):
    """A value that is not finite gives its row a scale of NaN (and NaN products), and no other row."""
    x, weight = make(1, 6, 130, dtype=BF16), make(2, 130, dtype=BF16)
    x[2, 77] = bad
    values, scales, _ = policy.rms_norm_int8(x, weight)
    assert torch.isnan(scales).tolist() == [False, False, True, False, False, False]
    w, ws = policy.quantize_weight(make(3, 20, 130))
    y = policy.linear_int8(values, scales, w, ws)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4, 5]]).all()
    y = policy.rms_norm(x, weight)
    assert torch.isnan(y[2, 77]) and torch.isfinite(y[[0, 1, 3, 4, 5]]).all()


# ---------------------------------------------------------------- the product


def ints(seed, *shape):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=gen, device="cuda", dtype=torch.int8)


def check_product(x, xs, w, ws, bias, dtype):
    y = policy.linear_int8(x, xs, w, ws, bias, dtype=dtype)
    exact = (x.cpu().double() @ w.cpu().double().T) * xs.cpu().double()[..., None] * ws.cpu().double()
    ref = exact + (0 if bias is None else bias.cpu().double())
    past = 65520 if dtype == F16 else math.inf  # what rounds to infinity
    ref = torch.where(ref.abs() >= past, ref.sign() * math.inf, ref)
    # the sum as a float, two products and an addition: four roundings of float32
    near(y, ref, UNIT[dtype] * ref.abs() + 2.0 ** -21 * (exact.abs() + (0 if bias is None else bias.cpu().double().abs()))
         + TINY[dtype])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,channels,width", [
    (1, 1, 1), (1, 33, 15), (2, 16, 16), (3, 300, 17), (16, 100, 100), (17, 64, 520), (31, 5, 64), (33, 130, 1000),
    (64, 257, 130), (65, 65, 127), (100, 1, 129), (129, 200, 300), (1000, 31, 640), (257, 4100, 256), (4097, 1030, 144)])
def test_product(rows, channels, width, dtype):
    x, w = ints(1, rows, width), ints(2, channels, width)
    xs, ws = make(3, rows).abs() * 1e-2, make(4, channels).abs() * 1e-2
    check_product(x, xs, w, ws, make(5, channels, dtype=dtype), dtype)
    check_product(x, xs, w, ws, None, dtype)


@gpu
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_product_of_views(rows):
    """Rows of wider buffers (on and off 16 bytes), leading axes, a float32 bias with a 16-bit result."""
    x, w = ints(1, rows, 400), ints(2, 77, 400)
    xs, ws, bias = make(3, rows).abs(), make(4, 77).abs(), make(5, 77)
    for cut in (slice(16, 316), slice(5, 205), slice(0, 399, 3)):
        check_product(x[:, cut], xs, w[:, cut], ws, bias, F16 if cut.start else BF16)
    y = policy.linear_int8(x, xs, w, ws)
    assert torch.equal(policy.linear_int8(x.view(1, rows, 400), xs[None], w, ws)[0], y)
    assert torch.equal(policy.linear_int8(x[0], xs[0], w, ws), policy.linear_int8(x[:1], xs[:1], w, ws)[0])
    assert policy.linear_int8(x[:0], xs[:0], w, ws).shape == (0, 77)
    assert policy.linear_int8(x, xs, w[:0], ws[:0]).shape == (rows, 0)


@gpu
@pytest.mark.parametrize("rows", [1, 70])
def test_product_at_the_ends_of_the_range(rows):
    """The widest row of the lowest values: the largest sum there is, 131071 * 2^14, stays within 32 bits."""
    x = torch.full((rows, 131071), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(rows, device="cuda")
    y = policy.linear_int8(x, one, x[:1].repeat(3, 1), one[:1].repeat(3), dtype=F32)
    assert bool((y == float(torch.tensor(131071 * 16384, dtype=torch.float32))).all())


@gpu
def test_quantized_layer():
    """The two together against the layer in 64 bits: off by the half steps of both roundings at most."""
    x, res, gain = make(1, 70, 384, dtype=BF16), make(2, 70, 384, dtype=BF16), make(3, 384, dtype=BF16)
    weight = make(4, 90, 384, std=0.05)
    values, scales, _ = policy.rms_norm_int8(x, gain, res)
    w, ws = policy.quantize_weight(weight)
    y = policy.linear_int8(values, scales, w, ws, dtype=F32)
    _, _, _, n = formula(x, gain, res)
    wd, s, t = weight.cpu().double(), scales.cpu().double()[:, None], ws.cpu().double()
    ref = n @ wd.T
    bound = 0.51 * s * wd.abs().sum(1) + 0.51 * n.abs().sum(1, keepdim=True) * t + 0.27 * 384 * s * t
    near(y, ref, bound + 1e-4 * ref.abs())


@gpu
def test_captured_in_a_graph():
    x, weight, w = make(1, 300, 96, dtype=BF16), make(2, 96, dtype=BF16), make(3, 50, 96)
    w, ws = policy.quantize_weight(w)

    def work():
        y, r, inv = policy.rms_norm_forward(x, weight, x)
        values, scales, _ = policy.rms_norm_int8(x, weight, x)
        return [y, *policy.rms_norm_backward(y, r, weight, inv, x), policy.linear_int8(values, scales, w, ws)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for seed in range(3):
        x.copy_(make(20 + seed, 300, 96, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, work()):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- refusals


def refused(name, struct, **fields):
    a = struct()
    for key, value in fields.items():
        setattr(a, key, value)
    L = abi.lib()
    extra = (None, 0, None) if name == "goi_rms_norm_backward" else (None,)
    return getattr(L, name)(ctypes.byref(a), *extra), L.goi_last_error().decode()


NORM = dict(rows=2, width=64, type=abi.BF16, weight_type=abi.BF16, x=4096, weight=4096, y=4096, x_stride=64, y_stride=64)
BACK = dict(rows=2, width=64, type=abi.BF16, weight_type=abi.BF16, dy=4096, r=4096, weight=4096, inv=4096, dx=4096, dweight=4096)
INT8 = dict(rows=2, channels=3, width=64, type=abi.BF16, x=4096, w=4096, x_scales=4096, w_scales=4096, y=4096, x_stride=64,
            w_stride=64, y_stride=3)


@pytest.mark.parametrize("name,struct,base,change,code", [
    ("goi_rms_norm", abi.GoiNorm, NORM, dict(rows=-1), abi.GOI_E_ARG), ("goi_rms_norm", abi.GoiNorm, NORM, dict(width=0), abi.GOI_E_ARG),
    ("goi_rms_norm", abi.GoiNorm, NORM, dict(width=32769), abi.GOI_E_UNSUPPORTED),
    ("goi_rms_norm", abi.GoiNorm, NORM, dict(type=7), abi.GOI_E_UNSUPPORTED),
    ("goi_rms_norm", abi.GoiNorm, NORM, dict(weight_type=abi.F16), abi.GOI_E_UNSUPPORTED),
    ("goi_rms_norm", abi.GoiNorm, NORM, dict(x=None), abi.GOI_E_ARG), ("goi_rms_norm", abi.GoiNorm, NORM, dict(y=None), abi.GOI_E_ARG),
    ("goi_rms_norm", abi.GoiNorm, NORM, dict(values=4096), abi.GOI_E_ARG),
    ("goi_rms_norm", abi.GoiNorm, NORM, dict(residual=4096), abi.GOI_E_ARG),
    ("goi_rms_norm_backward", abi.GoiNormBackward, BACK, dict(dweight=None), abi.GOI_E_ARG),
    ("goi_rms_norm_backward", abi.GoiNormBackward, BACK, dict(inv=None), abi.GOI_E_ARG),
    ("goi_rms_norm_backward", abi.GoiNormBackward, BACK, dict(), abi.GOI_E_ARG),  # no workspace
    ("goi_linear_int8", abi.GoiInt8, INT8, dict(width=131072), abi.GOI_E_UNSUPPORTED),
    ("goi_linear_int8", abi.GoiInt8, INT8, dict(width=0), abi.GOI_E_ARG), ("goi_linear_int8", abi.GoiInt8, INT8, dict(rows=-2), abi.GOI_E_ARG),
    ("goi_linear_int8", abi.GoiInt8, INT8, dict(x=4104), abi.GOI_E_ARG), ("goi_linear_int8", abi.GoiInt8, INT8, dict(w_stride=72), abi.GOI_E_ARG),
    ("goi_linear_int8", abi.GoiInt8, INT8, dict(y=None), abi.GOI_E_ARG), ("goi_linear_int8", abi.GoiInt8, INT8, dict(type=9), abi.GOI_E_UNSUPPORTED),
    ("goi_linear_int8", abi.GoiInt8, INT8, dict(bias=4096, bias_type=abi.F16), abi.GOI_E_UNSUPPORTED),
])
def test_refusals_of_the_library(name, struct, base, change, code):
    got, message = refused(name, struct, **{**base, **change})
    assert got == code and message.startswith(name), (got, message)


@gpu
def test_refusals_of_the_package():
    x, w = make(1, 4, 64, dtype=BF16), make(2, 64, dtype=BF16)
    for args in ((x, w[:32]), (x, w.half()), (x.double(), w), (x, w, x[:2]), (x, w, x.float()), (x.cpu(), w)):
        with pytest.raises(ValueError):
            policy.rms_norm(*args)
    y, r, inv = policy.rms_norm_forward(x, w)
    for dy, i in ((y[:2], inv), (y.float(), inv), (y, inv[:2]), (y, inv.half())):
        with pytest.raises(ValueError):
            policy.rms_norm_backward(dy, r, w, i)
    v, s, _ = policy.rms_norm_int8(x, w)
    q, qs = policy.quantize_weight(make(3, 10, 64))
    bad = [(v.float(), s, q, qs), (v, s[:2], q, qs), (v, s.half(), q, qs), (v, s, q[:, :32], qs), (v, s, q, qs[:5]),
           (v, s, q, qs, make(4, 9)), (v, s, q, qs, make(4, 10, dtype=F16)), (v, s.cpu(), q, qs)]
    for args in bad:
        with pytest.raises(ValueError):
            policy.linear_int8(*args)
    with pytest.raises(ValueError):
        policy.linear_int8(v, s, q, qs, dtype=torch.float64)


def test_quantize_weight():
    """Each channel's largest magnitude at 127, zeros kept, on any device."""
    w = torch.tensor([[1.0, -2.0, 0.5], [0.0, 0.0, 0.0], [3e-40, 0.0, 0.0]])
    q, s = policy.quantize_weight(w)
    assert q[0].tolist() == [64, -127, 32] and q[1].tolist() == [0, 0, 0] and s[1] == 1.0
    assert abs(float(s[0]) - 2 / 127) < 1e-8
    with pytest.raises(ValueError):
        policy.quantize_weight(w[0])
