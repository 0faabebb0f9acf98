"""policy.attention's outputs and dq carry the rounding of the result alone.

P and dS go into the second products in two parts, the value rounded to the inputs' type (u) and what that left, rounded in its turn:
u^2 of the value. So |out - ref| <= u |ref| + (u^2 + e) sum P |v|, with e for float32, where one part would give u sum P |v|; dS adds
what delta is off by, which comes from out. float16 adds half its smallest subnormal for each rest.
"""
import pytest
from test_policy_attention import BF16, E32, F16, TINY, UNIT, episodes, policy, reference, table, tensors, torch

SIZES = [(1, 1, 1, 1, 8), (3, 100, 4, 2, 64), (2, 30, 4, 4, 32), (2, 257, 4, 2, 128), (1, 1100, 6, 2, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,t,h,g,d", SIZES)
def test_windows_are_rounded_once(n, t, h, g, d, dtype):
    u, tiny = UNIT[dtype], TINY[dtype]
    q, k, v, dout = tensors(n, t, t, h, g, d, dtype)
    args = dict(first=episodes(n, t, 0.02), **table(h, dtype=dtype))
    ref = reference(q, k, v, dout=dout, **args)[0]
    size = reference(q, k, v.abs(), **args)[0]["out"]  # sum P |v|
    total = v.double().abs().sum(1, keepdim=True).cpu().repeat_interleave(h // g, 2)  # the rests' subnormals
    e_out = u * ref["out"].abs() + (u * u + E32) * size + tiny * total + tiny
    out, stats = policy.attention_forward(q, k, v, **args)
    over = (out.cpu().double() - ref["out"]).abs() - 1.02 * e_out
    assert over.max() <= 0, f"out: {int((over > 0).sum())} of {over.numel()} over"

    dq = policy.attention_backward(dout, q, k, v, out, stats, **args)[0]
    # P and dS again, to bound dq by |dS| |k| and P |k|
    first, (q8, k8, v8, go) = args["first"].cpu().long(), (x.cpu().double() for x in (q, k, v, dout))
    kk, vv = (x.repeat_interleave(h // g, 2).permute(0, 2, 1, 3) for x in (k8, v8))
    qq, go, e = (x.permute(0, 2, 1, 3) for x in (q8, go, e_out))
    at = torch.arange(t)
    bucket = args["buckets"].cpu().long()[(at[:, None] - at).clamp(0, args["buckets"].numel() - 1)]
    s = qq @ kk.mT * d ** -0.5 + args["bias"].cpu().double()[:, bucket]
    p = s.masked_fill(((at > at[:, None]) | (at < first[:, :, None]))[:, None], -torch.inf).softmax(3)
    dp, sizes = go @ vv.mT, go.abs() @ vv.abs().mT
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    e_ds = p * (go.abs() * e).sum(3, keepdim=True) + E32 * p * (sizes + (p * sizes).sum(3, keepdim=True)) + u * u * ds.abs() + tiny
    want = ref["dq"]
    e_dq = ((e_ds @ kk.abs()) * d ** -0.5 * (1 + u)).permute(0, 2, 1, 3) + u * want.abs() + tiny
    over = (dq.cpu().double() - want).abs() - 1.02 * e_dq
    assert over.max() <= 0, f"dq: {int((over > 0).sum())} of {over.numel()} over"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tk,h,g,d", [(77, 8, 2, 64), (3000, 8, 1, 128), (1, 2, 1, 40)])
def test_steps_over_caches_are_rounded_once(tk, h, g, d, dtype):
    u, tiny = UNIT[dtype], TINY[dtype]
    q, k, v, _ = tensors(3, 1, tk, h, g, d, dtype)
    lengths = torch.tensor([tk, (tk + 1) // 2, 1], dtype=torch.int32, device="cuda")
    args = dict(lengths=lengths, **table(h, dtype=dtype))
    ref, size = (reference(q, k, x, **args)[0]["out"] for x in (v, v.abs()))
    total = v.double().abs().sum(1, keepdim=True).cpu().repeat_interleave(h // g, 2)
    over = (policy.attention(q, k, v, **args).cpu().double() - ref).abs() - 1.02 * (
        u * ref.abs() + (u * u + E32) * size + tiny * total + tiny)
    assert over.max() <= 0, f"{int((over > 0).sum())} of {over.numel()} over"
