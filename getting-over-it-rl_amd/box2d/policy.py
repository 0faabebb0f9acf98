"""Operators of a policy network over the worlds' histories, on the GPU: what a training or acting loop runs between two
steps of the worlds.

    out = policy.attention(q, k, v, bias=table, buckets=policy.distance_buckets(32, 128), first=episode_start)  # differentiable
    act = policy.attention(q1, k_cache, v_cache, bias=table, buckets=buckets, lengths=steps_held)                # one step

Hand-written kernels for gfx950 through the C ABI in include/goi_policy.h; no fallback. Every call runs on the current
stream of its tensors' device and waits for nothing. Tensors whose strides the kernels do not take (a last axis that is not
contiguous, rows that are not 16-byte aligned) are copied first. No counterpart in the reference's physics package, which leaves the
policy to its caller (README.md:22-24).
"""
import contextlib
import ctypes
import math

import torch

from . import _abi

_TYPES = {torch.float32: _abi.F32, torch.float16: _abi.F16, torch.bfloat16: _abi.BF16}


def _need(ok, message, *args):
    if not ok:
        raise ValueError(message.format(*args))


def _on_gpu(*tensors):
    """The one CUDA device of the tensors that are given."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        _need(torch.is_tensor(t) and t.is_cuda, "the policy operators take CUDA tensors")
        _need(dev is None or t.device == dev, "tensors on more than one device")
        dev = t.device
    return dev


def _guard(dev):
    return contextlib.nullcontext() if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _stream(dev):
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _rows(x):
    """x (worlds, steps, heads, dim) as the attention kernels read it, and its strides of worlds, steps and heads."""
    if x.data_ptr() % 16 or x.stride(3) != 1 or any(x.stride(d) % 8 and x.shape[d] > 1 for d in range(3)):
        x = x.clone(memory_format=torch.contiguous_format)
    s = x.stride()
    return x, _abi._I64x3(*(s[d] if x.shape[d] > 1 else 0 for d in range(3)))


def _ints(x, shape, name):
    if x is None:
        return None
    _need(x.dtype == torch.int32 and tuple(x.shape) == shape, "{} must be int32 of shape {}", name, shape)
    return x.contiguous()


def _ptr(x):
    return None if x is None else x.data_ptr()


def distance_buckets(count, reach, two_sided=False, device="cuda"):
    """The bucket of each distance for `attention`'s bias, int32: one bucket each for the distances below count / 2, then
    ranges that grow geometrically up to `reach`; every distance from `reach` on shares the last bucket. Distances 0 .. reach, or
    for two_sided -reach .. reach with the second half of the buckets for keys after the query."""
    if two_sided:
        _need(count % 2 == 0, "two-sided buckets come in pairs")
        one = distance_buckets(count // 2, reach, device="cpu")
        return torch.cat([one[1:].flip(0) + count // 2, one]).to(device)
    near = count // 2
    _need(count >= 2 and reach >= max(near, 1), "distance_buckets needs two buckets or more and a reach of count / 2 or more")
    d = torch.arange(reach + 1, dtype=torch.float64)
    if reach > near:
        far = near + ((d.clamp_min(1) / near).log() / math.log(reach / near) * (count - near)).floor()
    else:
        far = torch.full_like(d, count - 1)
    return torch.where(d < near, d, far.clamp(near, count - 1)).to(torch.int32).to(device)


def _attention_args(q, k, v, bias, buckets, first, lengths, causal, scale):
    """(GoiAttention, device, tensors to keep): the checked inputs of both directions."""
    dev = _on_gpu(q, k, v, bias, buckets, first, lengths)
    _need(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k and v are (worlds, steps, heads, dim)")
    n, tq, h, d = q.shape
    tk, g = k.shape[1], k.shape[2]
    _need(tuple(k.shape) == (n, tk, g, d) and k.shape == v.shape, "k and v must be ({}, steps, heads, {}) alike", n, d)
    _need(q.dtype in (torch.bfloat16, torch.float16) and k.dtype == q.dtype and v.dtype == q.dtype,
          "q, k and v must all be bfloat16 or all float16")
    a = _abi.GoiAttention()
    a.n_worlds, a.q_steps, a.k_steps, a.heads, a.kv_heads, a.dim = n, tq, tk, h, g, d
    a.type, a.causal = _TYPES[q.dtype], int(bool(causal))
    a.scale = d ** -0.5 if scale is None else float(scale)
    q, a.q_strides = _rows(q)
    k, a.k_strides = _rows(k)
    v, a.v_strides = _rows(v)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if bias is not None:
        _need(buckets is not None, "a bias needs the buckets of the distances")
        _need(bias.dim() == 2 and bias.shape[0] == h and bias.dtype in (q.dtype, torch.float32),
              "the bias is (heads, buckets), of q's type or float32")
        _need(buckets.dim() == 1 and buckets.dtype == torch.int32, "buckets must be one row of int32")
        bias, buckets = bias.contiguous(), buckets.contiguous()
        a.bias, a.buckets, a.bias_type = bias.data_ptr(), buckets.data_ptr(), _TYPES[bias.dtype]
        a.n_buckets, a.n_distances = bias.shape[1], buckets.shape[0]
    first = _ints(first, (n, tq), "first")
    lengths = _ints(lengths, (n,), "lengths")
    a.first, a.lengths = _ptr(first), _ptr(lengths)
    return a, dev, (q, k, v, bias, buckets, first, lengths)


def _attention_call(a, dev, backward):
    L = _abi.lib()
    size = ctypes.c_uint64()
    _abi.check(L.goi_attention_workspace(ctypes.byref(a), backward, ctypes.byref(size)), L)
    ws = torch.empty(size.value, dtype=torch.uint8, device=dev) if size.value else None
    call = L.goi_attention_backward if backward else L.goi_attention_forward
    with _guard(dev):
        _abi.check(call(ctypes.byref(a), _ptr(ws), size.value, _stream(dev)), L)


def attention_forward(q, k, v, bias=None, buckets=None, first=None, lengths=None, causal=True, scale=None, need_stats=True):
    """(out, stats) of `attention`, without a graph. stats (worlds, heads, steps, 2) float32 is what attention_backward needs
    (None with need_stats=False): each query's largest score times log2(e), and the sum of the powers of two of the scores
    relative to it; minus infinity and 0 where it sees no key."""
    a, dev, keep = _attention_args(q, k, v, bias, buckets, first, lengths, causal, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    out, a.out_strides = _rows(out)
    stats = torch.empty((q.shape[0], q.shape[2], q.shape[1], 2), dtype=torch.float32, device=dev) if need_stats else None
    a.out, a.stats = out.data_ptr(), _ptr(stats)
    _attention_call(a, dev, 0)
    del keep
    return out, stats


def attention_backward(dout, q, k, v, out, stats, bias=None, buckets=None, first=None, lengths=None, causal=True, scale=None):
    """(dq, dk, dv, dbias) of `attention` for the gradient dout of its output; out and stats are attention_forward's. dbias is
    None without a bias. Every sum has a fixed order: the same inputs give the same bits."""
    a, dev, keep = _attention_args(q, k, v, bias, buckets, first, lengths, causal, scale)
    _on_gpu(q, dout, out, stats)
    _need(dout.shape == q.shape and out.shape == q.shape and dout.dtype == q.dtype and out.dtype == q.dtype,
          "dout and out must be like q")
    _need(stats.dtype == torch.float32 and tuple(stats.shape) == (q.shape[0], q.shape[2], q.shape[1], 2),
          "stats must be float32 (worlds, heads, steps, 2)")
    dout, a.dout_strides = _rows(dout)
    out, a.out_strides = _rows(out)
    stats = stats.contiguous()
    a.dout, a.out, a.stats = dout.data_ptr(), out.data_ptr(), stats.data_ptr()
    grads = [torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k, v)]
    dbias = None if bias is None else torch.empty(bias.shape, dtype=bias.dtype, device=dev)
    (dq, a.dq_strides), (dk, a.dk_strides), (dv, a.dv_strides) = map(_rows, grads)
    a.dq, a.dk, a.dv, a.dbias = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dbias)
    _attention_call(a, dev, 1)
    del keep
    return dq, dk, dv, dbias


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, buckets, first, lengths, causal, scale):
        out, stats = attention_forward(q, k, v, bias, buckets, first, lengths, causal, scale)
        ctx.save_for_backward(q, k, v, out, stats, bias, buckets, first, lengths)
        ctx.how = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, stats, *rest = ctx.saved_tensors
        grads = attention_backward(dout, q, k, v, out, stats, *rest, *ctx.how)
        return (*grads, None, None, None, None, None)


def attention(q, k, v, bias=None, buckets=None, first=None, lengths=None, causal=True, scale=None):
    """Attention of each world's steps over its history; differentiable in q, k, v and bias.

    q (worlds, steps, heads, dim), k and v (worlds, key steps, key heads, dim), bfloat16 or float16, dim a multiple of 8 up
    to 128; heads a multiple of key heads: query head h reads key head h // (heads / key heads). The queries are the last steps of the
    world's history of lengths[world] keys (all key steps without lengths): query i stands at p = length - steps + i and
    sees the keys first[world, i] <= j <= p (causal) or first[world, i] <= j < length. One query per world over a cache is
    acting; as many queries as keys, with `first` the step at which each step's episode began, is training on a window.

    bias (heads, buckets) adds bias[head, buckets[p - j]] to the scaled scores (distances past the map's ends take its ends;
    without a causal order the map holds both directions, distance 0 in the middle). scale is dim ** -0.5 by default.
    A query that sees nothing gives zeros and no gradient. Returns a tensor like q."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, bias)):
        return _Attention.apply(q, k, v, bias, buckets, first, lengths, causal, scale)
    return attention_forward(q, k, v, bias, buckets, first, lengths, causal, scale, need_stats=False)[0]
