"""Attention over the points of a sphere, of SO(3) or of any set, with a learned bias by buckets of the relative position.

The reference mixes features locally (correlation with a kernel of small support, s2cnn/soft/so3_conv.py:36-58) and globally
only by the integral at the end (s2cnn/soft/so3_integrate.py:7-31, examples/molecules/s2cnn_model.py:125); it has no attention.
Here every point can attend to every other.  The bias depends on the pair through a bucket number alone: with buckets of the
angle between two points (`s2_angle_buckets`) the operator commutes with rotations as far as the grid does, and with the
logarithm of the quadrature weights as `key_bias` the sum over keys is the integral over the sphere.
"""
import ctypes
import math

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _hip

MAX_HEAD = 128
MAX_BUCKETS = 64


def _unit_last(t):
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _vectors(t):
    """`t` as the kernels read it: vectors contiguous, less than 2^26 entries apart."""
    return t if (t.stride(-1) == 1 or t.size(-1) == 1) and t.stride(-2) < 1 << 26 else t.contiguous()


def _like(t):
    """Uninitialised, of the shape and order of axes of `t`, vectors contiguous."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _strides(t):
    """Strides of (batch, head, vector); 0 for an axis of one entry, whatever the tensor says."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3]))


def _describe(q, k, v, table, buckets, key_bias, lengths, scale, dtype):
    a = _hip.Attention()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = _strides(q), _strides(k), _strides(v)
    a.batch, a.heads, a.n_q, a.d = q.shape
    a.kv_heads, a.n_k = k.size(1), k.size(2)
    a.dtype, a.scale = dtype, scale
    if table is not None:
        a.table, a.buckets, a.n_buckets = table.data_ptr(), buckets.data_ptr(), table.size(1)
        a.bucket_stride[:] = (buckets.stride(0) if buckets.dim() == 3 else 0, buckets.stride(-2))
    if key_bias is not None:
        a.key_bias, a.key_bias_stride = key_bias.data_ptr(), key_bias.stride(0) if key_bias.dim() == 2 else 0
    if lengths is not None:
        a.lengths = lengths.data_ptr()
    return a


def _run(name, a, backward, device):
    nbytes = _hip.lib().s2cnn_attention_workspace(ctypes.byref(a), backward)
    ws = _hip.workspace(nbytes, device) if nbytes else None
    _hip.call(name, ctypes.byref(a), _hip.ptr(ws) if nbytes else None, nbytes, _hip.stream_ptr())


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, key_bias, lengths, scale, dtype, needs_grad):  # pylint: disable=W
        q, k, v = _vectors(q), _vectors(k), _vectors(v)
        out = _like(q)
        stats = None
        exact = q.new_empty(q.shape, dtype=torch.float32) if needs_grad and q.dtype != torch.float32 else None     # out before its rounding
        if out.numel():
            a = _describe(q, k, v, table, buckets, key_bias, lengths, scale, dtype)
            a.out, a.out_stride[:] = out.data_ptr(), _strides(out)
            if needs_grad:
                stats = q.new_empty(_hip.lib().s2cnn_attention_stats_floats(ctypes.byref(a)), dtype=torch.float32)
                a.stats, a.out_f32 = stats.data_ptr(), exact.data_ptr() if exact is not None else None
            _run("s2cnn_attention_fwd", a, 0, q.device)
        if needs_grad:
            ctx.save_for_backward(q, k, v, table, buckets, key_bias, lengths, out, stats, exact)
            ctx.scale, ctx.dtype = scale, dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):  # pylint: disable=W
        q, k, v, table, buckets, key_bias, lengths, out, stats, exact = ctx.saved_tensors
        if not out.numel() or not k.size(2):
            return (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v),
                    torch.zeros_like(table) if table is not None else None) + (None,) * 6
        g = _vectors(g)
        gq = _like(q)
        wants_kv = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        gk, gv = (_like(k), _like(v)) if wants_kv else (None, None)
        gtable = torch.empty_like(table) if table is not None and ctx.needs_input_grad[3] else None
        a = _describe(q, k, v, table, buckets, key_bias, lengths, ctx.scale, ctx.dtype)
        a.out, a.out_stride[:], a.stats = out.data_ptr(), _strides(out), stats.data_ptr()
        a.out_f32 = exact.data_ptr() if exact is not None else None
        a.gout, a.gout_stride[:] = g.data_ptr(), _strides(g)
        a.gq, a.gq_stride[:] = gq.data_ptr(), _strides(gq)
        if wants_kv:
            a.gk, a.gk_stride[:], a.gv, a.gv_stride[:] = gk.data_ptr(), _strides(gk), gv.data_ptr(), _strides(gv)
        if gtable is not None:
            a.gtable = gtable.data_ptr()
        _run("s2cnn_attention_bwd", a, 1, q.device)
        return (gq if ctx.needs_input_grad[0] else None, gk if ctx.needs_input_grad[1] else None, gv if ctx.needs_input_grad[2] else None,
                gtable, None, None, None, None, None, None)


def attention(q, k, v, table=None, buckets=None, key_bias=None, lengths=None, scale=None):
    """
    softmax(scale q k^T + table[head, buckets] + key_bias) v, the softmax over the keys, differentiable in q, k, v and table.

    :param q: [batch, heads, n_q, d], d <= 128; float32, bfloat16 or float16, any strides (copied if the last axis is strided)
    :param k, v: [batch, kv_heads, n_k, d], kv_heads dividing heads: head h reads the keys of h // (heads // kv_heads)
    :param table: [heads, n_buckets], n_buckets <= 64, the type of q: the learned bias; with buckets
    :param buckets: [n_q, n_k] or [batch, n_q, n_k] int8: the bucket of every pair.  A number outside 0 .. n_buckets - 1
        excludes the pair; what k and v hold there has still to be finite, as 0 * inf is not 0
    :param key_bias: [n_k] or [batch, n_k] float32, not differentiated: logarithms of quadrature weights, or -inf for a key
        that takes no part (its k and v are not used at all)
    :param lengths: [batch] int32: keys from lengths[b] on take no part
    :param scale: 1 / sqrt(d) if None
    :return out: [batch, heads, n_q, d]; zero for a query all of whose keys are excluded (its gradients are zero too)

    Sums, the softmax and its gradient are float32; float32 operands are multiplied to the accuracy of float32, the others'
    probabilities are rounded to the type of v.  The backward pass recomputes the probabilities.  Results do not depend on the order of execution.
    """
    assert q.dim() == 4 and k.dim() == 4 and v.dim() == 4
    assert k.shape == v.shape
    assert q.size(0) == k.size(0) and q.size(3) == k.size(3)
    assert 1 <= q.size(3) <= MAX_HEAD
    assert k.size(1) > 0 and q.size(1) % k.size(1) == 0
    assert (table is None) == (buckets is None)
    n_q, n_k = q.size(2), k.size(2)
    if table is not None:
        assert table.dim() == 2 and table.size(0) == q.size(1) and 1 <= table.size(1) <= MAX_BUCKETS
        assert buckets.shape in ((n_q, n_k), (q.size(0), n_q, n_k))
    assert key_bias is None or key_bias.shape in ((n_k,), (q.size(0), n_k))
    assert lengths is None or lengths.shape == (q.size(0),)
    dtype = _hip.require_gpu_float(q, k, v, table)
    _hip.require_gpu_of(torch.int8, buckets)
    _hip.require_gpu_of(torch.float32, key_bias)
    _hip.require_gpu_of(torch.int32, lengths)
    assert key_bias is None or not key_bias.requires_grad, "key_bias is not differentiated"
    d = q.size(3)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if d < 4:                                            # the kernels read four entries at a time
        q, k, v = (torch.nn.functional.pad(t, (0, 4 - d)) for t in (q, k, v))
    if table is not None:
        table = table.contiguous()
        buckets = buckets if buckets.stride(-1) == 1 and buckets.stride(-2) < 1 << 26 else buckets.contiguous()
    if key_bias is not None:
        key_bias = _unit_last(key_bias)
    if lengths is not None:
        lengths = lengths.contiguous()
    needs_grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, table))
    out = _Attention.apply(q, k, v, table, buckets, key_bias, lengths, scale, dtype, needs_grad)
    return out[..., :d] if d < 4 else out


def s2_angle_buckets(points_q, points_k=None, n_buckets=32, max_angle=math.pi, device=None):
    """
    Buckets of the angle between points of the sphere, for `attention`: n_buckets of equal width up to max_angle, -1 beyond
    (the pair is excluded).  Computed once on the host in 64 bits, like the kernel grids.

    :param points_q, points_k: (beta, alpha) pairs, as the s2 grids return them (points_k: points_q if None)
    :return: [len(points_q), len(points_k)] int8
    """
    assert 1 <= n_buckets <= MAX_BUCKETS
    assert 0 < max_angle <= math.pi

    def vectors(points):
        beta, alpha = np.asarray(points, dtype=np.float64).reshape(-1, 2).T
        return np.stack([np.sin(beta) * np.cos(alpha), np.sin(beta) * np.sin(alpha), np.cos(beta)], -1)

    p = vectors(points_q)
    q = p if points_k is None else vectors(points_k)
    out = np.empty((len(p), len(q)), dtype=np.int8)
    for at in range(0, len(p), 256):                     # 256 rows at a time: half a megabyte of angles per 256 points
        d = np.linalg.norm(p[at:at + 256, None] - q[None], axis=-1)
        angle = 2.0 * np.arcsin(np.minimum(d / 2.0, 1.0))               # accurate for small angles, where the cosine is not
        index = np.minimum(np.floor(angle * (n_buckets / max_angle) + 1e-9), n_buckets - 1)
        out[at:at + 256] = np.where(angle <= max_angle + 1e-9, index, -1)
    return torch.from_numpy(out).to(device) if device is not None else torch.from_numpy(out)


def s2_log_weights(b, device=None):
    """[4 b^2] float32: logarithms of the quadrature weights of the points of the 2b x 2b SOFT grid of the sphere (in the
    order of `s2_soft_grid`), as the `key_bias` that turns the sum over keys into the integral."""
    from .wigner import quadrature_weights
    w = np.repeat(np.log(np.asarray(quadrature_weights(b), dtype=np.float64)), 2 * b)
    return torch.tensor(w, dtype=torch.float32, device=device)
