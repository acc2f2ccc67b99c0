"""Attention over the points of a sphere, of SO(3) or of any set, with a learned bias by buckets of the relative position.

The reference mixes features locally (correlation with a kernel of small support, s2cnn/soft/so3_conv.py:36-58) and globally
only by the integral at the end (s2cnn/soft/so3_integrate.py:7-31, examples/molecules/s2cnn_model.py:125); it has no attention.
Here every point can attend to every other.  The bias depends on the pair through a bucket number alone: with buckets of the
angle between two points (`s2_angle_buckets`) the operator commutes with rotations as far as the grid does, and with the
logarithm of the quadrature weights as `key_bias` the sum over keys is the integral over the sphere.
"""
import ctypes
import math
import struct
from functools import lru_cache

import numpy as np
import torch

from . import _hip

MAX_HEAD = 128
MAX_BUCKETS = 64
MAX_GROUP = 128                  # heads that share a key head where there are buckets: a workgroup holds the table's rows of all of them


def _vectors(t):
    """`t` as the kernels read it: vectors contiguous, less than 2^25 entries apart."""
    return t if (t.stride(-1) == 1 or t.size(-1) == 1) and t.stride(-2) < 1 << 25 else t.contiguous()


def _even(t, few):
    """`t` with the vectors of neighbouring heads one after the other where they are few (see `few` in _Attention): the kernels take them together."""
    return t if not few or t.size(2) == 1 or t.stride(1) == t.size(2) * t.stride(2) else t.contiguous()


def _like(t):
    """Uninitialised, of the shape and order of axes of `t`, vectors contiguous."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


@lru_cache(maxsize=1024)
def _plan(shape_q, shape_k, strides, bucket_stride, key_bias_stride, n_buckets, dtype, scale, backward):
    """(the library's struct without its pointers, floats of the statistics, bytes of the workspace) of a call of these sizes.
    strides: of q, k, v, out and, backward, the gradients of out, q, k, v, as torch gives them."""
    a = _hip.Attention()
    a.batch, a.heads, a.n_q, a.d = shape_q
    a.kv_heads, a.n_k = shape_k[1], shape_k[2]
    a.dtype, a.scale, a.n_buckets = dtype, scale, n_buckets
    a.bucket_stride[:], a.key_bias_stride = bucket_stride, key_bias_stride
    queries, keys = shape_q[:3], shape_k[:3]
    for name, shape, stride in zip(("q", "k", "v", "out", "gout", "gq", "gk", "gv"), (queries, keys, keys, queries, queries, queries, keys, keys), strides):
        # 0 for an axis of one entry, whatever the tensor says
        getattr(a, name + "_stride")[:] = tuple(s if n > 1 else 0 for s, n in zip(stride, shape))
    if n_buckets:
        a.table = a.buckets = 16                          # some address: the sizes depend on there being one
    lib, ref = _hip.lib(), ctypes.byref(a)
    sizes = lib.s2cnn_attention_stats_floats(ref), lib.s2cnn_attention_workspace(ref, backward)
    a.table = a.buckets = None
    return (bytes(a), *sizes)


_POINTERS = struct.Struct("15P")                         # the struct's first fields, in the order of _run's arguments


def _run(name, plan, device, q, k, v, table, buckets, key_bias, lengths, out, stats, out_f32, gout=None, gq=None, gk=None, gv=None, gtable=None):
    a = _hip.Attention.from_buffer_copy(plan[0])
    _POINTERS.pack_into(a, 0, *[0 if t is None else t.data_ptr() for t in
                                (q, k, v, table, buckets, key_bias, lengths, out, stats, out_f32, gout, gq, gk, gv, gtable)])
    ws = _hip.workspace(plan[2], device) if plan[2] else None
    _hip.call(name, ctypes.byref(a), _hip.ptr_or_none(ws), plan[2], _hip.stream_ptr())


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, key_bias, lengths, scale, dtype, needs_grad):  # pylint: disable=W
        few = buckets is None and q.size(2) < 32 and q.size(1) > k.size(1)       # queries of heads that share keys
        q, k, v = _even(_vectors(q), few), _vectors(k), _vectors(v)
        out = _like(q)
        sizes = ((buckets.stride(0) if buckets.dim() == 3 else 0, buckets.stride(-2) if q.size(2) > 1 else 0) if buckets is not None else (0, 0),
                 key_bias.stride(0) if key_bias is not None and key_bias.dim() == 2 else 0,
                 table.size(1) if table is not None else 0, dtype, scale)
        stats = exact = None
        if out.numel():
            plan = _plan(q.shape, k.shape, (q.stride(), k.stride(), v.stride(), out.stride()), *sizes, 0)
            if needs_grad:
                stats = q.new_empty(plan[1], dtype=torch.float32)
                exact = q.new_empty(q.shape, dtype=torch.float32) if dtype else None         # out before its rounding
            _run("s2cnn_attention_fwd", plan, q.device, q, k, v, table, buckets, key_bias, lengths, out, stats, exact)
        if needs_grad:
            ctx.save_for_backward(q, k, v, table, buckets, key_bias, lengths, out, stats, exact)
            ctx.sizes, ctx.few = sizes, few
        return out

    @staticmethod
    @_hip.once_differentiable
    def backward(ctx, g):  # pylint: disable=W
        q, k, v, table, buckets, key_bias, lengths, out, stats, exact = ctx.saved_tensors
        wants_q, wants_k, wants_v, wants_table = ctx.needs_input_grad[:4]
        if not out.numel() or not k.size(2):
            return (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v),
                    torch.zeros_like(table) if table is not None else None) + (None,) * 6
        g = _even(_vectors(g), ctx.few)
        gq = _like(q)
        gk, gv = (_like(k), _like(v)) if wants_k or wants_v else (None, None)
        gtable = torch.empty_like(table) if wants_table else None
        strides = (q.stride(), k.stride(), v.stride(), out.stride(), g.stride(), gq.stride()) + ((gk.stride(), gv.stride()) if gk is not None else ())
        plan = _plan(q.shape, k.shape, strides, *ctx.sizes, 1)
        _run("s2cnn_attention_bwd", plan, q.device, q, k, v, table, buckets, key_bias, lengths, out, stats, exact, g, gq, gk, gv, gtable)
        return (gq if wants_q else None, gk if wants_k else None, gv if wants_v else None, gtable, None, None, None, None, None, None)


def attention(q, k, v, table=None, buckets=None, key_bias=None, lengths=None, scale=None):
    """
    softmax(scale q k^T + table[head, buckets] + key_bias) v, the softmax over the keys, differentiable in q, k, v and table.

    :param q: [batch, heads, n_q, d], d <= 128; float32, bfloat16 or float16, any strides (copied if the last axis is strided)
    :param k, v: [batch, kv_heads, n_k, d], kv_heads dividing heads: head h reads the keys of h // (heads // kv_heads)
    :param table: [heads, n_buckets], n_buckets <= 64, the type of q: the learned bias; with buckets, and at most 128 heads a key head
    :param buckets: [n_q, n_k] or [batch, n_q, n_k] int8: the bucket of every pair.  A number outside 0 .. n_buckets - 1
        excludes the pair; what k and v hold there has still to be finite (see below), as 0 * inf is not 0
    :param key_bias: [n_k] or [batch, n_k] float32, not differentiated: logarithms of quadrature weights, or -inf for a key
        that takes no part (its k and v are not used at all)
    :param lengths: [batch] int32: keys from lengths[b] on take no part
    :param scale: 1 / sqrt(d) if None
    :return out: [batch, heads, n_q, d]; zero for a query all of whose keys are excluded (its gradients are zero too)

    Sums, the softmax and its gradient are float32; float32 operands are multiplied to the accuracy of float32.  Of the other types the results
    are rounded, and before them nothing to less than 16 bits (float16: 22): probabilities and their gradients, as two parts.  The backward pass
    recomputes the probabilities.  Results do not depend on the order of execution.

    What takes part has to be finite, in float32 below 3.38e38.  Of an infinite entry of v or q, and of k in float32, come NaN (or an infinity) in all that depends on it,
    where the formula may have an infinity, or no weight for that key: products are of parts of the operands, and an infinity has none.  A table's
    entry or a key bias may be -inf; those of the type's lowest value leave no weight beside others, and even weights among themselves.
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
        assert q.size(1) <= MAX_GROUP * k.size(1), "at most %d heads a key head with buckets" % MAX_GROUP
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
        buckets = _vectors(buckets)
    if key_bias is not None:
        key_bias = key_bias if key_bias.stride(-1) == 1 or n_k == 1 else key_bias.contiguous()
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
