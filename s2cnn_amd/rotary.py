"""Positions of queries and keys as rotations, and the normalisation of every head's vectors, for `attention`.

The reference has no attention (its layers mix places by correlation, s2cnn/soft/so3_conv.py:36-58).  `attention` learns a bias by the
angle of two points; with `rotary` before it the scores depend on the difference of two positions as well, in directions too: pairs of a vector's
entries are turned by angles that are linear in the position.  The angles come as a table of cosines and sines, formed once for a grid
(`s2_rotary_table`) or for positions of any kind (`rotary_table`).  `norm_rotary` gives every vector the same size first, so that scores stay
bounded, in the same pass.
"""
import ctypes
import math
import struct
from functools import lru_cache

import numpy as np
import torch

from . import _hip
from .attention import _like

MAX_HEAD = 256
MAX_VECTORS = 1 << 31
POSITIONS = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}

_SIDE, _SHARED = struct.Struct("5P"), struct.Struct("2P")             # the pointers of s2cnn_rotary_side_t, and of s2cnn_rotary_t behind its two sides


def _vectors(t):
    """`t` with contiguous vectors"""
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


@lru_cache(maxsize=1024)
def _plan(shapes, strides, table, index_stride, norm, interleaved, eps, dtype):
    """(the library's struct without its pointers, bytes of the workspace of the weights' gradients) of a call of these sizes.
    strides: per tensor of x, g and y, as torch gives them; table: its batch stride, rows and pairs."""
    a = _hip.Rotary()
    present = [(shape, of) for shape, of in zip(shapes, strides) if shape is not None]      # one tensor alone is the first
    a.batch, _, a.n, a.d = present[0][0]
    for side, (shape, of) in zip(a.side, present):
        side.heads = shape[1]
        for name, stride in zip(("x_stride", "g_stride", "y_stride"), of):
            getattr(side, name)[:] = stride[:3] if stride is not None else (0, 0, 0)
    a.table_stride, a.rows, a.pairs = table
    a.index_stride, a.norm, a.interleaved, a.eps, a.dtype = index_stride, norm, interleaved, eps, dtype
    a.table = 16 if a.pairs else None                       # some address: the sizes are refused without
    nbytes = _hip.lib().s2cnn_rotary_workspace(ctypes.byref(a))
    a.table = None
    return bytes(a), nbytes


def _run(backward, plan, tensors, table, index, sums):
    """tensors: (x, weight, g, y, gweight) of each side"""
    a = _hip.Rotary.from_buffer_copy(plan[0])
    tensors = [t for t in tensors if t is not None]
    for i, t in enumerate(tensors):
        _SIDE.pack_into(a, i * ctypes.sizeof(_hip.RotarySide), *[0 if x is None else x.data_ptr() for x in t])
    _SHARED.pack_into(a, 2 * ctypes.sizeof(_hip.RotarySide), 0 if table is None else table.data_ptr(), 0 if index is None else index.data_ptr())
    if not backward:
        _hip.call("s2cnn_rotary_fwd", ctypes.byref(a), _hip.stream_ptr())
        return
    ws = _hip.workspace(plan[1], tensors[0][2].device) if sums else None
    _hip.call("s2cnn_rotary_bwd", ctypes.byref(a), _hip.ptr_or_none(ws), plan[1] if sums else 0, _hip.stream_ptr())


def _sizes(table, index):
    return ((table.stride(0) if table is not None and table.dim() == 4 and table.size(0) > 1 else 0, *(table.shape[-3:-1] if table is not None else (0, 0))),
            index.stride(0) if index is not None and index.dim() == 2 and index.size(0) > 1 else 0)


def _forward(q, k, q_weight, k_weight, table, index, options):
    out = [None if x is None else _like(x) for x in (q, k)]
    if q.size(0) * q.size(2) == 0 or q.size(1) == 0 and (k is None or k.size(1) == 0):
        return out
    xs = [None if x is None or not x.numel() else x for x in (q, k)]
    plan = _plan(tuple(None if x is None else x.shape for x in xs), tuple(None if x is None else (x.stride(), None, y.stride()) for x, y in zip(xs, out)),
                 *_sizes(table, index), *options)
    _run(False, plan, [None if x is None else (x, w, None, y, None) for x, w, y in zip(xs, (q_weight, k_weight), out)], table, index, False)
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, index, options):  # pylint: disable=W
        ctx.set_materialize_grads(False)
        norm = options[0]
        ctx.save_for_backward(q if norm else None, k if norm else None, q_weight, k_weight, table, index)
        ctx.options = options
        return tuple(_forward(q, k, q_weight, k_weight, table, index, options))

    @staticmethod
    @_hip.once_differentiable
    def backward(ctx, *grads):  # pylint: disable=W
        *xs, q_weight, k_weight, table, index = ctx.saved_tensors
        weights = (q_weight, k_weight)
        gx, gw, tensors, shapes, strides = [None, None], [None, None], [None, None], [None, None], [None, None]
        for i, (x, w, g) in enumerate(zip(xs, weights, grads)):
            wants = ctx.needs_input_grad[2 + i] and w is not None
            if g is None or not (ctx.needs_input_grad[i] or wants):
                continue
            g = _vectors(g)
            gx[i] = _like(g if x is None else x)
            if wants:
                gw[i] = torch.empty_like(w) if g.numel() else torch.zeros_like(w)
            if g.numel():
                tensors[i] = (x, w, g, gx[i], gw[i])
                shapes[i], strides[i] = g.shape, (None if x is None else x.stride(), g.stride(), gx[i].stride())
        if any(t is not None for t in tensors):
            plan = _plan(tuple(shapes), tuple(strides), *_sizes(table, index), *ctx.options)
            _run(True, plan, tensors, table, index, any(t is not None and t[4] is not None for t in tensors))
        return (*(g if ctx.needs_input_grad[i] else None for i, g in enumerate(gx)), *gw, None, None, None)


def _call(q, k, q_weight, k_weight, table, index, norm, eps, interleaved):
    assert q.dim() == 4 and (k is None or k.dim() == 4)
    batch, _, n, d = q.shape
    assert k is None or (k.size(0), k.size(2), k.size(3)) == (batch, n, d)
    assert 1 <= d <= MAX_HEAD
    assert batch * n * max(q.size(1), 0 if k is None else k.size(1)) < MAX_VECTORS
    if table is not None:
        assert table.dim() in (3, 4) and table.size(-1) == 2 and 1 <= table.size(-2) <= d // 2
        assert table.dim() == 3 or table.size(0) == batch
        assert not table.requires_grad, "the table is not differentiated"
        if index is None:
            assert table.size(-3) == n
        else:
            assert index.shape in ((n,), (batch, n)) and table.size(-3) >= 1
    else:
        assert index is None
    dtype = _hip.require_gpu_float(q, k, q_weight, k_weight)
    _hip.require_gpu_of(torch.float32, table)
    _hip.require_gpu_of(torch.int32, index)
    q, k = _vectors(q), None if k is None else _vectors(k)
    table = table.contiguous() if table is not None else None
    index = index.contiguous() if index is not None else None
    options = (int(norm), int(interleaved), eps, dtype)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _Rotary.apply(q, k, q_weight, k_weight, table, index, options)
    return tuple(_forward(q, k, q_weight, k_weight, table, index, options))


def rotary(q, k, table, index=None, interleaved=False):
    """
    Queries and keys with pairs of their entries turned by the angles of their positions, differentiable in both:
    (a, b) -> (a cos - b sin, a sin + b cos) for the pairs (j, pairs + j), or with `interleaved` (2j, 2j + 1), j < pairs.  Entries from
    2 pairs on stay as they are.

    :param q: [batch, heads, n, d], d <= 256; float32, bfloat16 or float16, any strides (copied if the last axis is strided)
    :param k: [batch, kv_heads, n, d] of the same places, or None
    :param table: [rows, pairs, 2] or [batch, rows, pairs, 2] float32, cosines and sines (`rotary_table`); without an index row n is the place's, and
        there are n of them.  Not differentiated
    :param index: [n] or [batch, n] int32: the row of every place.  A place whose row is below zero is not turned (padding); of one from `rows` on
        what would be turned becomes NaN
    :return (q, k): the types and orders of axes of the arguments; arithmetic is float32, rounded once.  k: None for None
    """
    assert table is not None
    return _call(q, k, None, None, table, index, False, 0.0, interleaved)


def norm_rotary(q, k, q_weight=None, k_weight=None, table=None, index=None, eps=1e-6, interleaved=False):
    """
    Queries and keys with every vector x divided by sqrt(mean(x^2) + eps) and multiplied by a weight, then turned as by `rotary` (without a table:
    not), in one pass; differentiable in q, k and the weights.

    :param q, k, table, index, interleaved: as for `rotary`
    :param q_weight, k_weight: [d], the type of q, shared by the heads, or None
    :param eps: > 0
    :return (q, k): as for `rotary`.  Squares are summed in float32: entries are below 2^63 in size
    """
    eps = ctypes.c_float(eps).value
    assert 0.0 < eps < math.inf
    assert q_weight is None or q_weight.shape == q.shape[-1:]
    assert k_weight is None or (k is not None and k_weight.shape == k.shape[-1:])
    q_weight = q_weight.contiguous() if q_weight is not None else None
    k_weight = k_weight.contiguous() if k_weight is not None else None
    return _call(q, k, q_weight, k_weight, table, index, True, eps, interleaved)


def rotary_table(positions, frequencies, scale=1.0):
    """
    Cosines and sines for `rotary`: of the angles sum over axes of positions[..., axis] * frequencies[axis, pair].  Not differentiated.

    :param positions: [..., axes] float32, float64, int32 or int64: places on an axis, angles on the sphere, points in space
    :param frequencies: [axes, pairs] float64 in radians (`rotary_frequencies`, `s2_rotary_frequencies`), pairs <= 128
    :param scale: a factor of both, which multiplies scores by its square where queries and keys are turned with the table
    :return [..., pairs, 2]: float32.  Angles are formed in 64 bits: no place is too far for its angle to be accurate to 2^-24
        below 2^26 turns
    """
    assert positions.dim() >= 1 and frequencies.dim() == 2
    axes, pairs = frequencies.shape
    assert positions.size(-1) == axes >= 1 and 1 <= pairs <= MAX_HEAD // 2
    if positions.dtype not in POSITIONS:
        raise RuntimeError("positions of float32, float64, int32 or int64 only (got %s)" % positions.dtype)
    _hip.require_gpu_of(positions.dtype, positions)
    _hip.require_gpu_of(torch.float64, frequencies)
    assert not positions.requires_grad and not frequencies.requires_grad, "the table is not differentiated"
    positions, frequencies = positions.contiguous(), frequencies.contiguous()
    table = torch.empty(*positions.shape[:-1], pairs, 2, dtype=torch.float32, device=positions.device)
    n = positions.numel() // axes
    if n:
        _hip.call("s2cnn_rotary_table", positions.data_ptr(), POSITIONS[positions.dtype], frequencies.data_ptr(), table.data_ptr(), n, axes, pairs, scale,
                  _hip.stream_ptr())
    return table


def rotary_frequencies(pairs, base=10000.0, factor=1.0, original=None, fast=32.0, slow=1.0, device=None):
    """
    [1, pairs] float64: base^(-j / pairs), for places on one axis.

    :param factor: how many times longer the axis is than the one that a model was trained on.  All frequencies are divided by it; or, where `original`
        gives the length of that axis, those that turn less than `slow` times along it, and none that turns more than `fast` times, with a linear passage
        between them: near places stay as far apart as they were
    """
    assert 1 <= pairs <= MAX_HEAD // 2 and base > 0 and factor > 0 and 0 <= slow < fast
    f = base ** (-np.arange(pairs, dtype=np.float64) / pairs)
    kept = np.zeros(pairs) if original is None else np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
    return torch.tensor(f * (kept + (1.0 - kept) / factor), dtype=torch.float64, device=device).view(1, pairs)


def s2_rotary_frequencies(pairs, device=None):
    """[2, pairs] float64, for (beta, alpha) of the sphere: even pairs turn with alpha, odd ones with beta, 1, 2, 3 ... times.  Whole numbers, so that
    alpha and alpha + 2 pi are the same place: scores commute with rotations about the polar axis."""
    assert 1 <= pairs <= MAX_HEAD // 2
    f = torch.zeros(2, pairs, dtype=torch.float64)
    f[1, 0::2] = torch.arange(1, (pairs + 1) // 2 + 1, dtype=torch.float64)
    f[0, 1::2] = torch.arange(1, pairs // 2 + 1, dtype=torch.float64)
    return f.to(device) if device is not None else f


def s2_rotary_table(b, pairs, device=None):
    """[4 b^2, pairs, 2] float32: the table of the points of the 2b x 2b SOFT grid of the sphere (in the order of `s2_soft_grid`), by
    `s2_rotary_frequencies`.  Computed once on the host in 64 bits, like the kernel grids."""
    from .s2_grid import s2_soft_grid
    angles = np.asarray(s2_soft_grid(b), dtype=np.float64).reshape(-1, 2) @ s2_rotary_frequencies(pairs).numpy()
    return torch.tensor(np.stack([np.cos(angles), np.sin(angles)], -1), dtype=torch.float32, device=device)
