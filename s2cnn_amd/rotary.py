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
from torch.autograd import forward_ad

from . import _hip
from .attention import _like

MAX_HEAD = 256
MAX_VECTORS = 1 << 31
POSITIONS = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}

_POINTERS = struct.Struct("12P")                         # the first fields of s2cnn_rotary_t


def _vectors(t):
    """`t` with contiguous vectors"""
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


@lru_cache(maxsize=1024)
def _plan(shape, other, strides, table, index_stride, norm, interleaved, eps, dtype):
    """(the library's struct without its pointers, bytes of the workspace of the weights' gradients) of a call of these sizes.
    shape, other: of the first tensor and of the second, or None; strides: of x, g and y of the first, then of the second, as torch gives them, or None;
    table: its batch stride, rows and pairs; index_stride: None without an index."""
    a = _hip.Rotary()
    a.batch, a.heads[0], a.n, a.d = shape
    a.heads[1] = 0 if other is None else other[1]
    for i in range(len(strides) // 3):
        for to, stride in zip((a.x_stride, a.g_stride, a.y_stride), strides[3 * i:]):
            to[i][:] = stride[:3] if stride is not None else (0, 0, 0)
    a.table_stride, a.rows, a.pairs = table
    a.index_stride, a.norm, a.interleaved, a.eps, a.dtype = index_stride or 0, norm, interleaved, eps, dtype
    a.table = 16 if a.pairs else None                    # some addresses: the sizes are refused without, and fewer rows than places without an index
    a.index = None if index_stride is None else 16
    nbytes = _hip.lib().s2cnn_rotary_workspace(ctypes.byref(a))
    a.table = a.index = None
    return bytes(a), nbytes


def _at(t):
    return 0 if t is None else t.data_ptr()


def _run(plan, table, index, backward, x, w, g, y, gw=None, x2=None, w2=None, g2=None, y2=None, gw2=None):
    a = _hip.Rotary.from_buffer_copy(plan[0])
    _POINTERS.pack_into(a, 0, _at(x), _at(x2), _at(w), _at(w2), _at(g), _at(g2), y.data_ptr(), _at(y2), _at(gw), _at(gw2), _at(table), _at(index))
    if not backward:
        _hip.call("s2cnn_rotary_fwd", ctypes.byref(a), _hip.stream_ptr())
    elif gw is None and gw2 is None:
        _hip.call("s2cnn_rotary_bwd", ctypes.byref(a), None, 0, _hip.stream_ptr())
    else:
        ws = _hip.workspace(plan[1], y.device)
        _hip.call("s2cnn_rotary_bwd", ctypes.byref(a), ws.data_ptr(), plan[1], _hip.stream_ptr())


def _forward(q, k, q_weight, k_weight, table, index, sizes):
    """sizes: of the table and the index, and the options, as _plan takes them"""
    y = _like(q)
    z = None if k is None else _like(k)
    one, two = y.numel() > 0, z is not None and z.numel() > 0
    if one and two:
        plan = _plan(q.shape, k.shape, (q.stride(), None, y.stride(), k.stride(), None, z.stride()), *sizes)
        _run(plan, table, index, False, q, q_weight, None, y, None, k, k_weight, None, z)
    elif one:
        _run(_plan(q.shape, None, (q.stride(), None, y.stride()), *sizes), table, index, False, q, q_weight, None, y)
    elif two:
        _run(_plan(k.shape, None, (k.stride(), None, z.stride()), *sizes), table, index, False, k, k_weight, None, z)
    return y, z


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, index, sizes):  # pylint: disable=W
        ctx.set_materialize_grads(False)
        if sizes[2]:
            ctx.save_for_backward(q, k, q_weight, k_weight, table, index)
        else:
            ctx.save_for_backward(None, None, None, None, table, index)
        ctx.sizes = sizes
        return _forward(q, k, q_weight, k_weight, table, index, sizes)

    @staticmethod
    @_hip.once_differentiable
    def backward(ctx, g, g2):  # pylint: disable=W
        q, k, q_weight, k_weight, table, index = ctx.saved_tensors
        wants_q, wants_k, wants_qw, wants_kw = ctx.needs_input_grad[:4]
        sides, out = [], [None] * 7
        for i, x, w, g, wants_x, wants_w in ((0, q, q_weight, g, wants_q, wants_qw), (1, k, k_weight, g2, wants_k, wants_kw)):
            if g is None or not (wants_x or wants_w):
                continue
            g = _vectors(g)
            y = _like(g if x is None else x)
            some = g.numel() > 0
            gw = None if not wants_w else torch.empty_like(w) if some else torch.zeros_like(w)
            out[i], out[2 + i] = y if wants_x else None, gw
            if some:
                sides.append((x, w, g, y, gw))
        if sides:
            strides = tuple(None if t is None else t.stride() for side in sides for t in (side[0], side[2], side[3]))
            plan = _plan(sides[0][2].shape, sides[1][2].shape if len(sides) > 1 else None, strides, *ctx.sizes)
            _run(plan, table, index, True, *sides[0], *(sides[1] if len(sides) > 1 else ()))
        return tuple(out)


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
            assert index.shape in ((n,), (batch, n)) and 1 <= table.size(-3) < MAX_VECTORS
    else:
        assert index is None
    dtype = _hip.require_gpu_float(q, k, q_weight, k_weight)
    _hip.require_gpu_of(torch.float32, table)
    _hip.require_gpu_of(torch.int32, index)
    q, k = _vectors(q), None if k is None else _vectors(k)
    if table is not None:
        table = table.contiguous()
        if table.data_ptr() & 7:                         # a view at an odd float
            table = table.clone()
    index = index.contiguous() if index is not None else None
    sizes = ((0, 0, 0) if table is None else (table.stride(0) if table.dim() == 4 and batch > 1 else 0, *table.shape[-3:-1]),
             None if index is None else 0 if index.dim() == 1 or batch == 1 else n, int(norm), int(interleaved), eps, dtype)
    # tangents of forward mode, which is on under no_grad as well, are refused there
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _Rotary.apply(q, k, q_weight, k_weight, table, index, sizes)
    return _forward(q, k, q_weight, k_weight, table, index, sizes)


def rotary(q, k, table, index=None, interleaved=False):
    """
    Queries and keys with pairs of their entries turned by the angles of their positions, differentiable in both:
    (a, b) -> (a cos - b sin, a sin + b cos) for the pairs (j, pairs + j), or with `interleaved` (2j, 2j + 1), j < pairs.  Entries from
    2 pairs on stay as they are.

    :param q: [batch, heads, n, d], d <= 256; float32, bfloat16 or float16, any strides (copied if the last axis is strided)
    :param k: [batch, kv_heads, n, d] of the same places, or None
    :param table: [rows, pairs, 2] or [batch, rows, pairs, 2] float32, cosines and sines (`rotary_table`); without an index row n is the place's, and
        there are n of them, with one any number below 2^31.  Not differentiated
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
    :param eps: >= 2^-126
    :return (q, k): as for `rotary`.  Squares are summed in float32: a vector's have to stay below 2^127 together (entries below 2^59 in size do for any d);
        beyond, the vector becomes zero or NaN
    """
    eps = ctypes.c_float(eps).value
    assert 2.0 ** -126 <= eps < math.inf
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
    :return [..., pairs, 2]: float32.  Angles are formed in 64 bits, with up to three roundings of each axis's part: where that is below 2^24 turns an angle is
        off by less than 2^-24, and an entry by less than 3 * 2^-24 of the scale; beyond, in proportion more
    """
    assert positions.dim() >= 1 and frequencies.dim() == 2
    axes, pairs = frequencies.shape
    assert positions.size(-1) == axes >= 1 and 1 <= pairs <= MAX_HEAD // 2
    if positions.dtype not in POSITIONS:
        raise RuntimeError("positions of float32, float64, int32 or int64 only (got %s)" % positions.dtype)
    _hip.require_gpu_of(positions.dtype, positions)
    _hip.require_gpu_of(torch.float64, frequencies)
    assert not positions.requires_grad and not frequencies.requires_grad, "the table is not differentiated"
    assert not _hip.have_tangents(positions, frequencies), "the table is not differentiated"
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
        between them: near places stay as far apart as they were (Peng, Quesnelle, Fan, Shippole, "YaRN: efficient context window extension of large
        language models", 2023; its factor of the scores is the square of `rotary_table`'s scale)
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
