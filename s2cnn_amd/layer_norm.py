"""Layer normalisation over the feature axis, dropout whose mask is never stored, and the step of a transformer block that joins
both with a residual.

The reference normalises with nn.BatchNorm3d between its layers (examples/shrec17/model.py:28-34) and has no dropout; a block
of `attention` and pointwise layers over the points of a sphere is trained with these.  Random numbers come from a
counter: the mask is a function of the seed and of an element's index, formed again in the backward pass.
"""
from functools import lru_cache

import torch

from . import _hip


def _seed_args(seed):
    """(number, address) of a seed that is a number or a tensor on the GPU."""
    if torch.is_tensor(seed):
        return 0, seed.data_ptr()
    return seed & 0xFFFFFFFFFFFFFFFF, None


def _check_dropout(p, seed):
    assert 0.0 <= p < 1.0
    if torch.is_tensor(seed):
        assert seed.numel() == 1
    else:
        assert isinstance(seed, int)


def _require_seed(seed):
    if torch.is_tensor(seed):
        _hip.require_gpu_of(torch.int64, seed)


@lru_cache(maxsize=1024)
def _workspace_floats(rows, features, dtype):
    return _hip.lib().s2cnn_layer_norm_bwd_workspace(rows, features, dtype) // 4


@lru_cache(maxsize=1024)
def _stats_floats(rows, features, dtype, step):
    return _hip.lib().s2cnn_layer_norm_stats_floats(rows, features, dtype, step)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, dtype):  # pylint: disable=W
        ctx.p, ctx.dtype = p, dtype
        ctx.seed = None if torch.is_tensor(seed) else seed
        ctx.save_for_backward(*((seed,) if torch.is_tensor(seed) else ()))
        return _Dropout.run(x, p, seed, dtype)

    @staticmethod
    @_hip.once_differentiable
    def backward(ctx, g):  # pylint: disable=W
        return _Dropout.run(g, ctx.p, ctx.saved_tensors[0] if ctx.seed is None else ctx.seed, ctx.dtype), None, None, None

    @staticmethod
    def run(x, p, seed, dtype):
        x = x.contiguous()
        y = torch.empty_like(x)
        if x.numel():
            number, at = _seed_args(seed)
            _hip.call("s2cnn_dropout", x.data_ptr(), y.data_ptr(), x.numel(), p, number, at, dtype, _hip.stream_ptr())
        return y


def dropout(x, p, seed):
    """
    x with elements set to zero with probability p and the others divided by the probability of staying (as torch's dropout
    in training), differentiable.

    :param x: float32, bfloat16 or float16, any shape
    :param p: in [0, 1), taken to the nearest multiple of 2^-16 below one
    :param seed: an int, or an int64 tensor of one element on the GPU that is read when the kernel runs (so that a captured
        graph drops others at each replay).  Equal seeds and sizes drop equal elements: give each call of a step its own
    :return y: contiguous; element i of it depends on seed and i alone (include/s2cnn_hip.h has the generator)
    """
    _check_dropout(p, seed)
    dtype = _hip.require_gpu_float(x)
    _require_seed(seed)
    return _Dropout.apply(x, float(p), seed, dtype)


class _LayerNorm(torch.autograd.Function):
    """(x, weight, bias) -> y, or with a residual (x, residual, ...) -> (h, y), h = residual + dropout(x)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, seed, dtype, needs_grad):  # pylint: disable=W
        ctx.set_materialize_grads(False)
        features = x.size(-1)
        rows = x.numel() // features
        x = x.contiguous()
        residual = residual.contiguous() if residual is not None else None
        y = torch.empty_like(x)
        h = torch.empty_like(x) if residual is not None else None
        stats = x.new_empty(_stats_floats(rows, features, dtype, residual is not None), dtype=torch.float32) if needs_grad else None
        number, at = _seed_args(seed)
        if rows:
            _hip.call("s2cnn_layer_norm_fwd", x.data_ptr(), _hip.ptr_or_none(residual), _hip.ptr_or_none(weight), _hip.ptr_or_none(bias),
                      _hip.ptr_or_none(h), y.data_ptr(), _hip.ptr_or_none(stats), rows, features, eps, p, number, at, dtype, _hip.stream_ptr())
        if needs_grad:
            ctx.save_for_backward(x if h is None else h, weight, stats, seed if torch.is_tensor(seed) else None)
            ctx.p, ctx.seed, ctx.dtype = p, seed if not torch.is_tensor(seed) else None, dtype
        return y if h is None else (h, y)

    @staticmethod
    @_hip.once_differentiable
    def backward(ctx, *grads):  # pylint: disable=W
        h, weight, stats, seed = ctx.saved_tensors
        step = len(grads) == 2
        g_h, g = grads if step else (None, grads[0])
        if g is None and g_h is None:
            return (None,) * 9
        seed = ctx.seed if seed is None else seed
        g = g.contiguous() if g is not None else torch.zeros_like(h)
        g_h = g_h.contiguous() if g_h is not None else None
        features = h.size(-1)
        rows = h.numel() // features
        wants_x, wants_residual, wants_weight, wants_bias = ctx.needs_input_grad[:4]
        wants_x = wants_x or (not step) or not wants_residual                # one of the two is always written
        gx = torch.empty_like(h) if wants_x else None
        gresidual = torch.empty_like(h) if step and wants_residual else None
        new = h.new_empty if rows else h.new_zeros
        gw = new(features) if wants_weight else None
        gb = new(features) if wants_bias else None
        if rows:
            floats = _workspace_floats(rows, features, ctx.dtype) if wants_weight or wants_bias else 0
            ws = h.new_empty(floats, dtype=torch.float32) if floats else None
            number, at = _seed_args(seed)
            _hip.call("s2cnn_layer_norm_bwd", h.data_ptr(), g.data_ptr(), _hip.ptr_or_none(g_h), _hip.ptr_or_none(weight), stats.data_ptr(),
                      _hip.ptr_or_none(gx), _hip.ptr_or_none(gresidual), _hip.ptr_or_none(gw), _hip.ptr_or_none(gb), _hip.ptr_or_none(ws), 4 * floats,
                      rows, features, ctx.p, number, at, int(step), ctx.dtype, _hip.stream_ptr())
        return gx, gresidual, gw, gb, None, None, None, None, None


@lru_cache(maxsize=1024)
def _column_sums_bytes(rows, features, dtype):
    return _hip.lib().s2cnn_column_sums_workspace(rows, features, dtype)


def column_sums(x):
    """Sums of x [..., features] (float32, bfloat16 or float16) over all other axes, float32.  Not differentiable: the gradient of a bias."""
    dtype = _hip.require_gpu_float(x)
    features = x.size(-1)
    rows = x.numel() // features
    if not rows:
        return x.new_zeros(features, dtype=torch.float32)
    x = x.contiguous()
    out = x.new_empty(features, dtype=torch.float32)
    nbytes = _column_sums_bytes(rows, features, dtype)
    ws = _hip.workspace(nbytes, x.device)
    _hip.call("s2cnn_column_sums", x.data_ptr(), out.data_ptr(), ws.data_ptr(), nbytes, rows, features, dtype, _hip.stream_ptr())
    return out


def _check_affine(x, weight, bias):
    assert x.dim() >= 1 and x.size(-1) >= 1
    assert weight is None or weight.shape == x.shape[-1:]
    assert bias is None or bias.shape == x.shape[-1:]


def _run(x, residual, weight, bias, eps, p, seed, dtype):
    needs_grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias))
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    return _LayerNorm.apply(x, residual, weight, bias, float(eps), float(p), seed, dtype, needs_grad)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """
    (x - mean) / sqrt(variance + eps) * weight + bias over the last axis, differentiable in x, weight and bias.

    :param x: [..., features]; float32, bfloat16 or float16 (statistics and sums are float32)
    :param weight, bias: [features], the type of x, or None
    :return y: contiguous, the type of x
    """
    _check_affine(x, weight, bias)
    dtype = _hip.require_gpu_float(x, weight, bias)
    return _run(x, None, weight, bias, eps, 0.0, 0, dtype)


def dropout_add_layer_norm(x, residual, p, seed, weight=None, bias=None, eps=1e-5):
    """
    h = residual + dropout(x, p, seed), y = layer_norm(h, weight, bias, eps) in one pass: what stands between two sublayers.

    :param x, residual: [..., features] of one shape and type
    :return (h, y): contiguous; y is formed from h before h is rounded to the type of x, and the gradients from 7 bits more of h than that rounding
        leaves (float32: from h): where a row's offset is d of its deviations, its normalised entries are off by d 2^-16 there (float16: d 2^-19)
    """
    assert residual.shape == x.shape
    _check_affine(x, weight, bias)
    _check_dropout(p, seed)
    dtype = _hip.require_gpu_float(x, residual, weight, bias)
    _require_seed(seed)
    return _run(x, residual, weight, bias, eps, p, seed, dtype)
