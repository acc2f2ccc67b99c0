"""Layers of a transformer over the points of the sphere: every point attends to every other (or to those within an angle), with a
learned bias by the angle of the two and with the quadrature weights of the points, and a learned query attends to all of them
in place of the integral.  The reference has neither (its layers mix places by correlation with a local kernel,
s2cnn/soft/so3_conv.py:36-58, and by the integral at the end, so3_integrate.py:7-31); they go between its layers and its head.

Rotations about the polar axis by a grid step permute the points of a ring and leave angles and weights as they are: the
block commutes with them exactly, with other rotations as far as the grid resolves the signal.
"""
import math

import torch
import torch.nn.functional as F
from torch import nn

from .. import _hip
from ..attention import attention, s2_angle_buckets, s2_log_weights
from ..layer_norm import column_sums, dropout_add_layer_norm, layer_norm
from ..rotary import norm_rotary, rotary as turned, s2_rotary_table
from ..s2_grid import s2_soft_grid


class _BiasGradient(torch.autograd.Function):
    """y, which has had the bias added to its last axis (without a gradient), and the gradient of the bias."""

    @staticmethod
    def forward(ctx, y, bias):  # pylint: disable=W
        ctx.dtype = bias.dtype
        return y.view_as(y)

    @staticmethod
    @_hip.once_differentiable
    def backward(ctx, g):  # pylint: disable=W
        return g, column_sums(g).to(ctx.dtype)


class _Expand(torch.autograd.Function):
    """x [...] for each of n signals: [n, ...], one storage."""

    @staticmethod
    def forward(ctx, x, n):  # pylint: disable=W
        return x.expand(n, *x.shape)

    @staticmethod
    @_hip.once_differentiable
    def backward(ctx, g):  # pylint: disable=W
        return column_sums(g.reshape(g.size(0), -1)).to(g.dtype).view(g.shape[1:]), None


def _sums_of_its_own(x, parameter):
    """Whether the gradient of a parameter that all rows of x share is summed by the library: while a graph is captured.  torch's sum over many
    rows clears a counter with a memset, and replays of a graph with such a node have other gradients from the second on.  Not otherwise:
    nodes of autograd in Python cost an eager step of two blocks 0.12 ms of 2.6."""
    return x.is_cuda and x.dtype in _hip.FLOATS and torch.cuda.is_current_stream_capturing() and parameter.requires_grad and torch.is_grad_enabled()


class Linear(nn.Linear):
    """nn.Linear that can be captured into a graph with its gradients."""

    def forward(self, x):  # pylint: disable=W
        if self.bias is None or not _sums_of_its_own(x, self.bias):
            return super().forward(x)
        return _BiasGradient.apply(F.linear(x, self.weight, self.bias.detach()), self.bias)


class _Norm(nn.Module):
    """Weight and bias of a layer normalisation; the names of nn.LayerNorm."""

    def __init__(self, features):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(features))
        self.bias = nn.Parameter(torch.zeros(features))


class _PointWeights(nn.Module):
    """Logarithms of the quadrature weights, float32 whatever type the module is converted to (`Module.to` leaves integers alone):
    rounded to 16 bits they would be off by a hundredth."""

    def __init__(self, b):
        super().__init__()
        self.register_buffer("bits", s2_log_weights(b).view(torch.int32), persistent=False)

    def forward(self):  # pylint: disable=W
        return self.bits.view(torch.float32)


class _PointTurns(_PointWeights):
    """Cosines and sines of the points' rotations, float32 in the same way."""

    def __init__(self, b, pairs):
        nn.Module.__init__(self)
        self.register_buffer("bits", s2_rotary_table(b, pairs).view(torch.int32), persistent=False)


class S2TransformerBlock(nn.Module):
    """Attention over the 4 b^2 points of the 2b x 2b grid and a pointwise network, each with a residual and a normalisation
    before it.  Between the sublayers the residual, the dropout and the next normalisation are one pass over the features.

    The block takes and gives the pair (h, y): the residual stream, and its normalisation by the block's first norm.  `norm`
    makes the first pair of a stack; the last normalisation of a block is that of the block after it (`next_norm`).

    qk_norm: the queries and keys of each head are normalised, with a learned weight, before their products.  rotary: they are turned by the places of
    the points (`s2_rotary_table`), so that scores depend on the direction from one point to another too, along the circles of latitude and
    across them; rotations about the polar axis still permute the points of a ring, others no longer commute with the block.
    """

    def __init__(self, features, heads, b, n_buckets=32, max_angle=math.pi, hidden=None, dropout=0.0, qk_norm=False, rotary=False):
        super().__init__()
        assert features % heads == 0
        assert not rotary or features // heads >= 2
        self.features, self.heads, self.b, self.dropout = features, heads, b, dropout
        hidden = 2 * features if hidden is None else hidden
        self.norm1, self.norm2 = _Norm(features), _Norm(features)
        self.qkv, self.out = Linear(features, 3 * features), Linear(features, features)
        self.expand, self.contract = Linear(features, hidden), Linear(hidden, features)
        self.bias_table = nn.Parameter(torch.zeros(heads, n_buckets))
        self.register_buffer("buckets", s2_angle_buckets(s2_soft_grid(b), n_buckets=n_buckets, max_angle=max_angle), persistent=False)
        self.log_weights = _PointWeights(b)
        self.qk_norm = qk_norm
        if qk_norm:
            self.q_weight, self.k_weight = (nn.Parameter(torch.ones(features // heads)) for _ in range(2))
        self.turns = _PointTurns(b, features // heads // 2) if rotary else None

    def _placed(self, q, k):
        """Queries and keys as the attention takes them."""
        table = self.turns() if self.turns is not None else None
        if self.qk_norm:
            return norm_rotary(q, k, self.q_weight.to(q.dtype), self.k_weight.to(q.dtype), table)
        return (q, k) if table is None else turned(q, k, table)

    def norm(self, h):
        """(h, y) of the residual stream h [batch, points, features]"""
        return h, layer_norm(h, self.norm1.weight, self.norm1.bias)

    def _step(self, x, h, seed, norm):
        p = self.dropout if self.training else 0.0
        return dropout_add_layer_norm(x.to(h.dtype), h, p, seed, norm.weight, norm.bias)

    def forward(self, h, y, next_norm, seeds):  # pylint: disable=W
        """(h, y) [batch, points, features] -> (h, y), y normalised by next_norm; seeds: two seeds for the dropout of this call"""
        batch, points, features = h.shape
        assert points == 4 * self.b ** 2
        q, k, v = self.qkv(y).view(batch, points, 3, self.heads, features // self.heads).permute(2, 0, 3, 1, 4)
        q, k = self._placed(q, k)
        x = attention(q, k, v, table=self.bias_table.to(q.dtype), buckets=self.buckets, key_bias=self.log_weights())
        x = self.out(x.transpose(1, 2).reshape(batch, points, features))
        h, y = self._step(x, h, seeds[0], self.norm2)
        x = self.contract(F.relu(self.expand(y)))
        return self._step(x, h, seeds[1], next_norm)


class S2AttentionPool(nn.Module):
    """One learned query per head attends to all points, with their quadrature weights: [batch, points, features] ->
    [batch, features].  With queries of zeros (as at the start) it is the integral of the values over the sphere."""

    def __init__(self, features, heads, b):
        super().__init__()
        assert features % heads == 0
        self.heads = heads
        self.query = nn.Parameter(torch.zeros(heads, 1, features // heads))
        self.kv = Linear(features, 2 * features)
        self.log_weights = _PointWeights(b)

    def forward(self, y):  # pylint: disable=W
        batch, points, features = y.shape
        k, v = self.kv(y).view(batch, points, 2, self.heads, features // self.heads).permute(2, 0, 3, 1, 4)
        q = self.query.to(k.dtype)
        q = _Expand.apply(q, batch) if _sums_of_its_own(k, q) else q.expand(batch, -1, -1, -1)
        return attention(q, k, v, key_bias=self.log_weights()).reshape(batch, features)


class S2Transformer(nn.Module):
    """A stack of blocks and the pooling after it: [batch, features, 2b, 2b] -> [batch, features].  `drops` counts the forward passes on
    the device, so that each training step drops others, replayed from a graph too.

    A pass that is run again in the backward pass, to save memory, has to drop what the first one did: its seeds are taken before it and
    given to both, `checkpoint(model, x, model.next_seeds())`.  Without them it is refused there.

    What is dropped is a function of `seed` and of the count alone, not of torch's generator: stacks of one network, the ranks of a
    data-parallel job and runs that are to differ need a `seed` each (`torch.initial_seed() + rank`, say).  Its low 32 bits count, and stacks
    in which they differ never use the same number.  It is the program's to keep, as the learning rate is: no part of the state dict.

    qk_norm, rotary: of the blocks."""

    def __init__(self, features, heads, b, layers, n_buckets=32, max_angle=math.pi, dropout=0.0, seed=0, qk_norm=False, rotary=False):
        super().__init__()
        self.blocks = nn.ModuleList(S2TransformerBlock(features, heads, b, n_buckets, max_angle, dropout=dropout, qk_norm=qk_norm, rotary=rotary)
                                    for _ in range(layers))
        self.last_norm = _Norm(features)
        self.pool = S2AttentionPool(features, heads, b)
        self.register_buffer("drops", torch.zeros(1, dtype=torch.int64))
        high = (seed & 0xFFFFFFFF) << 32                                    # the count takes the low 32 bits
        self.base = high - (1 << 64) if high >> 63 else high                # no buffer: data-parallel jobs hand those of one rank to all
        self.register_buffer("calls", torch.arange(2 * layers), persistent=False)

    def next_seeds(self):
        """The seeds of the dropouts of one pass in training, [2 layers]: others at each call."""
        self.drops.add_(1)
        return torch.add(self.calls, self.drops, alpha=2 * len(self.blocks)).add_(self.base)

    def forward(self, x, seeds=None):  # pylint: disable=W
        """seeds: from next_seeds, or None to count one pass on"""
        if self.training and seeds is None:
            if torch._C._current_graph_task_id() != -1 and any(block.dropout for block in self.blocks):
                raise RuntimeError("S2Transformer run again in the backward pass: it would drop other elements than before; give it the seeds of next_seeds()")
            seeds = self.next_seeds()
        seeds = (seeds if self.training else self.calls).split(1)
        h = x.flatten(2).transpose(1, 2).contiguous()                       # [batch, points, features]
        h, y = self.blocks[0].norm(h)
        for i, block in enumerate(self.blocks):
            following = self.blocks[i + 1].norm1 if i + 1 < len(self.blocks) else self.last_norm
            h, y = block(h, y, following, seeds[2 * i:2 * i + 2])
        return self.pool(y)
