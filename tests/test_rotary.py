"""rotary, norm_rotary and rotary_table (s2cnn_amd/rotary.py) against complex products and the formulas in 64 bits on the CPU.

Tolerances, in the 2-norm.  u = 2^-24, 2^-8, 2^-11 is the unit roundoff of float32, bfloat16, float16.  A turned entry is two products and a sum, whose
roundings are together at most 3 u of the pair's size; cosines and sines are read, not formed: 4 * 2^-24.  With the normalisation come the sum of up to 256
squares (random roundings: below 8 u), a root and up to four products: 16 * 2^-24.  16-bit results are rounded once more, by at most u.  The gradient
subtracts a mean of the vector's entries: 16 * 2^-24 of the size of what is subtracted on top.  Sums over vectors are float32 sums:
16 * 2^-24 of the 2-norm of the sums of magnitudes on top (n at most some thousand, in parts).  Entries of the table: an angle to 2^-53 of its
turns (below 2^26), its rest in float32 (2^-25 of a quarter turn) and one or two roundings of a value up to one: 4 * 2^-24 each."""
import ctypes
import importlib
import math

import pytest
import torch
from torch.autograd import forward_ad

import s2cnn_amd

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
LAYOUTS = pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
UNIT = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
EPS = 1e-6

# batch, heads, kv_heads, n, d, pairs
SHAPES = [(2, 3, 1, 5, 2, 1), (1, 1, 1, 1, 3, 1), (3, 2, 2, 7, 7, 3), (2, 4, 2, 9, 8, 4), (2, 6, 6, 50, 16, 8), (3, 5, 5, 40, 20, 10), (2, 3, 3, 11, 20, 3),
          (1, 7, 1, 13, 31, 15), (2, 2, 1, 30, 33, 16), (2, 3, 3, 21, 50, 25), (2, 8, 2, 65, 64, 32), (2, 8, 8, 33, 64, 24), (1, 4, 4, 20, 64, 5), (1, 4, 2, 17, 100, 50),
          (2, 6, 3, 14, 113, 28), (2, 8, 2, 40, 128, 64), (1, 3, 3, 10, 129, 64), (1, 2, 2, 9, 254, 125), (1, 2, 1, 11, 255, 120), (2, 2, 2, 19, 256, 128),
          (1, 1, 1, 3000, 24, 12)]
IDS = ["x".join(map(str, s)) for s in SHAPES]


def _close(got, want, dtype, what, chain=4, extra=0.0):
    assert got.dtype == dtype and got.shape == want.shape, what
    got = got.detach().cpu().double()
    allowed = (chain * 2.0 ** -24 + UNIT[dtype]) * want.norm().item() + 16 * 2.0 ** -24 * float(extra)
    assert torch.isfinite(got).all() and (got - want).norm().item() <= allowed, (what, (got - want).norm().item(), allowed)


def _turned(x, table, interleaved, back=False):
    """x [..., d] in 64 bits, turned by the complex numbers of the table [..., pairs, 2]"""
    p = table.size(-2)
    z = torch.view_as_complex(table.double().contiguous())
    z = z.conj() if back else z
    first, second = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if interleaved else (slice(0, p), slice(p, 2 * p))
    w = torch.complex(x[..., first], x[..., second]) * z
    y = x.clone()
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _gradients(x, weight, g):
    """(y before the rotation, gx, gw, sizes of the two parts of gx, magnitudes of gw) of the normalisation"""
    d = x.size(-1)
    size = torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS)
    u = g * weight
    mean = (u * x).sum(-1, keepdim=True) / d
    gx = u / size - x * mean / size ** 3
    gw = g * x / size
    return x / size * weight, gx, gw.sum((0, 1, 2)), (u / size).norm() + (x * mean / size ** 3).norm(), gw.abs().sum((0, 1, 2)).norm()


def _table(rows, pairs, batch=None):
    g = torch.Generator().manual_seed(rows * 100 + pairs)
    angles = torch.rand(*((batch,) if batch else ()), rows, pairs, generator=g, dtype=torch.float64) * 2 * math.pi
    return torch.stack([angles.cos(), angles.sin()], -1).float()


def _make(shape, dtype, seed=0):
    """q, k as views of a projection's output, weights, gradients with the heads' axis outside"""
    b, h, hk, n, d, _ = shape
    gen = torch.Generator().manual_seed(sum(shape) * 10007 + seed)
    x = (torch.randn(b, n, h + 2 * hk, d, generator=gen) * 1.5 + 0.25).to(dtype).cuda()
    weights = [(torch.randn(d, generator=gen) * 0.2 + 1).to(dtype).cuda() for _ in range(2)]
    grads = [torch.randn(b, heads, n, d, generator=gen).to(dtype).cuda() for heads in (h, hk)]
    return x[:, :, :h].transpose(1, 2), x[:, :, h:h + hk].transpose(1, 2), weights, grads


def _cpu(*tensors):
    return [t.detach().cpu().double() for t in tensors]


@pytest.mark.gpu
@TYPES
@LAYOUTS
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_rotary(hip, shape, interleaved, dtype):
    q, k, _, (gq, gk) = _make(shape, dtype)
    table = _table(shape[3], shape[5])
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    out = s2cnn_amd.rotary(q, k, table.cuda(), interleaved=interleaved)
    grads = torch.autograd.grad(out, [q, k], [gq, gk])
    for x, y, g, gx, name in zip((q, k), out, (gq, gk), grads, "qk"):
        xd, gd = _cpu(x, g)
        _close(y, _turned(xd, table, interleaved), dtype, name)
        _close(gx, _turned(gd, table, interleaved, back=True), dtype, "gradient of " + name)
        assert torch.equal(y[..., 2 * shape[5]:], x[..., 2 * shape[5]:])
    with torch.no_grad():
        alone, none = s2cnn_amd.rotary(k, None, table.cuda(), interleaved=interleaved)
    assert none is None and torch.equal(alone, out[1])
    only, = torch.autograd.grad(s2cnn_amd.rotary(q, k, table.cuda(), interleaved=interleaved)[1], [k], gk)
    assert torch.equal(only, grads[1])


@pytest.mark.gpu
@TYPES
@LAYOUTS
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_norm_rotary(hip, shape, interleaved, dtype):
    q, k, weights, gs = _make(shape, dtype, seed=1)
    table = _table(shape[3], shape[5])
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights)]
    out = s2cnn_amd.norm_rotary(*leaves, table.cuda(), eps=EPS, interleaved=interleaved)
    grads = torch.autograd.grad(out, leaves, gs)
    for i, name in enumerate("qk"):
        x, w, g = _cpu(leaves[i], leaves[2 + i], gs[i])
        y, gx, gw, parts, magnitudes = _gradients(x, w, _turned(g, table, interleaved, back=True))
        _close(out[i], _turned(y, table, interleaved), dtype, name, 16)
        _close(grads[i], gx, dtype, "gradient of " + name, 16, parts)
        _close(grads[2 + i], gw, dtype, "gradient of the weight of " + name, 16, magnitudes)
    again = torch.autograd.grad(s2cnn_amd.norm_rotary(*leaves, table.cuda(), eps=EPS, interleaved=interleaved), leaves, gs)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(s2cnn_amd.norm_rotary(*leaves, table.cuda(), eps=EPS, interleaved=interleaved), out))


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("shape", [(2, 3, 1, 5, 1, 0), (2, 4, 2, 30, 20, 0), (1, 2, 2, 7, 33, 0), (3, 8, 4, 50, 128, 0)], ids=lambda s: "x".join(map(str, s)))
@LAYOUTS
def test_norm_without_table_or_weights(hip, shape, interleaved, dtype):
    q, k, _, gs = _make(shape, dtype, seed=2)
    leaves = [t.detach().requires_grad_() for t in (q, k)]
    out = s2cnn_amd.norm_rotary(*leaves, eps=EPS, interleaved=interleaved)
    grads = torch.autograd.grad(out, leaves, gs)
    for i, name in enumerate("qk"):
        x, g = _cpu(leaves[i], gs[i])
        y, gx, _, parts, _ = _gradients(x, torch.ones(shape[4], dtype=torch.float64), g)
        _close(out[i], y, dtype, name, 16)
        _close(grads[i], gx, dtype, "gradient of " + name, 16, parts)


@pytest.mark.gpu
@LAYOUTS
@pytest.mark.parametrize("per_batch", [False, True])
@pytest.mark.parametrize("normed", [False, True])
def test_rows_by_index(hip, normed, per_batch, interleaved):
    """Rows in any order, twice, below zero (not turned) and behind the last (NaN), tables and indexes for each signal or for all."""
    b, h, hk, n, d, pairs, rows = 3, 4, 2, 10, 40, 18, 23
    q, k, weights, gs = _make((b, h, hk, n, d, pairs), F32, seed=3)
    weights = weights if normed else []
    for tables in (None, b):
        table = _table(rows, pairs, tables)
        index = torch.randint(0, rows, (b, n) if per_batch else (n,), generator=torch.Generator().manual_seed(7), dtype=torch.int32)
        index[..., 0], index[..., 1], index[..., 2], index[..., 3] = 0, rows - 1, -1, -2 ** 31
        taken = table[torch.arange(b).view(b, 1), index.expand(b, n).long().clamp(min=0)] if tables else table[index.expand(b, n).long().clamp(min=0)]
        taken = torch.where((index.expand(b, n) < 0).view(b, n, 1, 1), torch.tensor([1.0, 0.0]), taken).unsqueeze(1)
        leaves = [t.detach().requires_grad_() for t in (q, k, *weights)]
        run = s2cnn_amd.norm_rotary if normed else s2cnn_amd.rotary
        kw = {"eps": EPS} if normed else {}
        out = run(*leaves, table.cuda(), index=index.cuda(), interleaved=interleaved, **kw)
        grads = torch.autograd.grad(out, leaves, gs)
        for i in range(2):
            x, g = _cpu(leaves[i], gs[i])
            g = _turned(g, taken, interleaved, back=True)
            if not normed:
                _close(out[i], _turned(x, taken, interleaved), F32, "y")
                _close(grads[i], g, F32, "gx")
                continue
            y, gx, gw, parts, magnitudes = _gradients(x, weights[i].cpu().double(), g)
            _close(out[i], _turned(y, taken, interleaved), F32, "y", 16)
            _close(grads[i], gx, F32, "gx", 16, parts)
            _close(grads[2 + i], gw, F32, "gw", 16, magnitudes)
        wrong = index.clone()
        wrong[..., 5] = rows
        wrong[..., 6] = 2 ** 31 - 1
        with torch.no_grad():
            bad = run(*leaves, table.cuda(), index=wrong.cuda(), interleaved=interleaved, **kw)
        for a, y in zip(bad, out):
            assert a[:, :, 5:7, :2 * pairs].isnan().all() and torch.isfinite(a[:, :, 5:7, 2 * pairs:]).all()
            assert torch.equal(a[:, :, :5], y[:, :, :5]) and torch.equal(a[:, :, 7:], y[:, :, 7:])


@pytest.mark.gpu
@LAYOUTS
@pytest.mark.parametrize("per_batch", [False, True])
def test_gradients_with_fewer_rows_than_places(hip, per_batch, interleaved):
    """Packed sequences and places that share rows: weights' gradients too, with one index for all signals or one for each."""
    b, h, hk, n, d, pairs, rows = 3, 4, 2, 40, 24, 10, 7
    q, k, weights, gs = _make((b, h, hk, n, d, pairs), F32, seed=4)
    table = _table(rows, pairs)
    index = torch.randint(0, rows, (b, n) if per_batch else (n,), generator=torch.Generator().manual_seed(8), dtype=torch.int32)
    taken = table[index.expand(b, n).long()].unsqueeze(1)
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights)]
    out = s2cnn_amd.norm_rotary(*leaves, table.cuda(), index=index.cuda(), eps=EPS, interleaved=interleaved)
    grads = torch.autograd.grad(out, leaves, gs)
    for i in range(2):
        x, w, g = _cpu(leaves[i], weights[i], gs[i])
        y, gx, gw, parts, magnitudes = _gradients(x, w, _turned(g, taken, interleaved, back=True))
        _close(out[i], _turned(y, taken, interleaved), F32, "y", 16)
        _close(grads[i], gx, F32, "gx", 16, parts)
        _close(grads[2 + i], gw, F32, "gw", 16, magnitudes)


@pytest.mark.gpu
@TYPES
def test_orders_of_axes(hip, dtype):
    """Any strides: heads outside or inside, expanded, every other vector, a strided last axis, addresses at odd entries."""
    b, h, n, d, pairs = 2, 3, 8, 24, 12
    table = _table(n, pairs).cuda()
    gen = torch.Generator().manual_seed(0)
    base = torch.randn(b, h, n, d, generator=gen).to(dtype).cuda()
    w = (torch.randn(d, generator=gen) + 1).to(dtype).cuda()
    want = s2cnn_amd.norm_rotary(base, None, w, table=table)[0]
    flat, wide = (torch.empty(1 + 2 * b * h * n * (d + 3) * size, dtype=dtype, device="cuda") for size in (1, 2))
    views = [base.transpose(1, 2).contiguous().transpose(1, 2), base.permute(2, 0, 3, 1).contiguous().permute(1, 3, 0, 2),
             flat[1:].as_strided((b, h, n, d), (2 * h * n * (d + 3), (d + 3) * n, d + 3, 1)).copy_(base),
             wide.as_strided((b, h, n, d), (2 * d, 2 * b * d, 2 * b * d * h, 2)).copy_(base)]
    for v in views:
        assert torch.equal(v, base)
        y = s2cnn_amd.norm_rotary(v, None, w, table=table)[0]
        assert torch.equal(y, want)
        leaf = v.detach().requires_grad_()
        y = s2cnn_amd.norm_rotary(leaf, None, w, table=table)[0]
        one, = torch.autograd.grad(y, leaf, torch.ones((), dtype=dtype, device="cuda").expand_as(y))
        leaf = base.detach().requires_grad_()
        two, = torch.autograd.grad(s2cnn_amd.norm_rotary(leaf, None, w, table=table)[0], leaf, torch.ones_like(y).contiguous())
        assert torch.equal(one, two)
    once = base[:1, :1].expand(b, h, n, d)
    assert torch.equal(s2cnn_amd.rotary(once, None, table)[0], s2cnn_amd.rotary(once.contiguous(), None, table)[0])


@pytest.mark.gpu
def test_gradients_by_differences(hip):
    """float32: central differences of the loss along random directions, at steps where the second-order rest and the roundings are some 1e-4."""
    b, h, hk, n, d, pairs = 2, 3, 1, 6, 22, 9
    q, k, weights, gs = _make((b, h, hk, n, d, pairs), F32, seed=5)
    table = _table(n, pairs).cuda()
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights)]
    loss = lambda ts: sum((y.double() * g.double()).sum() for y, g in zip(s2cnn_amd.norm_rotary(*ts, table, eps=EPS), gs))
    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator().manual_seed(9)
    for i, t in enumerate(leaves):
        way = torch.randn(t.shape, generator=gen).cuda()
        step = 2.0 ** -7
        with torch.no_grad():
            up, down = (loss([x + s * step * way if j == i else x for j, x in enumerate(leaves)]) for s in (1, -1))
        slope = (up - down) / (2 * step)
        assert abs(slope - (grads[i].double() * way.double()).sum()) <= 2e-3 * (grads[i].double().norm() * way.double().norm() / math.sqrt(t.numel()) + 1)


@pytest.mark.gpu
def test_large_small_and_infinite_entries(hip):
    x = torch.zeros(1, 1, 6, 16, device="cuda")
    x[0, 0, 1] = 1e15
    x[0, 0, 2] = 1e-30
    x[0, 0, 3, 0] = float("inf")
    x[0, 0, 4, 0] = float("nan")
    x[0, 0, 5] = 1.0
    table = _table(6, 8).cuda()
    y = s2cnn_amd.norm_rotary(x, None, table=table)[0][0, 0]
    assert (y[0] == 0).all() and torch.isfinite(y[1:3]).all() and torch.isfinite(y[5]).all() and y[3:5].isnan().any(-1).all()
    assert abs(y[1].norm().item() - 4) < 1e-5 and y[2].abs().max() < 1e-26
    least = s2cnn_amd.norm_rotary(x, None, table=table, eps=2.0 ** -126)[0][0, 0]
    assert (least[0] == 0).all() and torch.isfinite(least[2]).all() and abs(least[5].norm().item() - 4) < 1e-5
    turned = s2cnn_amd.rotary(x, None, table)[0][0, 0]
    assert torch.isfinite(turned[[0, 1, 2, 5]]).all() and torch.isfinite(turned[3, 1:8]).all() and torch.isfinite(turned[3, 9:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [256, 255, 4, 1])
def test_largest_entries_of_a_normalisation(hip, d, dtype):
    """All entries just below the documented 2^59, at the largest d too, forward and backward; one entry of a single one just below 2^63.5."""
    gen = torch.Generator().manual_seed(d)
    below = 1 - 2.0 ** -8
    x = torch.where(torch.rand(1, 2, 5, d, generator=gen) < 0.5, -below, below).double()
    x[:, 1] *= torch.rand(1, 5, d, generator=gen)
    x *= 2.0 ** 59
    if d == 1:
        x.copy_(x.sign() * below * 2.0 ** 63.5)
    x = x.to(dtype)
    pairs = d // 2
    table = _table(5, pairs) if pairs else None
    g, w = torch.randn(1, 2, 5, d, generator=gen).to(dtype), (torch.rand(d, generator=gen) + 0.5).to(dtype)
    leaf = x.cuda().requires_grad_()
    y = s2cnn_amd.norm_rotary(leaf, None, w.cuda(), table=table.cuda() if pairs else None, eps=EPS)[0]
    gx, = torch.autograd.grad(y, leaf, g.cuda())
    xd, gd = x.double(), _turned(g.double(), table, False, back=True) if pairs else g.double()
    want, want_gx, _, parts, _ = _gradients(xd, w.double(), gd)
    _close(y, _turned(want, table, False) if pairs else want, dtype, "y", 16)
    _close(gx * 2.0 ** 40, want_gx * 2.0 ** 40, dtype, "gx", 16, parts * 2.0 ** 40)
    assert float(y.detach().float().norm()) > 1


@pytest.mark.gpu
@TYPES
@LAYOUTS
@pytest.mark.parametrize("d,pairs", [(64, 24), (64, 8), (40, 3), (23, 9), (7, 3), (128, 13)])
def test_what_is_not_turned_stays_bit_by_bit(hip, d, pairs, interleaved, dtype):
    """Entries behind the pairs, and vectors whose row is below zero, beside infinities, what is no number and zeros with a sign; gradients likewise."""
    n = 9
    gen = torch.Generator().manual_seed(d)
    x, g = (torch.randn(2, 2, n, d, generator=gen) for _ in range(2))
    for t in (x, g):
        t[torch.rand(t.shape, generator=gen) < 0.2] = -0.0
        t[torch.rand(t.shape, generator=gen) < 0.1] = math.inf
        t[torch.rand(t.shape, generator=gen) < 0.1] = math.nan
        t[..., 2 * pairs] = -math.inf
    x, g = (t.to(dtype).cuda() for t in (x, g))
    table = _table(n, pairs).cuda()
    index = torch.arange(n, dtype=torch.int32)
    index[::3] = -1
    leaf = x.detach().requires_grad_()
    y = s2cnn_amd.rotary(leaf, None, table, index=index.cuda(), interleaved=interleaved)[0]
    gx, = torch.autograd.grad(y, leaf, g)
    bits = torch.int32 if dtype == F32 else torch.int16
    for got, of in ((y.detach(), x), (gx, g)):
        assert torch.equal(got[..., 2 * pairs:].contiguous().view(bits), of[..., 2 * pairs:].contiguous().view(bits))
        assert torch.equal(got[:, :, ::3].contiguous().view(bits), of[:, :, ::3].contiguous().view(bits))
        # a pair with only finite entries has a finite result
        halves = (lambda t: (t[..., :2 * pairs:2], t[..., 1:2 * pairs:2])) if interleaved else (lambda t: (t[..., :pairs], t[..., pairs:2 * pairs]))
        one, two = (torch.isfinite(h)[:, :, 1::3] for h in halves(of))
        assert all(torch.equal(torch.isfinite(h)[:, :, 1::3], one & two) for h in halves(got))


@pytest.mark.gpu
@TYPES
def test_nothing_beside_the_vectors_is_written_or_read(hip, dtype):
    """Vectors with gaps between them that hold NaN, results in a tensor of the same form."""
    b, h, n, d, pairs = 2, 2, 5, 21, 9
    buffer = torch.full((b, n, h, d + 5), float("nan"), dtype=dtype, device="cuda")
    q = buffer[..., 2:2 + d].transpose(1, 2)
    q.copy_(torch.randn(b, h, n, d, generator=torch.Generator().manual_seed(1)))
    table = _table(n, pairs).cuda()
    for interleaved in (False, True):
        y = s2cnn_amd.norm_rotary(q, None, table=table, interleaved=interleaved)[0]
        assert torch.isfinite(y).all() and torch.equal(y, s2cnn_amd.norm_rotary(q.contiguous(), None, table=table, interleaved=interleaved)[0])


@pytest.mark.gpu
def test_many_vectors_and_far_offsets(hip):
    """More vectors than the workgroups take at once, and offsets past 2^32 bytes, against the same vectors in pieces."""
    n, d = 70001, 64
    table = _table(n, 32).cuda()
    base = torch.empty(2, n, 320, d, dtype=BF16, device="cuda")                    # 5.7 GB
    q, k = base[:, :, :2].transpose(1, 2), base[:, :, 317:].transpose(1, 2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for t in (q, k):
        t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
    y, z = s2cnn_amd.norm_rotary(q, k, table=table)
    for at in (0, 31111, n - 1000):
        part, other = s2cnn_amd.norm_rotary(q[:, :, at:at + 1000].contiguous(), k[:, :, at:at + 1000].contiguous(), table=table[at:at + 1000])
        assert torch.equal(y[:, :, at:at + 1000], part) and torch.equal(z[:, :, at:at + 1000], other)


@pytest.mark.gpu
@LAYOUTS
def test_tensors_larger_than_the_caches(hip, interleaved):
    """From 256 MB on accesses go past the caches: the same bits as in pieces, forward and backward."""
    n, d, pairs = 300001, 64, 32
    table = _table(n, pairs).cuda()
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, g = (torch.randn(1, n, 8, d, device="cuda", generator=gen).bfloat16().transpose(1, 2) for _ in range(2))
    w = (torch.rand(d, device="cuda", generator=gen) + 0.5).bfloat16()

    def both(x, g, table):
        x = x.detach().requires_grad_()
        y = s2cnn_amd.norm_rotary(x, None, w, table=table, interleaved=interleaved)[0]
        return y.detach(), torch.autograd.grad(y, x, g)[0], s2cnn_amd.rotary(x.detach(), None, table, interleaved=interleaved)[0]

    whole = both(x, g, table)
    for at in (0, 123457, n - 1000):
        part = both(*(t[:, :, at:at + 1000] for t in (x, g)), table[at:at + 1000])
        assert all(torch.equal(a[:, :, at:at + 1000], b) for a, b in zip(whole, part))


@pytest.mark.gpu
def test_tables_at_any_address_and_stride(hip):
    n, d, pairs = 20, 24, 9
    table = _table(n, pairs).cuda()
    x = torch.randn(2, 3, n, d, generator=torch.Generator().manual_seed(2)).cuda()
    want = s2cnn_amd.rotary(x, None, table)[0]
    flat = torch.empty(1 + table.numel(), device="cuda")
    for t in (flat[1:].view(table.shape).copy_(table), table.permute(2, 0, 1).contiguous().permute(1, 2, 0), table.expand(2, n, pairs, 2),
              torch.cat([table, table], -1)[..., :2]):
        assert torch.equal(t.expand_as(table) if t.dim() == 3 else t[0], table) and torch.equal(s2cnn_amd.rotary(x, None, t)[0], want)


@pytest.mark.gpu
def test_empty_tensors(hip):
    table = _table(4, 3).cuda()
    w = torch.ones(6, device="cuda", requires_grad=True)
    for shape, rows in (((0, 2, 4, 6), 4), ((2, 0, 4, 6), 4), ((2, 2, 0, 6), 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        other = torch.ones(shape[0], 1, shape[2], 6, device="cuda", requires_grad=True)
        y, z = s2cnn_amd.norm_rotary(x, other, w, w, table=table[:rows])
        assert y.shape == shape and z.shape == other.shape
        gx, gw = torch.autograd.grad(y.sum() + 0 * z.sum(), [x, w])
        assert gx.shape == shape and (gw == 0).all()
        assert s2cnn_amd.rotary(x, None, table[:rows])[0].shape == shape


@pytest.mark.gpu
def test_captured_steps_and_other_streams(hip):
    """Forward and backward pass captured into a graph, replayed with other inputs between eager calls, on a stream that is not the default one."""
    shape = (2, 4, 2, 100, 32, 16)
    table = _table(100, 16).cuda()
    (q, k, weights, gs), (q2, k2, _, gs2) = _make(shape, BF16, 6), _make(shape, BF16, 7)
    static = [q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_()]
    ws, grads_in = [w.detach().requires_grad_() for w in weights], [g.clone() for g in gs]

    def step(q, k, gs):
        out = s2cnn_amd.norm_rotary(q, k, *ws, table)
        grads = torch.autograd.grad(out, [q, k, *ws], gs)
        return (*(t.detach() for t in out), *grads)                    # no graph stays alive

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step(*static, grads_in)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*static, grads_in)
    for a, b, g in ((q, k, gs), (q2, k2, gs2), (q, k, gs)):
        want = step(a.detach().requires_grad_(), b.detach().requires_grad_(), g)
        with torch.no_grad():
            for to, of in zip((*static, *grads_in), (a, b, *g)):
                to.copy_(of)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, want))
    assert all(torch.equal(x, y) for x, y in zip(eager, want))


# ---- the table ------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.float64, torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("shape,axes,pairs", [((1,), 1, 1), ((3, 23), 3, 8), ((1000,), 1, 64), ((5, 7), 2, 33), ((300,), 2, 128), ((2, 3, 4), 1, 100)], ids=str)
def test_rotary_table(hip, shape, axes, pairs, kind):
    gen = torch.Generator().manual_seed(pairs)
    positions = torch.randint(-10 ** 6, 10 ** 6, (*shape, axes), generator=gen).to(kind) if kind not in (torch.float32, torch.float64) else \
        torch.randn(*shape, axes, generator=gen, dtype=torch.float64).mul_(100.0).to(kind)
    frequencies = torch.randn(axes, pairs, generator=gen, dtype=torch.float64)
    table = s2cnn_amd.rotary_table(positions.cuda(), frequencies.cuda(), scale=1.5)
    assert table.shape == (*shape, pairs, 2) and table.dtype == F32
    angles = (positions.double().unsqueeze(-1) * frequencies).sum(-2)
    # 64-bit angles of up to 2^22: off by 2^-30 themselves
    want = 1.5 * torch.stack([angles.cos(), angles.sin()], -1)
    assert (table.cpu().double() - want).abs().max() <= 1.5 * 4 * 2.0 ** -24
    assert (table.cpu().double().square().sum(-1) - 2.25).abs().max() <= 2.25 * 8 * 2.0 ** -24


@pytest.mark.gpu
def test_rotary_table_is_rounded_little_more_than_once(hip):
    """Entries that a sine's polynomial gives (below 0.7 in size), x in quarter turns, u = 2^-24: the result's rounding u / 2, x's 2^-26 by at most 1.45 (1.36
    where the result is above a half: 0.34 u), the product beyond pi/2 x, of at most 0.08: two roundings of its relative size and its own, 0.22 u, and what the
    polynomial leaves, below 0.04 u: 1.1 u in all.  Cosines' (above 0.71): the result's u / 2, x's 2^-26 by at most 1.12 (0.28 u), the square's and
    two more of at most 0.31: 0.5 u: 1.3 u.  Far places: the angle's own three roundings of 2^24 turns, 0.6 u."""
    places = torch.linspace(-9.0, 9.0, 1000003, dtype=torch.float64).view(-1, 1)
    f = torch.ones(1, 1, dtype=torch.float64)
    for base, more in ((0.0, 0.0), (2.0 ** 23 * 2 * math.pi, 0.3)):
        p = places + base
        got = s2cnn_amd.rotary_table(p.cuda(), f.cuda()).cpu().double().flatten()
        want = torch.stack([p.cos(), p.sin()], -1).flatten()
        off = (got - want).abs() * 2.0 ** 24
        assert off[want.abs() < 0.7].max() <= 1.1 + more and off[want.abs() > 0.71].max() <= 1.3 + more


@pytest.mark.gpu
def test_rotary_table_of_quarter_turns_and_far_places(hip):
    f = torch.tensor([[math.pi / 2, 2 * math.pi, 1.0]], dtype=torch.float64).cuda()
    t = s2cnn_amd.rotary_table(torch.arange(-4, 9).view(-1, 1).cuda(), f).cpu()
    for i, n in enumerate(range(-4, 9)):
        assert (t[i, 0] - torch.tensor([[1.0, 0.0], [0.0, 1.0], [-1.0, 0.0], [0.0, -1.0]][n % 4])).abs().max() < 1e-6
        assert (t[i, 1] - torch.tensor([1.0, 0.0])).abs().max() < 1e-6
    far = torch.tensor([[2 ** 31], [2 ** 28 + 1], [-(2 ** 30)]])
    t = s2cnn_amd.rotary_table(far.cuda(), f[:, 2:]).cpu().double()
    for i, n in enumerate(far.flatten().tolist()):        # 2^29 turns: 2^-24 of a turn left of 53 bits, times 2 pi
        assert abs(t[i, 0, 0].item() - math.cos(n)) < 4e-6 and abs(t[i, 0, 1].item() - math.sin(n)) < 4e-6
    assert s2cnn_amd.rotary_table(torch.full((2, 1), float("inf"), device="cuda"), f).isnan().all()
    assert s2cnn_amd.rotary_table(torch.zeros(0, 1, device="cuda"), f).shape == (0, 3, 2)


@pytest.mark.gpu
def test_scores_depend_on_differences_of_positions(hip):
    """What it is for: q . k is the same for all pairs of places as far apart; on the sphere it commutes with a turn about the polar axis."""
    d, n = 32, 50
    gen = torch.Generator().manual_seed(0)
    q, k = (torch.randn(1, 1, 1, d, generator=gen).expand(1, 1, n, d).cuda() for _ in range(2))
    table = s2cnn_amd.rotary_table(torch.arange(n).view(n, 1).cuda(), s2cnn_amd.rotary_frequencies(d // 2, device="cuda"))
    y, z = s2cnn_amd.rotary(q, k, table)
    scores = y[0, 0].double() @ z[0, 0].double().T
    for gap in (0, 3, 17):
        line = torch.diagonal(scores, gap)
        assert (line - line[0]).abs().max() < 1e-4
    b = 3
    table = s2cnn_amd.s2_rotary_table(b, d // 2).cuda()
    q, k = (t[:, :, :1].expand(1, 1, 4 * b * b, d) for t in (q, k))
    y, z = s2cnn_amd.rotary(q, k, table)
    scores = (y[0, 0].double() @ z[0, 0].double().T).view(2 * b, 2 * b, 2 * b, 2 * b)
    assert (scores - scores.roll((1, 1), (1, 3))).abs().max() < 1e-4


# ---- without a GPU --------------------------------------------------------------------------------------------------
def test_frequencies():
    f = s2cnn_amd.rotary_frequencies(4, base=16.0)
    assert f.shape == (1, 4) and f.dtype == torch.float64 and torch.allclose(f, torch.tensor([[1.0, 0.5, 0.25, 0.125]], dtype=torch.float64))
    assert torch.allclose(s2cnn_amd.rotary_frequencies(4, base=16.0, factor=4.0), f / 4)
    g = s2cnn_amd.rotary_frequencies(64, factor=4.0, original=4096)
    f = s2cnn_amd.rotary_frequencies(64)
    turns = 4096 * f / (2 * math.pi)
    assert (g[turns >= 32] == f[turns >= 32]).all() and torch.allclose(g[turns <= 1], f[turns <= 1] / 4) and (g <= f).all() and (g >= f / 4 * (1 - 1e-12)).all()
    assert (g[0, 1:] < g[0, :-1]).all()
    s = s2cnn_amd.s2_rotary_frequencies(5)
    assert s.tolist() == [[0, 1, 0, 2, 0], [1, 0, 2, 0, 3]]
    t = s2cnn_amd.s2_rotary_table(2, 3)
    beta, alpha = torch.tensor(s2cnn_amd.s2_soft_grid(2), dtype=torch.float64).T
    assert t.shape == (16, 3, 2) and torch.allclose(t[:, 1, 0].double(), beta.cos(), atol=1e-6) and torch.allclose(t[:, 2, 1].double(), (2 * alpha).sin(), atol=1e-6)


def test_refusals_before_the_gpu():
    q, k, table = torch.zeros(2, 4, 5, 8), torch.zeros(2, 2, 5, 8), torch.zeros(5, 4, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.rotary(q, k, table)
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.norm_rotary(q, k)
    for bad in (lambda: s2cnn_amd.rotary(q, k, None), lambda: s2cnn_amd.rotary(q[0], k, table), lambda: s2cnn_amd.rotary(q, k[:, :, :4], table),
                lambda: s2cnn_amd.rotary(q, k[..., :6], table), lambda: s2cnn_amd.rotary(q, k[:1], table), lambda: s2cnn_amd.rotary(q, k, torch.zeros(5, 5, 2)),
                lambda: s2cnn_amd.rotary(q, k, table[:4]), lambda: s2cnn_amd.rotary(q, k, torch.zeros(6, 4, 2)), lambda: s2cnn_amd.rotary(q, k, torch.zeros(3, 5, 4, 2)),
                lambda: s2cnn_amd.rotary(q, k, torch.zeros(5, 4, 3)), lambda: s2cnn_amd.rotary(q, k, torch.zeros(5, 0, 2)),
                lambda: s2cnn_amd.rotary(q, k, table, index=torch.zeros(4, dtype=torch.int32)), lambda: s2cnn_amd.rotary(q, k, table.requires_grad_()),
                lambda: s2cnn_amd.norm_rotary(q, k, index=torch.zeros(5, dtype=torch.int32)), lambda: s2cnn_amd.norm_rotary(q, k, torch.ones(7)),
                lambda: s2cnn_amd.norm_rotary(q, k, None, torch.ones(2, 8)), lambda: s2cnn_amd.norm_rotary(q, None, None, torch.ones(8)),
                lambda: s2cnn_amd.norm_rotary(q, k, eps=0.0), lambda: s2cnn_amd.norm_rotary(q, k, eps=1e-60), lambda: s2cnn_amd.norm_rotary(q, k, eps=1e-39), lambda: s2cnn_amd.norm_rotary(q, k, eps=float("nan")),
                lambda: s2cnn_amd.rotary(torch.zeros(1, 1, 1, 258), None, torch.zeros(1, 128, 2)),
                lambda: s2cnn_amd.rotary_table(torch.zeros(4, 2), torch.zeros(1, 3, dtype=torch.float64)),
                lambda: s2cnn_amd.rotary_table(torch.zeros(4, 1), torch.zeros(1, 129, dtype=torch.float64)),
                lambda: s2cnn_amd.rotary_table(torch.zeros(4, 0), torch.zeros(0, 3, dtype=torch.float64)),
                lambda: s2cnn_amd.rotary_frequencies(0), lambda: s2cnn_amd.rotary_frequencies(4, factor=0.0), lambda: s2cnn_amd.rotary_frequencies(4, fast=1.0)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError, match="positions"):
        s2cnn_amd.rotary_table(torch.zeros(4, 1, dtype=torch.int16), torch.zeros(1, 3, dtype=torch.float64))


def test_tables_of_too_many_rows_are_refused():
    """Rows are numbered by int32: 2^32 + 5 of them would be taken for five, and the others for none."""
    q, index = torch.zeros(1, 1, 3, 2), torch.zeros(3, dtype=torch.int32)
    for rows in (1 << 31, (1 << 32) + 5):
        with pytest.raises(AssertionError):
            s2cnn_amd.rotary(q, None, torch.zeros(1, 1, 2).expand(rows, 1, 2), index=index)
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.rotary(q, None, torch.zeros(1, 1, 2).expand((1 << 31) - 1, 1, 2), index=index)


@pytest.mark.gpu
def test_refusals_of_types(hip):
    q, table = torch.zeros(2, 4, 5, 8, device="cuda"), torch.zeros(5, 4, 2, device="cuda")
    for bad in (lambda: s2cnn_amd.rotary(q, q.bfloat16(), table), lambda: s2cnn_amd.rotary(q.double(), None, table), lambda: s2cnn_amd.rotary(q, q, table.double()),
                lambda: s2cnn_amd.rotary(q, q, table.cpu()), lambda: s2cnn_amd.rotary(q, q.cpu(), table),
                lambda: s2cnn_amd.rotary(q, q, table, index=torch.zeros(5, dtype=torch.int64, device="cuda")),
                lambda: s2cnn_amd.norm_rotary(q, q, torch.ones(8, device="cuda").half()),
                lambda: s2cnn_amd.rotary_table(torch.zeros(4, 1, device="cuda"), torch.zeros(1, 3, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    x = q.requires_grad_()
    y, = torch.autograd.grad(s2cnn_amd.rotary(x, None, table)[0].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiat"):
        torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("index_stride", [0, 100])
def test_workspaces_with_fewer_rows_than_places(index_stride):
    """With an index a table may have any number of rows: the workspace of the weights' gradients does not depend on it."""
    plan = importlib.import_module("s2cnn_amd.rotary")._plan
    strides = ((6400 * 4, 6400, 64, 1),) * 3
    of = lambda rows, index: plan((2, 4, 100, 64), None, strides, (0, rows, 32), index, 1, 0, EPS, 0)[1]
    assert of(50, index_stride) == of(100, index_stride) == of(100, None) > 0
    assert of(50, None) == 0                                               # without an index refused


@pytest.mark.gpu
@pytest.mark.parametrize("with_grad", [False, True])
def test_tangents_of_forward_mode_are_refused(hip, with_grad):
    """None is lost without a word, with and without gradients of the other mode; inside a level without tangents all is as outside."""
    x, w, table = torch.randn(2, 4, 5, 8).cuda(), torch.ones(8, device="cuda"), _table(5, 4).cuda()
    places, f = torch.arange(5.0, device="cuda").view(5, 1), torch.ones(1, 4, dtype=torch.float64, device="cuda")
    want = s2cnn_amd.norm_rotary(x, x, w, w, table) + s2cnn_amd.rotary(x, x, table) + (s2cnn_amd.rotary_table(places, f),)
    with forward_ad.dual_level(), torch.set_grad_enabled(with_grad):
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: s2cnn_amd.rotary(dual(x), None, table), lambda: s2cnn_amd.rotary(x, dual(x), table), lambda: s2cnn_amd.rotary(x, None, dual(table)),
                     lambda: s2cnn_amd.norm_rotary(dual(x), x, w, w, table), lambda: s2cnn_amd.norm_rotary(x, x, dual(w), w), lambda: s2cnn_amd.norm_rotary(x, x, w, dual(w), table)):
            with pytest.raises(NotImplementedError, match="forward mode"):
                call()
        for call in (lambda: s2cnn_amd.rotary_table(dual(places), f), lambda: s2cnn_amd.rotary_table(places, dual(f))):
            with pytest.raises(AssertionError, match="not differentiated"):
                call()
        got = s2cnn_amd.norm_rotary(x, x, w, w, table) + s2cnn_amd.rotary(x, x, table) + (s2cnn_amd.rotary_table(places, f),)
        assert s2cnn_amd.rotary_table(torch.arange(5, device="cuda").view(5, 1), f).equal(want[-1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_entry_points_refuse_sizes():
    """The C entries, before any launch."""
    from s2cnn_amd import _hip
    lib = _hip.lib()
    fake = 0x1000

    def make(**kw):
        a = _hip.Rotary()
        a.batch, a.n, a.d, a.pairs, a.rows, a.eps, a.table = 2, 3, 16, 8, 3, 1e-6, fake
        a.heads[0], a.x[0], a.g[0], a.y[0] = 4, fake, fake, fake
        for name, v in kw.items():
            if name.startswith("side_"):
                getattr(a, name[5:])[0] = v
            else:
                setattr(a, name, v)
        return ctypes.byref(a)

    for kw, rc in (({"d": 257}, -1), ({"d": 15}, -1), ({"pairs": -1}, -1), ({"n": 0}, -1), ({"batch": 0}, -1), ({"n": 4}, -1), ({"rows": 0, "index": fake}, -1),
                   ({"table": None}, -1), ({"pairs": 0}, -1), ({"dtype": 3}, -1), ({"side_heads": 0}, -1), ({"side_x": None}, -1), ({"side_y": None}, -1),
                   ({"norm": 1, "eps": 0.0}, -1), ({"side_weight": fake}, -1), ({"batch": 1 << 30, "n": 2}, -1), ({"batch": 1 << 20, "side_heads": 1 << 11}, -1),
                   ({"side_x": fake + 2}, -3), ({"table": fake + 4}, -3), ({"table_stride": 3}, -3), ({"index": fake + 2}, -3), ({"side_gweight": fake}, -1)):
        assert lib.s2cnn_rotary_fwd(make(**kw), None) == rc, kw
    assert lib.s2cnn_rotary_fwd(None, None) == -1
    assert lib.s2cnn_rotary_bwd(make(side_g=None), None, 0, None) == -1
    assert lib.s2cnn_rotary_bwd(make(norm=1, side_gweight=fake), None, 0, None) == -2
    assert lib.s2cnn_rotary_workspace(make()) == 0 and lib.s2cnn_rotary_workspace(make(norm=1)) > 0 and lib.s2cnn_rotary_workspace(make(norm=1, d=300)) == 0
    assert lib.s2cnn_rotary_table(fake, 4, fake, fake, 3, 1, 4, 1.0, None) == -1 and lib.s2cnn_rotary_table(fake, 0, fake, fake, 0, 1, 4, 1.0, None) == -1
    assert lib.s2cnn_rotary_table(fake, 0, fake, fake, 3, 1, 129, 1.0, None) == -1 and lib.s2cnn_rotary_table(fake + 4, 1, fake, fake, 3, 1, 4, 1.0, None) == -3
    assert lib.s2cnn_rotary_table(None, 0, fake, fake, 3, 1, 4, 1.0, None) == -1
