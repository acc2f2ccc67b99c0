"""layer_norm, dropout and dropout_add_layer_norm (s2cnn_amd/layer_norm.py) against the definitions in 64 bits on the CPU, the
generator in Python's integers.

Tolerances.  u = 2^-24, 2^-8, 2^-11 is the unit roundoff of float32, bfloat16, float16.  A float32 result is a chain of some ten
roundings of values not larger than a few of its own: 16 u in the 2-norm; 16-bit results are rounded once (0.45 u on average) and the
gradients of the step use the rounded h as well: 2 u.  Sums over the rows are float32 sums of n values: 16 * 2^-24 of the 2-norm of
the sums of magnitudes on top."""
import math

import numpy as np
import pytest
import torch

import s2cnn_amd

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
TOL = {F32: 16 * 2.0 ** -24, BF16: 2 * 2.0 ** -8, F16: 2 * 2.0 ** -11}
EPS = 1e-5


def _philox(counter, key):
    """Philox4x32-10 of a counter below 2^64."""
    m = 0xFFFFFFFF
    c, k = [counter & m, counter >> 32, 0, 0], [key & m, key >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def _factors(n, p, seed):
    drop = min(65535, round(p * 65536))
    bits = []
    for c in range((n + 7) // 8):
        for w in _philox(c, seed & (2 ** 64 - 1)):
            bits += [w & 0xFFFF, w >> 16]
    return torch.tensor(np.array(bits[:n]) >= drop).double() * (65536 / (65536 - drop))


def _close(got, want, dtype, what, mag=None):
    assert got.dtype == dtype and got.shape == want.shape, what
    got = got.detach().cpu().double()
    allowed = TOL[dtype] * want.norm().item() + (16 * 2.0 ** -24 * mag.norm().item() if mag is not None else 0.0)
    assert torch.isfinite(got).all() and (got - want).norm().item() <= allowed, (what, (got - want).norm().item(), allowed)


def _gradients(h, w, g):
    """(dh, dw, db, sums of magnitudes of the last two)"""
    n = h.size(1)
    mean = h.mean(1, keepdim=True)
    sd = torch.sqrt(((h - mean) ** 2).mean(1, keepdim=True) + EPS)
    xh = (h - mean) / sd
    u = g * w
    dh = (u - u.sum(1, keepdim=True) / n - xh * (u * xh).sum(1, keepdim=True) / n) / sd
    return dh, (g * xh).sum(0), g.sum(0), (g * xh).abs().sum(0), g.abs().sum(0)


def _make(rows, features, dtype, seed=0):
    gen = torch.Generator().manual_seed(rows * 10007 + features + seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    return [t.to(dtype).cuda() for t in (r(rows, features) * 1.5 + 0.25, r(features) * 0.2 + 1, r(features) * 0.2, r(rows, features))], r


SHAPES = [(1, 1), (3, 2), (7, 5), (5, 8), (300, 20), (64, 33), (1000, 64), (777, 100), (50, 129), (40, 257), (257, 350), (33, 512), (70, 1000), (9, 1024),
          (20, 2047), (6, 2048), (5, 4096), (3, 5000), (2, 8192), (7, 9001)]
SHAPE_IDS = ["%dx%d" % s for s in SHAPES]


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("shape", SHAPES, ids=SHAPE_IDS)
def test_layer_norm(hip, shape, dtype):
    (x, w, b, g), _ = _make(*shape, dtype)
    for t in (x, w, b):
        t.requires_grad_()
    y = s2cnn_amd.layer_norm(x, w, b, eps=EPS)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], g)
    xd, wd, bd, gd = (t.detach().cpu().double() for t in (x, w, b, g))
    mean = xd.mean(1, keepdim=True)
    want = (xd - mean) / torch.sqrt(((xd - mean) ** 2).mean(1, keepdim=True) + EPS) * wd + bd
    dx, dw, db, mw, mb = _gradients(xd, wd, gd)
    _close(y, want, dtype, "y")
    # rows of one or two features have no gradient: what is left is the roundings of what cancels
    scale = (gd * wd).abs() / torch.sqrt(((xd - mean) ** 2).mean(1, keepdim=True) + EPS)
    _close(gx, dx, dtype, "gx", scale + scale.mean(1, keepdim=True))
    _close(gw, dw, dtype, "gw", mw)
    _close(gb, db, dtype, "gb", mb)
    with torch.no_grad():
        assert torch.equal(s2cnn_amd.layer_norm(x, w, b, eps=EPS), y)
        plain = s2cnn_amd.layer_norm(x)
    _close(plain, (want - bd) / wd if (wd != 0).all() else want, dtype, "without weights")


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("shape", SHAPES[2:12] + [(5, 1000), (3, 4099), (2, 9000)], ids=lambda s: "%dx%d" % s)
def test_step(hip, shape, dtype):
    (x, w, b, g), r = _make(*shape, dtype, seed=1)
    res, g_h = (r(*shape).to(dtype).cuda() for _ in range(2))
    p, seed = 0.3, 2 ** 40 + 17
    for t in (x, res, w, b):
        t.requires_grad_()
    h, y = s2cnn_amd.dropout_add_layer_norm(x, res, p, seed, w, b, eps=EPS)
    gx, gr, gw, gb = torch.autograd.grad([h, y], [x, res, w, b], [g_h, g])
    xd, rd, wd, bd, gd, ghd = (t.detach().cpu().double() for t in (x, res, w, b, g, g_h))
    f = _factors(x.numel(), p, seed).view(shape)
    hd = rd + xd * f
    mean = hd.mean(1, keepdim=True)
    sd = torch.sqrt(((hd - mean) ** 2).mean(1, keepdim=True) + EPS)
    dh, dw, db, mw, mb = _gradients(hd, wd, gd)
    _close(h, hd, dtype, "h")
    _close(y, (hd - mean) / sd * wd + bd, dtype, "y")
    _close(gr, dh + ghd, dtype, "gr", (gd * wd).abs() / sd)
    _close(gx, (dh + ghd) * f, dtype, "gx", (gd * wd).abs() / sd)
    _close(gw, dw, dtype, "gw", mw)
    _close(gb, db, dtype, "gb", mb)
    # the pieces: what of it one by one gives
    assert torch.equal((gx == 0) | (f.cuda() != 0), torch.ones_like(gx, dtype=torch.bool))
    only_y = torch.autograd.grad(s2cnn_amd.dropout_add_layer_norm(x, res, p, seed, w, b, eps=EPS)[1], [x, res], g)
    _close(only_y[1], dh, dtype, "gradient of y alone", (gd * wd).abs() / sd)
    only_h = torch.autograd.grad(s2cnn_amd.dropout_add_layer_norm(x, res, p, seed, w, b, eps=EPS)[0], [x, res], g_h)
    _close(only_h[0], ghd * f, dtype, "gradient of h alone")
    assert torch.equal(only_h[1], g_h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,unit", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)], ids=["bf16", "f16"])
@pytest.mark.parametrize("shape", [(600, 200), (301, 77), (12, 9001)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("size", [2.0 ** -6, 1.0, 2.0 ** 6])
def test_sixteen_bit_step_is_rounded_once(hip, shape, size, dtype, unit):
    """A rounding is off by a uniform part of half a spacing: 0.43 u in the 2-norm over many numbers, with a spread of 1 / sqrt(2 n) over n of
    them, four of which are allowed.  The gradients are those of h before its rounding, of which the backward pass has 7 more bits.
    Rows of any magnitude, with zeros among them."""
    (x, w, b, g), r = _make(*shape, dtype, seed=4)
    res, g_h = (r(*shape).to(dtype).cuda() for _ in range(2))
    with torch.no_grad():
        x *= size
        res *= size
        x[:, ::3] = 0
        res[:, ::6] = 0
        w.fill_(1.0)
    for t in (x, res, w, b):
        t.requires_grad_()
    p, seed = 0.25, 3
    _, y = s2cnn_amd.dropout_add_layer_norm(x, res, p, seed, w, b, eps=EPS)
    gx, gr, gw, gb = torch.autograd.grad(y, [x, res, w, b], g)
    xd, rd, wd, gd = (t.detach().cpu().double() for t in (x, res, w, g))
    f = _factors(x.numel(), p, seed).view(shape)
    dh, dw, db, _, _ = _gradients(rd + xd * f, wd, gd)
    for got, want in ((gr, dh), (gx, dh * f), (gw, dw), (gb, db)):
        assert (got.detach().cpu().double() - want).norm() <= 0.45 * unit * (1 + 4 / (2 * want.numel()) ** 0.5) * want.norm()


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 4097, 100003])
def test_dropout(hip, n, dtype):
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype).cuda().requires_grad_()
    g = torch.randn(n, generator=torch.Generator().manual_seed(n + 1)).to(dtype).cuda()
    for p, seed in ((0.1, 0), (0.5, -3), (0.999, 2 ** 63 + 5)):
        f = _factors(n, p, seed)
        y = s2cnn_amd.dropout(x, p, seed)
        gx, = torch.autograd.grad(y, x, g)
        for got, of in ((y, x), (gx, g)):
            want = (of.detach().cpu().float() * f.float()).to(dtype)
            assert torch.equal(got.cpu(), want)
    assert torch.equal(s2cnn_amd.dropout(x, 0.0, 1), x)
    assert torch.equal(s2cnn_amd.dropout(x, 1e-7, 1), x)                     # no multiple of 2^-16 but zero


@pytest.mark.gpu
@TYPES
def test_dropout_of_large_tensors(hip, dtype):
    """Sizes that go past the caches (float32) and beyond one round of the workgroups: the head and the tail against the generator in integers,
    all of it against pieces, whose elements are those of the same index."""
    n, p, seed = (1 << 26) + 1003, 0.3, 21
    x = torch.ones(n, dtype=dtype, device="cuda")
    y = s2cnn_amd.dropout(x, p, seed)
    head = _factors(40000, p, seed).to(dtype)
    assert torch.equal(y[:40000].cpu(), head)
    first = (n - 4000) // 8 * 8
    drop, bits = round(p * 65536), []
    for c in range(first // 8, (n + 7) // 8):
        for w in _philox(c, seed):
            bits += [w & 0xFFFF, w >> 16]
    tail = (torch.tensor(np.array(bits[:n - first]) >= drop).double() * (65536 / (65536 - drop))).to(dtype)
    assert torch.equal(y[first:].cpu(), tail)
    kept = (y != 0).double().mean().item()
    assert abs(kept - (1 - drop / 65536)) < 6 * (0.3 * 0.7 / n) ** 0.5
    for m in (1 << 20, (1 << 22) + 5):                                            # pieces from the start
        assert torch.equal(s2cnn_amd.dropout(x[:m], p, seed), y[:m])


def test_generator_known_answer():
    """The published answer of Philox4x32-10 for a zero counter and key, and for all bits set in the words used here."""
    assert _philox(0, 0) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


@pytest.mark.gpu
def test_dropped_share_and_independence(hip):
    """Binomial: 2^22 elements at p = 0.25 drop a share of 0.25 with a standard deviation of 2.1e-4; 6 of them allowed.  Two seeds, and
    neighbours under one seed, agree as independent ones do (0.0625 both dropped, deviation 1.2e-4)."""
    n = 1 << 22
    x = torch.ones(n, device="cuda")
    a, b = (s2cnn_amd.dropout(x, 0.25, s) == 0 for s in (5, 6))
    assert abs(a.double().mean().item() - 0.25) < 1.3e-3
    assert abs((a & b).double().mean().item() - 0.0625) < 8e-4
    for shift in (1, 2, 8, 64):
        assert abs((a[shift:] & a[:-shift]).double().mean().item() - 0.0625) < 8e-4


@pytest.mark.gpu
def test_what_is_dropped_may_hold_anything(hip):
    n, p, seed = 5000, 0.5, 9
    f = _factors(n, p, seed).cuda()
    x = torch.randn(n, device="cuda")
    x[f == 0] = math.nan
    y = s2cnn_amd.dropout(x, p, seed)
    assert (y[f == 0] == 0).all() and torch.equal(y[f != 0], (x * f.float())[f != 0])
    h, _ = s2cnn_amd.dropout_add_layer_norm(x.view(50, 100), torch.ones(50, 100, device="cuda"), p, seed)
    assert torch.isfinite(h).all()


@pytest.mark.gpu
def test_seed_on_the_device(hip):
    x = torch.randn(3, 700, device="cuda", requires_grad=True)
    g = torch.randn(3, 700, device="cuda")
    seed = torch.tensor([2 ** 45 + 3], device="cuda")
    y, want = s2cnn_amd.dropout(x, 0.2, seed), s2cnn_amd.dropout(x, 0.2, 2 ** 45 + 3)
    assert torch.equal(y, want) and torch.equal(torch.autograd.grad(y, x, g)[0], torch.autograd.grad(want, x, g)[0])
    a, b = (s2cnn_amd.dropout_add_layer_norm(x, x.detach(), 0.2, s)[1] for s in (seed, 2 ** 45 + 3))
    assert torch.equal(a, b) and torch.equal(torch.autograd.grad(a, x, g)[0], torch.autograd.grad(b, x, g)[0])


@pytest.mark.gpu
def test_replays_from_a_graph_with_another_mask_each(hip):
    """A captured step whose seed is a counter on the device: each replay drops what the eager call with that seed drops."""
    gen = torch.Generator().manual_seed(1)
    x, res, w, g = (torch.randn(*s, generator=gen).cuda() for s in ((200, 100), (200, 100), (100,), (200, 100)))
    x.requires_grad_()
    w.requires_grad_()
    counter = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step(seed):
        h, y = s2cnn_amd.dropout_add_layer_norm(x, res, 0.25, seed, w)
        return (h, y, *torch.autograd.grad(y, [x, w], g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(counter.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        counter.add_(1)
        static = step(counter.clone())
    counter.zero_()
    seen = []
    for k in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, step(k)):
            assert torch.equal(a, b)
        seen.append(static[0].clone())
    assert not torch.equal(seen[0], seen[1])


@pytest.mark.gpu
@TYPES
def test_layouts(hip, dtype):
    """Strided inputs and gradients, leading axes, and rows that start at any entry."""
    gen = torch.Generator().manual_seed(4)
    base = torch.randn(6, 5, 3, 24, generator=gen).to(dtype).cuda()
    w = torch.randn(48, generator=gen).to(dtype).cuda()[::2]
    g = torch.randn(6, 5, 3, 24, generator=gen).to(dtype).cuda()
    storage = torch.zeros(base.numel() + 5, dtype=dtype, device="cuda")
    want = None
    for x, gg in ((base, g), (base.transpose(0, 2).contiguous().transpose(0, 2), g.transpose(1, 2).contiguous().transpose(1, 2)),
                  (storage[3:3 + base.numel()].view_as(base).copy_(base), storage.new_zeros(base.numel() + 1)[1:].view_as(g).copy_(g)),
                  (torch.stack([base, base], -1)[..., 0], g)):
        x = x.detach().requires_grad_()
        y = s2cnn_amd.layer_norm(x, w)
        got = (y, *torch.autograd.grad(y, x, gg), *torch.autograd.grad(s2cnn_amd.dropout(x, 0.4, 3), x, gg),
               *s2cnn_amd.dropout_add_layer_norm(x, x.detach(), 0.4, 3, w))
        want = want or got
        for a, b in zip(got, want):
            assert a.shape == b.shape and torch.equal(a, b)
    x = base.detach().requires_grad_()
    gx, = torch.autograd.grad(s2cnn_amd.layer_norm(x, w).sum(), x)          # an expanded gradient
    gy, = torch.autograd.grad(s2cnn_amd.layer_norm(x, w), x, torch.ones_like(x))
    assert torch.equal(gx, gy)


@pytest.mark.gpu
def test_same_bits_every_time_and_on_other_streams(hip):
    (x, w, b, g), _ = _make(5000, 100, F32)
    for t in (x, w, b):
        t.requires_grad_()
    want = torch.autograd.grad(s2cnn_amd.layer_norm(x, w, b), [x, w, b], g)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = torch.autograd.grad(s2cnn_amd.layer_norm(x, w, b), [x, w, b], g)
        torch.cuda.current_stream().wait_stream(side)
        for a, c in zip(got, want):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Central differences along random directions of length one, steps of 2^-6: their error is a third derivative (of the
    order of the gradient) times 2^-12 / 6, roundings 2^-17: 2e-3 allowed."""
    (x, w, b, g), r = _make(12, 30, F32, seed=5)
    args = {"x": x, "residual": r(12, 30).cuda(), "weight": w, "bias": b}
    for t in args.values():
        t.requires_grad_()

    def value(**a):
        h, y = s2cnn_amd.dropout_add_layer_norm(a["x"], a["residual"], 0.25, 3, a["weight"], a["bias"])
        return (y.double() * g.double()).sum() + 0.5 * (h.double() ** 2).sum()

    grads = torch.autograd.grad(value(**args), list(args.values()))
    gen = torch.Generator().manual_seed(6)
    for (n, t), grad in zip(args.items(), grads):
        u = torch.randn(t.shape, generator=gen).cuda()
        u /= u.norm()
        with torch.no_grad():
            f = [value(**{**args, n: t + s * 2.0 ** -6 * u}).item() for s in (1, -1)]
        assert abs((f[0] - f[1]) * 2.0 ** 5 - (grad.double() * u.double()).sum().item()) <= 2e-3 * max(1.0, grad.norm().item()), n


@pytest.mark.gpu
def test_large_offsets_of_the_rows(hip):
    """Rows far from zero: the variance is formed from centred values.  An offset of 1000 leaves 2^-24 * 1000 of a value of one: 6e-5,
    some 4 times in a result."""
    x = torch.randn(40, 100, generator=torch.Generator().manual_seed(2)).cuda() + 1000
    xd = x.cpu().double()
    want = (xd - xd.mean(1, keepdim=True)) / torch.sqrt(xd.var(1, unbiased=False, keepdim=True) + EPS)
    assert (s2cnn_amd.layer_norm(x).cpu().double() - want).abs().max().item() < 2.4e-4 * 4
    flat = s2cnn_amd.layer_norm(torch.full((3, 64), 7.0, device="cuda"))
    assert (flat == 0).all()                                                     # no variance: eps alone


@pytest.mark.gpu
def test_some_gradients_only_and_empty_sizes(hip):
    (x, w, b, g), _ = _make(50, 40, F32)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(s2cnn_amd.layer_norm(*full), full, g)
    for i in range(3):
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(s2cnn_amd.layer_norm(*part), part[i], g)[0], want[i])
        h, y = s2cnn_amd.dropout_add_layer_norm(part[0], x, 0.1, 1, part[1], part[2])
        assert torch.autograd.grad(y, part[i], g)[0].shape == part[i].shape
    res = x.clone().requires_grad_()
    assert torch.autograd.grad(s2cnn_amd.dropout_add_layer_norm(x, res, 0.1, 1, w, b)[1], res, g)[0].shape == x.shape
    e = torch.zeros(0, 40, device="cuda", requires_grad=True)
    wg = w.clone().requires_grad_()
    y = s2cnn_amd.layer_norm(e, wg)
    assert y.shape == e.shape and (torch.autograd.grad(y.sum(), wg)[0] == 0).all()
    assert s2cnn_amd.dropout(e, 0.5, 1).shape == e.shape
    assert s2cnn_amd.dropout_add_layer_norm(e, e, 0.5, 1)[0].shape == e.shape


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (64, 63), (65, 64), (1000, 65), (1600, 192), (4097, 7), (100003, 20), (17, 3001), (2, 70001)], ids=lambda s: "%dx%d" % s)
def test_column_sums(hip, shape, dtype):
    """Sums over the rows, strided and contiguous; float32 whatever the type."""
    from s2cnn_amd.layer_norm import column_sums
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).to(dtype).cuda()
    want, mag = x.cpu().double().sum(0), x.cpu().double().abs().sum(0)
    for t in (x, x.t().contiguous().t(), x.view(1, *shape)):
        got = column_sums(t)
        _close(got, want, F32, "sums", mag)
        assert torch.equal(got, column_sums(x))
    assert (column_sums(x[:0]) == 0).all() and column_sums(x[:0]).shape == shape[1:]


@pytest.mark.gpu
def test_column_sums_replayed_from_a_graph(hip):
    from s2cnn_amd.layer_norm import column_sums
    x = torch.randn(1600, 192, device="cuda")
    column_sums(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = column_sums(x)
    for k in range(4):
        x.mul_(1.0 + 0.1 * k)
        want = column_sums(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(static, want)


def test_column_sums_refused_without_a_gpu():
    from s2cnn_amd import _hip
    from s2cnn_amd.layer_norm import column_sums
    lib, f = _hip.lib(), 0x1000
    n = lib.s2cnn_column_sums_workspace(1600, 192, 0)
    assert n > 0 and lib.s2cnn_column_sums_workspace(0, 192, 0) == 0 and lib.s2cnn_column_sums_workspace(4, 0, 0) == 0
    call = lambda x=f, out=f, ws=f, size=n, rows=1600, features=192, dtype=0: lib.s2cnn_column_sums(x, out, ws, size, rows, features, dtype, None)
    assert call(x=None) == -1 and call(out=None) == -1 and call(rows=0) == -1 and call(features=0) == -1 and call(dtype=3) == -1
    assert call(x=f + 2) == -3 and call(out=f + 2) == -3 and call(size=n - 1) == -2 and call(ws=None) == -2 and call(ws=f + 8) == -2
    with pytest.raises(RuntimeError, match="no CPU path"):
        column_sums(torch.zeros(2, 3))


def test_refusals():
    z = torch.zeros
    for f in (lambda: s2cnn_amd.layer_norm(z(2, 0)), lambda: s2cnn_amd.layer_norm(z(())), lambda: s2cnn_amd.layer_norm(z(2, 3), z(4)),
              lambda: s2cnn_amd.layer_norm(z(2, 3), z(3), z(2)), lambda: s2cnn_amd.dropout(z(3), 1.0, 0), lambda: s2cnn_amd.dropout(z(3), -0.1, 0),
              lambda: s2cnn_amd.dropout(z(3), 0.5, 0.5), lambda: s2cnn_amd.dropout(z(3), 0.5, z(2, dtype=torch.int64)),
              lambda: s2cnn_amd.dropout_add_layer_norm(z(2, 3), z(3, 2), 0.5, 0), lambda: s2cnn_amd.dropout_add_layer_norm(z(2, 3), z(2, 3), 1.5, 0)):
        with pytest.raises(AssertionError):
            f()
    for f in (lambda: s2cnn_amd.layer_norm(z(2, 3)), lambda: s2cnn_amd.dropout(z(3), 0.5, 0), lambda: s2cnn_amd.dropout_add_layer_norm(z(2, 3), z(2, 3), 0.5, 0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


@pytest.mark.gpu
def test_refusals_of_types(hip):
    z = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)
    for f in (lambda: s2cnn_amd.layer_norm(z(2, 3, dtype=torch.float64)), lambda: s2cnn_amd.layer_norm(z(2, 3), z(3, dtype=BF16)),
              lambda: s2cnn_amd.dropout(z(3), 0.5, z(1, dtype=torch.int32)), lambda: s2cnn_amd.dropout(z(3), 0.5, torch.zeros(1, dtype=torch.int64)),
              lambda: s2cnn_amd.dropout_add_layer_norm(z(2, 3), z(2, 3, dtype=F16), 0.5, 0)):
        with pytest.raises(RuntimeError):
            f()


def test_entry_points_refuse_without_a_gpu():
    from s2cnn_amd import _hip
    lib = _hip.lib()
    f = 0x1000
    assert lib.s2cnn_dropout(f, f, 0, 0.5, 0, None, 0, None) == -1
    assert lib.s2cnn_dropout(f, f, 8, 1.0, 0, None, 0, None) == -1
    assert lib.s2cnn_dropout(f, f, 8, float("nan"), 0, None, 0, None) == -1
    assert lib.s2cnn_dropout(f, f, 8, 0.5, 0, None, 3, None) == -1
    assert lib.s2cnn_dropout(f + 2, f, 8, 0.5, 0, None, 0, None) == -3
    assert lib.s2cnn_dropout(f, f, 8, 0.5, 0, f + 4, 0, None) == -3
    fwd = lambda x=f, res=None, h=None, rows=4, features=8, p=0.0, dtype=0: lib.s2cnn_layer_norm_fwd(x, res, None, None, h, f, None, rows, features, 1e-5, p, 0, None, dtype, None)
    assert fwd(x=None) == -1 and fwd(res=f) == -1 and fwd(h=f) == -1 and fwd(rows=0) == -1 and fwd(features=0) == -1 and fwd(p=0.5) == -1 and fwd(dtype=7) == -1
    assert fwd(x=f + 1) == -3
    bwd = lambda h=f, gx=f, gr=None, gw=None, step=0, p=0.0, n=0: lib.s2cnn_layer_norm_bwd(h, f, None, None, f, gx, gr, gw, None, None, n, 4, 8, p, 0, None, step, 0, None)
    assert bwd(h=None) == -1 and bwd(gx=None) == -1 and bwd(gr=f) == -1 and bwd(p=0.5) == -1 and bwd(gx=None, step=1) == -1
    assert bwd(gw=f) == -2
    assert lib.s2cnn_layer_norm_bwd_workspace(4, 8, 0) > 0 and lib.s2cnn_layer_norm_bwd_workspace(0, 8, 0) == 0
