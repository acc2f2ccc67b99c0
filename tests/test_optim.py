"""adamw_step, adamw_states, grad_norm and AdamW (s2cnn_amd/optim.py) against the formulas in 64 bits, 8-bit codes against numpy's single float32
operations bit for bit.

Tolerances of one step from given tensors, in the 2-norm, w = 2^-24: the moments are two products and a sum (v: three), each off by at most w of its
result: 3 w of |m| b1 + |g| (1 - b1), 4 w for v.  With a clipping factor, rounded twice, and its product: 3 w (v: 6 w) more.  The update m / (1 - b1^t) / (root +
eps) lr adds a root and a reciprocal that are off by at most 2 w each, two factors (1 - b^t, of an exponent off by 2 w: 8 w together) and four products:
24 w of its size, with half of v's error in the root.  p itself is one product and a sum: 2 w, and its rounding to 16 bits u = 2^-8, 2^-11.
The norm is rounded once from 64 bits: 2 w."""
import copy
import ctypes
import io
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import s2cnn_amd

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
UNIT = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
W = 2.0 ** -24
SHAPES = [(1,), (3,), (0,), (255,), (256,), (257,), (4095,), (4096,), (4097,), (5, 7), (100, 33), (2, 3, 5), (20001,)]
HYPER = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def _random(shapes, dtype, seed, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * size).to(dtype).cuda() for s in shapes]


def _zeros(shapes, bits):
    """first, second, scales of moments of zero"""
    if bits == 32:
        return [torch.zeros(s, device="cuda") for s in shapes], [torch.zeros(s, device="cuda") for s in shapes], None
    codes = [[torch.zeros(s, dtype=torch.uint8, device="cuda") for s in shapes] for _ in range(2)]
    return [t.view(torch.float8_e4m3fn) for t in codes[0]], codes[1], [torch.zeros(-(-math.prod(s) // 256), 2, device="cuda") for s in shapes]


def _cpu(tensors):
    return [t.detach().cpu().double() for t in tensors]


def _expected(p, g, m, v, step, lr, betas, eps, weight_decay, factor=1.0):
    """(p, m, v, update) after a step, in 64 bits"""
    g = g * factor
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    update = lr * (m / (1 - betas[0] ** step)) / (torch.sqrt(v / (1 - betas[1] ** step)) + eps)
    return p - lr * weight_decay * p - update, m, v, update


def _close(got, want, allowed, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    assert (got - want).norm().item() <= allowed, (what, (got - want).norm().item(), allowed)


def _check_step(before, after, step, dtype, factor=1.0, clipped=0, **hyper):
    """before, after: (p, m, v) lists and gradients in between, values of what was held"""
    (ps, gs, ms, vs), (qs, ns, us) = before, after
    for i, (p, g, m, v) in enumerate(zip(ps, gs, ms, vs)):
        if not p.numel():
            continue
        want, wm, wv, update = _expected(p, g, m, v, step, factor=factor, **hyper)
        b1, b2 = hyper["betas"]
        mag_m, mag_v = (b1 * m.abs() + (1 - b1) * (factor * g).abs()).norm().item(), wv.norm().item()
        if ns is not None:
            _close(ns[i], wm, (3 + clipped) * W * mag_m, "m %d" % i)
            _close(us[i], wv, (4 + 2 * clipped) * W * mag_v, "v %d" % i)
        size = (update.abs() + hyper["lr"] * (b1 * m.abs() + (1 - b1) * (factor * g).abs()) / (1 - b1 ** step) / (torch.sqrt(wv / (1 - b2 ** step)) + hyper["eps"])).norm().item()
        _close(qs[i], want, (UNIT[dtype] + 2 * W) * want.norm().item() + 2 * W * p.norm().item() + (24 + 2 * clipped) * W * size, "p %d" % i)


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("clip", [False, True])
def test_steps_in_32_bits(hip, dtype, masters, clip):
    if masters and dtype == F32:
        masters = False
    exact = _random(SHAPES, F32, 1)
    params = [p.to(dtype) for p in exact]
    held = exact if masters else None
    first, second, _ = _zeros(SHAPES, 32)
    for step in range(1, 5):
        grads = _random(SHAPES, dtype, 10 + step, 0.1)
        norm = s2cnn_amd.grad_norm(grads) if clip else None
        want_norm = math.sqrt(sum(g.square().sum().item() for g in _cpu(grads)))
        factor = min(1.0, 2.0 / want_norm) if clip else 1.0
        before = _cpu(held if masters else params), _cpu(grads), _cpu(first), _cpu(second)
        s2cnn_amd.adamw_step(params, grads, first, second, step, masters=held, norm=norm, max_norm=2.0 if clip else None, **HYPER)
        _check_step(before, (_cpu(held if masters else params), first, second), step, F32 if masters else dtype, factor, 3 if clip else 0, **HYPER)
        if clip:
            assert norm.dtype == F32 and norm.shape == () and abs(norm.item() - want_norm) <= 2 * W * want_norm and factor < 1
        if masters:
            assert all(torch.equal(p, h.to(dtype)) for p, h in zip(params, held))


# ---- 8 bits: the definition in numpy's float32 ----------------------------------------------------------------------
def _philox(n, seed, step):
    """Two 16-bit numbers for each of n entries (a multiple of four)"""
    mask, c = np.uint64(0xFFFFFFFF), [np.arange(n // 4, dtype=np.uint64) for _ in range(4)]
    c[1] = c[0] >> np.uint64(32)
    c[0] = c[0] & mask
    c[2], c[3] = np.full_like(c[0], step & 0xFFFFFFFF), np.full_like(c[0], step >> 32)
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(c, 1).reshape(-1)
    return (words & np.uint64(0xFFFF)).astype(np.int64), (words >> np.uint64(16)).astype(np.int64)


VALUES = np.array([c if c < 8 else (8 + c % 8) * 2.0 ** (c // 8 - 1) for c in range(256)])


def _rounded(x, top, u, most):
    """(codes, factor) of one block of float32 values x >= 0"""
    s = np.float32(x.max() * np.float32(1.0 / VALUES[top]))
    if s < np.float32(2.0 ** -126):
        return np.zeros(len(x), np.int64), np.float32(0)
    y = (x * (np.float32(1) / s)).astype(np.float64)
    e = np.maximum(np.floor(np.log2(np.maximum(y, 1e-300))).astype(np.int64), 3)
    part = (y * 2.0 ** (3 - e)).astype(np.float32) + (u * 2.0 ** -16).astype(np.float32)           # a float32 sum
    return np.minimum((e - 3) * 8 + np.floor(part).astype(np.int64), most), s


class _EightBits:
    """The moments of a list of tensors, stepped one after the other"""

    def __init__(self, shapes):
        self.sizes = [math.prod(s) for s in shapes]
        self.m = [np.zeros(n, np.int64) for n in self.sizes]
        self.v = [np.zeros(n, np.int64) for n in self.sizes]
        self.scales = [np.zeros((-(-n // 256), 2), np.float32) for n in self.sizes]

    def step(self, grads, step, seed, betas, factor=None):
        """The moments before their rounding, of the steps' gradients"""
        um, uv = _philox(sum(-(-n // 256) * 256 for n in self.sizes), seed, step)
        f, at, exact = np.float32, 0, []
        for i, n in enumerate(self.sizes):
            g = grads[i].detach().cpu().float().numpy().reshape(-1)
            if factor is not None:
                g = g * f(factor)
            s = np.repeat(self.scales[i], 256, 0)[:n]
            sign = np.where(self.m[i] >= 128, -1, 1)
            m = (sign * VALUES[self.m[i] & 127]).astype(f) * s[:, 0]
            v = VALUES[self.v[i]].astype(f) * s[:, 1]
            m = m * f(betas[0]) + g * f(1 - betas[0])
            v = v * f(betas[1]) + (g * g) * f(1 - betas[1])
            exact.append((m, v))
            for b in range(0, n, 256):
                part = slice(b, min(b + 256, n))
                random = slice(at + b, at + min(b + 256, n))
                cm, sm = _rounded(np.abs(m[part]), 126, um[random], 126)
                cv, sv = _rounded(v[part], 255, uv[random], 255)
                if sv > 0:
                    cv = np.where(v[part] > 0, np.maximum(cv, 1), cv)
                self.m[i][part], self.v[i][part] = cm + 128 * (m[part] < 0), cv
                self.scales[i][b // 256] = sm, sv
            at += -(-n // 256) * 256
        return exact

    def equals(self, first, second, scales):
        for i, n in enumerate(self.sizes):
            assert np.array_equal(first[i].view(torch.uint8).cpu().numpy().reshape(-1), self.m[i]), i
            assert np.array_equal(second[i].cpu().numpy().reshape(-1), self.v[i]), i
            assert np.array_equal(scales[i].cpu().numpy(), self.scales[i]), i

    def values(self, i):
        s = np.repeat(self.scales[i], 256, 0)[:self.sizes[i]]
        m = np.where(self.m[i] >= 128, -1, 1) * VALUES[self.m[i] & 127]
        return m.astype(np.float32) * s[:, 0], VALUES[self.v[i]].astype(np.float32) * s[:, 1]


def test_the_two_definitions_of_a_code_agree():
    """float8_e4m3fn in units of 2^-9 is f; a value of the lattice is left as it is by any random number, others lie between their neighbours."""
    codes = torch.arange(127, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy() * 512, VALUES[:127])
    for u in (0, 65535):
        c, s = _rounded(VALUES.astype(np.float32), 255, np.full(256, u), 255)
        assert s == 1 and np.array_equal(c, np.arange(256))
    x = np.float32([1000.3, VALUES[255]])
    low, high = (_rounded(x, 255, np.full(2, u), 255)[0][0] for u in (0, 65535))
    assert high == low + 1 and VALUES[low] <= x[0] <= VALUES[high]


@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("clip", [False, True])
def test_steps_in_8_bits(hip, dtype, masters, clip):
    """Codes and factors bit for bit; parameters from the moments before their rounding."""
    if masters and dtype == F32:
        masters = False
    exact = _random(SHAPES, F32, 2)
    params = [p.to(dtype) for p in exact]
    held = exact if masters else None
    first, second, scales = _zeros(SHAPES, 8)
    model, seed = _EightBits(SHAPES), 2 ** 33 + 5
    for step in (1, 2, 3, 2 ** 32 + 7):
        grads = _random(SHAPES, dtype, 20 + step % 1000, 0.1)
        for g in grads[3:]:                                              # entries of very different sizes, and zeros
            g.view(-1)[::7] *= 1e-3
            g.view(-1)[::11] = 0
        norm = s2cnn_amd.grad_norm(grads) if clip else None
        factor = min(1.0, float(np.float32(2.0) / np.float32(norm.item()))) if clip else None
        before = _cpu(held if masters else params), _cpu(grads)
        moments = [model.values(i) for i in range(len(SHAPES))]
        s2cnn_amd.adamw_step(params, grads, first, second, step, masters=held, scales=scales, norm=norm, max_norm=2.0 if clip else None, seed=seed, **HYPER)
        model.step(grads, step, seed, HYPER["betas"], factor)
        model.equals(first, second, scales)
        ms, vs = ([torch.from_numpy(moments[i][j]).double().view(s) for i, s in enumerate(SHAPES)] for j in (0, 1))
        _check_step((*before, ms, vs), (_cpu(held if masters else params), None, None), step, F32 if masters else dtype, factor or 1.0, 3 if clip else 0, **HYPER)
        m, v = s2cnn_amd.adamw_states(first, second, scales)
        for i, s in enumerate(SHAPES):
            want = model.values(i)
            assert m[i].shape == v[i].shape == s and np.array_equal(m[i].cpu().numpy().reshape(-1), want[0]) and np.array_equal(v[i].cpu().numpy().reshape(-1), want[1])


@pytest.mark.gpu
def test_random_rounding_has_the_right_mean(hip):
    """Many blocks of one value beside a larger one: the mean of what is held against the value.  An entry is spread over at most one spacing, 1/8 of
    itself: the mean of n is off by at most 6 / 16 / sqrt(n) but with a probability of 1e-8."""
    n, betas = 256 * 4000, (0.9, 0.999)
    g = torch.full((n,), 0.01, device="cuda")
    g[::256] = 1.0
    for step, seed in ((1, 0), (9, 123456789)):
        first, second, scales = _zeros([(n,)], 8)
        p = torch.zeros(n, device="cuda")
        s2cnn_amd.adamw_step([p], [g], first, second, step, betas=betas, scales=scales, seed=seed)
        (m,), (v,) = s2cnn_amd.adamw_states(first, second, scales)
        for got, want in ((m, 0.1 * 0.01), (v, 0.001 * 0.01 ** 2)):
            small = got.view(-1, 256)[:, 1:].double().flatten()
            assert small.unique().numel() <= 2 and (small / want - 1).abs().max() <= 1 / 8
            assert abs(small.mean().item() / want - 1) <= 6 / 16 / math.sqrt(small.numel()) + 1e-5


@pytest.mark.gpu
def test_gradients_whose_squares_are_subnormal(hip):
    """An eps far below them: the quotient of the moments is one, as exactly as the square is (2^-13 of 2^-136, half of it in the root)."""
    for size in (2.0 ** -68, 2.0 ** -64, 2.0 ** -40, 2.0 ** 60):
        p, g = torch.zeros(600, device="cuda"), torch.full((600,), size, device="cuda")
        m, v = torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
        s2cnn_amd.adamw_step([p], [g], [m], [v], 1, lr=1.0, betas=(0.0, 0.0), eps=1e-30, weight_decay=0.0)
        assert (p + 1).abs().max() <= 2.0 ** -13, size


@pytest.mark.gpu
def test_small_second_moments_never_vanish(hip):
    g = torch.full((300,), 1e-12, device="cuda")
    g[0], g[7], g[299] = 1.0, 0.0, 0.0
    first, second, scales = _zeros([(300,)], 8)
    p = torch.zeros(300, device="cuda")
    s2cnn_amd.adamw_step([p], [g], first, second, 1, scales=scales)
    codes = second[0].cpu()
    assert codes[0] == 255 and codes[7] == 0 and (codes[1:7] == 1).all() and (codes[8:256] == 1).all()
    assert codes[299] == 0 and (scales[0][1, 1] > 0) == bool((codes[256:299] > 0).all())
    assert torch.isfinite(p).all() and p.abs().max() <= 1.001e-3
    # blocks whose factors would be below 2^-126 are zero, moments and factors
    first, second, scales = _zeros([(300,)], 8)
    g = torch.full((300,), 1e-37, device="cuda")
    s2cnn_amd.adamw_step([p], [g], first, second, 1, scales=scales)
    assert (first[0].view(torch.uint8) == 0).all() and (second[0] == 0).all() and (scales[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@TYPES
def test_many_tensors_at_odd_addresses(hip, bits, dtype):
    """More tensors than one launch takes, as views that begin anywhere; what lies between them stays.  8 bits: the random numbers go on from launch to
    launch as in one list."""
    sizes = [(i * 37) % 700 + 1 for i in range(130)]
    total = sum(sizes) + 3 * len(sizes)
    rand = torch.Generator().manual_seed(3)

    def views(dtype, fill):
        flat = torch.full((total,), fill, device="cuda").to(dtype)
        at, out = 1, []
        for n in sizes:
            out.append(flat[at:at + n])
            at += n + 3
        return flat, out

    def inside(flat):
        mask = torch.zeros(total, dtype=torch.bool)
        at = 1
        for n in sizes:
            mask[at:at + n] = True
            at += n + 3
        return flat.cpu()[mask], flat.cpu()[~mask]

    p, params = views(dtype, 0.0)
    g, grads = views(dtype, 0.0)
    g.copy_(torch.randn(total, generator=rand))
    p.copy_(torch.randn(total, generator=rand))
    masters = None
    if dtype != F32:
        m32, masters = views(F32, 0.0)
        m32.copy_(p)
    _, _, scales = _zeros([(n,) for n in sizes], 8)
    if bits == 32:
        a, first = views(F32, 0.0)
        b, second = views(F32, 0.0)
        scales = None
    else:
        a, first = views(torch.uint8, 0)
        b, second = views(torch.uint8, 0)
        first = [t.view(torch.float8_e4m3fn) for t in first]
    outside = [inside(t)[1].clone() for t in (p, a, b)]
    clean = [x.clone() for x in params]
    other = _zeros([(n,) for n in sizes], bits)
    other_masters = [m.clone() for m in masters] if masters else None
    s2cnn_amd.adamw_step(params, grads, first, second, 3, masters=masters, scales=scales, seed=4)
    for x, y in zip(outside, (p, a, b)):
        assert torch.equal(x, inside(y)[1])
    s2cnn_amd.adamw_step(clean, [x.clone() for x in grads], other[0], other[1], 3, masters=other_masters, scales=other[2], seed=4)
    for i in range(len(sizes)):
        assert torch.equal(clean[i], params[i]) and torch.equal(first[i].view(torch.uint8), other[0][i].view(torch.uint8)) and torch.equal(second[i], other[1][i])
        assert masters is None or torch.equal(masters[i], other_masters[i])
    if bits == 8:
        model = _EightBits([(n,) for n in sizes])
        model.step(grads, 3, 4, (0.9, 0.999))
        model.equals(first, second, scales)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_steps_without_a_finite_norm_are_left_out(hip, bits):
    shapes = [(300,), (5000,)]
    params, grads = _random(shapes, F32, 1), _random(shapes, F32, 2)
    first, second, scales = _zeros(shapes, bits)
    s2cnn_amd.adamw_step(params, grads, first, second, 1, scales=scales)
    tensors = params + first + second + (scales or [])
    before = [t.clone() for t in tensors]
    for bad in (float("inf"), float("nan"), -float("inf")):
        grads[1][77] = bad
        norm = s2cnn_amd.grad_norm(grads)
        assert not torch.isfinite(norm)
        s2cnn_amd.adamw_step(params, grads, first, second, 2, scales=scales, norm=norm, max_norm=1.0)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, tensors))
    # zero gradients: a factor of one
    norm = s2cnn_amd.grad_norm([torch.zeros(3, device="cuda")])
    assert norm.item() == 0
    grads[1][77] = 0.0
    clone = [[t.clone() for t in x] if x else None for x in (params, first, second, scales)]
    s2cnn_amd.adamw_step(params, grads, first, second, 2, scales=scales, norm=norm, max_norm=1.0)
    s2cnn_amd.adamw_step(clone[0], grads, clone[1], clone[2], 2, scales=clone[3])
    assert all(torch.equal(a, b) for a, b in zip(params, clone[0]))
    # without a norm: 32 bits hold what there is entry by entry, 8 bits lose the block of 256
    grads[0][3] = float("nan")
    s2cnn_amd.adamw_step(params, grads, first, second, 3, scales=scales)
    m = first if bits == 32 else s2cnn_amd.adamw_states(first, second, scales)[0]
    assert m[0][:256].isnan().sum() == (1 if bits == 32 else 256) and torch.isfinite(m[0][256:]).all() and torch.isfinite(m[1]).all()
    assert params[0].isnan().nonzero().flatten().tolist() == [3]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_masters_hold_small_steps_and_follow_the_program(hip, dtype):
    shapes = [(1000,)]
    params, grads = [torch.ones(1000, dtype=dtype, device="cuda")], [torch.ones(1000, dtype=dtype, device="cuda")]
    masters = [p.float() for p in params]
    first, second, _ = _zeros(shapes, 32)
    for step in range(1, 101):                                               # steps of 1e-5: far below a rounding
        s2cnn_amd.adamw_step(params, grads, first, second, step, lr=1e-5, weight_decay=0.0, masters=masters)
    assert (masters[0] - (1 - 1e-3)).abs().max() < 1e-5 and torch.equal(params[0], masters[0].to(dtype))
    params[0][10:20] = 5.0
    kept = masters[0].clone()
    s2cnn_amd.adamw_step(params, grads, first, second, 101, lr=1e-5, weight_decay=0.0, masters=masters)
    assert (masters[0][10:20] - (5 - 1e-5)).abs().max() < 2e-6
    assert (masters[0][:10] - kept[:10] + 1e-5).abs().max() < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@TYPES
@pytest.mark.parametrize("weight_decay", [0.0, 0.1])
def test_infinite_parameters_stay(hip, weight_decay, dtype, bits):
    """Masks among the parameters, as torch's p (1 - lr weight_decay) leaves them; the type's lowest values move; what is no number stays none."""
    lowest = torch.finfo(dtype).min
    start = torch.tensor([-math.inf, math.inf, math.nan, lowest, -lowest, 1.0] * 50).to(dtype).cuda()
    for size in (0.0, 1.0):
        p, masters = [start.clone()], [start.float()] if dtype != F32 else None
        first, second, scales = _zeros([start.shape], bits)
        for step in (1, 2):
            g = [torch.full_like(start, size)]
            s2cnn_amd.adamw_step(p, g, first, second, step, lr=0.5, weight_decay=weight_decay, masters=masters, scales=scales)
        for t in p + (masters or []):
            assert torch.equal(t[0::6], start[0::6].to(t.dtype)) and torch.equal(t[1::6], start[1::6].to(t.dtype)) and t[2::6].isnan().all()
            assert torch.isfinite(t.view(-1, 6)[:, 3:]).all() and (t[3::6] < 0).all() and (t[4::6] > 0).all()
            if size == 0.0:                                                              # with gradients a master of float16 moves from -65504 by two steps of 0.5
                assert (t[3::6] == lowest).all() == (t[5::6] == 1).all() == (weight_decay == 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_numbers_on_the_device_and_captured_steps(hip, bits):
    """The step and the learning rate as tensors give the same results as numbers; a captured step reads them at every replay."""
    shapes = [(40, 30), (77,), (5000,)]
    grads = _random(shapes, F32, 5, 0.01)
    sides = []
    for _ in range(3):
        sides.append((_random(shapes, F32, 4), *_zeros(shapes, bits)))
    rates = [0.01, 0.003, 0.02, 0.001]
    count, lr = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros((), device="cuda")

    def run(side, step, lr):
        params, first, second, scales = side
        s2cnn_amd.adamw_step(params, grads, first, second, step, lr=lr, scales=scales, norm=s2cnn_amd.grad_norm(grads), max_norm=0.5, seed=8)

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        s2cnn_amd.grad_norm(grads)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count.add_(1)
        run(sides[2], count, lr)
    for i, rate in enumerate(rates):
        rate = ctypes.c_float(rate).value
        for g in grads:
            g.mul_(1.1)
        lr.fill_(rate)
        graph.replay()
        run(sides[0], i + 1, rate)
        run(sides[1], torch.tensor([i + 1], device="cuda"), torch.tensor(rate, device="cuda"))
        torch.cuda.synchronize()
        flat = [[t for x in side if x for t in x] for side in sides]
        for a, b, c in zip(*flat):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(a.view(torch.uint8), c.view(torch.uint8))


@pytest.mark.gpu
def test_graphs_that_saved_a_parameter_notice_the_step(hip):
    """As after any operation in place: a backward pass through the old value is refused, not made with the new one."""
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    loss = (p * p).sum()
    s2cnn_amd.adamw_step([p], [torch.ones(5, device="cuda")], [torch.zeros(5, device="cuda")], [torch.zeros(5, device="cuda")], 1)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


@pytest.mark.gpu
def test_two_graphs_and_streams_between_each_other(hip):
    """Captured steps of two lists, replayed in turns on two streams with eager norms between them: each as by itself."""
    shapes = [(3000,), (77, 5)]
    lists = [(_random(shapes, F32, i), _random(shapes, F32, 10 + i, 0.1), *_zeros(shapes, 8)) for i in range(2)]
    alone = [[[t.clone() for t in x] for x in side] for side in lists]
    counts = [torch.zeros(1, dtype=torch.int64, device="cuda") for _ in range(2)]
    graphs, norms = [torch.cuda.CUDAGraph() for _ in range(2)], [None, None]

    def step(side, count, seed):
        params, grads, first, second, scales = side
        norm = s2cnn_amd.grad_norm(grads)
        s2cnn_amd.adamw_step(params, grads, first, second, count, scales=scales, norm=norm, max_norm=0.3, seed=seed)
        return norm

    s2cnn_amd.grad_norm(lists[0][1])
    torch.cuda.synchronize()
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            counts[i].add_(1)
            norms[i] = step(lists[i], counts[i], i)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        other = s2cnn_amd.grad_norm(lists[1][1])
        torch.cuda.synchronize()
        assert torch.equal(other, norms[1])
    for i in range(2):
        for turn in range(4):
            step(alone[i], turn + 1, i)
        for a, b in zip(lists[i], alone[i]):
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


# ---- the norm -------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_grad_norm(hip):
    sizes = [1, 2, 7, 8, 9, 0, 1000, 16383, 16384, 16385, 32769, 300001]
    gen = torch.Generator().manual_seed(0)
    mixed = []
    for i, n in enumerate(sizes):
        for dtype in (F32, BF16, F16):
            t = torch.randn(n, generator=gen).to(dtype).cuda()
            one = s2cnn_amd.grad_norm([t])
            want = t.double().norm().item()
            assert one.dtype == F32 and one.shape == () and abs(one.item() - want) <= 2 * W * want, (n, dtype)
            if n:
                mixed += [t, torch.cat([t, t])[1:1 + n]]
    many = mixed * 8                                                      # several launches
    assert len(many) > 400
    want = math.sqrt(sum(t.double().square().sum().item() for t in many))
    got = s2cnn_amd.grad_norm(many)
    assert abs(got.item() - want) <= 2 * W * want and torch.equal(got, s2cnn_amd.grad_norm(iter(many)))
    assert s2cnn_amd.grad_norm([]).item() == 0 and s2cnn_amd.grad_norm([torch.zeros(0, device="cuda")]).item() == 0
    strided = torch.randn(50, 60, generator=gen).cuda().T
    assert abs(s2cnn_amd.grad_norm([strided]).item() - strided.double().norm().item()) <= 2 * W * strided.double().norm().item()


@pytest.mark.gpu
def test_grad_norm_of_lists_larger_than_the_caches(hip):
    """From 256 MB on they are read past the caches."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    for dtype, n in ((F32, 70000001), (BF16, 140000003)):
        t = torch.randn(n, device="cuda", generator=gen).to(dtype)
        want = math.sqrt(sum(p.double().square().sum().item() for p in t.split(1 << 24)))
        assert abs(s2cnn_amd.grad_norm([t]).item() - want) <= 2 * W * want
        assert torch.equal(s2cnn_amd.grad_norm([t[:1 << 20]]), s2cnn_amd.grad_norm([t[:1 << 20].clone()]))


@pytest.mark.gpu
def test_grad_norm_of_extreme_values(hip):
    for value in (1e30, 1e-30, 3e38, 1e-44):
        t = torch.full((1000,), value, device="cuda")
        want = t[0].double().item() * math.sqrt(1000)
        got = s2cnn_amd.grad_norm([t]).item()
        assert got == math.inf if want > 3.5e38 else abs(got - want) <= 2 * W * want + 2.0 ** -149
    for value in (float("inf"), float("nan")):
        t = torch.ones(20000, device="cuda")
        t[19999] = value
        assert not math.isfinite(s2cnn_amd.grad_norm([torch.ones(5, device="cuda"), t]).item())


@pytest.mark.gpu
def test_grad_norm_is_not_differentiated(hip):
    """What would have a graph, or a tangent, is refused and not cut off without a word: a penalty on it would train nothing."""
    x = torch.nn.Parameter(torch.randn(300, 5, device="cuda"))
    g, = torch.autograd.grad(x.pow(3).sum(), x, create_graph=True)
    for tensors in ([g], [x], [x.detach(), x], [x.T], [x.detach().half(), g]):
        with pytest.raises(AssertionError, match="not differentiated"):
            s2cnn_amd.grad_norm(tensors)
        with torch.no_grad():
            norm = s2cnn_amd.grad_norm(tensors)
        assert torch.equal(norm, s2cnn_amd.grad_norm([t.detach() for t in tensors])) and not norm.requires_grad
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(AssertionError, match="not differentiated"):
            s2cnn_amd.grad_norm([x, forward_ad.make_dual(x.detach(), torch.ones_like(x))])
        assert torch.equal(s2cnn_amd.grad_norm([x]), s2cnn_amd.grad_norm([x.detach()]))


# ---- the optimizer --------------------------------------------------------------------------------------------------
def _network(dtype=F32):
    torch.manual_seed(3)
    return torch.nn.Sequential(torch.nn.Linear(20, 33), torch.nn.ReLU(), torch.nn.Linear(33, 7)).cuda().to(dtype)


def _backward(net, i):
    net.zero_grad(set_to_none=True)
    x = torch.randn(16, 20, generator=torch.Generator().manual_seed(i)).to(next(net.parameters()).dtype).cuda()
    net(x).square().mean().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [None, 0.05])
def test_optimizer_follows_torchs(hip, clip):
    """float32 against torch's own in 64 bits on the CPU with the same gradients: ten steps, each off by what _check_step allows of the update, and
    the tensors' own roundings."""
    net = _network()
    ref = [p.detach().cpu().double().requires_grad_() for p in net.parameters()]
    opt = s2cnn_amd.AdamW([{"params": list(net[0].parameters())}, {"params": list(net[2].parameters()), "lr": 0.003, "weight_decay": 0.0}], lr=0.01, betas=(0.8, 0.95),
                          weight_decay=0.1, max_norm=clip)
    want = torch.optim.AdamW([{"params": ref[:2]}, {"params": ref[2:], "lr": 0.003, "weight_decay": 0.0}], lr=0.01, betas=(0.8, 0.95), weight_decay=0.1)
    schedules = [torch.optim.lr_scheduler.ExponentialLR(o, 0.9) for o in (opt, want)]
    for i in range(10):
        _backward(net, i)
        if i in (3, 4):
            net[2].bias.grad = None                                        # left out of two steps
        for p, r in zip(net.parameters(), ref):
            r.grad = None if p.grad is None else p.grad.detach().cpu().double()
        if clip:
            norm = torch.nn.utils.clip_grad_norm_(ref, clip)
        assert opt.step() is None
        want.step()
        if clip:
            assert abs(opt.norm.item() - norm.item()) <= 4 * W * norm.item() + 1e-6 * norm.item()
        for s in schedules:
            s.step()
    for p, r in zip(net.parameters(), ref):
        # torch clips by max_norm / (norm + 1e-6): 2e-5 of the gradients here, which the quotient of the moments mostly cancels
        allowed = 10 * (4 * W * r.detach().norm().item() + 64 * W * 0.01 * math.sqrt(r.numel())) + (1e-5 * 0.1 * math.sqrt(r.numel()) if clip else 0)
        assert (p.detach().cpu().double() - r.detach()).norm().item() <= allowed
    assert opt.step(lambda: 5.0) == 5.0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@TYPES
def test_state_dicts(hip, bits, dtype):
    """Saved, loaded into another optimizer of another network of the same form, and on: the same bits; types stay."""
    net = _network(dtype)
    opt = s2cnn_amd.AdamW(net.parameters(), lr=0.01, state_bits=bits, max_norm=1.0, seed=9)
    for i in range(3):
        _backward(net, i)
        if i == 1:
            net[2].bias.grad = None
        opt.step()
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    other = copy.deepcopy(net)
    again = s2cnn_amd.AdamW(other.parameters(), state_bits=40 - bits, max_norm=1.0, seed=9)
    again.load_state_dict(torch.load(file, weights_only=True))
    for a, b in zip(opt.state.values(), again.state.values()):
        assert a.keys() == b.keys() and all(a[k].dtype == b[k].dtype and a[k].data_ptr() != b[k].data_ptr() for k in a)
        assert a["first"].dtype == (torch.float8_e4m3fn if bits == 8 else F32) and ("master" in a) == (dtype != F32)
    assert again.param_groups[0]["lr"] == 0.01 and len({id(s["step"]) for s in again.state.values()}) == 2
    for i in range(3, 6):
        for n, o in ((net, opt), (other, again)):
            _backward(n, i)
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(net.parameters(), other.parameters()))
    assert [s["step"].item() for s in opt.state.values()] == [6, 6, 6, 5]


@pytest.mark.parametrize("bits", [8, 32])
def test_hooks_of_loading(bits):
    """What a hook before the loading gives is loaded, in the states' types; what one after it writes stays.  Hooks are the program's: none is left."""
    def make():
        p = torch.nn.Parameter(torch.ones(300, dtype=BF16))
        return p, s2cnn_amd.AdamW([p], state_bits=bits)

    p, opt = make()
    opt.state[p] = opt._new_state(p, opt.param_groups[0], torch.full((1,), 3))
    opt.state[p]["first"].view(torch.uint8).fill_(7)
    saved = opt.state_dict()
    q, other = make()

    def before(_, state_dict):
        return {**state_dict, "state": {i: {**s, "second": s["second"] + 5, "step": s["step"] + 1} for i, s in state_dict["state"].items()}}

    def after(o):
        assert (o.state[q]["second"] == 5).all()
        o.state[q]["master"].fill_(2.0)

    kept = [other.register_load_state_dict_pre_hook(before), other.register_load_state_dict_post_hook(after)]
    for times in range(2):
        other.load_state_dict(saved)
        state = other.state[q]
        assert state["step"].item() == 4 and state["step"].dtype == torch.int64 and (state["second"] == 5).all() and (state["master"] == 2).all()
        assert state["first"].dtype == opt.state[p]["first"].dtype and state["second"].dtype == opt.state[p]["second"].dtype and state["master"].dtype == F32
        assert torch.equal(state["first"].view(torch.uint8), opt.state[p]["first"].view(torch.uint8)) and state["first"].data_ptr() != opt.state[p]["first"].data_ptr()
        assert (opt.state[p]["second"] == 0).all() and opt.state[p]["step"].item() == 3
    for hook in kept:
        hook.remove()
    with pytest.raises(ValueError):
        other.load_state_dict({"state": {}, "param_groups": []})
    other.load_state_dict(saved)
    assert (other.state[q]["second"] == 0).all() and (other.state[q]["master"] == 1).all() and other.state[q]["step"].item() == 3
    assert not other._optimizer_load_state_dict_pre_hooks and not other._optimizer_load_state_dict_post_hooks


@pytest.mark.gpu
def test_loaded_groups_count_their_own_steps(hip):
    """Two groups of as many steps, saved and loaded: one step counts one in each."""
    params = [torch.nn.Parameter(torch.ones(30, device="cuda")) for _ in range(4)]
    make = lambda: s2cnn_amd.AdamW([{"params": params[:2]}, {"params": params[2:], "lr": 0.5}], lr=0.1)
    for p in params:
        p.grad = torch.ones_like(p)
    opt = make()
    opt.step()
    again = make()
    again.load_state_dict(opt.state_dict())
    again.step()
    assert [again.state[p]["step"].item() for p in params] == [2] * 4 and len({id(again.state[p]["step"]) for p in params}) == 2
    assert [opt.state[p]["step"].item() for p in params] == [1] * 4


@pytest.mark.gpu
def test_lists_of_a_step_round_apart(hip):
    """Groups of equal gradients, moments in 8 bits: the first list's codes are those of adamw_step with the seed, the others' are rounded at random numbers of
    their own.  A code is one of two: of n independent ones, each rounded up with the same probability on both sides, at least n / 100 differ where it
    lies between 0.1 and 0.9 for a tenth of them (n / 10 * 2 * 0.09 = n / 55 expected; the spread is below sqrt(n))."""
    n = 20000
    g = torch.randn(n, generator=torch.Generator().manual_seed(2)).cuda()
    params = [torch.nn.Parameter(torch.ones(n, device="cuda", dtype=d)) for d in (F32, F32, F32, BF16)]
    opt = s2cnn_amd.AdamW([{"params": params[:1]}, {"params": params[1:2], "weight_decay": 0.0}, {"params": params[2:]}], state_bits=8, seed=-3)
    for p in params:
        p.grad = g.to(p.dtype)
    opt.step()
    first, second, scales = _zeros([(n,)], 8)
    s2cnn_amd.adamw_step([torch.ones(n, device="cuda")], [g], first, second, 1, scales=scales, seed=-3)
    codes = [[opt.state[p][k].view(torch.uint8) for k in ("first", "second")] for p in params]
    assert torch.equal(codes[0][0], first[0].view(torch.uint8)) and torch.equal(codes[0][1], second[0])
    for i in range(4):
        for j in range(i):
            for a, b in zip(codes[i], codes[j]):
                assert (a != b).sum().item() > n / 100, (i, j)


@pytest.mark.gpu
@pytest.mark.parametrize("option,then", [("state_bits", 8), ("state_bits", 32), ("masters", False), ("masters", True)])
def test_options_changed_between_first_steps(hip, option, then):
    """Parameters keep what they were first stepped with; loaded with equal counts they go on together, each as it is held."""
    before = {"state_bits": 40 - then} if option == "state_bits" else {"masters": not then}
    params = [torch.nn.Parameter(torch.ones(300, device="cuda", dtype=BF16)) for _ in range(3)]
    opt = s2cnn_amd.AdamW(params, lr=0.1, **before)
    params[0].grad = torch.ones_like(params[0])
    opt.step()
    params[0].grad = None
    opt.param_groups[0][option] = then
    for p in params[1:]:
        p.grad = torch.ones_like(p)
    opt.step()
    again = s2cnn_amd.AdamW(params, lr=0.1)
    again.load_state_dict(opt.state_dict())
    held = [set(again.state[p]) for p in params]
    assert held[1] == held[2] != held[0] and len({id(again.state[p]["step"]) for p in params}) == 1
    kept = [p.detach().clone() for p in params]
    params[0].grad = torch.ones_like(params[0])
    for o in (again, again):
        o.step()
    assert all(again.state[p]["step"].item() == 3 for p in params) and all((p < k).all() for p, k in zip(params, kept))
    assert [set(again.state[p]) for p in params] == held and torch.equal(params[1], params[2])
    assert all(torch.equal(p, again.state[p]["master"].to(BF16)) for p in params if "master" in again.state[p])


@pytest.mark.gpu
def test_groups_types_and_steps_left_out(hip):
    """Parameters of two types and a group in 8 bits; a step without a finite norm is neither made nor counted."""
    a, b, c = (torch.nn.Parameter(torch.ones(300, device="cuda", dtype=d)) for d in (F32, BF16, F32))
    opt = s2cnn_amd.AdamW([a, b], lr=0.1, max_norm=1.0)
    opt.add_param_group({"params": [c], "state_bits": 8, "weight_decay": 0.5})
    for p in (a, b, c):
        p.grad = torch.ones_like(p)
    opt.step()
    kept = [p.detach().clone() for p in (a, b, c)]
    assert all((p < 1).all() for p in kept) and (kept[2] < kept[0]).all() and abs(opt.norm.item() - 30) < 1e-4
    a.grad[5] = float("inf")
    opt.step()
    assert all(torch.equal(p, k) for p, k in zip((a, b, c), kept)) and all(s["step"].item() == 1 for s in opt.state.values())
    a.grad[5] = 1.0
    opt.step()
    assert all((p < k).all() for p, k in zip((a, b, c), kept)) and all(s["step"].item() == 2 for s in opt.state.values())
    assert opt.state[c]["first"].dtype == torch.float8_e4m3fn and opt.state[b]["master"].dtype == F32


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [None, 1.0])
def test_refused_steps_are_neither_made_nor_counted(hip, clip):
    """What one list is refused for leaves the lists before it, and all counts, as they were."""
    params = [torch.nn.Parameter(torch.ones(4, 3, device="cuda")) for _ in range(3)]
    opt = s2cnn_amd.AdamW([{"params": params[:1]}, {"params": params[1:]}], lr=0.1, max_norm=clip)
    for p in params:
        p.grad = torch.ones_like(p)
    opt.step()
    kept = [p.detach().clone() for p in params]
    group, data = opt.param_groups[1], params[2].data

    def unchanged():
        assert all(torch.equal(p, k) for p, k in zip(params, kept))
        assert all(opt.state[p]["step"].item() == 1 for p in params) and all((opt.state[p]["first"] == opt.state[params[0]]["first"][0, 0]).all() for p in params)

    group["lr"] = -1.0
    with pytest.raises(AssertionError):
        opt.step()
    unchanged()
    group["lr"] = 0.1
    params[2].data = data.T
    with pytest.raises(RuntimeError, match="contiguous"):
        opt.step()
    params[2].data = data
    unchanged()
    opt.step()
    assert all(opt.state[p]["step"].item() == 2 for p in params) and all((p < k).all() for p, k in zip(params, kept))


@pytest.mark.gpu
def test_captured_training_steps(hip):
    """Backward pass, norm and step in one graph, against the same steps made eagerly."""
    nets = [_network() for _ in range(2)]
    opts = [s2cnn_amd.AdamW(n.parameters(), lr=0.01, state_bits=8, max_norm=0.5) for n in nets]
    x = torch.randn(16, 20, device="cuda")

    def step(net, opt):
        opt.zero_grad(set_to_none=True)
        net(x).square().mean().backward()
        opt.step()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(nets[0], opts[0])
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        step(nets[1], opts[1])
    graph = torch.cuda.CUDAGraph()
    opts[0].zero_grad(set_to_none=True)
    with torch.cuda.graph(graph):
        step(nets[0], opts[0])
    for _ in range(4):
        graph.replay()
        step(nets[1], opts[1])
        torch.cuda.synchronize()
        for p, q in zip(nets[0].parameters(), nets[1].parameters()):
            assert (p - q).norm() <= 1e-5 * q.norm()
    assert {s["step"].item() for o in opts for s in o.state.values()} == {6}


@pytest.mark.gpu
def test_captured_steps_need_a_step_before(hip):
    """A capture that would make moments, or begin a count of steps, is refused; the program goes on with eager steps."""
    net = _network()
    params = list(net.parameters())
    opt = s2cnn_amd.AdamW(params, lr=0.01)
    for p in params:
        p.grad = torch.ones_like(p)

    def refused(match):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=match):
            with torch.cuda.graph(graph):
                opt.step()

    refused("begins with a parameter")
    assert not any(opt.state[p] for p in params if p in opt.state)
    opt.step()
    params[1].grad = None
    refused("leaves a parameter out")
    before = [p.detach().clone() for p in params]
    opt.step()
    assert [opt.state[p]["step"].item() for p in params] == [2, 1, 2, 2] and torch.equal(before[1], params[1]) and not torch.equal(before[0], params[0])


@pytest.mark.gpu
def test_moments_of_a_parameter(hip):
    """Of 8 bits within a spacing (1/8) of those of 32, after one step; None before it."""
    g = torch.randn(40, 30, generator=torch.Generator().manual_seed(1)).cuda()
    got = []
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(40, 30, device="cuda"))
        opt = s2cnn_amd.AdamW([p], state_bits=bits)
        assert opt.moments(p) is None
        p.grad = g.clone()
        opt.step()
        got.append(opt.moments(p))
    for a, b, of in zip(*got, (0.1 * g, 0.001 * g * g)):
        assert a.dtype == b.dtype == F32 and a.shape == b.shape == p.shape
        assert (a - of).abs().max() <= 8 * W * of.abs().max()
        assert ((a - b).abs() <= a.abs() / 8 + 1e-4 * a.abs().max()).all()


@pytest.mark.gpu
def test_copies_of_an_optimizer(hip):
    """copy.deepcopy and pickles keep the clipping and the seed."""
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = s2cnn_amd.AdamW([p], lr=0.1, state_bits=8, max_norm=0.5, seed=7)
    opt.step()
    twin = copy.deepcopy(opt)
    q = twin.param_groups[0]["params"][0]
    q.grad = p.grad.clone()
    for o in (opt, twin):
        o.step()
    assert twin.max_norm == 0.5 and twin.seed == 7 and torch.equal(p, q) and torch.equal(opt.state[p]["second"], twin.state[q]["second"])


# ---- refusals -------------------------------------------------------------------------------------------------------
def test_refusals_before_the_gpu():
    t = [torch.zeros(3)]
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.grad_norm(t)
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.adamw_step(t, t, t, t, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.adamw_states([torch.zeros(3).to(torch.float8_e4m3fn)], [torch.zeros(3, dtype=torch.uint8)], [torch.zeros(1, 2)])
    for kw in ({"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": 0.0}, {"eps": 1e-31}, {"weight_decay": -1.0}, {"lr": -1.0}, {"lr": float("nan")}, {"seed": 0.5},
               {"norm": torch.zeros(())}, {"max_norm": 1.0}, {"norm": torch.zeros(()), "max_norm": 0.0}, {"norm": torch.zeros(2), "max_norm": 1.0}, {"lr": torch.zeros(2)}):
        with pytest.raises(AssertionError):
            s2cnn_amd.adamw_step(t, t, t, t, 1, **kw)
    for step in (0, -1, 1.5, torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(AssertionError):
            s2cnn_amd.adamw_step(t, t, t, t, step)
    with pytest.raises(AssertionError):
        s2cnn_amd.adamw_step(t, t + t, t, t, 1)
    s2cnn_amd.adamw_step([], [], [], [], 1)
    assert s2cnn_amd.adamw_states([], [], []) == ([], [])
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in ({"state_bits": 16}, {"betas": (0.9, 1.0)}, {"eps": 0.0}, {"max_norm": 0.0}, {"lr": -1.0}, {"weight_decay": float("inf")}):
        with pytest.raises(AssertionError):
            s2cnn_amd.AdamW(p, **kw)
    with pytest.raises(RuntimeError):
        s2cnn_amd.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])


def test_refused_groups_are_not_added():
    p, q = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    opt = s2cnn_amd.AdamW([p])
    for group in ({"params": [q], "state_bits": 16}, {"params": [q], "eps": 0.0}, {"params": [q], "lr": -1.0},
                  {"params": [torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))]}):
        with pytest.raises((AssertionError, RuntimeError)):
            opt.add_param_group(group)
        assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [q], "state_bits": 8})
    assert [len(g["params"]) for g in opt.param_groups] == [1, 1]


@pytest.mark.gpu
def test_refusals_of_tensors(hip):
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    step = s2cnn_amd.adamw_step
    good = lambda: ([z(4, 3)], [z(4, 3)], [z(4, 3)], [z(4, 3)])
    step(*good(), 1)
    for i, wrong in ((0, z(4, 3).half()), (0, z(4, 3).double()), (0, z(3, 4).T), (1, z(4, 3).half()), (1, torch.zeros(4, 3)), (2, z(4, 3).half()), (2, z(3, 4).T),
                     (3, z(4, 3, d=torch.uint8)), (3, torch.zeros(4, 3))):
        lists = good()
        lists[i][0] = wrong
        with pytest.raises(RuntimeError):
            step(*lists, 1)
    for i, wrong in ((0, z(3, 5)), (1, z(13)), (2, z(4, 2)), (3, z(13))):
        lists = good()
        lists[i][0] = wrong
        with pytest.raises(AssertionError):
            step(*lists, 1)
    p = z(5)
    with pytest.raises(AssertionError, match="twice"):
        step([p, z(5), p], [z(5)] * 3, [z(5) for _ in range(3)], [z(5) for _ in range(3)], 1)
    with pytest.raises(AssertionError, match="masters"):
        step(*good(), 1, masters=[z(4, 3)])
    eight = lambda: ([z(300)], [z(300)], [z(300, d=torch.uint8).view(torch.float8_e4m3fn)], [z(300, d=torch.uint8)], 1)
    step(*eight(), scales=[z(2, 2)])
    for scales in ([z(1, 2)], [z(2, 1)], []):
        with pytest.raises(AssertionError):
            step(*eight(), scales=scales)
    for scales in (None, [z(2, 2, d=torch.float64)], [z(2, 2).T], [torch.zeros(2, 2)]):
        with pytest.raises(RuntimeError):
            step(*eight(), scales=scales)
    for kw in ({"norm": z(1).double(), "max_norm": 1.0}, {"norm": torch.zeros(1), "max_norm": 1.0}, {"lr": z(1).double()}):
        with pytest.raises(RuntimeError):
            step(*good(), 1, **kw)
    with pytest.raises(RuntimeError):
        step(*good(), z(1))
    with pytest.raises(RuntimeError):
        s2cnn_amd.grad_norm([z(3), z(3).double()])
    with pytest.raises(RuntimeError):
        s2cnn_amd.grad_norm([z(3), torch.zeros(3)])


def test_lists_of_tensors():
    """What s2cnn_tensor_list says of tensors in host memory (device type 1 of DLPack), against torch's own words."""
    from array import array
    from s2cnn_amd import _hip
    fn, describe = _hip.tensor_list()
    at = lambda a: a.buffer_info()[0]

    def run(tensors, code=2, bits=32, known=None):
        objects, out = array("Q", map(id, tensors)), array("Q", bytes(8 * len(tensors)))
        n = array("q", bytes(8 * len(tensors))) if known is None else array("q", known)
        return fn(describe, at(objects), len(tensors), code, bits, 1, 0, at(out), at(n), int(known is not None)), list(out), list(n)

    base = torch.zeros(4, 6)
    good = [base, torch.nn.Parameter(torch.zeros(3)), torch.zeros(()), base.view(-1)[5:], torch.zeros(2, 0, 3), base[2:3, :], base[:1].T, torch.zeros(5, 1, 2)[:, 0]]
    rc, addresses, n = run(good)
    assert rc == 0 and n == [t.numel() for t in good] and addresses == [t.data_ptr() for t in good]
    assert run(good, known=n)[0] == 0 and run(good, known=n[:3] + [1] + n[4:])[0] == 4
    for wrong in (base.T, base[:, 1:], base.expand(2, 4, 6), torch.zeros(3, dtype=torch.float64), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.complex64)):
        assert run([base, wrong, base])[0] == 2
    assert run([base.half()], 2, 16)[0] == run([base.bfloat16()], 4, 16)[0] == run([base.to(torch.float8_e4m3fn)], 10, 8)[0] == run([base.byte()], 1, 8)[0] == 0
    assert run([base.bfloat16()], 2, 16)[0] == run([base.to(torch.float8_e5m2)], 10, 8)[0] == run([base.char()], 1, 8)[0] == 1
    with pytest.raises(Exception):
        run([torch.zeros(2, device="meta")])
    assert fn(None, None, 0, 2, 32, 1, 0, None, None, 0) == -1 and fn(describe, None, 1, 2, 32, 1, 0, None, None, 0) == -1 and fn(describe, None, -1, 2, 32, 1, 0, None, None, 0) == -1


@pytest.mark.gpu
def test_lists_without_the_exchange_interface(hip, monkeypatch):
    """Tensor by tensor, as for subclasses of tensors: the same results and refusals."""
    from s2cnn_amd import _hip
    shapes = [(300,), (7, 3), (0,)]
    sides = []
    for direct in (True, False):
        if not direct:
            monkeypatch.setattr(_hip, "tensor_list", lambda: None)
        params, grads, (first, second, scales) = _random(shapes, BF16, 1), _random(shapes, BF16, 2), _zeros(shapes, 8)
        grads[1] = grads[1].T.contiguous().T
        masters = [p.float() for p in params]
        s2cnn_amd.adamw_step(params, grads, first, second, 1, masters=masters, scales=scales, norm=s2cnn_amd.grad_norm(grads), max_norm=1.0)
        m, v = s2cnn_amd.adamw_states(first, second, scales)
        sides.append(params + masters + m + v)
        for bad in ((grads[0].float(), 1), (params[1].T, 0), (first[0].view(torch.uint8), 2)):
            lists = [list(x) for x in (params, grads, first, second)]
            lists[bad[1]][0] = bad[0]
            with pytest.raises(RuntimeError):
                s2cnn_amd.adamw_step(*lists, 1, masters=masters, scales=scales)
    assert all(torch.equal(a, b) for a, b in zip(*sides))


def test_entry_points_refuse_lists():
    """The C entries, before any launch."""
    from s2cnn_amd import _hip
    lib = _hip.lib()
    null, fake = (ctypes.c_void_p * 1)(0), (ctypes.c_void_p * 1)(0x1000)
    odd = (ctypes.c_void_p * 1)(0x1002)
    n = (ctypes.c_long * 1)(5)
    at = lambda x: ctypes.cast(x, ctypes.c_void_p).value

    def run(**kw):
        a = _hip.AdamW()
        a.p = a.g = a.first = a.second = at(fake)
        a.n, a.count, a.dtype, a.bits, a.step = at(n), 1, 0, 32, 1
        a.lr, a.beta1, a.beta2, a.eps = 1e-3, 0.9, 0.99, 1e-8
        for k, v in kw.items():
            setattr(a, k, at(v) if isinstance(v, ctypes.Array) else v)
        return lib.s2cnn_adamw_step(ctypes.byref(a), None)

    for kw, rc in (({"count": -1}, -1), ({"dtype": 3}, -1), ({"bits": 16}, -1), ({"bits": 8}, -1), ({"scales": fake}, -1), ({"masters": fake}, -1), ({"p": null}, -1),
                   ({"g": null}, -1), ({"first": null}, -1), ({"second": null}, -1), ({"p": None}, -1), ({"n": None}, -1), ({"n": (ctypes.c_long * 1)(-1)}, -1),
                   ({"n": (ctypes.c_long * 1)(1 << 42)}, -1), ({"step": 0}, -1), ({"beta1": 1.0}, -1), ({"beta2": -0.5}, -1), ({"eps": 0.0}, -1), ({"lr": -1.0}, -1),
                   ({"lr": float("nan")}, -1), ({"weight_decay": -1.0}, -1), ({"norm": 0x1000}, -1), ({"norm": 0x1002, "max_norm": 1.0}, -3), ({"lr_at": 0x1002}, -3),
                   ({"step_at": 0x1004}, -3), ({"p": odd}, -3), ({"second": odd}, -3), ({"dtype": 1, "masters": odd}, -3), ({"dtype": 1, "masters": null}, -1),
                   ({"bits": 8, "scales": (ctypes.c_void_p * 1)(0x1004)}, -3), ({"bits": 8, "scales": null}, -1)):
        assert run(**kw) == rc, kw
    assert lib.s2cnn_adamw_step(None, None) == -1
    assert run(count=0) == 0                                                                # nothing to do
    f, o, z = at(fake), at(odd), at(null)
    assert lib.s2cnn_adamw_states(f, f, f, f, f, at(n), -1, None) == -1 and lib.s2cnn_adamw_states(f, f, z, f, f, at(n), 1, None) == -1
    assert lib.s2cnn_adamw_states(f, f, f, o, f, at(n), 1, None) == -3 and lib.s2cnn_adamw_states(None, None, None, None, None, None, 0, None) == 0
    kinds = (ctypes.c_int * 1)(0)
    assert lib.s2cnn_grad_norm_workspace(at(n), at(kinds), 1) == 8 and lib.s2cnn_grad_norm_workspace(at(n), at((ctypes.c_int * 1)(3)), 1) == 0
    assert lib.s2cnn_grad_norm_workspace(None, None, 1) == 0 and lib.s2cnn_grad_norm_workspace(at((ctypes.c_long * 1)(8193)), at(kinds), 1) == 16
    assert lib.s2cnn_grad_norm(z, at(n), at(kinds), 1, 0x1000, 0x1000, 8, None) == -1 and lib.s2cnn_grad_norm(f, at(n), at(kinds), 1, 0x1000, 0x1000, 7, None) == -2
    assert lib.s2cnn_grad_norm(o, at(n), at(kinds), 1, 0x1000, 0x1000, 8, None) == -3 and lib.s2cnn_grad_norm(f, at(n), at(kinds), 1, 0x1002, 0x1000, 8, None) == -3
    assert lib.s2cnn_grad_norm(f, at(n), at(kinds), 1, None, 0x1000, 8, None) == -1 and lib.s2cnn_grad_norm(f, at(n), at(kinds), 1, 0x1000, None, 8, None) == -2


def test_entry_points_refuse_tensors_twice():
    """One that is written by two workgroups of a launch, in one list or in two; refused on the host.  Tensors without entries may be anything."""
    from s2cnn_amd import _hip
    lib = _hip.lib()
    names = ("p", "g", "first", "second", "scales", "masters")

    def run(count, same=None, empty=()):
        arrays = {k: [0x1000000 * (j + 1) + 0x1000 * i for i in range(count)] for j, k in enumerate(names)}
        if same:
            (a, i), (b, j) = same
            arrays[a][i] = arrays[b][j]
        a, keep = _hip.AdamW(), []
        for k, v in arrays.items():
            keep.append((ctypes.c_void_p * count)(*v))
            setattr(a, k, ctypes.cast(keep[-1], ctypes.c_void_p).value)
        keep.append((ctypes.c_long * count)(*(0 if i in empty or not same else 5 for i in range(count))))
        a.n, a.count, a.dtype, a.bits, a.step = ctypes.cast(keep[-1], ctypes.c_void_p).value, count, 1, 8, 1
        a.lr, a.beta1, a.beta2, a.eps = 1e-3, 0.9, 0.99, 1e-8
        return lib.s2cnn_adamw_step(ctypes.byref(a), None)

    written = [k for k in names if k != "g"]
    for count in (2, 3, 56, 57, 500):
        for a in written:
            assert run(count, ((a, 0), (a, count - 1))) == -1
            for b in written:
                if a != b:
                    assert run(count, ((a, 0), (b, 1))) == run(count, ((a, 1), (b, 1))) == -1
        assert run(count, (("p", 0), ("p", 1)), empty=range(count)) != -1         # nothing to do: not refused (where there is no GPU its status tells of that)


def test_sizes_that_fit_a_launch():
    """A launch has fewer than 2^32 threads: tensors of more are refused, the largest is not."""
    from s2cnn_amd import _hip
    lib = _hip.lib()
    most = (1 << 35) - 2048
    odd, fake = ((ctypes.c_void_p * 1)(x) for x in (0x1002, 0x1000))
    kind = (ctypes.c_int * 1)(0)
    for entries, rc in ((most, -3), (most + 1, -1)):                                        # at the address 0x1002 the largest is refused all the same
        n = (ctypes.c_long * 1)(entries)
        a = _hip.AdamW()
        a.p, a.g, a.first, a.second, a.n = (ctypes.cast(x, ctypes.c_void_p).value for x in (odd, fake, fake, fake, n))
        a.count, a.dtype, a.bits, a.step, a.lr, a.beta1, a.beta2, a.eps = 1, 0, 32, 1, 1e-3, 0.9, 0.99, 1e-8
        assert lib.s2cnn_adamw_step(ctypes.byref(a), None) == rc
        assert lib.s2cnn_adamw_states(fake, fake, fake, odd, fake, n, 1, None) == rc
        assert lib.s2cnn_grad_norm(odd, n, kind, 1, 0x1000, 0x1000, 8, None) == rc
        assert (lib.s2cnn_grad_norm_workspace(n, kind, 1) > 0) == (rc == -3)


@pytest.mark.gpu
def test_moments_given_twice_are_refused(hip):
    z = lambda: torch.zeros(300, device="cuda")
    params, grads, first, second = ([z() for _ in range(3)] for _ in range(4))
    g = grads[:1] * 3                                                                       # gradients are only read
    s2cnn_amd.adamw_step(params, g, first, second, 1)
    for lists in ((params, g, [first[0], first[1], first[0]], second), (params, g, first, first), (params, g, first, [second[0], second[1], params[0]])):
        with pytest.raises(RuntimeError):
            s2cnn_amd.adamw_step(*lists, 1)


@pytest.mark.gpu
def test_lists_of_more_than_a_launch(hip):
    """One tensor 33 times, of 2^19 workgroups each: more than 2^32 threads, in two launches.  Counts of ones are exact."""
    t = torch.ones(1 << 33, dtype=BF16, device="cuda")
    assert s2cnn_amd.grad_norm([t] * 33).item() == np.float32(math.sqrt(33 * 2.0 ** 33))


@pytest.mark.gpu
def test_loaded_rates_are_on_the_gpu(hip):
    """A rate that is a tensor, from a checkpoint that was read to the host."""
    p = torch.nn.Parameter(torch.ones(30, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = s2cnn_amd.AdamW([p], lr=torch.full((1,), 0.25, device="cuda"))
    opt.step()
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    saved = torch.load(file, weights_only=True, map_location="cpu")
    again = s2cnn_amd.AdamW([p], lr=torch.zeros(1, device="cuda"))
    again.load_state_dict(saved)
    before = p.detach().clone()
    again.step()
    assert again.param_groups[0]["lr"].is_cuda and again.param_groups[0]["lr"].item() == 0.25 and not torch.equal(before, p)
    assert not saved["param_groups"][0]["lr"].is_cuda
