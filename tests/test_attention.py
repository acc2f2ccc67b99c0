"""attention (s2cnn_amd/attention.py): forward and gradients against the definition in 64 bits on the CPU.

Tolerances.  u = 2^-24, 2^-8, 2^-11 is the unit roundoff of float32, bfloat16, float16.  float32: a score of magnitude up to
about 8 carries some 8 roundings of that size, so a probability is off by at most 64 u, a gradient by twice that: 128 u in the
2-norm.  The 16-bit types: the result is rounded, an error of 0.45 u on average, and 2 u allowed; what comes before is exact to well
within that.  Differences that cancel (a softmax over one key has no gradient)
are float32 sums: 4 * 2^-24 of the sum of magnitudes on top."""
import math

import pytest
import torch

import s2cnn_amd

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 128 * 2.0 ** -24, BF16: 2 * 2.0 ** -8, F16: 2 * 2.0 ** -11}


def _reference(q, k, v, table=None, buckets=None, key_bias=None, lengths=None, scale=None, g=None):
    """Everything in 64 bits on the CPU; with g also the gradients and, per gradient, the sum of magnitudes."""
    dt = torch.float64
    q, k, v = (t.detach().cpu().to(dt) for t in (q, k, v))
    b, h, nq, d = q.shape
    hk, nk = k.shape[1:3]
    scale = 1 / math.sqrt(d) if scale is None else scale
    kk, vv = (t.repeat_interleave(h // hk, 1) for t in (k, v))
    out_of = torch.zeros(b, 1, nq, nk, dtype=torch.bool)
    if lengths is not None:
        out_of |= (torch.arange(nk) >= lengths.cpu().view(-1, 1)).view(b, 1, 1, nk)
    x_add = torch.zeros(b, h, nq, nk, dtype=dt)
    if buckets is not None:
        n = buckets.cpu().long()
        n = n if n.dim() == 3 else n.unsqueeze(0)
        bad = (n < 0) | (n >= table.size(1))
        out_of |= bad.unsqueeze(1)
        n = n.masked_fill(bad, 0).expand(b, nq, nk)
        x_add += table.detach().cpu().to(dt)[:, n].transpose(0, 1)
    if key_bias is not None:
        kb = key_bias.cpu().to(dt)
        kb = (kb if kb.dim() == 2 else kb.unsqueeze(0)).view(-1, 1, 1, nk)
        out_of |= kb == -math.inf
        x_add = x_add + kb.masked_fill(kb == -math.inf, 0)
    dead = out_of.all(2).all(1) if nq else torch.zeros(b, nk, dtype=torch.bool)      # keys nobody sees: whatever they hold
    kk, vv = (t.masked_fill(dead.view(b, 1, nk, 1), 0) for t in (kk, vv))
    x = (scale * (q @ kk.transpose(-1, -2)) + x_add).masked_fill(out_of, -math.inf)
    top = x.amax(-1, keepdim=True) if nk else torch.zeros(b, h, nq, 1, dtype=dt)
    e = torch.exp(x - top.masked_fill(top == -math.inf, 0))
    s = e.sum(-1, keepdim=True)
    p = e / s.masked_fill(s == 0, 1)
    out = p @ vv
    if g is None:
        return out
    g = g.detach().cpu().to(dt).masked_fill(s == 0, 0)
    dp = g @ vv.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    mag = p * (g.abs() @ vv.abs().transpose(-1, -2) + (g.abs() * out.abs()).sum(-1, keepdim=True))

    def per_key(t):
        return t.view(b, hk, h // hk, nk, d).sum(2)

    grads = {"q": scale * ds @ kk, "k": per_key(scale * ds.transpose(-1, -2) @ q), "v": per_key(p.transpose(-1, -2) @ g)}
    mags = {"q": scale * mag @ kk.abs(), "k": per_key(scale * mag.transpose(-1, -2) @ q.abs()), "v": torch.zeros_like(grads["v"])}
    if buckets is not None:
        hot = torch.nn.functional.one_hot(n, table.size(1)).to(dt) * (~bad).to(dt).expand(b, nq, nk).unsqueeze(-1)
        grads["table"] = torch.einsum("bhij,bijn->hn", ds, hot)
        mags["table"] = torch.einsum("bhij,bijn->hn", mag, hot)
    return out, grads, mags


def _close(got, want, dtype, what, mag=None):
    assert got.dtype == dtype and got.shape == want.shape, what
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    allowed = TOL[dtype] * want.norm().item() + (4 * 2.0 ** -24 * mag.norm().item() if mag is not None else 0.0)
    assert (got - want).norm().item() <= allowed, (what, (got - want).norm().item(), allowed)
    top = TOL[dtype] * 8 * want.abs().max().item() + (32 * 2.0 ** -24 * mag.abs().max().item() if mag is not None else 0.0)
    assert (got - want).abs().max().item() <= top, (what, "largest", (got - want).abs().max().item(), top)


def _inputs(b, h, hk, nq, nk, d, dtype, nb=0, per_batch=False, excluded=0.0, key_bias=None, ragged=False, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * nq + 13 * nk + d)
    s = {"q": torch.randn(b, nq, h, d, generator=g).to(dtype).cuda().transpose(1, 2),
         "k": torch.randn(b, nk, hk, d, generator=g).to(dtype).cuda().transpose(1, 2),
         "v": torch.randn(b, nk, hk, d, generator=g).to(dtype).cuda().transpose(1, 2)}
    if nb:
        s["table"] = torch.randn(h, nb, generator=g).to(dtype).cuda()
        n = torch.randint(0, nb, ((b,) if per_batch else ()) + (nq, nk), generator=g)
        s["buckets"] = torch.where(torch.rand(n.shape, generator=g) < excluded, torch.full_like(n, -1), n).to(torch.int8).cuda()
    if key_bias:
        s["key_bias"] = torch.randn(((b,) if key_bias == "batch" else ()) + (nk,), generator=g).cuda()
    if ragged:
        lengths = torch.randint(0, nk + 1, (b,), generator=g)
        lengths[0] = nk
        if b > 1:
            lengths[1] = 0
        s["lengths"] = lengths.int().cuda()
    return s, torch.randn(b, h, nq, d, generator=g).to(dtype).cuda()


def _check(s, g, dtype, what="", **kw):
    names = [n for n in ("q", "k", "v", "table") if n in s]
    with torch.no_grad():
        plain = s2cnn_amd.attention(**s, **kw)                  # without statistics
    for n in names:
        s[n].requires_grad_()
    out = s2cnn_amd.attention(**s, **kw)
    grads = torch.autograd.grad(out, [s[n] for n in names], g)
    want, want_grads, mags = _reference(**s, **kw, g=g)
    assert torch.equal(plain, out.detach()), what
    _close(out, want, dtype, what + " out")
    for n, t in zip(names, grads):
        _close(t, want_grads[n], dtype, what + " gradient of " + n, mags[n])
    return out, dict(zip(names, grads))


SIZES = [  # batch, heads, kv_heads, n_q, n_k, d
    (2, 2, 2, 1, 1, 8), (3, 2, 1, 1, 2, 16), (2, 3, 3, 31, 33, 32), (2, 4, 2, 23, 23, 16), (1, 2, 2, 64, 64, 64), (2, 2, 2, 129, 65, 40),
    (1, 6, 3, 100, 257, 100), (1, 2, 1, 130, 96, 128), (1, 1, 1, 5, 700, 20), (1, 8, 2, 1, 1500, 50), (1, 2, 2, 700, 3, 33),
    (2, 4, 1, 33, 40, 1), (1, 2, 2, 400, 400, 20), (1, 1, 1, 2, 31, 127),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=["x".join(map(str, s)) for s in SIZES])
def test_forward_and_gradients(hip, size, dtype):
    for i, kind in enumerate([dict(), dict(nb=32, key_bias="all"), dict(nb=7, per_batch=True, excluded=0.3, key_bias="batch", ragged=True)]):
        s, g = _inputs(*size, dtype, seed=i, **kind)
        _check(s, g, dtype, str(kind))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 65, 100, 127, 128])
def test_wide_heads_with_few_columns(hip, d, dtype):
    """Few queries, few keys, one and several tiles of the other side: the workgroups of one wave, which have the most per lane."""
    for i, (nq, nk) in enumerate([(1, 32), (2, 31), (3, 33), (31, 64), (32, 100), (1, 300), (5, 129), (64, 1), (100, 32), (257, 31), (40, 20)]):
        for kind in (dict(), dict(nb=11, excluded=0.2, key_bias="batch", ragged=True)):
            s, g = _inputs(2, 2, 1, nq, nk, d, dtype, seed=i, **kind)
            _check(s, g, dtype, "%d %d %s" % (nq, nk, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(300, 1, 1, 20, 1030, 20), (9, 33, 33, 40, 1030, 20), (11, 26, 13, 33, 1090, 100), (1, 290, 145, 30, 1100, 64), (2, 2, 2, 33, 4000, 50)],
                         ids=lambda s: "x".join(map(str, s)))
def test_long_rows_in_parts(hip, size, dtype):
    """Sizes whose long rows are cut although every compute unit has a workgroup (parts joined four entries a lane), and into many parts
    where few have one; lengths of zero and such that leave a part empty, rows without keys in one part or in all."""
    s, g = _inputs(*size, dtype, nb=5, excluded=0.1, key_bias="all", ragged=size[0] > 1)
    nk = size[4]
    s["buckets"][1, : nk // 2] = -1
    s["buckets"][2, nk // 2:] = -1
    s["buckets"][3] = -1
    out, _ = _check(s, g, dtype)
    assert (out[:, :, 3] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("nq", [1, 5, 40])
def test_heads_that_share_keys_taken_together(hip, nq, dtype):
    """No buckets: the queries of a key head's heads as those of one, where they lie one after the other (or are copied so, being few), with key
    biases, lengths, gradients in another layout than the outputs, and a query expanded over the signals."""
    s, g = _inputs(3, 6, 2, nq, 200, 20, dtype, key_bias="batch", ragged=True)
    for layout in (s["q"], s["q"].contiguous()):
        for gradient in (g, g.transpose(1, 2).contiguous().transpose(1, 2)):
            _check({**{n: t.detach() for n, t in s.items()}, "q": layout.detach()}, gradient, dtype)
    one = s["q"][:1].detach().contiguous()
    _check({**{n: t.detach() for n, t in s.items()}, "q": one.expand(3, -1, -1, -1)}, g, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_sixteen_bit_results_are_rounded_once(hip, dtype):
    """A rounding is off by a uniform part of half a spacing, 2^-8 to 2^-9 of a bfloat16: 0.43 u in the 2-norm.  Everything before it is
    float32 or two parts (2^-16 of a probability): 0.5 u allowed."""
    s, g = _inputs(2, 4, 2, 300, 500, 64, dtype, nb=32, excluded=0.1, key_bias="all")
    for n in ("q", "k", "v"):
        s[n].requires_grad_()
    out = s2cnn_amd.attention(**s)
    grads = torch.autograd.grad(out, [s[n] for n in ("q", "k", "v")], g)
    want, want_grads, _ = _reference(**s, g=g)
    for got, exact in ((out, want), *((t, want_grads[n]) for n, t in zip(("q", "k", "v"), grads))):
        assert (got.detach().cpu().double() - exact).norm() <= TOL[dtype] / 4 * exact.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("nb", [1, 2, 63, 64])
def test_tables_of_every_size(hip, nb):
    s, g = _inputs(2, 3, 3, 70, 90, 24, F32, nb=nb, excluded=0.1)
    _check(s, g, F32)


@pytest.mark.gpu
def test_buckets_outside_the_table_exclude(hip):
    s, g = _inputs(1, 2, 2, 40, 50, 16, F32, nb=9)
    n = s["buckets"]
    n[:, ::5] = -128
    n[:, 1::5] = 9
    n[:, 2::5] = 127
    _check(s, g, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
def test_queries_without_keys(hip, dtype):
    """Rows that see nothing: by buckets, by length zero, by key biases; outputs and gradients zero, also for a gradient of NaN
    there, and nothing of them in the other gradients."""
    s, g = _inputs(3, 2, 1, 37, 45, 16, dtype, nb=5, per_batch=True, ragged=True)
    s["buckets"][0, 3] = -1
    s["buckets"][2, ::2] = -1
    s["key_bias"] = torch.zeros(3, 45, device="cuda")
    s["lengths"][2] = 40
    out, grads = _check(s, g, dtype)
    assert (out[0, :, 3] == 0).all() and (out[1] == 0).all() and (out[2, :, ::2] == 0).all()
    assert (grads["q"][0, :, 3] == 0).all() and (grads["k"][1] == 0).all()
    g[0, :, 3], g[1], g[2, :, ::2] = math.nan, math.nan, math.nan
    again = torch.autograd.grad(s2cnn_amd.attention(**s), [s[n] for n in grads], g)
    for a, b in zip(again, grads.values()):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_keys_that_take_no_part_may_hold_anything(hip, dtype):
    s, g = _inputs(2, 2, 2, 35, 77, 24, dtype, nb=4, key_bias="batch", ragged=True)
    s["lengths"][1] = 50
    s["key_bias"][:, 5:20] = -math.inf
    clean, grads = _check(s, g, dtype)
    with torch.no_grad():
        for n, value in (("k", math.nan), ("v", math.inf)):
            s[n][:, :, 5:20] = value
            s[n][1, :, 50:] = math.nan
    out, again = _check(s, g, dtype)
    assert torch.equal(out, clean)
    for n in grads:
        assert torch.equal(again[n], grads[n]), n
    assert (again["k"][:, :, 5:20] == 0).all() and (again["v"][1, :, 50:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("nq", [5, 150])
def test_what_is_not_finite_stays_where_it_is_and_is_not_lost(hip, nq, value, dtype):
    """An infinite value, or one that is no number, of a key that takes part: no finite number in that entry of the output, the other entries as
    ever.  In a query: nowhere but in its row.  In the gradient of a query: nowhere but in the gradients of its row and of the keys."""
    s, g = _inputs(1, 2, 2, nq, 77, 24, dtype)
    out, grads = _check(dict(s), g, dtype)
    with torch.no_grad():
        v = s["v"].clone()
        v[0, 1, 70, 3] = value
        got = s2cnn_amd.attention(s["q"], s["k"], v)
        assert not torch.isfinite(got[0, 1, :, 3]).any()
        got[0, 1, :, 3] = out[0, 1, :, 3]
        assert torch.equal(got, out)
        q = s["q"].clone()
        q[0, 1, 2, 5] = value
        got = s2cnn_amd.attention(q, s["k"], s["v"])
        assert not torch.isfinite(got[0, 1, 2]).any()
        got[0, 1, 2] = out[0, 1, 2]
        assert torch.equal(got, out)
    g = g.clone()
    g[0, 1, 2, 5] = value
    again = torch.autograd.grad(s2cnn_amd.attention(s["q"], s["k"], s["v"]), [s["q"], s["k"], s["v"]], g)
    assert not torch.isfinite(again[0][0, 1, 2]).any() and not torch.isfinite(again[2][0, 1, :, 5]).any()
    assert torch.equal(again[0][:, 0], grads["q"][:, 0]) and torch.equal(again[1][:, 0], grads["k"][:, 0]) and torch.equal(again[2][:, 0], grads["v"][:, 0])


@pytest.mark.gpu
def test_lowest_value_as_a_mask(hip):
    """Key biases of float32's lowest value: no weight beside other keys, even weights where all keys have it."""
    s, g = _inputs(2, 2, 2, 9, 70, 16, F32, key_bias="batch")
    low = torch.finfo(torch.float32).min
    s["key_bias"][0, 10:60] = low
    s["key_bias"][1] = low
    out = s2cnn_amd.attention(**s)
    keep = list(range(10)) + list(range(60, 70))
    want = _reference(s["q"][:1], s["k"][:1, :, keep], s["v"][:1, :, keep], key_bias=s["key_bias"][:1, keep])
    _close(out[:1], want, F32, "beside others")
    _close(out[1], s["v"][1].cpu().double().mean(1, keepdim=True).expand(-1, 9, -1), F32, "all of them")
    s["v"].requires_grad_()
    gv, = torch.autograd.grad(s2cnn_amd.attention(**s), s["v"], g)
    _close(gv[1], g[1].cpu().double().sum(1, keepdim=True).expand(-1, 70, -1) / 70, F32, "gradient")


@pytest.mark.gpu
def test_infinite_entries_of_the_table_exclude(hip):
    s, g = _inputs(1, 2, 2, 40, 64, 16, F32, nb=4)
    s["table"][:, 2] = -math.inf
    out = s2cnn_amd.attention(**s)
    n = s["buckets"].clone()
    n[n == 2] = -1
    assert torch.equal(out, s2cnn_amd.attention(s["q"], s["k"], s["v"], table=s["table"], buckets=n))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("nq,nk", [(9, 70), (150, 70), (2, 1500)])
def test_lowest_value_in_the_table(hip, nq, nk, dtype):
    """Entries of the type's lowest value: no weight beside other pairs, even weights in a row that has no others (of float16 it is a bias as any
    other; 64 bits lose the scores beside that of the others, too), on keys of the lowest bias as well."""
    for low_keys in (False, True):
        s, g = _inputs(2, 2, 1, nq, nk, 16, dtype, nb=4, excluded=0.1, key_bias="all")
        s["table"][:, 2] = torch.finfo(dtype).min
        if dtype != F16:
            s["buckets"][1] = 2
        if low_keys:
            s["key_bias"][3:40] = torch.finfo(F32).min
        out, grads = _check(s, g, dtype)
        if dtype != F16 and not low_keys:
            _close(out[:, :, 1], s["v"].cpu().double().mean(2).expand(-1, 2, -1), dtype, "even")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_layouts(hip, dtype):
    """Contiguous, heads split off a joint projection, unaligned, reversed axes, a strided last axis, shared (expanded) inputs."""
    b, h, n, d = 2, 3, 50, 24
    gen = torch.Generator().manual_seed(3)
    base, g = _inputs(b, h, h, n, n, d, dtype, nb=6, seed=5)
    want, wq = _check(dict(base), g, dtype)
    joint = torch.randn(b, n, 3, h, d, generator=gen).to(dtype).cuda()
    unaligned = torch.zeros(b * h * n * (d + 1) + 3, dtype=dtype, device="cuda")[3:].view(b, h, n, d + 1)[..., :d]
    strided = torch.zeros(b, h, n, 2 * d, dtype=dtype, device="cuda")[..., ::2]
    turned = torch.zeros(n, d, h, b, dtype=dtype, device="cuda").permute(3, 2, 0, 1)
    for to in (joint[:, :, 1].transpose(1, 2), unaligned, strided, turned, torch.empty(b, h, n, d, dtype=dtype, device="cuda")):
        s = {key: t.detach() for key, t in base.items()}
        for key in ("q", "k", "v"):
            moved = to.clone(memory_format=torch.preserve_format) if key != "v" else to
            s[key] = moved.copy_(base[key].detach())
        gg = torch.empty_like(to).copy_(g)
        out, grads = _check(s, gg, dtype)
        assert torch.equal(out, want)
        for key in grads:
            assert torch.equal(grads[key], wq[key]), key
    # one query vector for all, one gradient for all
    s = {key: t.detach() for key, t in base.items()}
    one = s["q"][:1, :1, :1].contiguous().requires_grad_()
    out = s2cnn_amd.attention(one.expand(b, h, n, d), s["k"], s["v"], table=s["table"], buckets=s["buckets"])
    g1 = torch.ones(1, dtype=dtype, device="cuda").expand(out.shape)
    got, = torch.autograd.grad(out, one, g1)
    s["q"] = one.detach().expand(b, h, n, d)
    ref, grads, mags = _reference(**s, g=g1)
    _close(out, ref, dtype, "expanded")
    allowed = (TOL[dtype] * grads["q"].norm() + 2.0 ** -22 * mags["q"].norm()).item() * math.sqrt(b * h * n)   # a sum of so many
    assert (got.cpu().double() - grads["q"].sum((0, 1, 2), keepdim=True)).norm().item() <= allowed


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Directional derivatives of a scalar of the output by central differences of the operator itself.  With steps of 2^-6 the
    difference's own error is 2^-12 / 6 of a third derivative (of the order of the value), its rounding 2^-17: 2e-3 allowed."""
    s, g = _inputs(1, 2, 1, 20, 30, 8, F32, nb=4, excluded=0.2, key_bias="all", seed=2)
    _, grads = _check(s, g, F32)
    gen = torch.Generator().manual_seed(11)
    for n, grad in grads.items():
        u = torch.randn(s[n].shape, generator=gen).cuda()
        u /= u.norm()
        with torch.no_grad():
            f = [(s2cnn_amd.attention(**{**s, n: s[n] + sign * 2.0 ** -6 * u}).double() * g.double()).sum().item() for sign in (1, -1)]
        want = (grad.double() * u.double()).sum().item()
        assert abs((f[0] - f[1]) * 2.0 ** 5 - want) <= 2e-3 * max(1.0, grad.norm().item()), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("factor", [1e-4, 30.0])
def test_small_and_large_gradients(hip, dtype, factor):
    """A scaled gradient gives scaled results to the same accuracy: float16's few exponents are not in the way."""
    s, g = _inputs(1, 2, 1, 90, 800, 32, dtype, nb=8)
    g = (g.double() * factor).to(dtype)
    names = ["q", "k", "v", "table"]
    for n in names:
        s[n].requires_grad_()
    grads = torch.autograd.grad(s2cnn_amd.attention(**s), names and [s[n] for n in names], g)
    _, want, mags = _reference(**s, g=g)
    for n, t in zip(names, grads):
        spacing = 2.0 ** -25 * math.sqrt(t.numel()) if dtype == F16 else 0.0       # results below float16's smallest normal number
        err = (t.cpu().double() - want[n]).norm().item()
        assert err <= TOL[dtype] * want[n].norm().item() + 2.0 ** -22 * mags[n].norm().item() + spacing, n


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk,length,d,value", [(3, 32768, 2, 128, 16.0), (3, 32768, 2, 128, 500.0), (70, 4096, 2, 64, 64.0), (70, 4096, 4096, 64, 64.0),
                                                  (40, 1024, 2, 64, 128.0), (3, 64, 64, 64, 500.0), (150, 2, 2, 20, 500.0)])
def test_float16_gradients_of_large_values(hip, nq, nk, length, d, value):
    """Two keys that share a row, their values +-`value` in every entry, and a gradient of ones: gradients of scores up to d value / 2, which
    float16 holds, times the power of two that rows of n_k keys have, which it would not.  And values of that size for all keys.  The
    output of the two keys is a difference that cancels: sums of magnitudes on top, as for gradients."""
    s, g = _inputs(1, 2, 1, nq, nk, d, F16, key_bias="all")
    s["lengths"] = torch.tensor([length], dtype=torch.int32, device="cuda")
    wide = {**s, "v": (s["v"].float() * (value / 8)).half()}
    s["k"][:, :, 1] = s["k"][:, :, 0]
    s["key_bias"][:2] = 10.0
    s["v"][:, :, 0], s["v"][:, :, 1] = value, -value
    for what, t, gradient in (("two keys", s, torch.ones_like(g)), ("all keys", wide, g), ("a small gradient", wide, g * 2.0 ** -6)):
        t = {n: x.detach() for n, x in t.items()}
        names = ["q", "k", "v"]
        for n in names:
            t[n].requires_grad_()
        out = s2cnn_amd.attention(**t)
        grads = torch.autograd.grad(out, [t[n] for n in names], gradient)
        want, want_grads, mags = _reference(**t, g=gradient)
        _close(out, want, F16, what + " out", _reference(**{**t, "v": t["v"].abs()}))
        for n, x in zip(names, grads):
            _close(x, want_grads[n], F16, what + " gradient of " + n, mags[n])


@pytest.mark.gpu
def test_scale_and_large_scores(hip):
    """Scores up to about 90 (a softmax that one key holds): 2^-24 of such a score, some 8 times, is 4e-5 of a probability."""
    s, g = _inputs(1, 2, 2, 40, 200, 32, F32)
    out = s2cnn_amd.attention(**s, scale=4.0)
    want = _reference(**s, scale=4.0)
    assert (out.cpu().double() - want).norm() <= 4e-5 * want.norm()
    assert torch.equal(s2cnn_amd.attention(**s, scale=0.0)[..., :1, :], s2cnn_amd.attention(**s, scale=0.0)[..., 7:8, :])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [-0.5, 1e-3, 2.0, 0.0])
@pytest.mark.parametrize("size", [(2, 4, 2, 3, 70, 24), (2, 4, 2, 150, 140, 24), (2, 2, 1, 1, 900, 100), (1, 2, 2, 40, 60, 2)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_at_other_scales(hip, size, scale, dtype):
    """Negative, small, large and no scale, with a table, key biases and lengths: the 16-bit types take its sign into the queries, its magnitude
    into the scores and its inverse into the biases.  float32's allowance is for scores of 8 and grows with them.  float16 gradients of a
    small scale lie below its smallest normal number: spacings of 2^-24 on top."""
    for kind in (dict(), dict(nb=5, excluded=0.1, key_bias="batch", ragged=True)):
        s, g = _inputs(*size, dtype, **kind)
        names = [n for n in ("q", "k", "v", "table") if n in s]
        for n in names:
            s[n].requires_grad_()
        out = s2cnn_amd.attention(**s, scale=scale)
        grads = torch.autograd.grad(out, [s[n] for n in names], g)
        want, want_grads, mags = _reference(**s, scale=scale, g=g)
        top = abs(scale) * s["q"].detach().norm(dim=-1).max().item() * s["k"].detach().norm(dim=-1).max().item()
        tol = TOL[dtype] * (max(1.0, top / 8) if dtype == F32 else 1.0)
        for what, t, exact, mag in [("out", out, want, None)] + [(n, t, want_grads[n], mags[n]) for n, t in zip(names, grads)]:
            spacing = 2.0 ** -25 * math.sqrt(t.numel()) if dtype == F16 else 0.0
            extra = 4 * 2.0 ** -24 * mag.norm().item() if mag is not None else 0.0
            err = (t.detach().cpu().double() - exact).norm().item()
            assert err <= tol * exact.norm().item() + extra + spacing, (what, kind, err, exact.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("nq,nk,d", [(9, 150, 16), (150, 150, 16), (70, 40, 100)])
@pytest.mark.parametrize("bias", [-1e4, -1e6, 1e6])
def test_probabilities_of_both_passes_are_the_same(hip, bias, nq, nk, d, dtype):
    """A large bias on every key, by the keys or by the table, leaves a score few bits, and the two passes have to round it alike: with values of
    one the outputs are one, and the gradients of the values add up to that of the outputs.  The probabilities of a row add up to one but for
    some 8 roundings of float32, and what is returned is rounded: TOL of the sum of magnitudes."""
    for by_table in (False, True):
        s, g = _inputs(1, 4, 2, nq, nk, d, dtype, nb=3, key_bias="all")
        if by_table:
            limit = torch.finfo(dtype).max / 4
            s["table"] = torch.full_like(s["table"], max(-limit, min(limit, bias)))
        else:
            s["key_bias"] = torch.full_like(s["key_bias"], bias)
        s["v"] = torch.ones_like(s["v"]).requires_grad_()
        out = s2cnn_amd.attention(**s)
        gv, = torch.autograd.grad(out, s["v"], g)
        assert (out.double() - 1).abs().max().item() <= TOL[dtype]
        sums = g.double().sum(2).view(1, 2, 2, d).sum(2)
        mags = g.double().abs().sum(2).view(1, 2, 2, d).sum(2)
        assert ((gv.double().sum(2) - sums).abs() <= TOL[dtype] * mags).all(), ((gv.double().sum(2) - sums).abs() / mags).max().item() / TOL[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", [(F32, 3e4), (F32, 1e3), (BF16, 1e3), (F16, 1e3), (BF16, 3e4), (BF16, 1e6), (F16, 4e3)],
                         ids=["f32-3e4", "f32-1e3", "bf16", "f16", "bf16-3e4", "bf16-1e6", "f16-4e3"])
@pytest.mark.parametrize("nq", [9, 150])
def test_gradients_of_large_scores(hip, nq, dtype, size):
    """Queries and keys of a thousand and more: scores of 10^7 to 10^13, which round to hundreds and lie further apart than that: one key has the row."""
    s, g = _inputs(1, 2, 2, nq, 150, 64, dtype)
    s["q"] *= size
    s["k"] *= size
    _check(s, g, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30, -1e9, -1e8, -1e5])
def test_masked_keys_beside_others(hip, low, dtype):
    """Keys that a large negative bias leaves without weight, whole tiles of them before and after the others, in one pass and in parts."""
    for nq, nk, kind in ((9, 150, {}), (150, 150, dict(nb=5)), (1, 1500, {}), (40, 1500, dict(nb=5, excluded=0.1))):
        s, g = _inputs(1, 2, 2, nq, nk, 16, dtype, key_bias="all", **kind)
        s["key_bias"][:70] = low
        s["key_bias"][-40:] = low
        _check(s, g, dtype, "%d %d" % (nq, nk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [None, 3.0, 1e-3])
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30, -1e9, -1e7, 1e9, 1e30])
def test_every_key_has_the_same_large_bias(hip, low, scale, dtype):
    """Weights that add up to one in both passes (see test_probabilities_of_both_passes_are_the_same), and even ones where the bias leaves nothing
    of the scores, 2^-24 of 10^30 being far more than any.  Each of the values' gradients is rounded: below float16's smallest normal number by
    2^-25."""
    for nq, nk in ((9, 150), (150, 150), (1, 1500)):
        s, g = _inputs(1, 2, 2, nq, nk, 16, dtype)
        s["key_bias"] = torch.full((nk,), low, device="cuda")
        values = s["v"]
        if abs(low) >= 1e30:
            _close(s2cnn_amd.attention(**s, scale=scale), values.cpu().double().mean(2, keepdim=True).expand(-1, -1, nq, -1), dtype, "even")
        s["v"] = torch.ones_like(values)
        for n in ("q", "k", "v"):
            s[n].requires_grad_()
        out = s2cnn_amd.attention(**s, scale=scale)
        assert (out.double() - 1).abs().max().item() <= TOL[dtype]
        gq, gk, gv = torch.autograd.grad(out, [s["q"], s["k"], s["v"]], g)
        spacing = nk * 2.0 ** -25 if dtype == F16 else 0.0
        assert ((gv.double().sum(2) - g.double().sum(2)).abs() <= TOL[dtype] * g.double().abs().sum(2) + spacing).all()
        assert torch.isfinite(gq).all() and torch.isfinite(gk).all()


@pytest.mark.gpu
def test_same_bits_every_time_and_on_other_streams(hip):
    s, g = _inputs(2, 4, 2, 200, 300, 32, F32, nb=32, excluded=0.1, key_bias="all", ragged=True)
    out, grads = _check(s, g, F32)
    names = list(grads)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = s2cnn_amd.attention(**s)
            got = torch.autograd.grad(again, [s[n] for n in names], g)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(again, out)
        for n, t in zip(names, got):
            assert torch.equal(t, grads[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("size", [(2, 4, 2, 200, 300, 64), (1, 8, 2, 2, 3000, 50), (3, 6, 3, 130, 700, 100)], ids=lambda s: "x".join(map(str, s)))
def test_same_bits_every_time_in_sixteen_bits(hip, size, dtype):
    """Other calls in between, so that workspaces and outputs lie in memory that held something else."""
    s, g = _inputs(*size, dtype, nb=32, excluded=0.1, key_bias="all", ragged=size[0] > 1)
    other, other_g = _inputs(*size, dtype, nb=32, excluded=0.1, key_bias="all", seed=1)
    want, grads = _check(s, g, dtype)
    for _ in range(3):
        _check({n: t.detach() for n, t in other.items()}, other_g, dtype)
        out = s2cnn_amd.attention(**s)
        again = torch.autograd.grad(out, [s[n] for n in grads], g)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(again, grads.values()))


@pytest.mark.gpu
def test_replays_from_a_graph(hip):
    s, g = _inputs(2, 4, 1, 3, 900, 20, F32, nb=6, key_bias="all")              # split over the keys: several kernels
    names = ["q", "k", "v", "table"]
    for n in names:
        s[n].requires_grad_()

    def step():
        out = s2cnn_amd.attention(**s)
        return (out, *torch.autograd.grad(out, [s[n] for n in names], g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for k in range(4):
        with torch.no_grad():
            for n in names:
                s[n].mul_(0.9 + 0.05 * k)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_some_gradients_only_and_empty_sizes(hip):
    s, g = _inputs(2, 4, 2, 30, 40, 16, F32, nb=5)
    _, all_grads = _check({n: t.clone() for n, t in s.items()}, g, F32)
    for names in (["v"], ["q"], ["table"], ["k", "table"]):
        t = {n: x.detach().clone() for n, x in s.items()}
        for n in names:
            t[n].requires_grad_()
        for n, grad in zip(names, torch.autograd.grad(s2cnn_amd.attention(**t), [t[n] for n in names], g)):
            assert torch.equal(grad, all_grads[n]), n
    z = lambda *shape: torch.zeros(*shape, device="cuda", requires_grad=True)
    q, k = z(2, 2, 5, 8), z(2, 2, 0, 8)
    out = s2cnn_amd.attention(q, k, k)
    assert out.shape == (2, 2, 5, 8) and (out == 0).all()
    gq, gk = torch.autograd.grad(out.sum(), [q, k])
    assert (gq == 0).all() and gk.shape == k.shape
    for shape in ((0, 2, 5, 8), (2, 2, 0, 8)):
        q, k = z(*shape), z(shape[0], 2, 7, 8)
        out = s2cnn_amd.attention(q, k, k)
        assert out.shape == shape
        assert (torch.autograd.grad(out.sum(), k)[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_no_keys_with_a_table(hip, dtype):
    """n_k = 0 with buckets (an empty tensor, which has no address), key biases and lengths: zeros, as without them."""
    for per_batch in (False, True):
        s, g = _inputs(2, 4, 2, 5, 0, 8, dtype, nb=3, per_batch=per_batch, key_bias="all")
        s["lengths"] = torch.zeros(2, dtype=torch.int32, device="cuda")
        with torch.no_grad():
            assert (s2cnn_amd.attention(**s) == 0).all()
        names = ["q", "k", "v", "table"]
        for n in names:
            s[n].requires_grad_()
        out = s2cnn_amd.attention(**s)
        assert out.shape == (2, 4, 5, 8) and (out == 0).all()
        for n, grad in zip(names, torch.autograd.grad(out, [s[n] for n in names], g)):
            assert grad.shape == s[n].shape and (grad == 0).all()


@pytest.mark.gpu
def test_double_backward_is_refused(hip):
    s, g = _inputs(1, 1, 1, 4, 5, 8, F32)
    q = s["q"].requires_grad_()
    gq, = torch.autograd.grad(s2cnn_amd.attention(**s), q, g.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        gq.sum().backward()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(hip):
    """Keys and values that start, and end, more than 2^31 entries into their storage; one query per head over a long axis."""
    n, d, stride = 600, 16, 1 << 22
    store = torch.empty(n * stride + d, dtype=torch.bfloat16, device="cuda")             # 5 GB
    k = store.as_strided((1, 1, n, d), (0, 0, stride, 1))
    gen = torch.Generator().manual_seed(0)
    q, kk = torch.randn(1, 2, 40, d, generator=gen).to(BF16).cuda(), torch.randn(1, 1, n, d, generator=gen).to(BF16).cuda()
    k.copy_(kk)
    assert torch.equal(s2cnn_amd.attention(q, k, k), s2cnn_amd.attention(q, kk, kk))
    assert torch.equal(s2cnn_amd.attention(q[:, :, :1], k, k), s2cnn_amd.attention(q[:, :, :1], kk, kk))


def test_refusals():
    """Shapes are checked before devices (as the reference's asserts are), devices and types before anything is launched."""
    z = torch.zeros
    q = z(2, 4, 5, 8)
    k = z(2, 2, 6, 8)
    bad = [
        (z(4, 5, 8), k, k), (q, z(2, 3, 6, 8), z(2, 3, 6, 8)), (q, k, z(2, 2, 7, 8)), (q, z(3, 2, 6, 8), z(3, 2, 6, 8)),
        (q, z(2, 2, 6, 9), z(2, 2, 6, 9)), (z(2, 4, 5, 129), z(2, 2, 6, 129), z(2, 2, 6, 129)), (z(2, 4, 5, 0), z(2, 2, 6, 0), z(2, 2, 6, 0)),
    ]
    for args in bad:
        with pytest.raises(AssertionError):
            s2cnn_amd.attention(*args)
    n = z(5, 6, dtype=torch.int8)
    for kw in (dict(table=z(4, 3)), dict(buckets=n), dict(table=z(3, 3), buckets=n), dict(table=z(4, 65), buckets=n), dict(table=z(4, 0), buckets=n),
               dict(table=z(4, 3), buckets=z(6, 5, dtype=torch.int8)), dict(table=z(4, 3), buckets=z(3, 5, 6, dtype=torch.int8)),
               dict(key_bias=z(5)), dict(key_bias=z(3, 6)), dict(lengths=z(3, dtype=torch.int32))):
        with pytest.raises(AssertionError):
            s2cnn_amd.attention(q, k, k, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.attention(q, k, k)


@pytest.mark.gpu
def test_refusals_of_types(hip):
    z = lambda *shape, **kw: torch.zeros(*shape, device="cuda", **kw)
    q, k, n = z(1, 2, 5, 8), z(1, 2, 6, 8), z(5, 6, dtype=torch.int8)
    for args, kw in (((q.double(), k.double(), k.double()), {}), ((q, k.half(), k), {}), ((q, k, k.cpu()), {}),
                     ((q, k, k), dict(table=z(2, 3, dtype=BF16), buckets=n)), ((q, k, k), dict(table=z(2, 3), buckets=n.int())),
                     ((q, k, k), dict(key_bias=z(6, dtype=F16))), ((q, k, k), dict(lengths=z(1, dtype=torch.int64)))):
        with pytest.raises(RuntimeError):
            s2cnn_amd.attention(*args, **kw)
    with pytest.raises(AssertionError):
        s2cnn_amd.attention(q, k, k, key_bias=z(6, requires_grad=True))


def test_entry_points_refuse_without_a_gpu():
    import ctypes
    from s2cnn_amd import _hip
    lib = _hip.lib()

    def a(**kw):
        t = _hip.Attention(q=0x1000, k=0x1000, v=0x1000, out=0x1000, stats=0x1000, gout=0x1000, gq=0x1000, gk=0x1000, gv=0x1000,
                           batch=1, heads=2, kv_heads=1, n_q=4, n_k=5, d=8, scale=1.0)
        for n, v in kw.items():
            setattr(t, n, v)
        return ctypes.byref(t)

    for kw in (dict(d=129), dict(d=0), dict(kv_heads=3), dict(n_q=0), dict(n_k=-1), dict(dtype=3), dict(batch=0), dict(buckets=0x1000), dict(n_buckets=3),
               dict(buckets=0x1000, table=0x1000, n_buckets=65), dict(n_q=1 << 30, heads=4), dict(q=0), dict(out=0), dict(k=0)):
        assert lib.s2cnn_attention_fwd(a(**kw), None, 0, None) == -1, kw
    assert lib.s2cnn_attention_fwd(a(q=0x1002), None, 0, None) == -3
    assert lib.s2cnn_attention_bwd(a(), None, 0, None) == -2
    for kw in (dict(n_k=0), dict(stats=0), dict(gk=0), dict(gq=0), dict(gtable=0x1000), dict(gout=0)):
        assert lib.s2cnn_attention_bwd(a(**kw), None, 0, None) == -1, kw
    long_axis = a(n_q=1, n_k=100000)
    assert lib.s2cnn_attention_workspace(long_axis, 0) > 0                      # the keys are split
    assert lib.s2cnn_attention_fwd(long_axis, None, 0, None) == -2
    assert lib.s2cnn_attention_workspace(a(d=0), 1) == 0


@pytest.mark.gpu
def test_vectors_and_buckets_of_one_row_far_apart(hip):
    """One query, or key, of a storage whose rows are 2^25 entries apart: the stride of an axis of one entry is nobody's limit."""
    s, g = _inputs(2, 2, 1, 1, 50, 16, F32, nb=4, excluded=0.2)
    wide = torch.full((2, 1 << 25), 3, dtype=torch.int8, device="cuda")
    wide[1, 7:57] = s["buckets"][0]
    want, grads = _check(dict(s), g, F32)
    out, again = _check({**{n: t.detach() for n, t in s.items()}, "buckets": wide[1:, 7:57]}, g, F32)
    assert torch.equal(out, want) and all(torch.equal(again[n], grads[n]) for n in grads)
    far = torch.empty(2 * (1 << 25), dtype=BF16, device="cuda").as_strided((1, 2, 1, 16), (0, 16, 1 << 25, 1))
    s, g = _inputs(1, 2, 2, 1, 1, 16, BF16)
    far.copy_(s["q"])
    for n in ("q", "k", "v"):
        _check({**{m: t.detach() for m, t in s.items()}, n: far}, g, BF16)


def _sizes(**kw):
    """floats of the statistics of a call of these sizes, 0 if it is refused (host only)"""
    import ctypes
    from s2cnn_amd import _hip
    a = _hip.Attention(**{**dict(batch=1, heads=2, kv_heads=1, n_q=4, n_k=5, d=8, scale=1.0), **kw})
    return _hip.lib().s2cnn_attention_stats_floats(ctypes.byref(a))


def test_heads_that_share_a_key_head_with_buckets():
    """128 of them at most: refused by name, and by the entry; any number without buckets."""
    z = torch.zeros
    n = z(1, 1, dtype=torch.int8)
    with pytest.raises(AssertionError, match="128"):
        s2cnn_amd.attention(z(1, 129, 1, 8), z(1, 1, 1, 8), z(1, 1, 1, 8), table=z(129, 3), buckets=n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        s2cnn_amd.attention(z(1, 256, 1, 8), z(1, 2, 1, 8), z(1, 2, 1, 8), table=z(256, 3), buckets=n)
    with_buckets = dict(table=0x1000, buckets=0x1000, n_buckets=3)
    assert _sizes(heads=129, **with_buckets) == 0 and _sizes(heads=128, **with_buckets) > 0 and _sizes(heads=129) > 0


@pytest.mark.gpu
def test_most_heads_a_key_head(hip):
    s, g = _inputs(1, 128, 1, 3, 40, 128, F32, nb=64)
    _check(s, g, F32, "128 heads, 64 buckets")
    s, g = _inputs(1, 129, 1, 3, 40, 16, F32)
    _check(s, g, F32, "129 heads")


def test_no_keys_need_no_buckets():
    assert _sizes(n_k=0, table=0x1000, n_buckets=3) > 0
    assert _sizes(table=0x1000, n_buckets=3) == 0 and _sizes(n_k=0, buckets=0x1000, n_buckets=3) == 0


def test_angle_buckets():
    """Against the definition, and their rotation invariance: points and their rotations have the same buckets."""
    import numpy as np
    points = s2cnn_amd.s2_soft_grid(4)
    n = s2cnn_amd.s2_angle_buckets(points, n_buckets=16)
    assert n.shape == (64, 64) and n.dtype == torch.int8
    assert (n.diagonal() == 0).all() and torch.equal(n, n.t()) and int(n.min()) == 0 and int(n.max()) <= 15
    p = np.array(points)
    xyz = np.stack([np.sin(p[:, 0]) * np.cos(p[:, 1]), np.sin(p[:, 0]) * np.sin(p[:, 1]), np.cos(p[:, 0])], 1)
    angle = np.arctan2(np.linalg.norm(np.cross(xyz[:, None], xyz[None]), axis=-1), xyz @ xyz.T)
    inside = np.abs(angle * 16 / np.pi - np.round(angle * 16 / np.pi)) > 1e-6                       # not at a boundary of two buckets
    assert (n.numpy()[inside] == np.floor(angle * 16 / np.pi)[inside]).all()
    near = s2cnn_amd.s2_angle_buckets(points, n_buckets=5, max_angle=0.8)
    assert ((near.numpy() < 0) == (angle > 0.8)).all() and int(near.max()) == 4
    turned = [(b, a + 0.3) for b, a in points]
    assert torch.equal(s2cnn_amd.s2_angle_buckets(turned, n_buckets=5, max_angle=0.8), near)
    assert s2cnn_amd.s2_angle_buckets(points[:3], points).shape == (3, 64)
    with pytest.raises(AssertionError):
        s2cnn_amd.s2_angle_buckets(points, n_buckets=65)


def test_log_weights():
    w = s2cnn_amd.s2_log_weights(5)
    assert w.shape == (100,) and w.dtype == torch.float32
    assert abs(float(w.double().exp().view(10, 10)[:, 0].sum()) - 1 / 100) < 1e-6
