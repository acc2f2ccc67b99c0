"""The transformer over the points of the sphere (s2cnn_amd/soft/s2_transformer.py) against its formulas in 64 bits on the CPU, its
symmetry, its training step eager and replayed from a graph.

Tolerance of outputs and gradients: ten products, normalisations and attentions one after the other, each of which may add what a
float32 attention may (128 * 2^-24 in the 2-norm), twice that for gradients: 1e-4 and 2e-4."""
import io
import math

import pytest
import torch
import torch.nn.functional as F

import s2cnn_amd
from s2cnn_amd import harness


def _stack(**kw):
    torch.manual_seed(5)
    model = s2cnn_amd.S2Transformer(**{**dict(features=24, heads=3, b=3, layers=2, n_buckets=6), **kw})
    for name, p in model.named_parameters():             # nothing left at zero or one
        if name.endswith("bias_table") or name.endswith("query") or "norm" in name:
            p.data += 0.5 * torch.randn(p.shape)
    return model


def _plain(model, x, masks, heads):
    """The same function in torch's own operators; masks: what each dropout multiplies by."""
    def norm(h, m):
        return F.layer_norm(h, h.shape[-1:], m.weight, m.bias)

    def split(t, n):
        return t.unflatten(-1, (n, heads, t.shape[-1] // (n * heads))).permute(2, 0, 3, 1, 4)

    h = x.flatten(2).transpose(1, 2)
    for i, block in enumerate(model.blocks):
        q, k, v = split(block.qkv(norm(h, block.norm1)), 3)
        n = block.buckets.long()
        s = q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1]) + block.bias_table[:, n.clamp(min=0)] + block.log_weights().to(q.dtype)
        a = torch.softmax(s.masked_fill(n < 0, -math.inf), -1) @ v
        h = h + masks[2 * i] * block.out(a.transpose(1, 2).flatten(2))
        h = h + masks[2 * i + 1] * block.contract(F.relu(block.expand(norm(h, block.norm2))))
    k, v = split(model.pool.kv(norm(h, model.last_norm)), 2)
    s = (model.pool.query * k).sum(-1) / math.sqrt(k.shape[-1]) + model.pool.log_weights().to(k.dtype)
    return (torch.softmax(s, -1).unsqueeze(-1) * v).sum(-2).flatten(1)


def _relative(a, b):
    a, b = a.detach().double().cpu(), b.detach()
    return float((a - b).norm() / b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("p,angle", [(0.0, math.pi), (0.25, 1.2)])
def test_equals_the_formulas(hip, p, angle):
    model = _stack(max_angle=angle, dropout=p)
    plain = _stack(max_angle=angle, dropout=p).double()
    x, g = torch.randn(2, 24, 6, 6), torch.randn(2, 24)
    model.cuda()
    xg = x.cuda().requires_grad_()
    xp = x.double().requires_grad_()
    y = model(xg)
    y.backward(g.cuda())
    seeds = [4 + i for i in range(4)]                    # first call: drops = 1, four dropouts a call
    masks = [s2cnn_amd.dropout(torch.ones(2, 36, 24, device="cuda"), p, s).double().cpu() for s in seeds]
    want = _plain(plain, xp, masks, 3)
    want.backward(g.double())
    assert _relative(y, want) < 1e-4
    assert _relative(xg.grad, xp.grad) < 2e-4
    for (name, a), b in zip(model.named_parameters(), plain.parameters()):
        assert _relative(a.grad, b.grad) < 2e-4 or float(b.grad.norm()) < 1e-9, name


@pytest.mark.gpu
def test_invariant_under_rotations_about_the_axis(hip):
    """A rotation by a grid step about the polar axis permutes the points of each ring: the blocks permute with them, the pooling
    does not see it.  Sums in another order: 1e-4 as above."""
    model = _stack(b=4, n_buckets=16).cuda().eval()
    x = torch.randn(2, 24, 8, 8, device="cuda")
    with torch.no_grad():
        a, b = model(x), model(x.roll(3, -1))
    assert _relative(b, a.double().cpu()) < 1e-4


@pytest.mark.gpu
def test_pooling_starts_as_the_integral(hip):
    """Queries of zeros: the mean of the values with the quadrature weights."""
    torch.manual_seed(1)
    pool = s2cnn_amd.S2AttentionPool(16, 2, 5).cuda()
    y = torch.randn(3, 100, 16, device="cuda")
    w = pool.log_weights().double().exp()
    want = torch.einsum("p,bpf->bf", w / w.sum(), pool.kv(y)[..., 16:].double())
    assert _relative(pool(y), want.detach().cpu()) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sixteen_bit_and_autocast(hip, dtype):
    """Twenty roundings one after the other, each of half a unit: 10 units of the type in the 2-norm."""
    model, plain = _stack(), _stack().double()
    x = torch.randn(2, 24, 6, 6)
    want = _plain(plain, x.double(), [1.0] * 4, 3).detach()
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    with torch.no_grad():
        model.cuda().eval()
        with torch.autocast("cuda", dtype=dtype):
            cast = model(x.cuda())
        assert _relative(cast, want) < 10 * unit
        assert _relative(model.to(dtype)(x.cuda().to(dtype)), want) < 10 * unit


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cast", [False, True], ids=["module", "autocast"])
def test_sixteen_bit_gradients(hip, cast, dtype):
    """As test_sixteen_bit_and_autocast, twice as many roundings on the way to a gradient: 20 units of the type in the 2-norm of all gradients of
    the parameters together, and of the input's."""
    model, plain = _stack(), _stack().double()
    gen = torch.Generator().manual_seed(6)
    x, g = torch.randn(2, 24, 6, 6, generator=gen), torch.randn(2, 24, generator=gen)
    xp = x.double().requires_grad_()
    _plain(plain, xp, [1.0] * 4, 3).backward(g.double())
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    model.cuda()
    if cast:
        xg = x.cuda().requires_grad_()
        with torch.autocast("cuda", dtype=dtype):
            y = model(xg)
    else:
        model.to(dtype)
        xg = x.cuda().to(dtype).requires_grad_()
        y = model(xg)
    y.backward(g.cuda().to(y.dtype))
    assert _relative(xg.grad, xp.grad) < 20 * unit
    a, b = (torch.cat([p.grad.detach().double().cpu().flatten() for p in m.parameters()]) for m in (model, plain))
    assert _relative(a, b) < 20 * unit


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_run_again_in_the_backward_pass(hip, reentrant):
    """With its seeds given, a pass that is formed again in the backward pass gives the gradients of the one that is kept; without them it is
    refused (two passes may have been counted since), unless nothing is dropped."""
    from torch.utils.checkpoint import checkpoint
    model = _stack(dropout=0.25).cuda()
    gen = torch.Generator().manual_seed(3)
    x, g = torch.randn(2, 24, 6, 6, generator=gen).cuda(), torch.randn(2, 24, generator=gen).cuda()

    def gradients(f):
        model.zero_grad()
        xs = x.clone().requires_grad_()
        y = f(xs)
        y.backward(g)
        return [y.detach(), xs.grad] + [p.grad for p in model.parameters()]

    seeds = model.next_seeds()
    want = gradients(lambda t: model(t, seeds))
    for a, b in zip(gradients(lambda t: checkpoint(model, t, seeds, use_reentrant=reentrant)), want):
        assert torch.equal(a, b)
    blocks = torch.cat([model(x, s) for s in (seeds, model.next_seeds())])
    assert torch.equal(blocks[:2], want[0]) and not torch.equal(blocks[2:], want[0])
    with pytest.raises(RuntimeError, match="next_seeds"):
        gradients(lambda t: checkpoint(model, t, use_reentrant=reentrant))
    for block in model.blocks:
        block.dropout = 0.0
    for a, b in zip(gradients(lambda t: checkpoint(model, t, use_reentrant=reentrant)), gradients(model)):
        assert torch.equal(a, b)


def test_seeds_of_stacks():
    """Stacks of other seeds, of whatever depth, share no number in any of their passes; one of the same seed repeats them; without one they count
    from the number of calls, as ever.  `seed` may be any integer."""
    def first(seed, layers=2, passes=50):
        model = s2cnn_amd.S2Transformer(8, 2, 2, layers, dropout=0.1, **({} if seed is None else {"seed": seed}))
        return [n for _ in range(passes) for n in model.next_seeds().tolist()]

    assert first(None)[:4] == [4, 5, 6, 7] and first(0) == first(None)
    seeds = (0, 1, 2, 12345, -1, 2 ** 31, 2 ** 32 - 2)
    numbers = [n for seed in seeds for n in first(seed, 1 + seed % 3)]
    assert len(set(numbers)) == len(numbers)
    assert first(7) == first(7) and first(7) == first(7 + 2 ** 40)


def test_seeds_of_ranks_whose_buffers_are_those_of_one():
    """What a data-parallel job does before each pass: the buffers of rank 0 go to all ranks, which still drop other elements."""
    ranks = [s2cnn_amd.S2Transformer(8, 2, 2, 2, dropout=0.1, seed=3 + rank) for rank in range(3)]
    seen = []
    for _ in range(4):
        for model in ranks[1:]:
            for a, b in zip(ranks[0].buffers(), model.buffers()):
                b.copy_(a)
        seen += [n for model in ranks for n in model.next_seeds().tolist()]
    assert len(set(seen)) == len(seen) == 4 * 3 * 4


@pytest.mark.gpu
def test_stacks_of_one_network_drop_other_elements(hip):
    x = torch.randn(2, 24, 6, 6, generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        a, b, again = (_stack(dropout=0.25, **kw).cuda()(x) for kw in (dict(), dict(seed=1), dict(seed=1)))
    assert not torch.equal(a, b) and torch.equal(b, again)


@pytest.mark.gpu
def test_network_trains_and_reloads(hip):
    model, losses, _ = harness.train_steps("sphere_transformer", batch=8, steps=8, warmup=0, lr=0.02)
    print("sphere transformer losses:", ["%.4f" % l for l in losses], flush=True)
    assert all(l == l for l in losses) and losses[-1] < losses[0]
    x, _ = harness.synthetic_batch("sphere_transformer", 8, "cuda:0")
    model.eval()
    with torch.no_grad():
        want = model(x)
    buf = io.BytesIO()
    torch.save(model.state_dict(), buf)
    buf.seek(0)
    twin = harness.NETWORKS["sphere_transformer"][0]().cuda()
    twin.load_state_dict(torch.load(buf, weights_only=True))
    twin.eval()
    with torch.no_grad():
        assert torch.equal(twin(x), want)


@pytest.mark.gpu
def test_step_replayed_from_a_graph(hip):
    """Each replay drops other elements than the one before: the losses are those of as many eager steps."""
    _, eager, _ = harness.train_steps("sphere_transformer", batch=4, steps=5, warmup=3, lr=0.02)
    _, replayed, _ = harness.train_steps_replayed("sphere_transformer", batch=4, steps=5, warmup=3, lr=0.02)
    print("eager", ["%.5f" % l for l in eager[3:]], "replayed", ["%.5f" % l for l in replayed], flush=True)
    assert max(abs(a - b) for a, b in zip(eager[3:], replayed)) < 1e-4 * abs(eager[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cast", [False, True], ids=["", "autocast"])
def test_linear_captured_with_its_gradients(hip, cast, dtype):
    """nn.Linear outside of a capture; captured, the outputs and the gradients of the input and the weight are its own bit by bit, in every replay,
    and the bias's is the sum of the gradient's rows: float32 sums, rounded to the type."""
    from s2cnn_amd.soft.s2_transformer import Linear
    gen = torch.Generator().manual_seed(8)
    a, b = Linear(96, 192).to(dtype).cuda(), torch.nn.Linear(96, 192).to(dtype).cuda()
    b.load_state_dict(a.state_dict())
    x, g = (torch.randn(4, 400, n, generator=gen).to(dtype).cuda() for n in (96, 192))
    x.requires_grad_()

    def run(m):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=cast, cache_enabled=False):
            y = m(x)
        return (y, *torch.autograd.grad(y, [x, m.weight, m.bias], g.to(y.dtype)))

    for m in (a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(m)
        torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(run(a), run(b)):
        assert torch.equal(u, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run(a)
    unit = 2.0 ** -8 if cast or dtype == torch.bfloat16 else 2.0 ** -20
    for k in range(4):
        with torch.no_grad():
            g.mul_(1.0 + 0.25 * k)
        want = run(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(static[:3], want):
            assert torch.equal(u, v), k
        assert static[3].dtype == want[3].dtype
        assert _relative(static[3], g.to(static[0].dtype).double().sum((0, 1)).cpu()) <= unit, k


@pytest.mark.gpu
def test_replays_between_eager_steps(hip, monkeypatch):
    """The captured training step, and a twin that makes the same steps eagerly between its replays (with synchronisations, and other work that
    allocates and clears memory): losses, gradients and weights of each are the other's.  The twin sums its biases' gradients as captured work
    does, so that all kernels are the same, sums in the same order."""
    from s2cnn_amd.soft import s2_transformer
    monkeypatch.setattr(s2_transformer, "_sums_of_its_own", lambda x, parameter: True)
    x, y = harness.synthetic_batch("sphere_transformer", 4, "cuda:0")
    loss_fn = harness.NETWORKS["sphere_transformer"][3]

    def make():
        torch.manual_seed(0)
        model = harness.NETWORKS["sphere_transformer"][0]().cuda().train()
        opt = torch.optim.SGD(model.parameters(), lr=0.02, momentum=0.9)

        def step():
            opt.zero_grad(set_to_none=True)
            loss = loss_fn(model(x), y)
            loss.backward()
            opt.step()
            return loss
        return model, opt, step

    (model, opt, step), (twin, _, twin_step) = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step(), twin_step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    opt.zero_grad(set_to_none=True)
    with torch.cuda.graph(graph):
        static = step()
    for k in range(5):
        want = twin_step()
        torch.cuda.synchronize()
        junk = [torch.randn(1 << 20, device="cuda").sum() for _ in range(4)] + [torch.zeros(777, device="cuda")]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.isfinite(j).all() for j in junk)
        assert abs(float(static) - float(want)) <= 1e-6 * abs(float(want)), k
        for (name, a), b in zip(model.named_parameters(), twin.parameters()):
            assert _relative(a.grad, b.grad.double().cpu()) < 1e-5, (k, name)
            assert _relative(a, b.double().cpu()) < 1e-5, (k, name)


def test_refusals():
    with pytest.raises(AssertionError):
        s2cnn_amd.S2TransformerBlock(25, 3, 3)
    with pytest.raises(AssertionError):
        s2cnn_amd.S2AttentionPool(25, 3, 3)
    block = s2cnn_amd.S2TransformerBlock(24, 3, 3)
    with pytest.raises(AssertionError):
        block(torch.zeros(1, 35, 24), torch.zeros(1, 35, 24), block.norm1, (1, 2))
