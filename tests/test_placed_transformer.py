"""The transformer over the points of the sphere with normalised and turned queries and keys, against its formulas in 64 bits on the CPU, and its training
with AdamW, eager and replayed from a graph.

Tolerances as in test_s2_transformer.py: 1e-4 of outputs and 2e-4 of gradients in the 2-norm; 10 and 20 units of a 16-bit type, whose two further
roundings a block are within those."""
import math

import pytest
import torch
import torch.nn.functional as F

import s2cnn_amd
from s2cnn_amd import harness

PLACED = [dict(qk_norm=True, rotary=True), dict(qk_norm=True), dict(rotary=True)]
IDS = ["both", "norm", "rotary"]


def _stack(**kw):
    torch.manual_seed(5)
    model = s2cnn_amd.S2Transformer(**{**dict(features=30, heads=3, b=3, layers=2, n_buckets=6), **kw})
    for name, p in model.named_parameters():             # nothing left at zero or one
        if name.endswith(("bias_table", "query", "q_weight", "k_weight")) or "norm" in name:
            p.data += 0.5 * torch.randn(p.shape)
    return model


def _turned(x, b):
    """x [..., points, d] with its halves' pairs turned by the points' angles"""
    pairs = x.size(-1) // 2
    beta, alpha = torch.tensor(s2cnn_amd.s2_soft_grid(b), dtype=torch.float64).T
    angles = torch.stack([(j // 2 + 1) * (alpha if j % 2 == 0 else beta) for j in range(pairs)], -1)
    a, c = x[..., :pairs], x[..., pairs:2 * pairs]
    return torch.cat([a * angles.cos() - c * angles.sin(), a * angles.sin() + c * angles.cos(), x[..., 2 * pairs:]], -1)


def _plain(model, x, heads, qk_norm=False, rotary=False):
    """The same function in torch's own operators, 64 bits on the CPU"""
    norm = lambda h, m: F.layer_norm(h, h.shape[-1:], m.weight, m.bias)
    h = x.flatten(2).transpose(1, 2)
    y = norm(h, model.blocks[0].norm1)
    batch, points, features = h.shape
    for i, block in enumerate(model.blocks):
        q, k, v = block.qkv(y).view(batch, points, 3, heads, -1).permute(2, 0, 3, 1, 4)
        if qk_norm:
            q, k = (t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w for t, w in ((q, block.q_weight), (k, block.k_weight)))
        if rotary:
            q, k = _turned(q, block.b), _turned(k, block.b)
        index = block.buckets.long()
        scores = q @ k.transpose(-1, -2) / math.sqrt(q.size(-1)) + block.bias_table[:, index.clamp(min=0)] + block.log_weights().double()
        p = torch.softmax(scores.masked_fill(index < 0, -math.inf), -1)
        h = h + block.out((p @ v).transpose(1, 2).reshape(batch, points, features))
        h = h + block.contract(F.relu(block.expand(norm(h, block.norm2))))
        y = norm(h, model.blocks[i + 1].norm1 if i + 1 < len(model.blocks) else model.last_norm)
    k, v = model.pool.kv(y).view(batch, points, 2, heads, -1).permute(2, 0, 3, 1, 4)
    scores = model.pool.query @ k.transpose(-1, -2) / math.sqrt(k.size(-1)) + model.pool.log_weights().double()
    return (torch.softmax(scores, -1) @ v).reshape(batch, features)


def _relative(a, b):
    b = b.detach().double()
    return ((a.detach().double().cpu() - b).norm() / b.norm()).item()


def test_parameters_only_where_asked_for():
    """State dicts of stacks without them are what they were; turns are no parameters and no part of the state."""
    names = lambda **kw: set(_stack(**kw).state_dict())
    assert names() == names(rotary=True)
    assert names(qk_norm=True) - names() == {"blocks.%d.%s_weight" % (i, c) for i in range(2) for c in "qk"}
    model = _stack(rotary=True).to(torch.bfloat16)
    assert torch.equal(model.blocks[0].turns(), s2cnn_amd.s2_rotary_table(3, 5))
    with pytest.raises(AssertionError):
        s2cnn_amd.S2TransformerBlock(6, 6, 2, rotary=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", PLACED, ids=IDS)
def test_stack_and_its_gradients(hip, kw):
    model, plain = _stack(**kw).cuda().eval(), _stack(**kw).double()
    gen = torch.Generator().manual_seed(6)
    x, g = torch.randn(2, 30, 6, 6, generator=gen), torch.randn(2, 30, generator=gen)
    xg, xp = x.cuda().requires_grad_(), x.double().requires_grad_()
    y, want = model(xg), _plain(plain, xp, 3, **kw)
    y.backward(g.cuda())
    want.backward(g.double())
    assert _relative(y, want) < 1e-4
    assert _relative(xg.grad, xp.grad) < 2e-4
    for (name, a), b in zip(model.named_parameters(), plain.parameters()):
        assert _relative(a.grad, b.grad) < 2e-4 or float(b.grad.norm()) < 1e-9, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cast", [False, True], ids=["module", "autocast"])
def test_sixteen_bit_stack(hip, cast, dtype):
    kw = PLACED[0]
    model, plain = _stack(**kw).cuda(), _stack(**kw).double()
    gen = torch.Generator().manual_seed(6)
    x, g = torch.randn(2, 30, 6, 6, generator=gen), torch.randn(2, 30, generator=gen)
    xp = x.double().requires_grad_()
    want = _plain(plain, xp, 3, **kw)
    want.backward(g.double())
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    if cast:
        xg = x.cuda().requires_grad_()
        with torch.autocast("cuda", dtype=dtype):
            y = model(xg)
    else:
        model.to(dtype)
        xg = x.cuda().to(dtype).requires_grad_()
        y = model(xg)
    y.backward(g.cuda().to(y.dtype))
    assert _relative(y, want) < 10 * unit
    assert _relative(xg.grad, xp.grad) < 20 * unit
    a, b = (torch.cat([p.grad.detach().double().cpu().flatten() for p in m.parameters()]) for m in (model, plain))
    assert _relative(a, b) < 20 * unit


@pytest.mark.gpu
def test_invariant_under_rotations_about_the_axis(hip):
    """Frequencies of alpha are whole numbers: a rotation by a grid step permutes the points of each ring and no more."""
    model = _stack(b=4, n_buckets=16, **PLACED[0]).cuda().eval()
    x = torch.randn(2, 30, 8, 8, device="cuda")
    with torch.no_grad():
        a, b = model(x), model(x.roll(3, -1))
    assert _relative(b, a.double().cpu()) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["adamw", "adamw_8bit"])
def test_training_steps_run_eager_and_replayed(hip, optimizer):
    """The network's step with this optimizer runs both ways; replays take the same steps as eager ones (dropout depends on the count of passes, which both
    have): losses of the first replayed steps as those of the eager run after as many, to 1e-3 of float32 sums in another order through four steps."""
    _, eager, _ = harness.train_steps("sphere_transformer_rotary", batch=4, steps=6, warmup=0, lr=1e-3, optimizer=optimizer)
    model, replayed, _ = harness.train_steps_replayed("sphere_transformer_rotary", batch=4, steps=3, warmup=3, lr=1e-3, optimizer=optimizer)
    assert all(math.isfinite(v) for v in eager + replayed)
    for a, b in zip(eager[3:], replayed):
        assert abs(a - b) <= 1e-3 * abs(a)
    assert all(torch.isfinite(p).all() for p in model.parameters())


@pytest.mark.gpu
def test_masters_and_eight_bits_train_a_network_in_sixteen(hip):
    """A stack in bfloat16, three steps: parameters move and stay their masters' roundings."""
    model = _stack(**PLACED[0]).cuda().to(torch.bfloat16)
    before = [p.detach().clone() for p in model.parameters()]
    opt = s2cnn_amd.AdamW(model.parameters(), lr=1e-2, state_bits=8, max_norm=1.0)
    x = torch.randn(2, 30, 6, 6, device="cuda", dtype=torch.bfloat16)
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        model(x).float().square().mean().backward()
        opt.step()
    assert torch.isfinite(opt.norm)
    for p, b in zip(model.parameters(), before):
        assert torch.isfinite(p).all() and torch.equal(p, opt.state[p]["master"].bfloat16())
        assert not torch.equal(p, b)
