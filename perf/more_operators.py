"""Operators of a transformer's attention and of its training step: tables of rotations by position, the rotation of queries and keys,
the same with each head's vectors normalised before it, the norm of a list of gradients, and an AdamW step over a list of tensors with
states of 32 or of 8 bits.

`listed()` names the cases, `draw(rng)` gives more of the same ranges, `prepare` makes what a program holds before the call,
`run` is one pass (plain torch operations in 32 bits, 64 for angles and sums of squares, or with `own` the package's operators), `exact`
the same from the definitions in 64 bits, `work` what a pass cannot do without.

States in 8 bits.  Blocks of 256 entries of a tensor have a factor s each; an entry is s f(c) of a code c, f(c) = c for c < 8 and
(8 + c % 8) 2^(c / 8 - 1) (rounded down) beyond: three bits after the leading one.  First moments have a sign and codes up to 126 in units of 2^-9, which is
the type float8_e4m3fn; second moments codes up to 255.  s = (largest entry of the block) / (f of the largest code), and zero (with all codes)
where that is below 2^-126.  An entry x is rounded up or down at random: with y = x / s, and e = max(3, exponent of y), it becomes
floor(y 2^(3 - e) + u) 2^(e - 3), u a multiple of 2^-16 from a generator (below); second moments above zero get at least code 1.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NORM_EPS = 1e-6
BLOCK = 256
TOP_FIRST, TOP_SECOND = 448.0, 15.0 * 2.0 ** 30
LR, BETAS, ADAM_EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01


def listed():
    return [
        # rotations by the place of every atom of a batch of molecules, three axes, eight pairs: the smallest call
        {"name": "table_atoms", "op": "table", "positions": "f32", "batch": 64, "n": 23, "axes": 3, "pairs": 8, "scale": 1.0},
        # all positions of a long axis for heads of 128 entries
        {"name": "table_long", "op": "table", "positions": "i64", "batch": 1, "n": 262144, "axes": 1, "pairs": 64, "scale": 1.25},
        # one new vector per sequence, each at a position of its own, from a table of all of them
        {"name": "rotary_infer_single_bf16", "op": "rotary", "train": False, "dtype": "bf16", "batch": 64, "heads": 16, "kv_heads": 4, "n": 1, "d": 64,
         "pairs": 32, "interleaved": True, "rows": 32768, "index": True},
        # the points of the sphere at b = 32, 24 of 32 pairs turned, forward and backward
        {"name": "rotary_train_s2_b32", "op": "rotary", "train": True, "dtype": "f32", "batch": 4, "heads": 8, "kv_heads": 8, "n": 4096, "d": 64,
         "pairs": 24, "interleaved": False, "rows": 4096, "index": False},
        # the points at b = 10 (the resolution the digit and shape networks end with), 100 features in 5 heads
        {"name": "norm_rotary_train_s2_b10", "op": "norm_rotary", "train": True, "dtype": "f32", "batch": 32, "heads": 5, "kv_heads": 5, "n": 400,
         "d": 20, "pairs": 10, "interleaved": False, "rows": 400, "index": False},
        # b = 16 with wide heads in bfloat16, key heads shared
        {"name": "norm_rotary_train_s2_b16_bf16", "op": "norm_rotary", "train": True, "dtype": "bf16", "batch": 16, "heads": 8, "kv_heads": 2, "n": 1024,
         "d": 64, "pairs": 32, "interleaved": True, "rows": 1024, "index": False},
        # long sequences, heads as wide as the attention takes them
        {"name": "norm_rotary_train_long_bf16", "op": "norm_rotary", "train": True, "dtype": "bf16", "batch": 4, "heads": 32, "kv_heads": 8, "n": 8192,
         "d": 128, "pairs": 64, "interleaved": False, "rows": 8192, "index": False},
        # one new vector per sequence in half precision
        {"name": "norm_rotary_infer_single_f16", "op": "norm_rotary", "train": False, "dtype": "f16", "batch": 128, "heads": 32, "kv_heads": 8, "n": 1,
         "d": 128, "pairs": 64, "interleaved": False, "rows": 8192, "index": True},
        # the norm of the gradients of a large stack, in bfloat16
        {"name": "grad_norm_stack_bf16", "op": "grad_norm", "dtype": "bf16", "features": 1280, "layers": 8, "hidden": 2560, "heads": 10},
        # the tensors of the network of two blocks of 96 features, gradients clipped: latency
        {"name": "adamw_small", "op": "adamw", "dtype": "f32", "bits": 32, "masters": False, "clip": True, "features": 96, "layers": 2, "hidden": 192, "heads": 6},
        # twelve blocks in bfloat16 with states in 8 bits and the parameters in 32 beside them, gradients clipped
        {"name": "adamw_stack_8bit_bf16", "op": "adamw", "dtype": "bf16", "bits": 8, "masters": True, "clip": True, "features": 512, "layers": 12,
         "hidden": 1024, "heads": 8},
        # four wide blocks in float32: the largest case
        {"name": "adamw_large", "op": "adamw", "dtype": "f32", "bits": 32, "masters": False, "clip": False, "features": 2048, "layers": 4, "hidden": 4096,
         "heads": 16},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    limit = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["table", "rotary", "rotary", "norm_rotary", "norm_rotary", "norm_rotary", "grad_norm", "adamw", "adamw", "adamw"])
        if op == "table":
            axes = rng.choice([1, 1, 2, 3])
            case = {"op": op, "positions": rng.choice(["f32", "f64", "i32", "i64"]), "batch": _log_int(rng, 1, 64), "n": _log_int(rng, 1, 262144),
                    "axes": axes, "pairs": _log_int(rng, 1, 64), "scale": rng.choice([1.0, 1.25])}
        elif op in ("rotary", "norm_rotary"):
            kv_heads, n, d = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, _log_int(rng, 2, 8192), _log_int(rng, 2, 8192)]), _log_int(rng, 8, 128)
            d += d % 2 if rng.random() < 0.7 else 0
            index = n == 1 or rng.random() < 0.3
            case = {"op": op, "train": n > 1 and rng.random() < 0.7, "dtype": rng.choice(["f32", "bf16", "f16"]), "batch": _log_int(rng, 1, 128),
                    "heads": kv_heads * rng.choice([1, 1, 2, 4]), "kv_heads": kv_heads, "n": n, "d": d,
                    "pairs": rng.choice([d // 2, d // 2, max(1, d // 4), rng.randint(1, d // 2)]), "interleaved": rng.random() < 0.5,
                    "rows": n + _log_int(rng, 1, 32768) if index else n, "index": index}
        else:
            features, heads = 0, rng.choice([1, 2, 4, 5, 8])
            features = heads * _log_int(rng, 4, 256)
            case = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "features": features, "layers": rng.randint(1, 12),
                    "hidden": features * rng.choice([1, 2, 4]), "heads": heads}
            if op == "adamw":
                case.update(bits=rng.choice([8, 32]), clip=rng.random() < 0.5, masters=case["dtype"] != "f32" and rng.random() < 0.6)
        if work(case)["bytes"] <= limit:
            return case


def _shapes(case):
    """The parameters of a stack of transformer blocks."""
    f, h = case["features"], case["hidden"]
    block = [(f,), (f,), (3 * f, f), (3 * f,), (f, f), (f,), (case["heads"], 32), (f,), (f,), (h, f), (h,), (f, h), (f,)]
    return block * case["layers"] + [(f,), (f,)]


def _entries(case):
    return sum(math.prod(s) for s in _shapes(case))


def work(case):
    if case["op"] == "table":
        rows = case["batch"] * case["n"]
        size = 8 if case["positions"] in ("i64", "f64") else 4
        return {"bytes": rows * (case["axes"] * size + case["pairs"] * 8) + case["axes"] * case["pairs"] * 8, "flops": rows * case["pairs"] * 40}
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("rotary", "norm_rotary"):
        entries = case["batch"] * (case["heads"] + case["kv_heads"]) * case["n"] * case["d"]
        rows = min(case["rows"], case["batch"] * case["n"]) if case["index"] else case["n"]
        tensors = 2 + ((2 if case["op"] == "rotary" else 3) if case["train"] else 0)      # x, y; gy, gx and x again
        return {"bytes": tensors * entries * size + rows * case["pairs"] * 8, "flops": entries * (20 if case["train"] else 8)}
    n = _entries(case)
    if case["op"] == "grad_norm":
        return {"bytes": n * size, "flops": 2 * n}
    states = 16 if case["bits"] == 32 else 4 + 8                  # read and written; 8 bits: and their values written
    return {"bytes": n * (3 * size + states + (8 if case["masters"] else 0)), "flops": 20 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _frequencies(axes, pairs, dev):
    """[axes, pairs] in 64 bits: falling geometrically from 1 to 1e-4, turned over the axes pair by pair where there are several."""
    f = 1e4 ** (-torch.arange(pairs, dtype=torch.float64, device=dev) / pairs)
    return f * (torch.arange(pairs, device=dev) % axes == torch.arange(axes, device=dev).view(-1, 1)) if axes > 1 else f.view(1, -1)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    state = {"case": case, "seed": seed}
    if case["op"] == "table":
        shape = (case["batch"], case["n"], case["axes"])
        if case["positions"] in ("i32", "i64"):      # consecutive places behind what is there already
            p = torch.arange(case["n"], device=dev).view(1, -1, 1) + torch.randint(0, 65536, (case["batch"], 1, case["axes"]), device=dev, generator=g)
            state["positions"] = p.to(torch.int32 if case["positions"] == "i32" else torch.int64)
        else:
            state["positions"] = (normal(*shape) * 3.0).to(torch.float32 if case["positions"] == "f32" else torch.float64)
        state["frequencies"] = _frequencies(case["axes"], case["pairs"], dev)
        return state
    dt = TYPES[case["dtype"]]
    if case["op"] in ("rotary", "norm_rotary"):
        b, h, hk, n, d = (case[k] for k in ("batch", "heads", "kv_heads", "n", "d"))
        # queries, keys and values are split off a projection's output, so that they are strided views as in a program
        x = (normal(b, n, h + 2 * hk, d) * 1.5 + 0.1).to(dt)
        state["q"], state["k"] = x[:, :, :h].transpose(1, 2), x[:, :, h:h + hk].transpose(1, 2)
        angles = torch.arange(case["rows"], device=dev, dtype=torch.float64).view(-1, 1) * _frequencies(1, case["pairs"], dev)
        state["table"] = torch.stack([angles.cos(), angles.sin()], -1).float()
        state["index"] = torch.randint(0, case["rows"], (b, n), device=dev, generator=g, dtype=torch.int32) if case["index"] else None
        if case["op"] == "norm_rotary":
            state["q_weight"], state["k_weight"] = ((normal(d) * 0.2 + 1.0).to(dt) for _ in range(2))
        if case["train"]:
            state["gq"], state["gk"] = (normal(b, n, heads, d).to(dt).transpose(1, 2) for heads in (h, hk))
            for name in ("q", "k", "q_weight", "k_weight"):
                if name in state:
                    state[name].requires_grad_()
        return state
    # Parameters, gradients and states as views of one buffer each, every tensor at a multiple of 256 entries
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + -(-s // BLOCK) * BLOCK)
    total = starts[-1]
    inside = torch.zeros(total + 1, dtype=torch.int32, device=dev)        # 1 at the tensors' entries, 0 between them
    at = torch.tensor([starts[:-1], [a + n for a, n in zip(starts, sizes)]], device=dev)
    inside.index_add_(0, at[0], torch.ones_like(at[0], dtype=torch.int32))
    inside.index_add_(0, at[1], -torch.ones_like(at[1], dtype=torch.int32))
    inside = inside.cumsum(0)[:total].float()

    def views(flat):
        return [flat[a:a + n].view(s) for a, n, s in zip(starts, sizes, shapes)]

    spread = torch.repeat_interleave(torch.exp(normal(total // BLOCK)), BLOCK)            # gradients differ from block to block
    flat = {"grad": (normal(total).mul_(spread).mul_(inside) * 1e-3).to(dt)}
    if case["op"] == "adamw":
        p = normal(total).mul_(inside) * 0.02
        flat["p"] = p.to(dt)
        if case["masters"]:
            flat["master"] = p
        state["step"] = 100 + seed % 1000
        if case["bits"] == 32:
            flat["first"] = normal(total).mul_(spread).mul_(inside) * 3e-4
            flat["second"] = (torch.rand(total, device=dev, generator=g) + 0.1).mul_(spread * spread).mul_(inside) * 1e-6
        else:
            flat["first"] = (normal(total) * 100.0).clamp_(-TOP_FIRST, TOP_FIRST).mul_(inside).to(torch.float8_e4m3fn)
            flat["second"] = (torch.randint(192, 256, (total,), device=dev, generator=g) * inside).to(torch.uint8)
            by_block = spread.view(-1, BLOCK)[:, 0]
            state["scales"] = torch.stack([by_block * (1e-3 / (TOP_FIRST * 512.0)), by_block * by_block * (4e-6 / TOP_SECOND)], 1)
            state["scale_views"] = [state["scales"][a // BLOCK:a // BLOCK - (-n // BLOCK)] for a, n in zip(starts, sizes)]
    state["flat"] = flat
    state["views"] = {name: views(t) for name, t in flat.items()}
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"table": _plain_table, "rotary": _plain_rotary, "norm_rotary": _plain_rotary, "grad_norm": _plain_grad_norm, "adamw": _plain_adamw}[state["case"]["op"]](state)


def _run_own(s):
    import s2cnn_amd
    case = s["case"]
    if case["op"] == "table":
        return {"table": s2cnn_amd.rotary_table(s["positions"], s["frequencies"], scale=case["scale"])}
    if case["op"] in ("rotary", "norm_rotary"):
        if case["op"] == "rotary":
            q, k = s2cnn_amd.rotary(s["q"], s["k"], s["table"], index=s["index"], interleaved=case["interleaved"])
            names = ["q", "k"]
        else:
            q, k = s2cnn_amd.norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"], index=s["index"], eps=NORM_EPS,
                                         interleaved=case["interleaved"])
            names = ["q", "k", "q_weight", "k_weight"]
        if not case["train"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad([q, k], [s[n] for n in names], [s["gq"], s["gk"]])
        return {"q": q, "k": k, **{"g" + n: t for n, t in zip(names, grads)}}
    v = s["views"]
    if case["op"] == "grad_norm":
        return {"norm": s2cnn_amd.grad_norm(v["grad"])}
    norm = s2cnn_amd.grad_norm(v["grad"]) if case["clip"] else None
    s2cnn_amd.adamw_step(v["p"], v["grad"], v["first"], v["second"], s["step"], lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY,
                         masters=v.get("master"), scales=s.get("scale_views"), norm=norm, max_norm=1.0 if case["clip"] else None, seed=s["seed"])
    out = {"p": s["flat"]["p"], "first": s["flat"]["first"], "second": s["flat"]["second"]}
    if case["masters"]:
        out["master"] = s["flat"]["master"]
    if case["clip"]:
        out["norm"] = norm
    if case["bits"] == 8:
        (out["first"],), (out["second"],) = s2cnn_amd.adamw_states([out["first"]], [out["second"]], [s["scales"]])
    return out


def _plain_table(s):
    angles = (s["positions"].double().unsqueeze(-1) * s["frequencies"]).sum(-2)
    return {"table": (torch.stack([angles.cos(), angles.sin()], -1) * s["case"]["scale"]).float()}


def _turned(x, table, interleaved, sign=1.0):
    """x [..., d] turned by the table's angles (sign -1: back), the entries behind the pairs as they are."""
    pairs = table.size(-2)
    head, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :pairs], head[..., pairs:])
    cos, sin = table[..., 0], table[..., 1] * sign
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, rest], -1)


def _plain_rotary(s):
    case = s["case"]
    table = s["table"] if s["index"] is None else s["table"][s["index"].long()].unsqueeze(1)
    out = {}
    for name in ("q", "k"):
        x, dt = s[name].float(), s[name].dtype
        if case["op"] == "rotary":
            out[name] = _turned(x, table, case["interleaved"]).to(dt)
            if case["train"]:
                out["g" + name] = _turned(s["g" + name].float(), table, case["interleaved"], -1.0).to(dt)
            continue
        w = s[name + "_weight"].float()
        r = (x.square().mean(-1, keepdim=True) + NORM_EPS).rsqrt()
        xh = x * r
        out[name] = _turned(xh * w, table, case["interleaved"]).to(dt)
        if case["train"]:
            g = _turned(s["g" + name].float(), table, case["interleaved"], -1.0)
            u = g * w
            out["g" + name] = (r * (u - xh * (u * xh).mean(-1, keepdim=True))).to(dt)
            out["g" + name + "_weight"] = (g * xh).sum((0, 1, 2)).to(dt)
    return out


def _norm(flat):
    return flat.double().square().sum().sqrt().float()


def _plain_grad_norm(s):
    return {"norm": _norm(s["flat"]["grad"])}


def _random(n, seed, step, dev):
    """Two multiples of 2^-16 below one for each of n entries: the halves of word i % 4 of Philox4x32-10 of counter (i / 4, step) and key seed."""
    mask = 0xFFFFFFFF
    index = torch.arange(n // 4, device=dev, dtype=torch.int64)
    c0, c1 = index & mask, index >> 32
    c2, c3 = torch.full_like(index, step & mask), torch.full_like(index, (step >> 32) & mask)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & mask) ^ c1 ^ k0, b & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack([c0, c1, c2, c3], 1).flatten()
    return (words & 0xFFFF).float() * 2.0 ** -16, (words >> 16).float() * 2.0 ** -16


def _value(codes):
    """f of codes, float32"""
    c = codes.int()
    return torch.where(c < 8, c, 8 + c % 8).float() * ((c // 8 + 126).clamp(min=127) << 23).view(torch.float32)


def _codes(x, inverse, u, most):
    """Codes of x >= 0 in units of 1 / inverse, rounded at random."""
    y = x * inverse
    part, e = torch.frexp(y)                                      # y = part 2^e, part from 1/2 up to 1
    above = e > 3
    return (torch.where(above, (e - 4) * 8, 0) + torch.floor(torch.where(above, part * 16.0, y) + u).int()).clamp(max=most)


def _scale(x, factor):
    """[blocks, 1]: the block's factor and its inverse, both zero where the factor is below 2^-126"""
    s = x.view(-1, BLOCK).abs().amax(1, keepdim=True) * factor
    fine = s >= 2.0 ** -126
    return torch.where(fine, s, torch.zeros_like(s)), torch.where(fine, s.reciprocal(), torch.zeros_like(s))


def _plain_adamw(s):
    case, flat = s["case"], s["flat"]
    g = flat["grad"].float()
    out = {"p": flat["p"]}
    if case["clip"]:
        out["norm"] = _norm(flat["grad"])
        g = g * torch.clamp(1.0 / out["norm"], max=1.0)
    if case["bits"] == 8:
        scales = torch.repeat_interleave(s["scales"], BLOCK, 0)
        m, v = flat["first"].float() * 512.0 * scales[:, 0], _value(flat["second"]) * scales[:, 1]
    else:
        m, v = flat["first"], flat["second"]
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + (g * g) * (1 - BETAS[1])
    p = flat["master"] if case["masters"] else flat["p"].float()
    size = LR / (1 - BETAS[0] ** s["step"])
    p = p * (1 - LR * DECAY) - size * (m / ((v / (1 - BETAS[1] ** s["step"])).sqrt() + ADAM_EPS))
    flat["p"].copy_(p)
    if case["masters"]:
        out["master"] = flat["master"].copy_(p)
    if case["bits"] == 32:
        out["first"], out["second"] = flat["first"].copy_(m), flat["second"].copy_(v)
        return out
    u_m, u_v = _random(m.numel(), s["seed"], s["step"], m.device)
    (sm, im), (sv, iv) = _scale(m, 1.0 / (TOP_FIRST * 512.0)), _scale(v, 1.0 / TOP_SECOND)
    cm = _codes(m.abs().view(-1, BLOCK), im, u_m.view(-1, BLOCK), 126)
    cv = _codes(v.view(-1, BLOCK), iv, u_v.view(-1, BLOCK), 255)
    cv = torch.where((v.view(-1, BLOCK) > 0) & (iv > 0), cv.clamp(min=1), cv)
    cm = cm + 128 * (m.view(-1, BLOCK) < 0).int()
    flat["first"].view(torch.uint8).copy_(cm.view(-1))
    flat["second"].copy_(cv.view(-1))
    s["scales"].copy_(torch.cat([sm, sv], 1))
    out["first"] = (flat["first"].float() * 512.0).view(-1, BLOCK).mul_(sm).view(-1)
    out["second"] = _value(cv).mul_(sv).view(-1)
    return out


# ---- 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        p = s["positions"].double()
        total = sum(p[..., a, None] * s["frequencies"][a] for a in range(case["axes"]))
        z = torch.polar(torch.full_like(total, case["scale"]), total)
        return {"table": torch.view_as_real(z)}
    if case["op"] in ("rotary", "norm_rotary"):
        return _exact_rotary(s)
    if case["op"] == "grad_norm":
        return {"norm": torch.linalg.vector_norm(s["flat"]["grad"].double())}
    f = {name: t.double() for name, t in s["flat"].items() if t.dtype != torch.uint8}
    p, g, result = f["master" if case["masters"] else "p"], f["grad"], {}
    if case["clip"]:
        total = torch.sqrt((g ** 2).sum())
        result["norm"] = total
        if total > 1.0:
            g = g / total
    m, v = f["first"], f.get("second")
    if case["bits"] == 8:
        c = s["flat"]["second"].double()
        v = torch.where(c < 8, c, (8 + torch.remainder(c, 8)) * 2.0 ** (torch.floor(c / 8) - 1))
        factors = s["scales"].double()
        m = (m.view(-1, BLOCK) * factors[:, :1] * 512).view(-1)
        v = (v.view(-1, BLOCK) * factors[:, 1:]).view(-1)
    m = m + (1 - BETAS[0]) * (g - m)
    v = v + (1 - BETAS[1]) * (g ** 2 - v)
    mh, vh = m / (1 - BETAS[0] ** s["step"]), v / (1 - BETAS[1] ** s["step"])
    p = p - LR * DECAY * p - LR * mh / (torch.sqrt(vh) + ADAM_EPS)
    result["p"] = p
    if case["masters"]:
        result["master"] = p
    # states in 8 bits are rounded at random numbers, next to which 64 bits may fall on the other side: no such value
    result["first"], result["second"] = (m, v) if case["bits"] == 32 else (None, None)
    return result


def _exact_rotary(s):
    case = s["case"]
    t = s["table"].double()
    turn = torch.complex(t[..., 0], t[..., 1])
    if s["index"] is not None:
        turn = turn[s["index"].long()].unsqueeze(1)
    pairs = case["pairs"]

    def rotate(z, by):
        w = z.clone()
        first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if case["interleaved"] else (slice(0, pairs), slice(pairs, 2 * pairs))
        c = torch.complex(z[..., first], z[..., second]) * by
        w[..., first], w[..., second] = c.real, c.imag
        return w

    result = {}
    for name in ("q", "k"):
        x = s[name].detach().double()
        g = rotate(s["g" + name].double(), turn.conj()) if case["train"] else None
        if case["op"] == "rotary":
            result[name] = rotate(x, turn)
            if case["train"]:
                result["g" + name] = g
            continue
        w, d = s[name + "_weight"].detach().double(), case["d"]
        size = torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + NORM_EPS)
        result[name] = rotate(x / size * w, turn)
        if case["train"]:
            u = g * w
            result["g" + name] = u / size - x * (u * x).sum(-1, keepdim=True) / (d * size ** 3)
            result["g" + name + "_weight"] = (g * x / size).sum((0, 1, 2))
    return result
