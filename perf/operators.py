"""The operators of a transformer block over the points of a sphere, of SO(3) or of a molecule: attention with a learned bias by
buckets of the angle (or distance) of two points, layer normalisation, dropout, and the step between two sublayers that joins
residual, dropout and normalisation.

`listed()` names the cases, `draw(rng)` gives more of the same ranges, `prepare` makes what a program holds before the call,
`run` is one pass (plain torch operations in 32 bits, or with `own` the package's operators), `exact` the same from the
definitions in 64 bits, `work` what a pass cannot do without.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def listed():
    return [
        # a training step on molecules: up to 23 atoms, buckets of the distances of each molecule's atoms, the smallest attention
        {"name": "attention_train_atoms", "op": "attention", "train": True, "dtype": "f32", "batch": 64, "heads": 4, "kv_heads": 4, "n_q": 23,
         "n_k": 23, "d": 16, "buckets": 16, "shared": False, "ragged": True, "radius": 4.0, "grid": False},
        # a layer on the sphere at b = 10 (the resolution the digit and shape networks end with), 100 features in 5 heads
        {"name": "attention_train_s2_b10", "op": "attention", "train": True, "dtype": "f32", "batch": 32, "heads": 5, "kv_heads": 5, "n_q": 400,
         "n_k": 400, "d": 20, "buckets": 32, "shared": True, "ragged": False, "radius": 4.0, "grid": True},
        # the same at b = 16 with wide heads in bfloat16, each point attending to the points within a radian
        {"name": "attention_train_s2_b16_bf16", "op": "attention", "train": True, "dtype": "bf16", "batch": 16, "heads": 8, "kv_heads": 2,
         "n_q": 1024, "n_k": 1024, "d": 64, "buckets": 32, "shared": True, "ragged": False, "radius": 1.0, "grid": True},
        # the full sphere at b = 32 in float32: the largest case
        {"name": "attention_train_s2_b32", "op": "attention", "train": True, "dtype": "f32", "batch": 4, "heads": 8, "kv_heads": 8, "n_q": 4096,
         "n_k": 4096, "d": 64, "buckets": 32, "shared": True, "ragged": False, "radius": 4.0, "grid": True},
        # one pooled query per signal over the 32^3 points of SO(3) at b = 16, in place of the integral: a single token over a long axis
        {"name": "attention_infer_pool_so3_b16", "op": "attention", "train": False, "dtype": "f32", "batch": 8, "heads": 8, "kv_heads": 2, "n_q": 1,
         "n_k": 32768, "d": 50, "buckets": 0, "shared": True, "ragged": False, "radius": 4.0, "grid": False},
        # odd point sets of another size each, evaluated in half precision, heads as wide as they come
        {"name": "attention_infer_points_f16", "op": "attention", "train": False, "dtype": "f16", "batch": 7, "heads": 6, "kv_heads": 3, "n_q": 1009,
         "n_k": 2501, "d": 100, "buckets": 48, "shared": True, "ragged": True, "radius": 4.0, "grid": False},
        # the features at the points of b = 10 for a batch of 32, forward and backward
        {"name": "norm_train_100", "op": "norm", "dtype": "f32", "rows": 12800, "features": 100},
        # wide features at many points in bfloat16
        {"name": "norm_train_1024_bf16", "op": "norm", "dtype": "bf16", "rows": 65536, "features": 1024},
        # activations of a layer at b = 32 (16 signals of 64 features on the 64 x 64 x 64 grid): the largest dropout
        {"name": "dropout_train_b32", "op": "dropout", "dtype": "f32", "n": 16 * 16 * 64 * 64 * 64, "p": 0.1},
        # a few thousand activations in bfloat16, an odd number of them: latency
        {"name": "dropout_train_small_bf16", "op": "dropout", "dtype": "bf16", "n": 23 * 64 * 5 + 7, "p": 0.3},
        # between two sublayers of the molecules' block
        {"name": "step_train_atoms", "op": "step", "dtype": "f32", "rows": 64 * 23, "features": 64, "p": 0.1},
        # between two sublayers at the points of b = 16, 512 features, batch 16
        {"name": "step_train_s2_b16_bf16", "op": "step", "dtype": "bf16", "rows": 16 * 1024, "features": 512, "p": 0.1},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def _draw_attention(rng):
    kind = rng.choice(["atoms", "sphere", "sphere", "points", "pool"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    case = {"op": "attention", "train": rng.random() < 0.6, "dtype": dtype, "batch": _log_int(rng, 1, 32), "heads": heads, "kv_heads": kv_heads}
    if kind == "atoms":
        n = rng.randint(2, 64)
        case.update(n_q=n, n_k=n, buckets=rng.randint(2, 64), shared=False, ragged=True, radius=4.0, grid=False)
    elif kind == "sphere":
        n = 4 * _log_int(rng, 4, 32) ** 2
        case.update(n_q=n, n_k=n, buckets=rng.randint(4, 64), shared=True, ragged=False, radius=rng.choice([1.0, 4.0]), grid=True)
    elif kind == "points":
        case.update(n_q=_log_int(rng, 1, 2047), n_k=_log_int(rng, 16, 8191), buckets=rng.choice([0, 16, 32]), shared=True,
                    ragged=rng.random() < 0.5, radius=4.0, grid=False)
    else:
        case.update(n_q=rng.choice([1, 1, 2, 5]), n_k=8 * rng.randint(3, 16) ** 3, buckets=0, shared=True, ragged=rng.random() < 0.3,
                    radius=4.0, grid=False)
    case["d"] = _log_int(rng, 8, 128)
    return case


def draw(rng):
    limit = _cost(listed()[3])
    while True:
        op = rng.choice(["attention", "attention", "attention", "norm", "dropout", "step"])
        if op == "attention":
            case = _draw_attention(rng)
        elif op == "dropout":
            case = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "n": _log_int(rng, 1000, 1 << 26) | 1, "p": rng.choice([0.05, 0.1, 0.25, 0.5])}
        else:
            case = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "rows": _log_int(rng, 16, 65535) | 1, "features": _log_int(rng, 8, 2048)}
            if op == "step":
                case["p"] = rng.choice([0.05, 0.1, 0.25, 0.5])
        if _cost(case) <= limit:
            return case


def _cost(case):
    w = work(case)
    return w["flops"] / 1e14 + w["bytes"] / 3e12


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "attention":
        b, h, hk, nq, nk, d = (case[k] for k in ("batch", "heads", "kv_heads", "n_q", "n_k", "d"))
        share = 0.5 if case["ragged"] else 1.0          # lengths are spread evenly over 0 .. n_k
        queries, keys = b * h * nq * d * size, 2 * b * hk * nk * d * size
        table = h * case["buckets"] * size
        buckets = (1 if case["shared"] else b) * nq * nk if case["buckets"] else 0
        once = 2 * queries + keys * share + table + buckets + 4 * nk
        pairs = b * h * nq * nk * share
        if not case["train"]:
            return {"bytes": once, "flops": 4 * pairs * d}
        return {"bytes": once + 2 * queries + keys + table, "flops": 12 * pairs * d}      # and dO read; dQ, dK, dV, dtable written
    if case["op"] == "dropout":
        return {"bytes": 4 * case["n"] * size, "flops": 2 * case["n"]}                     # x, g read; y, gx written
    n = case["rows"] * case["features"]
    tensors = 4 if case["op"] == "norm" else 8          # x, g, y, gx; step: x, residual, g_h, g_y, h, y, gx, g_residual
    return {"bytes": tensors * n * size + 4 * case["features"] * size, "flops": 20 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _points(case, n, dev, g):
    """n unit vectors and the logarithm of the area each stands for: the points of the 2b x 2b grid, or random ones."""
    if case["grid"]:
        b = math.isqrt(n) // 2
        beta = (2 * torch.arange(2 * b, device=dev, dtype=torch.float32) + 1) * math.pi / (4 * b)
        alpha = torch.arange(2 * b, device=dev, dtype=torch.float32) * math.pi / b
        beta, alpha = (t.reshape(-1) for t in torch.meshgrid(beta, alpha, indexing="ij"))
        xyz = torch.stack([beta.sin() * alpha.cos(), beta.sin() * alpha.sin(), beta.cos()], -1)
        return xyz, beta.sin().log()
    xyz = torch.randn(n, 3, device=dev, generator=g)
    return xyz / xyz.norm(dim=-1, keepdim=True), torch.rand(n, device=dev, generator=g).add(0.1).log()


def _buckets(p, q, n, radius):
    """Bucket of the angle of every pair; -1 beyond the radius."""
    angle = (p @ q.transpose(-1, -2)).clamp(-1.0, 1.0).arccos()
    index = (angle * (n / min(radius, math.pi))).floor().clamp(max=n - 1)
    return torch.where(angle <= radius, index, torch.full_like(index, -1.0)).to(torch.int8)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g).to(dt)

    state = {"case": case}
    if case["op"] == "attention":
        b, h, hk, nq, nk, d, nb = (case[k] for k in ("batch", "heads", "kv_heads", "n_q", "n_k", "d", "buckets"))
        # heads are split off a projection's output, so that they are strided views as in a program
        state["q"] = normal(b, nq, h, d).transpose(1, 2)
        state["k"] = normal(b, nk, hk, d).transpose(1, 2)
        state["v"] = normal(b, nk, hk, d).transpose(1, 2)
        points, area = _points(case, nk, dev, g)
        state["table"] = normal(h, nb) if nb else None
        state["buckets"] = None
        if nb and case["shared"]:
            state["buckets"] = _buckets(points if nq == nk else _points(case, nq, dev, g)[0], points, nb, case["radius"])
        elif nb:
            atoms = torch.randn(b, nk, 3, device=dev, generator=g)
            atoms = atoms / atoms.norm(dim=-1, keepdim=True)
            state["buckets"] = _buckets(atoms, atoms, nb, case["radius"])
        state["key_bias"] = area
        state["lengths"] = None
        if case["ragged"]:
            state["lengths"] = torch.randint(0, nk + 1, (b,), device=dev, generator=g, dtype=torch.int32)
            state["lengths"][0] = nk         # a batch is padded to its longest set
        names = ("q", "k", "v", "table")
        state["g"] = normal(b, h, nq, d)
    elif case["op"] == "dropout":
        state["x"], state["g"] = normal(case["n"]), normal(case["n"])
        names = ("x",)
    else:
        rows, features = case["rows"], case["features"]
        state["x"], state["g"] = normal(rows, features) * 1.5 + 0.25, normal(rows, features)
        state["weight"], state["bias"] = normal(features) * 0.2 + 1.0, normal(features) * 0.2
        names = ("x", "weight", "bias")
        if case["op"] == "step":
            state["residual"], state["g_h"] = normal(rows, features), normal(rows, features)
            names = ("x", "residual", "weight", "bias")
    state["seed"] = seed
    if case.get("train", True):
        for name in names:
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"attention": _plain_attention, "norm": _plain_norm, "dropout": _plain_dropout, "step": _plain_step}[state["case"]["op"]](state)


def _run_own(s):
    import s2cnn_amd
    case = s["case"]
    if case["op"] == "attention":
        out = s2cnn_amd.attention(s["q"], s["k"], s["v"], table=s["table"], buckets=s["buckets"], key_bias=s["key_bias"], lengths=s["lengths"])
        if not case["train"]:
            return {"out": out}
        names = ["q", "k", "v"] + (["table"] if s["table"] is not None else [])
        grads = torch.autograd.grad(out, [s[n] for n in names], s["g"])
        return {"out": out, **{"g" + n: t for n, t in zip(names, grads)}}
    if case["op"] == "norm":
        y = s2cnn_amd.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        gx, gw, gb = torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["g"])
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    if case["op"] == "dropout":
        y = s2cnn_amd.dropout(s["x"], case["p"], s["seed"])
        return {"y": y, "gx": torch.autograd.grad(y, s["x"], s["g"])[0]}
    h, y = s2cnn_amd.dropout_add_layer_norm(s["x"], s["residual"], case["p"], s["seed"], s["weight"], s["bias"], eps=EPS)
    gx, gr, gw, gb = torch.autograd.grad([h, y], [s["x"], s["residual"], s["weight"], s["bias"]], [s["g_h"], s["g"]])
    return {"h": h, "y": y, "gx": gx, "gresidual": gr, "gw": gw, "gb": gb}


def _plain_attention(s):
    case, dt = s["case"], s["q"].dtype
    b, h, hk, nq, nk, d, nb = (case[k] for k in ("batch", "heads", "kv_heads", "n_q", "n_k", "d", "buckets"))
    group = h // hk
    q = s["q"].float().reshape(b, hk, group * nq, d)
    k, v = s["k"].float().contiguous(), s["v"].float().contiguous()
    scale = 1.0 / math.sqrt(d)
    x = (q @ k.transpose(-1, -2).contiguous()).mul_(scale).view(b, hk, group, nq, nk)
    valid = torch.ones(1, 1, 1, 1, nk, dtype=torch.bool, device=q.device)
    index = None
    if s["lengths"] is not None:
        valid = (torch.arange(nk, device=q.device) < s["lengths"].view(b, 1)).view(b, 1, 1, 1, nk)
    if nb:
        index = s["buckets"].long()
        valid = valid & (index >= 0).view(-1, 1, 1, nq, nk)
        bias = s["table"].float()[:, index.clamp(min=0)]                                # [heads, (batch,) n_q, n_k]
        bias = bias.transpose(0, 1) if index.dim() == 3 else bias.unsqueeze(0)
        x += bias.view(-1, hk, group, nq, nk)
    x += s["key_bias"]
    x.masked_fill_(~valid, -math.inf)
    x -= x.amax(-1, keepdim=True).nan_to_num_(neginf=0.0)
    p = x.exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, torch.ones_like(total))
    p = p.view(b, hk, group * nq, nk)
    out = p @ v
    result = {"out": out.view(b, h, nq, d).to(dt)}
    if not case["train"]:
        return result
    g = s["g"].float().reshape(b, hk, group * nq, d)
    gv = p.transpose(-1, -2).contiguous() @ g
    dp = g @ v.transpose(-1, -2).contiguous()
    ds = dp.sub_((g * out).sum(-1, keepdim=True)).mul_(p)
    gq = (ds @ k) * scale
    gk = (ds.transpose(-1, -2).contiguous() @ q) * scale
    result.update(gq=gq.view(b, h, nq, d).to(dt), gk=gk.to(dt), gv=gv.to(dt))
    if nb:
        ds = ds.view(b, h, nq, nk)
        if index.dim() == 2:
            ds, index = ds.sum(0, keepdim=True), index.unsqueeze(0)
        hot = (index.unsqueeze(-1) == torch.arange(nb, device=q.device)).float()        # [batch or 1, n_q, n_k, buckets]
        rows = ds.transpose(1, 2).contiguous() @ hot                                    # [batch or 1, n_q, heads, buckets]
        result["gtable"] = rows.sum(1).sum(0).to(dt)
    return result


def _normalised(x):
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = (centred.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return centred * rstd, rstd


def _norm_gradients(xh, rstd, g, w):
    gw = g * w
    gx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return gx, (g * xh).sum(0), g.sum(0)


def _plain_norm(s):
    dt = s["x"].dtype
    w, g = s["weight"].float(), s["g"].float()
    xh, rstd = _normalised(s["x"].float())
    y = xh * w + s["bias"].float()
    return dict(zip(("y", "gx", "gw", "gb"), (t.to(dt) for t in (y, *_norm_gradients(xh, rstd, g, w)))))


def _kept(n, p, seed, dev):
    """The factor 0 or 1 / (1 - p) of each of n elements: Philox4x32-10 of (index / 8, seed), 16 bits an element."""
    mask = 0xFFFFFFFF
    index = torch.arange((n + 7) // 8, device=dev, dtype=torch.int64)
    c0, c1 = index & mask, index >> 32
    c2, c3 = torch.zeros_like(index), torch.zeros_like(index)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & mask) ^ c1 ^ k0, b & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 1)
    drop = min(65535, round(p * 65536))
    return (words.reshape(-1)[:n] >= drop).float() * (65536.0 / (65536 - drop))


def _plain_dropout(s):
    dt = s["x"].dtype
    factor = _kept(s["x"].numel(), s["case"]["p"], s["seed"], s["x"].device)
    return {"y": (s["x"].float() * factor).to(dt), "gx": (s["g"].float() * factor).to(dt)}


def _plain_step(s):
    dt = s["x"].dtype
    factor = _kept(s["x"].numel(), s["case"]["p"], s["seed"], s["x"].device).view_as(s["x"])
    h = s["residual"].float() + s["x"].float() * factor
    w, g = s["weight"].float(), s["g"].float()
    xh, rstd = _normalised(h)
    y = xh * w + s["bias"].float()
    gn, gw, gb = _norm_gradients(xh, rstd, g, w)
    gr = s["g_h"].float() + gn
    return {"h": h.to(dt), "y": y.to(dt), "gx": (gr * factor).to(dt), "gresidual": gr.to(dt), "gw": gw.to(dt), "gb": gb.to(dt)}


# ---- 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = {k: v.detach() if torch.is_tensor(v) else v for k, v in prepare(case, seed).items()}
    if case["op"] == "attention":
        return _exact_attention(s)
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    factor = _kept(d["x"].numel(), case["p"], seed, d["x"].device).double().view_as(d["x"]) if "p" in case else None
    if factor is not None:      # a factor of 65536 / (65536 - T), rounded to 32 bits above
        drop = min(65535, round(case["p"] * 65536))
        factor = torch.where(factor > 0, torch.full_like(factor, 65536 / (65536 - drop)), factor)
    if case["op"] == "dropout":
        return {"y": d["x"] * factor, "gx": d["g"] * factor}
    h = d["x"] if case["op"] == "norm" else d["residual"] + d["x"] * factor
    n = h.size(1)
    mean = h.sum(1, keepdim=True) / n
    var = ((h - mean) ** 2).sum(1, keepdim=True) / n
    sd = torch.sqrt(var + EPS)
    y = (h - mean) / sd * d["weight"] + d["bias"]
    u = d["g"] * d["weight"]
    a = u.sum(1, keepdim=True) / n
    c = (u * (h - mean)).sum(1, keepdim=True) / n
    gh = u / sd - a / sd - (h - mean) * c / sd ** 3
    gw, gb = (d["g"] * (h - mean) / sd).sum(0), d["g"].sum(0)
    if case["op"] == "norm":
        return {"y": y, "gx": gh, "gw": gw, "gb": gb}
    gh = gh + d["g_h"]
    return {"h": h, "y": y, "gx": gh * factor, "gresidual": gh, "gw": gw, "gb": gb}


def _exact_attention(s):
    case = s["case"]
    b, h, hk, nq, nk, d, nb = (case[k] for k in ("batch", "heads", "kv_heads", "n_q", "n_k", "d", "buckets"))
    group, scale = h // hk, d ** -0.5
    dev = s["q"].device
    q, k, v, g = (s[n].double().contiguous() for n in ("q", "k", "v", "g"))
    out, gq = torch.zeros_like(q), torch.zeros_like(q)
    gk, gv = torch.zeros_like(k), torch.zeros_like(v)
    gtable = torch.zeros(h, max(nb, 1), dtype=torch.float64, device=dev)
    for j in range(h):
        by_pair = torch.zeros(nq, nk, dtype=torch.float64, device=dev)
        for i in range(b):
            n = nk if s["lengths"] is None else int(s["lengths"][i])
            if n == 0:
                continue
            kk, vv = k[i, j // group, :n], v[i, j // group, :n]
            logits = scale * torch.mm(q[i, j], kk.t()) + s["key_bias"].double()[:n]
            if nb:
                index = s["buckets"] if case["shared"] else s["buckets"][i]
                index = index[:, :n].long()
                logits = torch.where(index < 0, torch.full_like(logits, -math.inf), logits + s["table"][j].double()[index.clamp(min=0)])
            top = torch.logsumexp(logits, -1, keepdim=True)
            p = torch.where(torch.isfinite(top), torch.exp(logits - top), torch.zeros_like(logits))
            out[i, j] = torch.mm(p, vv)
            if not case["train"]:
                continue
            dp = torch.mm(g[i, j], vv.t())
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            gq[i, j] = scale * torch.mm(ds, kk)
            gk[i, j // group, :n] += scale * torch.mm(ds.t(), q[i, j])
            gv[i, j // group, :n] += torch.mm(p.t(), g[i, j])
            if nb and case["shared"]:
                by_pair[:, :n] += ds
            elif nb:
                gtable[j] += torch.stack([ds[index == t].sum() for t in range(nb)])
        if nb and case["train"] and case["shared"]:
            gtable[j] = torch.stack([by_pair[s["buckets"] == t].sum() for t in range(nb)])
    if not case["train"]:
        return {"out": out}
    result = {"out": out, "gq": gq, "gk": gk, "gv": gv}
    if nb:
        result["gtable"] = gtable
    return result
