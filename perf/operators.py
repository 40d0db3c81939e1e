"""What the operators of a language-model head cost: layer norm, the 8-bit block-scaled product, log probabilities, AdamW.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes what a program has in hand before the
call, ``run()`` is one pass.  With ``own`` false ``run()`` computes the plain form (elementary torch operations in 32 bits, rounded
once); with ``own`` true it calls this package's kernels.  ``exact()`` gives the same outputs from the definition in 64 bits.
"""
import math
import random

import torch
import torch.nn.functional as F

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CODE, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
TILE = 128              # elements of the reduction that share a scale in the product
STATE_BLOCK = 256       # elements of a tensor that share a scale in an 8-bit optimizer state


# ---------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decoded token of a few streams: the latency of the smallest call
        {"name": "norm_token", "op": "norm", "rows": 4, "cols": 512, "dtype": "bf16", "wtype": "f32", "residual": True, "train": False},
        # a ragged batch in 32 bits, odd width, forward and backward
        {"name": "norm_train_ragged", "op": "norm", "rows": 2565, "cols": 1001, "dtype": "f32", "wtype": "f32", "residual": False, "train": True},
        # a training batch with the residual stream, forward and backward
        {"name": "norm_train_wide", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "wtype": "bf16", "residual": True, "train": True},
        # three decoded tokens through a wide layer: the weights are read once
        {"name": "product_token", "op": "product", "m": 3, "n": 16384, "k": 8192, "out": "bf16", "b_rows": False, "bias": True},
        # a ragged prompt, none of the sizes a multiple of a tile
        {"name": "product_ragged", "op": "product", "m": 1037, "n": 2057, "k": 1900, "out": "f32", "b_rows": True, "bias": False},
        # a long prompt through a square layer: the matrix cores are the limit
        {"name": "product_wide", "op": "product", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "b_rows": False, "bias": False},
        # a linear layer's training step: quantising both ways, the product and both of its gradients
        {"name": "linear_train", "op": "linear", "m": 8192, "n": 4096, "k": 4096, "dtype": "bf16"},
        # eight decoded tokens over a long vocabulary with alternatives
        {"name": "probs_token", "op": "probs", "outer": 8, "classes": 128000, "inner": 1, "dtype": "bf16", "top": 8, "train": False, "masked": True},
        # a training batch over an odd vocabulary, forward and backward, policy gradient and entropy bonus
        {"name": "probs_train", "op": "probs", "outer": 4096, "classes": 50257, "inner": 1, "dtype": "bf16", "top": 0, "train": True, "masked": False},
        # label maps of five agents' frames (11 classes, class dimension 1) with the runner-up of every pixel
        {"name": "probs_pixels", "op": "probs", "outer": 20, "classes": 11, "inner": 262144, "dtype": "f32", "top": 2, "train": True, "masked": False},
        # a small network's many tensors, states in 32 bits, gradients clipped to a norm
        {"name": "adamw_small", "op": "adamw", "tensors": 62, "elements": 2000000, "dtype": "f32", "bits": 32, "clip": True},
        # a large model's tensors, states in 8 bits
        {"name": "adamw_large_8bit", "op": "adamw", "tensors": 24, "elements": 134217728, "dtype": "f32", "bits": 8, "clip": False},
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["norm", "product", "linear", "probs", "probs", "adamw"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "norm":
        cols = _spread(rng, 16, 20000)
        rows = _spread(rng, 1, max(1, min(16384, 33554432 // cols)))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "wtype": rng.choice(["f32", dtype]),
                "residual": rng.random() < 0.5, "train": rng.random() < 0.6}
    if op == "product":
        return {"op": op, "m": _spread(rng, 1, 8192), "n": _spread(rng, 1, 8192), "k": _spread(rng, 16, 8192),
                "out": dtype, "b_rows": rng.random() < 0.3, "bias": rng.random() < 0.5}
    if op == "linear":
        return {"op": op, "m": _spread(rng, 1, 8192), "n": _spread(rng, 16, 4096), "k": _spread(rng, 16, 4096), "dtype": dtype}
    if op == "probs":
        top = rng.choice([0, 1, 2, 5, 8, 20])
        if rng.random() < 0.3:
            classes = rng.randint(max(2, top), 40)
            outer, inner = rng.randint(1, 8), _spread(rng, 2, 100000)
        else:
            classes = _spread(rng, max(2, top), 150000)
            outer, inner = _spread(rng, 1, max(1, min(8192, 134217728 // classes))), 1
        return {"op": op, "outer": outer, "classes": classes, "inner": inner, "dtype": dtype, "top": top,
                "train": rng.random() < 0.5, "masked": rng.random() < 0.4}
    return {"op": op, "tensors": rng.randint(1, 120), "elements": _spread(rng, 1000, 67108864), "dtype": dtype,
            "bits": rng.choice([8, 32]), "clip": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------- the inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _power_of_two(e):
    return (e + 127).clamp(0, 254).to(torch.uint8).view(SCALE)


def _exponent(amax, largest=448.0):
    """the smallest e with amax <= largest * 2^e; 0 for a block of zeros"""
    bits = amax.float().view(torch.int32)
    top = torch.tensor(largest, device=amax.device).view(torch.int32)
    e = (bits >> 23) - (top >> 23) + ((bits & 0x7FFFFF) > (top & 0x7FFFFF)).int()
    return torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e))


def _quantize(x, tile_rows):
    """f32 [R, C] -> (codes [R, C up to a multiple of 128], scales [R or R/128 rounded up, C/128 rounded up])"""
    R, C = x.shape
    pr, pc = (-R % tile_rows), (-C % TILE)
    t = F.pad(x, (0, pc, 0, pr)).view((R + pr) // tile_rows, tile_rows, (C + pc) // TILE, TILE)
    e = _exponent(t.abs().amax(dim=(1, 3)))
    codes = torch.ldexp(t, -e[:, None, :, None]).to(CODE).view(R + pr, C + pc)[:R]
    return codes.contiguous(), _power_of_two(e)


def _held(codes, scale, tile_rows):
    """what codes and scales stand for, f32"""
    R, C = codes.shape
    s = scale.float().repeat_interleave(tile_rows, 0)[:R].repeat_interleave(TILE, 1)
    return codes.float() * s


def _numels(tensors, elements):
    """the same mix of matrices and vectors for one (tensors, elements): every third tensor holds most of them"""
    r = random.Random(tensors * 7919 + elements)
    w = [math.exp(r.uniform(0.0, 1.5)) * (1.0 if i % 3 == 0 else 0.002) for i in range(tensors)]
    return [max(1, round(elements * v / sum(w))) for v in w]


def _prepare_norm(c, g):
    dt, wt = DTYPES[c["dtype"]], DTYPES[c["wtype"]]
    shape = (c["rows"], c["cols"])
    s = {"x": _normal(g, shape, dt, 1.5, 0.5), "w": _normal(g, c["cols"], wt, 0.2, 1.0), "b": _normal(g, c["cols"], wt, 0.2), "eps": 1e-5}
    if c["residual"]:
        s["r"] = _normal(g, shape, dt)
    if c["train"]:
        s["dy"] = _normal(g, shape, dt)
        if c["residual"]:
            s["dh"] = _normal(g, shape, dt)
    return s


def _prepare_product(c, g):
    x = _normal(g, (c["m"], c["k"])) * torch.exp(_normal(g, (c["m"], 1)))
    w = _normal(g, (c["n"], c["k"]), scale=c["k"] ** -0.5)
    a, sa = _quantize(x, 1)
    b, sb = _quantize(w, 1 if c["b_rows"] else TILE)
    return {"a": a, "sa": sa, "b": b, "sb": sb, "bias": _normal(g, c["n"]) if c["bias"] else None}


def _prepare_linear(c, g):
    dt = DTYPES[c["dtype"]]
    return {"x": _normal(g, (c["m"], c["k"]), dt).requires_grad_(), "w": _normal(g, (c["n"], c["k"]), scale=c["k"] ** -0.5).requires_grad_(),
            "b": _normal(g, c["n"]).requires_grad_(), "dy": _normal(g, (c["m"], c["n"]), dt)}


def _prepare_probs(c, g):
    shape = (c["outer"], c["classes"]) + ((c["inner"],) if c["inner"] > 1 else ())
    rest = shape[:1] + shape[2:]
    x = _normal(g, shape, DTYPES[c["dtype"]], 2.5)
    if c["masked"]:
        x.masked_fill_(torch.rand(shape, generator=g, device="cuda") < 0.3, -math.inf)
    t = torch.randint(0, c["classes"], rest, generator=g, device="cuda")
    t.masked_fill_(torch.rand(rest, generator=g, device="cuda") < 0.1, -100)
    s = {"x": x, "target": t}
    if c["train"]:
        s["g_logp"], s["g_entropy"] = _normal(g, rest), _normal(g, rest, scale=0.1)
        s["g_top"] = _normal(g, rest + (c["top"],)) if c["top"] else None
    return s


def _prepare_adamw(c, g):
    sizes = _numels(c["tensors"], c["elements"])
    places, at = [], 0
    for n in sizes:
        places.append((at, n))
        at += -(-n // STATE_BLOCK) * STATE_BLOCK
    dt = DTYPES[c["dtype"]]
    cut = lambda flat: [flat[o:o + n] for o, n in places]                       # noqa: E731
    inside = torch.zeros(at, device="cuda")
    for t in cut(inside):
        t.fill_(1.0)
    s = {"p_all": (_normal(g, at, scale=0.5) * inside).to(dt), "g_all": (_normal(g, at, scale=0.02) * inside).to(dt),
         "step_all": torch.full((len(sizes),), 9.0, device="cuda"), "sizes": sizes}
    m = _normal(g, at, scale=0.01) * inside
    v = (torch.rand(at, generator=g, device="cuda") * 4e-4 + 1e-6) * inside
    if c["bits"] == 8:
        em, ev = _exponent(m.view(-1, STATE_BLOCK).abs().amax(1)), _exponent(v.sqrt().view(-1, STATE_BLOCK).amax(1))
        s["m_all"] = torch.ldexp(m.view(-1, STATE_BLOCK), -em[:, None]).to(CODE).view(-1)
        s["v_all"] = torch.ldexp(v.sqrt().view(-1, STATE_BLOCK), -ev[:, None]).to(CODE).view(-1)
        s["ms_all"], s["vs_all"] = _power_of_two(em), _power_of_two(ev)
        s["ms"] = [s["ms_all"][o // STATE_BLOCK:-(-(o + n) // STATE_BLOCK)] for o, n in places]
        s["vs"] = [s["vs_all"][o // STATE_BLOCK:-(-(o + n) // STATE_BLOCK)] for o, n in places]
    else:
        s["m_all"], s["v_all"] = m, v
    s["p"], s["g"], s["m"], s["v"] = cut(s["p_all"]), cut(s["g_all"]), cut(s["m_all"]), cut(s["v_all"])
    s["step"] = list(s["step_all"].unbind())
    s["hyper"] = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01, "max_norm": 1.0 if c["clip"] else None}
    s["seed"] = 1234567
    return s


_PREPARE = {"norm": _prepare_norm, "product": _prepare_product, "linear": _prepare_linear, "probs": _prepare_probs, "adamw": _prepare_adamw}


def prepare(case, seed):
    s = _PREPARE[case["op"]](case, _generator(seed))
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------------------------------------- the plain forms

def _plain_norm(c, s):
    x = s["x"]
    h = (x.float() + s["r"].float()).to(x.dtype) if c["residual"] else x
    hf = h.float()
    mean = hf.mean(1, keepdim=True)
    d = hf - mean
    rstd = ((d * d).mean(1, keepdim=True) + s["eps"]).rsqrt()
    n = d * rstd
    out = {"y": (n * s["w"].float() + s["b"].float()).to(x.dtype)}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        dy = s["dy"].float()
        dn = dy * s["w"].float()
        dx = (dn - dn.mean(1, keepdim=True) - n * (dn * n).mean(1, keepdim=True)) * rstd
        if c["residual"]:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(x.dtype)
        out["dw"], out["db"] = (dy * n).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)
    return out


def _plain_product(c, s):
    y = _held(s["a"], s["sa"], 1) @ _held(s["b"], s["sb"], 1 if c["b_rows"] else TILE).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[c["out"]])


def _plain_linear(c, s):
    x, w, dy = s["x"].detach().float(), s["w"].detach(), s["dy"].float()
    wq = _held(*_quantize(w, TILE), TILE)[:, :c["k"]]
    y = _held(*_quantize(x, 1), 1)[:, :c["k"]] @ wq.t() + s["b"].detach()
    dx = _held(*_quantize(dy, 1), 1)[:, :c["n"]] @ wq
    dw = _held(*_quantize(dy.t().contiguous(), 1), 1) @ _held(*_quantize(x.t().contiguous(), 1), 1).t()
    return {"y": y.to(s["x"].dtype), "dx": dx.to(s["x"].dtype), "dw": dw, "db": dy.sum(0)}


def _plain_probs(c, s):
    x, t = s["x"].float(), s["target"]
    m = x.amax(1, keepdim=True)
    empty = m == -math.inf
    m = m.masked_fill(empty, 0.0)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    logs = torch.log(total)
    p = e / total.masked_fill(empty, 1.0)
    log_p = (x - m - logs).masked_fill(empty, -math.inf)
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(1, keepdim=True)
    keep = t != -100
    at = t.clamp_min(0).unsqueeze(1)
    out = {"logp": torch.where(keep, log_p.gather(1, at).squeeze(1), torch.zeros_like(keep, dtype=torch.float32)), "entropy": entropy.squeeze(1)}
    places = []
    if c["top"]:
        shape = [1, c["classes"]] + [1] * (x.dim() - 2)
        iota = torch.arange(c["classes"], device=x.device).view(shape)
        taken = torch.zeros_like(x, dtype=torch.bool)
        for _ in range(c["top"]):
            best = x.masked_fill(taken, -math.inf).amax(1, keepdim=True)
            place = torch.where((x == best) & ~taken, iota, c["classes"]).amin(1, keepdim=True)
            taken.scatter_(1, place, True)
            places.append(place)
        out["top_logp"] = torch.stack([log_p.gather(1, q).squeeze(1) for q in places], -1)
        out["top_index"] = torch.stack([q.squeeze(1) for q in places], -1)
    if c["train"]:
        g = (s["g_logp"] * keep).unsqueeze(1)
        each = torch.zeros_like(x).scatter_(1, at, g)
        whole = g
        for i, q in enumerate(places):
            gi = s["g_top"][..., i].unsqueeze(1)
            each.scatter_add_(1, q, gi)
            whole = whole + gi
        dx = each - p * whole - torch.where(p > 0, s["g_entropy"].unsqueeze(1) * p * (log_p + entropy), torch.zeros_like(p))
        out["dx"] = dx.masked_fill(empty, 0.0).to(s["x"].dtype)
    return out


def _dither(n, seed, step, device):
    """32 random bits for each element: a hash of (seed, step, place), every product modulo 2^32"""
    low = 0xFFFFFFFF
    i = torch.arange(n, device=device, dtype=torch.int64)
    key = (seed * 0x9E3779B1 + step.long() * 0x85EBCA6B) & low
    x = ((i & low) * 0xA3D8F62B + (i >> 32) * 0xC2B2AE35 + key) & low
    x = ((x ^ (x >> 15)) * 0xC58B3E95) & low
    x = ((x ^ (x >> 13)) * 0x9E3779B1) & low
    return x ^ (x >> 16)


def _encode(x, noise, positive):
    """f32 [n] and 20 random bits each -> e4m3 codes and block scales; a positive value keeps a positive code"""
    n = x.numel()
    t = F.pad(x, (0, -n % STATE_BLOCK)).view(-1, STATE_BLOCK)
    e = _exponent(t.abs().amax(1))
    t = torch.ldexp(t, -e[:, None]).view(-1)[:n]
    bits = (t.abs() * 2.0 ** -120).view(torch.int32)
    code = ((bits + noise.int()) >> 20).clamp(max=126)
    if positive:
        code = torch.where(t > 0, code.clamp(min=1), code)
    return torch.where(t < 0, code + 128, code).to(torch.uint8).view(CODE), _power_of_two(e)


def _state(codes, scale):
    return codes.float() * scale.float().repeat_interleave(STATE_BLOCK)[:codes.numel()]


def _plain_adamw(c, s):
    hp = s["hyper"]
    out, factor = {}, 1.0
    if c["clip"]:
        total = torch.stack([t.double().square().sum() for t in s["g"]]).sum().sqrt()
        out["norm"] = total.float()
        factor = (hp["max_norm"] / (total + 1e-6)).clamp(max=1.0).float()
    s["step_all"].add_(1.0)
    t = s["step_all"].double()
    bias1, bias2 = (1.0 - hp["beta1"] ** t).float(), (1.0 - hp["beta2"] ** t).sqrt().float()
    for i, p in enumerate(s["p"]):
        g, pf = s["g"][i].float() * factor, p.float()
        if c["bits"] == 8:
            m, root = _state(s["m"][i], s["ms"][i]), _state(s["v"][i], s["vs"][i])
            v = root * root
        else:
            m, v = s["m"][i], s["v"][i]
        m = hp["beta1"] * m + (1.0 - hp["beta1"]) * g
        v = hp["beta2"] * v + (1.0 - hp["beta2"]) * (g * g)
        root = v.sqrt()
        pf = pf * (1.0 - hp["lr"] * hp["weight_decay"]) - (hp["lr"] / bias1[i]) * (m / (root / bias2[i] + hp["eps"]))
        p.copy_(pf)
        if c["bits"] == 8:
            noise = _dither(p.numel(), s["seed"], s["step_all"][i], p.device)
            for x, code, scale, bits, positive in ((m, s["m"][i], s["ms"][i], ((noise & 0xFFFF) << 4) + 8, False),
                                                   (root, s["v"][i], s["vs"][i], ((noise >> 16) << 4) + 8, True)):
                new, new_scale = _encode(x, bits, positive)
                code.copy_(new)
                scale.copy_(new_scale)
        else:
            s["m"][i].copy_(m)
            s["v"][i].copy_(v)
    return _adamw_outputs(c, s, out)


def _adamw_outputs(c, s, out):
    out.update(p=s["p_all"], m=s["m_all"], v=s["v_all"], step=s["step_all"])
    if c["bits"] == 8:
        out.update(m_scale=s["ms_all"], v_scale=s["vs_all"])
    return out


_PLAIN = {"norm": _plain_norm, "product": _plain_product, "linear": _plain_linear, "probs": _plain_probs, "adamw": _plain_adamw}


# ---------------------------------------------------------------------------------------------------------------- the package's calls

def _own_norm(c, s):
    from multiagentperception_amd import ops
    y, h, mean, rstd = ops.layer_norm_forward(s["x"], s["w"], s["b"], s["eps"], residual=s.get("r"))
    out = {"y": y}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        out["dx"], out["dw"], out["db"] = ops.layer_norm_backward(s["dy"], h, s["w"], mean, rstd, dh=s.get("dh"))
    return out


def _own_product(c, s):
    from multiagentperception_amd import ops
    return ops.matmul_fp8(ops.Fp8Blocks(s["a"], s["sa"], c["k"]), ops.Fp8Blocks(s["b"], s["sb"], c["k"]), bias=s["bias"], out_dtype=DTYPES[c["out"]])


def _own_linear(c, s):
    from multiagentperception_amd import train_ops
    y = train_ops.linear_fp8(s["x"], s["w"], s["b"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _own_probs(c, s):
    from multiagentperception_amd import ops
    r = ops.log_probs_forward(s["x"], s["target"], top=c["top"], dim=1, ignore_index=-100)
    out = {"logp": r.logp, "entropy": r.entropy}
    if c["top"]:
        out["top_logp"], out["top_index"] = r.top_logp, r.top_index
    if c["train"]:
        out["dx"] = ops.log_probs_backward(s["x"], s["target"], r, g_logp=s["g_logp"], g_entropy=s["g_entropy"], g_top=s["g_top"], dim=1, ignore_index=-100)
    return out


def _own_adamw(c, s):
    from multiagentperception_amd import ops
    states = list(zip(s["m"], s["ms"], s["v"], s["vs"])) if c["bits"] == 8 else list(zip(s["m"], s["v"]))
    norm = ops.adamw_step(s["p"], s["g"], states, s["step"], seed=s["seed"], **s["hyper"])
    return _adamw_outputs(c, s, {"norm": norm} if c["clip"] else {})


_OWN = {"norm": _own_norm, "product": _own_product, "linear": _own_linear, "probs": _own_probs, "adamw": _own_adamw}


def run(state):
    c = state["case"]
    if own:
        return _OWN[c["op"]](c, state)
    with torch.no_grad():
        return _PLAIN[c["op"]](c, state)


# ---------------------------------------------------------------------------------------------------------------- the work

def work(c):
    if c["op"] == "norm":
        n, b = c["rows"] * c["cols"], BYTES[c["dtype"]]
        passes = (2 + 2 * c["residual"]) + (3 + c["residual"] if c["train"] else 0)
        return {"bytes": n * b * passes + c["cols"] * BYTES[c["wtype"]] * (4 if c["train"] else 2), "flops": n * (8 + (14 if c["train"] else 0))}
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": (m + n) * k + m * n * BYTES[c["out"]] + (m + (n if c["b_rows"] else n / TILE)) * k / TILE, "flops": 2 * m * n * k}
    if c["op"] == "linear":
        m, n, k, b = c["m"], c["n"], c["k"], BYTES[c["dtype"]]
        return {"bytes": 2 * m * (k + n) * b + 2 * n * k * 4 + 2 * n * 4, "flops": 6 * m * n * k}
    if c["op"] == "probs":
        rows, b = c["outer"] * c["inner"], BYTES[c["dtype"]]
        n = rows * c["classes"]
        each = 8 + 4 + 4 + 12 * c["top"] + ((8 + 4 * c["top"]) if c["train"] else 0)
        return {"bytes": n * b * (2 if c["train"] else 1) + rows * each, "flops": n * (6 + (8 if c["train"] else 0))}
    n, b = sum(_numels(c["tensors"], c["elements"])), BYTES[c["dtype"]]
    state = 16 if c["bits"] == 32 else 4 + 4 / STATE_BLOCK
    return {"bytes": n * (3 * b + state), "flops": n * 16}


# ---------------------------------------------------------------------------------------------------------------- 64 bits

def _exact_norm(c, s):
    f = lambda k: s[k].double()                                                  # noqa: E731
    h = f("x")
    if c["residual"]:
        h = (h + f("r")).to(s["x"].dtype).double()
    var, mean = torch.var_mean(h, dim=-1, unbiased=False, keepdim=True)
    sigma = torch.sqrt(var + s["eps"])
    xhat = (h - mean) / sigma
    out = {"y": f("w") * xhat + f("b")}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        up = f("dy") * f("w")
        D = c["cols"]
        dx = (D * up - up.sum(-1, keepdim=True) - xhat * (up * xhat).sum(-1, keepdim=True)) / (D * sigma)
        out["dx"] = dx + f("dh") if c["residual"] else dx
        out["dw"], out["db"] = torch.einsum("rc,rc->c", f("dy"), xhat), f("dy").sum(0)
    return out


def _values64(codes, scale):
    """codes and scales to the numbers they stand for, in 64 bits, by the codes' own fields"""
    table = torch.arange(256, device=codes.device)
    ex, man = (table >> 3) & 15, (table & 7).double()
    mag = torch.where(ex > 0, (1 + man / 8) * 2.0 ** (ex.double() - 7), man * 2.0 ** -9)
    table = torch.where(table >= 128, -mag, mag)
    v = table[codes.contiguous().view(torch.uint8).long()]
    p = 2.0 ** (scale.contiguous().view(torch.uint8).double() - 127)
    R, C = codes.shape
    each = -(-R // scale.shape[0]) if scale.shape[0] != R else 1
    each = TILE if each > 1 or (scale.shape[0] == 1 and R > 1) else 1
    rows, cols = torch.arange(R, device=codes.device) // each, torch.arange(C, device=codes.device) // TILE
    return v * p[rows][:, cols]


def _exact_product(c, s):
    y = torch.matmul(_values64(s["a"], s["sa"]), _values64(s["b"], s["sb"]).t().contiguous())
    return y if s["bias"] is None else y + s["bias"].double()


def _rounded64(x, tile_rows):
    """x (64 bits) to the nearest e4m3 multiples of its tiles' powers of two, ties to even"""
    R, C = x.shape
    rows, cols = torch.arange(R, device=x.device) // tile_rows, torch.arange(C, device=x.device) // TILE
    nr, nc = int(rows[-1]) + 1, int(cols[-1]) + 1
    tile = rows[:, None] * nc + cols[None, :]
    amax = torch.zeros(nr * nc, dtype=torch.float64, device=x.device).scatter_reduce_(0, tile.view(-1), x.abs().reshape(-1), "amax")
    e = torch.where(amax > 0, torch.ceil(torch.log2(amax / 448.0)), torch.zeros_like(amax))
    e = torch.where(amax > 448.0 * 2.0 ** e, e + 1, torch.where((amax > 0) & (amax <= 224.0 * 2.0 ** e), e - 1, e))
    unit = (2.0 ** e)[tile]
    u = x / unit
    _, k = torch.frexp(u)
    step = 2.0 ** (torch.clamp(k - 1, min=-6).double() - 3)
    return torch.round(u / step) * step * unit


def _exact_linear(c, s):
    x, w, dy = s["x"].detach().double(), s["w"].detach().double(), s["dy"].double()
    wq = _rounded64(w, TILE)
    return {"y": torch.matmul(_rounded64(x, 1), wq.t().contiguous()) + s["b"].detach().double(), "dx": torch.matmul(_rounded64(dy, 1), wq),
            "dw": torch.matmul(_rounded64(dy.t().contiguous(), 1), _rounded64(x.t().contiguous(), 1).t().contiguous()), "db": dy.sum(0)}


def _exact_probs(c, s):
    x, t = s["x"].double(), s["target"]
    lse = torch.logsumexp(x, 1, keepdim=True)
    empty = torch.isneginf(lse)
    lp = torch.where(empty, torch.full_like(x, -math.inf), x - torch.where(empty, torch.zeros_like(lse), lse))
    p = torch.exp(lp)
    H = (p * torch.where(p > 0, -lp, torch.zeros_like(lp))).sum(1)
    used = t >= 0
    lt = torch.gather(lp, 1, torch.where(used, t, torch.zeros_like(t)).unsqueeze(1))[:, 0]
    out = {"logp": torch.where(used, lt, torch.zeros_like(lt)), "entropy": H}
    top = None
    if c["top"]:
        top = torch.sort(x, dim=1, descending=True, stable=True)[1].narrow(1, 0, c["top"])
        out["top_logp"] = torch.gather(lp, 1, top).movedim(1, -1)
        out["top_index"] = top.movedim(1, -1).contiguous()
    if c["train"]:
        gl = torch.where(used, s["g_logp"].double(), torch.zeros_like(lt)).unsqueeze(1)
        d = -p * gl
        d.scatter_add_(1, torch.where(used, t, torch.zeros_like(t)).unsqueeze(1), gl)
        if c["top"]:
            gt = s["g_top"].double().movedim(-1, 1)
            d = (d - p * gt.sum(1, keepdim=True)).scatter_add(1, top, gt)
        d = d - s["g_entropy"].double().unsqueeze(1) * torch.where(p > 0, p * (lp + H.unsqueeze(1)), torch.zeros_like(p))
        out["dx"] = torch.where(empty, torch.zeros_like(d), d)
    return out


def _blocked64(x, noise, positive):
    """x (64 bits, [n]) rounded by the noise in [0, 1) to e4m3 multiples of its blocks' powers of two: (codes' values, scales)"""
    n = x.numel()
    t = torch.cat([x, x.new_zeros(-n % STATE_BLOCK)]).view(-1, STATE_BLOCK)
    top = t.float().abs().amax(1).double()                    # the scale belongs to the value in 32 bits that the block holds
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448.0)), torch.zeros_like(top))
    e = torch.where(top > 448.0 * 2.0 ** e, e + 1, torch.where((top > 0) & (top <= 224.0 * 2.0 ** e), e - 1, e))
    u = (t / (2.0 ** e)[:, None]).view(-1)[:n]
    _, k = torch.frexp(u)
    step = 2.0 ** (torch.clamp(k - 1, min=-6).double() - 3)
    q = torch.floor(u.abs() / step + noise) * step
    q = torch.clamp(q, max=448.0)
    if positive:
        q = torch.where(u > 0, torch.clamp(q, min=2.0 ** -9), q)
    return q * torch.sign(u), 2.0 ** e


def _exact_adamw(c, s):
    hp = s["hyper"]
    b1, b2 = hp["beta1"], hp["beta2"]
    out, factor = {}, 1.0
    if c["clip"]:
        norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in s["g"]))
        out["norm"] = norm
        factor = min(1.0, hp["max_norm"] / (norm + 1e-6))
    P, M, V = s["p_all"].double(), s["m_all"].double(), s["v_all"].double()
    MS, VS = (s["ms_all"].double(), s["vs_all"].double()) if c["bits"] == 8 else (None, None)
    at = 0
    for i, n in enumerate(s["sizes"]):
        t = float(s["step"][i]) + 1.0
        g, m, v = s["g"][i].double() * factor, M[at:at + n], V[at:at + n]
        blocks = slice(at // STATE_BLOCK, -(-(at + n) // STATE_BLOCK))
        if c["bits"] == 8:
            of = torch.arange(n, device=g.device) // STATE_BLOCK
            m, v = m * MS[blocks][of], (v * VS[blocks][of]) ** 2
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        P[at:at + n] = P[at:at + n] * (1 - hp["lr"] * hp["weight_decay"]) - hp["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + hp["eps"])
        if c["bits"] == 8:
            r = _dither(n, s["seed"], s["step"][i] + 1.0, g.device)
            M[at:at + n], MS[blocks] = _blocked64(m, ((r % 65536).double() + 0.5) / 65536, False)
            V[at:at + n], VS[blocks] = _blocked64(torch.sqrt(v), ((r // 65536).double() + 0.5) / 65536, True)
        else:
            M[at:at + n], V[at:at + n] = m, v
        at += -(-n // STATE_BLOCK) * STATE_BLOCK
    out.update(p=P, m=M, v=V, step=s["step_all"].double() + 1.0)
    if c["bits"] == 8:
        out.update(m_scale=MS, v_scale=VS)
    return out


_EXACT = {"norm": _exact_norm, "product": _exact_product, "linear": _exact_linear, "probs": _exact_probs, "adamw": _exact_adamw}


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["op"]](case, prepare(case, seed))
