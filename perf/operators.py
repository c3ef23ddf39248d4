"""Cases of three operators of a transformer's training step on long sequences, with their plain forms.

adamw       clipping by the global gradient norm and one AdamW step over a whole list of parameters, with the two moments
            held in 32 bits or in 8 bits (one byte a value and a scale for each block of 256 values)
gated_norm  the norm of a block's output, its gate and residual scale, the residual sum and the norm in front of the next
            block, forward and backward
window      attention that sees a window of keys around the query and a few first keys, forward and backward, and the form for
            single tokens that reads a cache

`own` chooses between the plain form (elementary torch operations in 32 bits) and the calls of probtalk_amd.train_ops.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 256                       # values that share a scale
M_BITS, V_BITS = 3, 4             # mantissa bits of a first / second moment's code; both have four exponent bits
TOP_M, TOP_V = 15 * 2 ** 14, 31 * 2 ** 14


def _up(n, m):
    return (n + m - 1) // m * m


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the parameters of one LayerNorm and its Linear's bias: a call that is all latency
        {"name": "adamw 32 one norm", "op": "adamw", "sizes": "norm", "elements": 0, "tensors": 3, "bits": 32, "dtype": "fp32"},
        # the whole 512-wide motion transformer: 6 decoder layers with their style blocks, embeddings and heads
        {"name": "adamw 32 decoder", "op": "adamw", "sizes": "decoder", "elements": 0, "tensors": 0, "bits": 32, "dtype": "fp32"},
        # the same parameters with the moments in a byte each
        {"name": "adamw 8 decoder", "op": "adamw", "sizes": "decoder", "elements": 0, "tensors": 0, "bits": 8, "dtype": "fp32"},
        # a larger model held in bf16: ragged tensors, as the embeddings and heads of odd vocabularies give
        {"name": "adamw 8 bf16 160M", "op": "adamw", "sizes": "ragged", "elements": 160_000_000, "tensors": 310, "bits": 8, "dtype": "bf16"},
        # one clip's 44 tokens while sampling
        {"name": "norm fp32 one clip", "op": "gated_norm", "rows": 44, "per_clip": 44, "cols": 512, "kind": "layer", "bias": True, "grad": False, "dtype": "fp32"},
        # the bench batch of the motion transformer, in training: 512 clips of 88 tokens, 512 wide
        {"name": "norm fp32 train", "op": "gated_norm", "rows": 512 * 88, "per_clip": 88, "cols": 512, "kind": "layer", "bias": True, "grad": True, "dtype": "fp32"},
        # a wide model's prompt, forward only; one gate for all rows
        {"name": "norm bf16 forward", "op": "gated_norm", "rows": 49_152, "per_clip": 49_152, "cols": 2048, "kind": "rms", "bias": False, "grad": False, "dtype": "bf16"},
        # a wide model in training
        {"name": "norm bf16 train", "op": "gated_norm", "rows": 16_384, "per_clip": 4096, "cols": 4096, "kind": "rms", "bias": False, "grad": True, "dtype": "bf16"},
        # one sequence being generated, 8 heads of 64
        {"name": "step one sequence", "op": "step", "batch": 1, "keys": 1500, "heads": 8, "kv_heads": 8, "dim": 64, "left": 511, "sinks": 4, "ragged": False, "dtype": "bf16"},
        # a full serving batch over a long cache, grouped heads, sequences of all lengths
        {"name": "step serving batch", "op": "step", "batch": 64, "keys": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "left": 4095, "sinks": 4, "ragged": True, "dtype": "bf16"},
        # whole utterances through the motion transformer's 8 heads of 64: both directions visible, padded to the longest
        {"name": "window fp32 train", "op": "window", "batch": 4, "rows": 1200, "heads": 8, "kv_heads": 8, "dim": 64, "left": 128, "right": 128, "sinks": 0, "ragged": True, "grad": True, "dtype": "fp32"},
        # a long sequence in training, causal, grouped heads
        {"name": "window bf16 train", "op": "window", "batch": 1, "rows": 8192, "heads": 16, "kv_heads": 4, "dim": 128, "left": 1023, "right": 0, "sinks": 4, "ragged": False, "grad": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adamw", "gated_norm", "step", "window"])
    if op == "adamw":
        tensors = _log(rng, 1, 400)
        return {"op": op, "sizes": "ragged", "elements": _log(rng, 50 * tensors, 120_000_000), "tensors": tensors, "bits": rng.choice([32, 8]),
                "dtype": rng.choice(["fp32", "bf16"])}
    if op == "gated_norm":
        cols = rng.choice([64, 512, 1024, _log(rng, 33, 8192), _log(rng, 33, 8192)])
        rows = _log(rng, 1, max(1, min(65_536, 60_000_000 // cols)))
        per = min(rows, rng.choice([1, rows, _log(rng, 1, rows)]))
        return {"op": op, "rows": rows // per * per, "per_clip": per, "cols": cols, "kind": rng.choice(["layer", "rms"]), "bias": rng.random() < 0.5,
                "grad": rng.random() < 0.6, "dtype": rng.choice(["fp32", "bf16"])}
    kv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 64, 80, 96, 128, 128])
    if op == "step":
        keys = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(128, 60 * 8192 * 8 * 128 // (keys * kv * dim))))
        return {"op": op, "batch": batch, "keys": keys, "heads": kv * group, "kv_heads": kv, "dim": dim, "left": _log(rng, 1, 4096), "sinks": rng.choice([0, 1, 4, 16]),
                "ragged": rng.random() < 0.7, "dtype": rng.choice(["fp32", "bf16", "bf16"])}
    dtype = rng.choice(["fp32", "bf16", "bf16"])
    rows = _log(rng, 1, 8192 if dtype == "bf16" else 2500)
    most = 16 * 8192 * 8192 if dtype == "bf16" else 8 * 2500 * 2500
    group = min(group, max(1, most // (kv * rows * rows)))
    kv = min(kv, max(1, most // (group * rows * rows)))
    batch = _log(rng, 1, max(1, min(32, most // (kv * group * rows * rows))))
    left = _log(rng, 1, 1024 if dtype == "bf16" else 256)
    return {"op": op, "batch": batch, "rows": rows, "heads": kv * group, "kv_heads": kv, "dim": dim, "left": left, "right": rng.choice([0, 0, left]),
            "sinks": rng.choice([0, 1, 4, 16]), "ragged": rng.random() < 0.5, "grad": rng.random() < 0.7, "dtype": dtype}


def _sizes(case):
    """The number of values of each parameter."""
    if case["sizes"] == "norm":
        return [512, 512, 1536]
    if case["sizes"] == "decoder":
        style = [1024 * 512, 1024, 512, 512, 512 * 512, 512]
        attn = [1536 * 512, 1536, 512 * 512, 512]
        layer = attn * 2 + [2048 * 512, 2048, 512 * 2048, 512] + [512, 512] * 3 + style * 3
        return [129 * 512, 4 * 512, 512 * 768, 512, 128 * 377, 128] + layer * 6 + [512 * 512, 512, 128 * 512, 128]
    r = np.random.RandomState(case["elements"] % 65_521 + case["tensors"])
    w = np.exp(1.5 * r.standard_normal(case["tensors"]))
    n = np.maximum(1, (w / w.sum() * case["elements"]).astype(np.int64))
    return [int(v) | 1 if i % 3 else int(v) for i, v in enumerate(n)]


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    s["type"] = dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, device=DEV, generator=g) * scale + shift).to(dtype)

    if case["op"] == "adamw":
        # each parameter starts at a multiple of a block inside one storage, so that whole storages can be compared; what lies
        # between two parameters is zero
        sizes = _sizes(case)
        at = np.concatenate([[0], np.cumsum([_up(n, BLOCK) for n in sizes])])
        total = int(at[-1])
        inside = torch.zeros(total, dtype=torch.bool, device=DEV)
        for a, n in zip(at, sizes):
            inside[int(a):int(a) + n] = True
        flat = {"param": normal(total, scale=0.05) * inside, "grad": normal(total, scale=1e-3) * inside}
        if case["bits"] == 32:
            flat["m"] = normal(total, scale=5e-4, dtype=torch.float32) * inside
            flat["v"] = (normal(total, scale=1e-3, dtype=torch.float32).square() * inside) * 0.5
        else:
            # codes in use: magnitudes over several octaves of the block's largest, sign in the top bit of a first moment
            flat["m"] = (torch.randint(0, 128, (total,), device=DEV, generator=g) | torch.randint(0, 2, (total,), device=DEV, generator=g) << 7).to(torch.uint8) * inside
            flat["v"] = torch.randint(40, 256, (total,), device=DEV, generator=g).to(torch.uint8) * inside
            nb = total // BLOCK
            scale = torch.rand(nb, 2, device=DEV, generator=g) + 0.5
            flat["scale"] = scale * torch.tensor([2e-3 / TOP_M, 4e-6 / TOP_V], device=DEV)
        s["flat"], s["total"] = flat, total
        s["lists"] = {k: [t[int(a):int(a) + n] for a, n in zip(at, sizes)] for k, t in flat.items() if k != "scale"}
        if case["bits"] == 8:
            s["lists"]["scale"] = [flat["scale"][int(a) // BLOCK:int(b) // BLOCK] for a, b in zip(at[:-1], at[1:])]
        s["hyper"] = {"step": 1000, "lr": 1e-4, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 1e-2}
        s["max_norm"], s["seed"] = 0.8e-3 * math.sqrt(sum(sizes)), int(seed) & 0xFFFF
        return s
    if case["op"] == "gated_norm":
        rows, cols, clips = case["rows"], case["cols"], case["rows"] // case["per_clip"]
        s["x"], s["t"] = normal(rows, cols, scale=1.5), normal(rows, cols, scale=0.7, shift=0.1)
        s["gate"] = normal(clips, cols, scale=0.3, shift=0.5)
        s["res_scale"] = normal(cols, scale=0.05, shift=0.3, dtype=torch.float32)
        for k in ("post", "pre"):
            s[k + "_weight"] = normal(cols, scale=0.1, shift=1.0, dtype=torch.float32)
            s[k + "_bias"] = normal(cols, scale=0.1, dtype=torch.float32) if case["bias"] else None
        s["leaves"] = [k for k in ("x", "t", "gate", "res_scale", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[k] is not None]
        if case["grad"]:
            s["dy"], s["dh"] = normal(rows, cols), normal(rows, cols)
            for k in s["leaves"]:
                s[k].requires_grad_()
        return s
    b, heads, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    n = case["keys"] if case["op"] == "step" else case["rows"]
    s["q"] = normal(b, heads, d, scale=1.5) if case["op"] == "step" else normal(b, n, heads, d, scale=1.5)
    s["k"], s["v"] = normal(b, n, kv, d), normal(b, n, kv, d)
    s["lengths"] = None
    if case["op"] == "step" or case["ragged"]:
        low = max(1, n // 4) if case["ragged"] else n
        s["lengths"] = torch.randint(low, n + 1, (b,), device=DEV, generator=g).to(torch.int32)
        s["lengths"][0] = n
    if case.get("grad"):
        s["do"] = normal(b, n, heads, d)
        for k in ("q", "k", "v"):
            s[k].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------------------ adamw
def _hash(c, key):
    """32 random bits of each counter, as int64."""
    x = ((c ^ key) * 0x9E3779B9) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 14)


def _key(seed, step):
    x = ((int(step) * 0x9E3779B9) ^ int(seed)) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 15)


def _value(code, mant, scale):
    """What a magnitude code stands for: below 2^mant the code itself, above it (2^mant + low bits) 2^(octave - 1), times the scale."""
    c = code.to(torch.int32)
    n = torch.where(c < 2 ** mant, c, (2 ** mant + (c & (2 ** mant - 1))) << ((c >> mant) - 1).clamp_min(0))
    return (n.to(torch.float32).view(-1, BLOCK) * scale.view(-1, 1)).view(-1)


def _code(x, mant, top, r):
    """(codes of |x|, scales): stochastic rounding with the 16 random bits r."""
    a = x.abs().view(-1, BLOCK)
    big = a.amax(1, keepdim=True)
    scale = torch.where(big < 2.0 ** -100, torch.zeros_like(big), big / torch.full_like(big, top))
    z = torch.where(scale > 0, a * torch.reciprocal(scale), torch.zeros_like(a)).clamp_max(top).view(-1)
    low = torch.floor(z + r.to(torch.float32) * 2.0 ** -16).to(torch.int64)
    high = ((z.view(torch.int32).to(torch.int64) + (r << (7 - mant))) >> (23 - mant)) - ((126 + mant) << mant)
    return torch.where(z < 2 ** mant, low, high), z, scale.view(-1)


def _adamw_plain(s):
    f, h, bits = s["flat"], s["hyper"], s["bits"]
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    b1, b2 = f32(h["betas"][0]), f32(h["betas"][1])
    c1, c2 = f32(1 - np.float32(b1)), f32(1 - np.float32(b2))
    step_size = h["lr"] / (1 - b1 ** h["step"])
    g = f["grad"].to(torch.float32)
    norm = g.double().square().sum().sqrt().to(torch.float32)
    coef = (torch.full_like(norm, s["max_norm"]) / (norm + 1e-6)).clamp_max(1.0)
    g = g * coef
    if bits == 8:
        key = _key(s["seed"], h["step"])
        bits_m = f["m"].to(torch.int64)
        m = _value(bits_m & 127, M_BITS, f["scale"][:, 0])
        m = torch.where(bits_m >= 128, -m, m)
        v = _value(f["v"], V_BITS, f["scale"][:, 1])
    else:
        m, v = f["m"], f["v"]
    m = m * b1 + g * c1
    v = v * b2 + (g * c2) * g
    p = f["param"].to(torch.float32) * (1 - h["lr"] * h["weight_decay"])
    p = p - step_size * (m / (v.sqrt() / math.sqrt(1 - b2 ** h["step"]) + h["eps"]))
    r = _hash(torch.arange(s["total"], device=DEV), _key(s["seed"], h["step"])) if bits == 8 or s["dtype"] == "bf16" else None
    if bits == 8:
        code, _, f["scale"][:, 0] = _code(m, M_BITS, TOP_M, r & 0xFFFF)
        f["m"].copy_(code | ((m < 0).to(torch.int64) << 7))
        code, z, f["scale"][:, 1] = _code(v, V_BITS, TOP_V, r >> 16)
        f["v"].copy_(torch.where(z > 0, code.clamp_min(1), code))
        code = f["m"].to(torch.int64)
        m = _value(code & 127, M_BITS, f["scale"][:, 0])
        m = torch.where(code >= 128, -m, m)
        v = _value(f["v"], V_BITS, f["scale"][:, 1])
    else:
        f["m"].copy_(m)
        f["v"].copy_(v)
        m, v = f["m"], f["v"]
    if s["dtype"] == "bf16":      # stochastic rounding: a step far below a half of bf16's last bit moves the mean all the same
        low = ((r * 0xBB67AE85) >> 16) & 0xFFFF
        p = ((p.view(torch.int32).to(torch.int64) + low).to(torch.int32) & -65536).view(torch.float32)
    f["param"].copy_(p)
    return {"norm": norm, "param": f["param"], "exp_avg": m, "exp_avg_sq": v}


def _adamw_own(s):
    from probtalk_amd import train_ops as T
    f, x = s["flat"], s["lists"]
    if "list" not in s:                       # an optimizer keeps it with its moments
        s["list"] = T.AdamWList(x["param"], x["m"], x["v"], x.get("scale"))
    norm = s["list"].step(x["grad"], max_norm=s["max_norm"], seed=s["seed"], **s["hyper"])
    m, v = T.moment_values(f["m"], f["v"], f["scale"]) if s["bits"] == 8 else (f["m"], f["v"])
    return {"norm": norm[0], "param": f["param"], "exp_avg": m, "exp_avg_sq": v}


def _adamw_exact(s):
    f, h = s["flat"], s["hyper"]
    b1, b2 = h["betas"]
    g = f["grad"].double()
    norm = g.square().sum().sqrt()
    g = g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    m, v = f["m"].double(), f["v"].double()
    if s["bits"] == 8:
        def decode(c, mant, scale):
            e = torch.div(c, 2 ** mant, rounding_mode="floor")
            mantissa = c - e * 2 ** mant
            return (torch.where(e == 0, mantissa, (mantissa + 2 ** mant) * 2.0 ** (e - 1)).view(-1, BLOCK) * scale.double().view(-1, 1)).view(-1)
        sign = torch.where(m >= 128, -1.0, 1.0)
        m, v = decode(m % 128, M_BITS, f["scale"][:, 0]) * sign, decode(v, V_BITS, f["scale"][:, 1])
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    p = f["param"].double() * (1 - h["lr"] * h["weight_decay"])
    p -= h["lr"] * (m / (1 - b1 ** h["step"])) / ((v / (1 - b2 ** h["step"])).sqrt() + h["eps"])
    if s["bits"] == 8:                        # which of two neighbouring codes a value takes depends on its last bits
        m = v = None
    return {"norm": norm, "param": p, "exp_avg": m, "exp_avg_sq": v}


# ------------------------------------------------------------------------------------------------------------- gated_norm
def _norm(x, kind, eps):
    """(normalised rows, 1 / standard deviation)."""
    c = x - x.mean(1, keepdim=True) if kind == "layer" else x
    rstd = torch.rsqrt(c.square().mean(1, keepdim=True) + eps)
    return c * rstd, rstd


def _norm_grad(d, n, rstd, kind):
    d = d - n * (d * n).mean(1, keepdim=True)
    return rstd * (d - d.mean(1, keepdim=True) if kind == "layer" else d)


EPS = 1e-5


def _gated_formula(s, wide):
    """y = x + a g N(t), h = N(y) and all gradients, computed in `wide`."""
    kind, per = s["kind"], s["per_clip"]
    x, t, gate, a, w1, w2 = (s[k].detach().to(wide) for k in ("x", "t", "gate", "res_scale", "post_weight", "pre_weight"))
    b1, b2 = (s[k].detach().to(wide) if s[k] is not None else 0 for k in ("post_bias", "pre_bias"))
    rows, cols = x.shape
    g = gate.view(-1, 1, cols).expand(-1, per, -1).reshape(rows, cols)
    tn, tr = _norm(t, kind, EPS)
    u = tn * w1 + b1
    y = x + a * g * u
    yn, yr = _norm(y, kind, EPS)
    out = {"y": y, "h": yn * w2 + b2}
    if not s["grad"]:
        return out
    dy, dh = s["dy"].to(wide), s["dh"].to(wide)
    dx = dy + _norm_grad(dh * w2, yn, yr, kind)
    du = dx * a * g
    out |= {"x": dx, "t": _norm_grad(du * w1, tn, tr, kind), "gate": (dx * a * u).view(-1, per, cols).sum(1), "res_scale": (dx * g * u).sum(0),
            "post_weight": (du * tn).sum(0), "pre_weight": (dh * yn).sum(0)}
    if s["bias"]:
        out |= {"post_bias": du.sum(0), "pre_bias": dh.sum(0)}
    return out


def _gated_plain(s):
    out = _gated_formula(s, torch.float32)
    return {k: v.to(s[k].dtype if k in s else s["type"]) for k, v in out.items()}


def _gated_own(s):
    from probtalk_amd import train_ops as T
    y, h = T.gated_norm(s["x"], s["t"], s["gate"], s["res_scale"], s["post_weight"], s["post_bias"], s["pre_weight"], s["pre_bias"], rows_per_clip=s["per_clip"],
                        kind=s["kind"], eps=EPS)
    out = {"y": y.detach(), "h": h.detach()}
    if s["grad"]:
        out |= dict(zip(s["leaves"], torch.autograd.grad((y, h), [s[k] for k in s["leaves"]], (s["dy"], s["dh"]))))
    return out


# ----------------------------------------------------------------------------------------------------------------- window
def _visible(s, rows, keys):
    """(B or 1, rows, keys): key j of a row at position i is seen if it is no further right than i + right, and no further left than i - left or one of the
    first keys, and inside its sequence."""
    i = torch.arange(keys - rows, keys, device=DEV).view(1, -1, 1)
    j = torch.arange(keys, device=DEV).view(1, 1, -1)
    seen = (j <= i + s["right"]) & ((j >= i - s["left"]) | (j < s["sinks"]))
    return seen if s["lengths"] is None else seen & (j < s["lengths"].view(-1, 1, 1))


def _softmax(sc, seen):
    sc = sc.masked_fill(~seen, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = (sc - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _window_formula(s, wide):
    q, k, v = (s[x].detach().to(wide).transpose(1, 2).contiguous() for x in ("q", "k", "v"))     # (B, H, N, D)
    b, heads, n, d = q.shape
    kv = k.shape[1]
    group = heads // kv
    q = q.view(b, kv, group * n, d)
    scale = 1 / math.sqrt(d)
    seen = _visible(s, n, n)[:, None, None]
    p = _softmax(torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).view(b, kv, group, n, n), seen).view(b, kv, group * n, n)
    o = torch.matmul(p, v)
    back = lambda x, h: x.reshape(b, h, n, d).transpose(1, 2)  # noqa: E731
    out = {"o": back(o, heads)}
    if not s["grad"]:
        return out
    do = s["do"].to(wide).transpose(1, 2).reshape(b, kv, group * n, d)
    out["v"] = back(torch.matmul(p.transpose(2, 3).contiguous(), do), kv)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = (ds - (do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    del p
    out["q"] = back(torch.matmul(ds, k), heads)
    out["k"] = back(torch.matmul(ds.transpose(2, 3).contiguous(), q), kv)
    return out


def _window_plain(s):
    return {k: x.to(s["type"]).contiguous() for k, x in _window_formula(s, torch.float32).items()}


def _window_own(s):
    from probtalk_amd import train_ops as T
    o = T.window_attention(s["q"], s["k"], s["v"], s["left"], s["right"], sinks=s["sinks"], lengths=s["lengths"])
    out = {"o": o.detach()}
    if s["grad"]:
        out["v"], out["q"], out["k"] = torch.autograd.grad(o, [s["v"], s["q"], s["k"]], s["do"])
    return out


def _step_formula(s, wide):
    """The visible keys only: the first ones and the window's, gathered from the cache."""
    b, heads, d = s["q"].shape
    kv = s["k"].shape[2]
    last = s["lengths"].to(torch.int64).view(-1, 1) - 1
    sinks = torch.arange(s["sinks"], device=DEV).expand(b, -1)
    win = last - torch.arange(min(s["left"] + 1, s["keys"]), device=DEV)
    seen = torch.cat([(sinks <= last) & (sinks < last - s["left"]), win >= 0], 1)
    at = torch.cat([sinks, win], 1).clamp(min=0, max=s["keys"] - 1)
    row = torch.arange(b, device=DEV).view(-1, 1)
    k, v = (s[x][row, at].to(wide).transpose(1, 2) for x in ("k", "v"))                          # (B, KV, visible, D)
    q = s["q"].to(wide).view(b, kv, heads // kv, d)
    p = _softmax(torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d), seen[:, None, None])
    return torch.matmul(p, v.contiguous()).view(b, heads, d)


def _step_own(s):
    from probtalk_amd import train_ops as T
    return T.window_attention_step(s["q"], s["k"], s["v"], s["lengths"], s["left"], sinks=s["sinks"])


# ------------------------------------------------------------------------------------------------------------------- calls
def run(s):
    op = s["op"]
    if own:
        return {"adamw": _adamw_own, "gated_norm": _gated_own, "window": _window_own, "step": _step_own}[op](s)
    with torch.no_grad():
        if op == "step":
            return _step_formula(s, torch.float32).to(s["type"])
        return {"adamw": _adamw_plain, "gated_norm": _gated_plain, "window": _window_plain}[op](s)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "adamw":
            return _adamw_exact(s)
        if case["op"] == "gated_norm":
            return _gated_exact(s)
        return _attention_exact(s)


def _gated_exact(s):
    """By torch's own differentiation of the definition, in 64 bits."""
    with torch.enable_grad():
        v = {k: s[k].detach().double().requires_grad_(s["grad"]) for k in s["leaves"]}

        def norm(x, w, b):
            if s["kind"] == "layer":
                x = x - x.mean(1, keepdim=True)
            x = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * w
            return x + b if b is not None else x

        u = norm(v["t"], v["post_weight"], v.get("post_bias")).view(-1, s["per_clip"], s["cols"])
        y = v["x"] + (v["res_scale"] * v["gate"].unsqueeze(1) * u).view(s["rows"], s["cols"])
        h = norm(y, v["pre_weight"], v.get("pre_bias"))
        out = {"y": y.detach(), "h": h.detach()}
        if s["grad"]:
            out |= dict(zip(s["leaves"], torch.autograd.grad((y, h), list(v.values()), (s["dy"].double(), s["dh"].double()))))
    return out


def _attention_exact(s):
    """Sequence by sequence and head by head, in 64 bits; the gradients by torch's own differentiation."""
    step = s["op"] == "step"
    q, k, v = (s[x].detach().double() for x in ("q", "k", "v"))
    q = q[:, None] if step else q
    b, n, heads, d = q.shape
    keys, group = k.shape[1], heads // k.shape[2]
    if b * heads * n * keys > 3e9:
        return None
    o, grads = torch.zeros_like(q), {"q": torch.zeros_like(q), "k": torch.zeros_like(k), "v": torch.zeros_like(v)}
    j = torch.arange(keys, device=DEV)
    for c in range(b):
        size = keys if s["lengths"] is None else int(s["lengths"][c])
        i = torch.tensor([size - 1], device=DEV) if step else torch.arange(n, device=DEV)
        right = 0 if step else s["right"]
        far = ((j > i[:, None] + right) | ((j < i[:, None] - s["left"]) & (j >= s["sinks"])) | (j >= size))
        for h in range(heads):
            with torch.enable_grad():
                x = [t.detach().clone().requires_grad_(bool(s.get("grad"))) for t in (q[c, :, h], k[c, :, h // group], v[c, :, h // group])]
                w = torch.exp(x[0] @ x[1].T / math.sqrt(d)).masked_fill(far, 0.0)
                r = (w / w.sum(1, keepdim=True).clamp_min(1e-300)) @ x[2]
                if s.get("grad"):
                    dq, dk, dv = torch.autograd.grad(r, x, s["do"][c, :, h].double())
                    grads["q"][c, :, h] += dq
                    grads["k"][c, :, h // group] += dk
                    grads["v"][c, :, h // group] += dv
            o[c, :, h] = r.detach()
    if step:
        return o[:, 0]
    return {"o": o} | (grads if s["grad"] else {})


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (3 * size + state), "flops": 20 * n}       # the parameter and the two moments in and out, the gradient in
    if case["op"] == "gated_norm":
        n, clips = case["rows"] * case["cols"], case["rows"] // case["per_clip"]
        gate = clips * case["cols"] * size
        return {"bytes": (4 * n * size + gate) * (2 if case["grad"] else 1), "flops": n * (60 if case["grad"] else 20)}   # x, t, y, h and their gradients
    b, heads, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    n = case["keys"] if case["op"] == "step" else case["rows"]
    share = 0.625 if case["ragged"] else 1.0                             # the mean length
    if case["op"] == "step":
        size_of = np.arange(max(1, n // 4), n + 1) if case["ragged"] else np.array([n])
        seen = float(np.minimum(size_of, np.minimum(size_of, case["left"] + 1) + case["sinks"]).mean()) * b
        return {"bytes": 2 * seen * kv * d * size + 2 * b * heads * d * size, "flops": 4 * seen * heads * d}
    i = np.arange(n, dtype=np.int64)
    last, first = np.minimum(i + case["right"], n - 1), np.maximum(i - case["left"], 0)
    seen = float((last - first + 1 + np.minimum(case["sinks"], first)).sum()) * b * share
    once = 2 * b * n * d * size * (heads + kv)                           # q, o, k, v; with the gradients the same again
    return {"bytes": 2 * once, "flops": 14 * seen * heads * d} if case["grad"] else {"bytes": once, "flops": 4 * seen * heads * d}
