"""The training operators beside the KDA recurrence, as cases to be timed and compared.

Two operators: the matrix product with bias, activation and residual in its epilogue (one layer,
``linear_act``, and a block's MLP of two, ``mlp``, each with its gradients), and the AdamW step
over a model's tensors at once with its states in 32 or in 8 bits (``adamw_step``).  ``run``
computes them in plain torch, in 32 bits, or through the framework's entry points when ``own``
is true.  ``exact`` computes the same from the definitions in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256  # elements that share an exponent in an 8-bit state
M_LOW, V_LOW = 15, 31  # binades of the 8-bit codes below the block's exponent


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # the output projection of one streamed token, added to the residual stream (latency)
        dict(name="linear_token", op="linear", train=False, m=1, k=768, n=768, dtype="bf16", act="none", bias=False,
             residual=True, pad=0),
        # the 400-class head over the pooled features of 8 clips, a training step
        dict(name="linear_head_train", op="linear", train=True, m=8, k=768, n=400, dtype="bf16", act="none", bias=True,
             residual=False, pad=0),
        # odd everything: ragged token count, widths that no 16-byte row holds, a strided view
        dict(name="linear_odd_train", op="linear", train=True, m=1003, k=781, n=203, dtype="fp16", act="silu", bias=True,
             residual=True, pad=3),
        # the fused q, k, v projection of 8 clips of 1568 tokens, a training step
        dict(name="linear_qkv_train", op="linear", train=True, m=12544, k=768, n=2304, dtype="bf16", act="none",
             bias=False, residual=False, pad=0),
        # a block's MLP on a few streamed tokens (the weights' bytes bound it)
        dict(name="mlp_tokens", op="mlp", train=False, m=16, k=2048, n=8192, dtype="bf16", act="gelu", bias=True,
             residual=True, pad=0),
        # a block's MLP on one segment of 4096 streamed tokens, 16 heads of 128
        dict(name="mlp_segment", op="mlp", train=False, m=4096, k=2048, n=8192, dtype="fp16", act="gelu_tanh", bias=True,
             residual=True, pad=0),
        # a block's MLP, training step on one clip
        dict(name="mlp_clip_train", op="mlp", train=True, m=1568, k=512, n=2048, dtype="bf16", act="gelu", bias=True,
             residual=True, pad=0),
        # a block's MLP, training step on 8 clips of 1568 tokens
        dict(name="mlp_train", op="mlp", train=True, m=12544, k=1024, n=4096, dtype="bf16", act="gelu", bias=True,
             residual=True, pad=0),
        # the step of a small model in float32: many tensors of a few elements each (latency)
        dict(name="adamw_small", op="adamw", width=128, hidden=512, depth=2, dtype="fp32", bits=32, clip=0.0, ema=0.0),
        # the step of float32 master weights with gradient clipping and the shadow average
        dict(name="adamw_fp32_clip_ema", op="adamw", width=768, hidden=2304, depth=12, dtype="fp32", bits=32, clip=1.0,
             ema=0.999),
        # the step of bf16 weights with 8-bit states, the largest model that the list holds
        dict(name="adamw_8bit", op="adamw", width=1024, hidden=4096, depth=12, dtype="bf16", bits=8, clip=0.0, ema=0.0),
        # the same with clipping, odd widths: blocks and vectors that end inside a tensor
        dict(name="adamw_8bit_odd_clip", op="adamw", width=391, hidden=1501, depth=6, dtype="fp32", bits=8, clip=0.5,
             ema=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: half of them a multiple of 64 as models have them, half any number."""
    w = _log(rng, lo, hi)
    return max(64, w // 64 * 64) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(["linear", "linear", "mlp", "adamw"])
    if op == "adamw":
        bits = rng.choice([32, 8])
        return dict(op=op, width=_width(rng, 64, 1024), hidden=_width(rng, 128, 4096), depth=rng.randint(1, 8),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), bits=bits, clip=rng.choice([0.0, 0.1, 1.0]),
                    ema=rng.choice([0.0, 0.999]))
    k, n = _width(rng, 64, 2048), _width(rng, 16, 4096)
    m = _log(rng, 1, 12544)
    m = max(1, min(m, 12544 * 1024 * 4096 // (k * n)))
    return dict(op=op, train=rng.random() < 0.6, m=m, k=k, n=n, dtype=rng.choice(["bf16", "fp16"]),
                act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), bias=rng.random() < 0.7,
                residual=rng.random() < 0.5, pad=rng.choice([0, 0, 0, 8, 5]))


def work(case):
    if case["op"] == "adamw":
        numel = sum(math.prod(s) for s in _shapes(case))
        e = 2 if case["dtype"] != "fp32" else 4
        state = 16.0 if case["bits"] == 32 else 4.0 * (1 + 1.0 / BLOCK) + 4.0  # 8 bits: returned as 16-bit values too
        per = 3 * e + state + (8 if case["ema"] else 0)
        return {"bytes": per * numel, "flops": 16.0 * numel}
    m, k, n, t = case["m"], case["k"], case["n"], case["train"]
    products = 2 if case["op"] == "mlp" else 1
    out = k if case["op"] == "mlp" else n
    weights = products * (k * n) + (((n + k) if case["op"] == "mlp" else n) if case["bias"] else 0)
    rows = m * k + m * out + (m * out if case["residual"] else 0)  # x, y, residual
    if t:
        rows += m * out + m * k + (m * out if case["residual"] else 0)  # dy, dx, the residual's gradient
        weights *= 2
    return {"bytes": 2.0 * (rows + weights), "flops": 2.0 * products * m * k * n * (3 if t else 1)}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _shapes(case):
    """The tensors of ``depth`` blocks of the video model at a width: projections, convolutions,
    gates, norms and the MLP."""
    w, h, heads = case["width"], case["hidden"], max(1, case["width"] // 64)
    block = [(w, w)] * 4 + [(64, w), (w, 64), (heads, w), (heads,), (w,)]
    block += [(w, 4), (w,)] * 3 + [(64, w), (w, 64), (w,), (64,)]
    block += [(w,), (w,), (w,), (w,), (h, w), (h,), (w, h), (w,)]
    return block * case["depth"]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _views(flat, shapes):
    """The tensors of a flat buffer, each starting at a multiple of BLOCK elements."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += -(-n // BLOCK) * BLOCK
    return out


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, g)
    dt, m, k, n, pad = DTYPES[case["dtype"]], case["m"], case["k"], case["n"], case["pad"]

    def normal(*s, scale=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * scale).to(dt)

    def uniform(*s, bound):
        return ((torch.rand(*s, generator=g, device="cuda") * 2 - 1) * bound).to(dt)

    out = k if case["op"] == "mlp" else n
    s = dict(case=case, x=normal(m, k + pad)[:, :k], w1=uniform(n, k, bound=k ** -0.5), b1=None, residual=None)
    if case["bias"]:
        s["b1"] = uniform(n, bound=0.5)
    if case["op"] == "mlp":
        s["w2"] = uniform(k, n, bound=n ** -0.5)
        s["b2"] = uniform(k, bound=0.5) if case["bias"] else None
    if case["residual"]:
        s["residual"] = normal(m, out)
    if case["train"]:
        s["dy"] = normal(m, out)
    return s


def _prepare_adamw(case, g):
    shapes, dt = _shapes(case), DTYPES[case["dtype"]]
    sizes = [math.prod(s) for s in shapes]
    total = sum(-(-n // BLOCK) * BLOCK for n in sizes)
    # gradients of one scale a tensor, between 1e-5 and 1e-2; elements of a tensor differ by some binades
    scale = torch.zeros(total, device="cuda")
    for v, e in zip(_views(scale, shapes), torch.rand(len(shapes), generator=g, device="cuda")):
        v.copy_((10.0 ** (3 * e - 5)).expand(v.shape))
    spread = torch.exp2(torch.randn(total, generator=g, device="cuda") * 2)
    normal = lambda: torch.randn(total, generator=g, device="cuda")  # noqa: E731
    live = scale > 0
    m = normal() * scale * spread * 0.3
    v = (scale * spread).square() * (0.25 + torch.rand(total, generator=g, device="cuda")) * live
    s = dict(case=case, sizes=sizes, step=100, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, wd=0.05, seed=1234,
             p=(normal() * 0.02 * live).to(dt), g=(normal() * scale * spread).to(dt))
    if case["ema"]:
        s["ema"] = (s["p"].float() + 1e-3 * normal()) * live
    del spread, scale
    if case["bits"] == 8:
        half = torch.full((total,), 1 << 19, dtype=torch.int32, device="cuda")
        s["m"], s["m_exp"] = _encode(m, half, M_LOW, True)
        s["v"], s["v_exp"] = _encode(v, half, V_LOW, False)
    else:
        s["m"], s["v"] = m, v
    # the lists of tensors as a training program holds them
    s["lists"] = {n: _views(s[n], shapes) for n in ("p", "g", "m", "v", "ema") if n in s}
    if case["bits"] == 8:
        blocks = [-(-n // BLOCK) for n in sizes]
        for n in ("m", "v"):
            s["lists"][n] = list(zip(s["lists"][n], torch.split(s[n + "_exp"], blocks)))
    return s


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return _own_adamw(s) if op == "adamw" else _own_linear(s)
    return _plain_adamw(s) if op == "adamw" else _plain_mlp(s) if op == "mlp" else _plain_linear(s)


def _own_linear(s):
    from mlx_vit_b200.linear import linear_act, mlp
    c = s["case"]
    names = ["x", "w1", "b1", "residual"] if c["op"] == "linear" else ["x", "w1", "b1", "w2", "b2", "residual"]
    t = {n: s[n] for n in names}
    if c["train"]:
        t = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    if c["op"] == "linear":
        y = linear_act(t["x"], t["w1"], t["b1"], c["act"], t["residual"])
    else:
        y = mlp(t["x"], t["w1"], t["b1"], t["w2"], t["b2"], c["act"], t["residual"])
    if not c["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [v for v in t.values() if v is not None], s["dy"])]


def _own_adamw(s):
    from mlx_vit_b200.optim import adamw_step, decode_state8
    c, t = s["case"], s["lists"]
    s["step"] += 1
    norm = adamw_step(t["p"], t["g"], t["m"], t["v"], step=s["step"], lr=s["lr"], betas=s["betas"], eps=s["eps"],
                      weight_decay=s["wd"], max_grad_norm=c["clip"] or None, emas=t.get("ema"),
                      ema_decay=c["ema"] or None, seed=s["seed"])
    out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if c["bits"] == 8:
        out["m"] = decode_state8(s["m"], s["m_exp"], signed=True)
        out["v"] = decode_state8(s["v"], s["v_exp"], signed=False)
    if c["ema"]:
        out["ema"] = s["ema"]
    if c["clip"]:
        out["norm"] = norm
    return out


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end ----
def _act(z, kind):
    if kind == "none":
        return z
    if kind == "relu":
        return z * (z > 0)
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))


def _act_grad(z, kind):
    if kind == "none":
        return torch.ones_like(z)
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    a = (2 / math.pi) ** 0.5
    t = torch.tanh(a * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)


def _affine(x, w, b):
    z = x @ w.t()
    return z if b is None else z + b.float()


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w1"].float()
    z = _affine(x, w, s["b1"])
    y = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not c["train"]:
        return [y.to(dt)]
    dz = s["dy"].float() * _act_grad(z, c["act"])
    out = [y, dz @ w, dz.t() @ x]
    if s["b1"] is not None:
        out.append(dz.sum(0))
    if s["residual"] is not None:
        out.append(s["dy"])
    return [t.to(dt) for t in out]


def _plain_mlp(s):
    c, dt = s["case"], s["x"].dtype
    x, w1, w2 = s["x"].float(), s["w1"].float(), s["w2"].float()
    z = _affine(x, w1, s["b1"])
    h = _act(z, c["act"])
    y = _affine(h, w2, s["b2"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not c["train"]:
        return [y.to(dt)]
    dy = s["dy"].float()
    dz = (dy @ w2) * _act_grad(z, c["act"])
    out = [y, dz @ w1, dz.t() @ x]
    if s["b1"] is not None:
        out.append(dz.sum(0))
    out.append(dy.t() @ h)
    if s["b2"] is not None:
        out.append(dy.sum(0))
    if s["residual"] is not None:
        out.append(s["dy"])
    return [t.to(dt) for t in out]


def _mix(h):
    """The finaliser of MurmurHash3 (32 bits), on int64 tensors or numbers."""
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random(seed, step, tensor, n, device):
    """The 32 random bits of each element of one tensor in one step."""
    key = _mix(_mix((seed + step * 0x9E3779B9) & 0xFFFFFFFF) ^ tensor)
    return _mix(torch.arange(n, dtype=torch.int64, device=device) ^ key)


def _decode(code, exp, low, signed):
    """The float32 values of 8-bit codes (a whole number of blocks)."""
    c = code.view(-1, BLOCK).int()
    e = exp.int()[:, None]
    mag = c & 127 if signed else c
    x = ((mag + 8 * (e - low)) << 20).view(torch.float32)
    x = torch.where((mag > 0) & (e > 0), x, torch.zeros_like(x))
    return (torch.where(c > 127, -x, x) if signed else x).view(-1)


def _encode(x, r20, low, signed):
    """Codes and exponents of float32 values (a whole number of blocks); r20: what is added below
    the code's last bit before it is cut off, 0 to 2^20 - 1."""
    x, r20 = x.view(-1, BLOCK), r20.view(-1, BLOCK)
    b = x.abs().view(torch.int32)
    top = b.amax(1, keepdim=True)
    e = torch.where(top >= 1 << 23, (top >> 23) + 1, torch.zeros_like(top))
    code = ((b + r20) >> 20) - 8 * (e - low)
    least = ((e - low) << 23) + (1 << 20)
    if signed:  # below the least code: that code or zero, by the same random bits
        up = r20.float() * 2.0 ** -20 * torch.clamp(least, min=0).view(torch.float32) < x.abs()
        code = torch.where(b < least, up.int(), code)
    else:  # never zero for a value above zero
        code = torch.where(b < least, torch.ones_like(code), code)
    code = torch.where(b < 1 << 23, torch.zeros_like(code), code)
    if signed:
        code = torch.where((x < 0) & (code > 0), code + 128, code)
    return code.to(torch.uint8).view(-1), e.to(torch.uint8).view(-1)


def _plain_adamw(s):
    c = s["case"]
    s["step"] += 1
    b1, b2 = s["betas"]
    out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    coef = None
    if c["clip"]:
        total = torch.stack([g.double().square().sum() for g in s["lists"]["g"]]).sum().sqrt()
        coef = torch.clamp(c["clip"] / (total + 1e-6), max=1.0).float()
        out["norm"] = total.float()
    c1 = s["lr"] / (1 - b1 ** s["step"])
    c2 = 1 / math.sqrt(1 - b2 ** s["step"])
    g = s["g"].float() if coef is None else s["g"].float() * coef
    eight = c["bits"] == 8
    m = _decode(s["m"], s["m_exp"], M_LOW, True) if eight else s["m"]
    v = _decode(s["v"], s["v_exp"], V_LOW, False) if eight else s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = s["p"].float() * (1 - s["lr"] * s["wd"]) - c1 * m / (v.sqrt() * c2 + s["eps"])
    s["p"].copy_(p)
    if eight:
        r = torch.cat([_random(s["seed"], s["step"], i, -(-n // BLOCK) * BLOCK, g.device) for i, n in enumerate(s["sizes"])])
        code, exp = _encode(m, ((r & 0xFFFF) * 16 + 8).int(), M_LOW, True)
        s["m"].copy_(code), s["m_exp"].copy_(exp)
        code, exp = _encode(v, ((r >> 16) * 16 + 8).int(), V_LOW, False)
        s["v"].copy_(code), s["v_exp"].copy_(exp)
        # three bits of mantissa and float32's exponent: the 16-bit values are exact
        out["m"] = _decode(s["m"], s["m_exp"], M_LOW, True).bfloat16()
        out["v"] = _decode(s["v"], s["v_exp"], V_LOW, False).bfloat16()
    else:
        s["m"].copy_(m), s["v"].copy_(v)
    if c["ema"]:
        s["ema"].copy_(s["ema"] * c["ema"] + s["p"].float() * (1 - c["ema"]))
        out["ema"] = s["ema"]
    return out


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_adamw(case, s) if case["op"] == "adamw" else _exact_product(case, s)


def _exact_product(case, s):
    d = {n: v.double().requires_grad_(case["train"]) for n, v in s.items() if isinstance(v, torch.Tensor)}
    kind = case["act"]

    def f(z):
        if kind == "relu":
            return torch.relu(z)
        if kind == "silu":
            return z * torch.sigmoid(z)
        if kind == "gelu":
            return z * torch.special.ndtr(z)
        if kind == "gelu_tanh":  # 1 + tanh(u) = 2 sigmoid(2 u)
            return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        return z

    def layer(x, w, b):
        z = torch.einsum("mk,nk->mn", x, w)
        return z + b if b is not None else z

    y = f(layer(d["x"], d["w1"], d.get("b1")))
    names = ["x", "w1", "b1", "residual"]
    if case["op"] == "mlp":
        y = layer(y, d["w2"], d.get("b2"))
        names = ["x", "w1", "b1", "w2", "b2", "residual"]
    if "residual" in d:
        y = y + d["residual"]
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [d[n] for n in names if n in d], d["dy"].detach())]


def _exact_values(code, exp, low, signed):
    code = code.reshape(-1, BLOCK).long()
    mag = code % 128 if signed else code
    x = (1 + (mag % 8).double() / 8) * 2.0 ** ((mag // 8) - low + exp.long()[:, None] - 127).double() * (mag > 0)
    return (x * (1 - 2.0 * (code // 128)) if signed else x).reshape(-1)


def _exact_rounded(x, u, low, signed):
    """x rounded to the 8-bit format: up with the probability that the fraction cut off has (u)."""
    x, u = x.reshape(-1, BLOCK), u.reshape(-1, BLOCK)
    a = x.abs()
    a = a * (a >= 2.0 ** -126)
    frac, e = torch.frexp(a.amax(1, keepdim=True))  # the block's largest = frac 2^e, frac in [0.5, 1)
    _, xe = torch.frexp(a)
    step = 2.0 ** (xe - 4).double()  # eight steps a binade
    y = torch.floor(a / step + u) * step
    least = 1.125 * 2.0 ** (e - low).double()
    y = torch.where(a < least, least * ((u * least < a) if signed else (a > 0)), y)
    return (torch.sign(x) * y).reshape(-1)


def _exact_adamw(case, s):
    step, (b1, b2) = s["step"] + 1, s["betas"]
    g, p = s["g"].double(), s["p"].double()
    out = {}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["clip"] / (float(norm) + 1e-6))
        out["norm"] = norm
    if case["bits"] == 8:
        m, v = _exact_values(s["m"], s["m_exp"], M_LOW, True), _exact_values(s["v"], s["v_exp"], V_LOW, False)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = p - s["lr"] * s["wd"] * p
    p = p - s["lr"] * (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + s["eps"])
    if case["ema"]:
        held = p.to(s["p"].dtype).double()  # the shadow follows the parameter as it is stored
        out["ema"] = case["ema"] * s["ema"].double() + (1 - case["ema"]) * held
    if case["bits"] == 8:
        def fmix(h):
            h = (h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B) & np.uint64(0xFFFFFFFF)
            h = (h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35) & np.uint64(0xFFFFFFFF)
            return h ^ (h >> np.uint64(16))
        mask, bits = (1 << 32) - 1, []
        key = fmix(np.array([(s["seed"] + step * 0x9E3779B9) & mask], dtype=np.uint64))
        for i, n in enumerate(s["sizes"]):
            k = fmix(key ^ np.uint64(i))
            bits.append(fmix(np.arange(-(-n // BLOCK) * BLOCK, dtype=np.uint64) ^ k).astype(np.uint32).view(np.int32))
        r = torch.from_numpy(np.concatenate(bits)).to(g.device).long() & mask
        m = _exact_rounded(m, ((r % 65536).double() + 0.5) / 65536, M_LOW, True)
        v = _exact_rounded(v, ((r // 65536).double() + 0.5) / 65536, V_LOW, False)
    return {**out, "p": p, "m": m, "v": v}
