"""Plain restatements of the AdamW step and of its 8-bit state format (numpy, CPU)."""
import numpy as np

BLOCK = 256
M32 = 0xFFFFFFFF


def mix(h):
    h = np.asarray(h, dtype=np.uint64)
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & np.uint64(M32)
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & np.uint64(M32)
    return h ^ (h >> np.uint64(16))


def random_bits(seed, step, tensor, n):
    key = mix(mix((seed + step * 0x9E3779B9) & M32) ^ np.uint64(tensor))
    return mix(np.arange(n, dtype=np.uint64) ^ key)


def decode(code, exp, low, signed):
    """float64 values of a state; a block whose exponent byte is 255 is NaN."""
    n = code.size
    c = code.astype(np.int64)
    e = np.repeat(exp.astype(np.int64), BLOCK)[:n]
    mag = c & 127 if signed else c
    x = (1 + (mag & 7) / 8.0) * np.exp2((mag >> 3) - low + e - 127.0)
    x = np.where((mag == 0) | (e == 0), 0.0, x)
    if signed:
        x = np.where(c > 127, -x, x)
    return np.where(e == 255, np.nan, x)


def encode(x, r16, low, signed):
    """Codes and exponents of float32 values, in 64-bit arithmetic: up with the probability of the
    fraction cut off.  Finite values only."""
    n = x.size
    full = -(-n // BLOCK) * BLOCK
    a = np.zeros(full)
    a[:n] = np.abs(x.astype(np.float64))
    a[a < 2.0 ** -126] = 0
    u = np.zeros(full)
    u[:n] = (r16.astype(np.float64) + 0.5) / 65536
    top = a.reshape(-1, BLOCK).max(1)
    e = np.where(top > 0, np.frexp(top)[1] + 127, 0)  # top < 2^(e - 127)
    eb = np.repeat(e, BLOCK)
    xe = np.where(a > 0, np.frexp(a)[1], 0)
    q = np.floor(a / np.exp2(xe - 4.0) + u)  # 8 .. 16 eighths of the binade
    xe, q = np.where(q == 16, xe + 1, xe), np.where(q == 16, 8, q)
    code = 8 * (xe - 1 - (eb - 127) + low) + (q - 8)
    least = 1.125 * np.exp2(eb - 127.0 - low)
    code = np.where(a < least, (u * least < a) if signed else 1, code)
    code = np.where(a > 0, code, 0).astype(np.int64)
    assert (code >= 0).all() and (code <= 8 * low).all()
    sign = np.zeros(full, np.int64)
    sign[:n] = (x < 0) * 128 if signed else 0
    code = np.where(code > 0, code + sign, 0)
    return code[:n].astype(np.uint8), e.astype(np.uint8)


def adamw64(p, g, m, v, step, lr, b1, b2, eps, wd, bias=True, coef=1.0):
    """The formulas in float64."""
    g = g * coef
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    c1, c2 = (1 - b1 ** step, 1 - b2 ** step) if bias else (1.0, 1.0)
    return p * (1 - lr * wd) - lr * (m / c1) / (np.sqrt(v / c2) + eps), m, v


def moments32(g, m, v, b1, b2, coef=1.0):
    """m and v as separately rounded float32 operations, the step's own definition."""
    f = np.float32
    g = g.astype(f) * f(coef)
    return m.astype(f) * f(b1) + g * f(1 - b1), v.astype(f) * f(b2) + (g * g) * f(1 - b2)
