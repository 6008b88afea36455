"""AdamW from its definition, in 64 bits and plain Python / NumPy (test infrastructure): torch.optim.AdamW's update with
clip_grad_norm_ ahead of it, the 8-bit block formats of include/mscl_hip.h as explicit grids of values, and their stochastic rounding as
a choice between two neighbours on the grid."""
import numpy as np

BLOCK = 256


def hash32(x):
    """finaliser of MurmurHash3 (Appleby, public domain) on uint64 arrays of 32-bit values"""
    m = np.uint64(0xFFFFFFFF)
    x = x.astype(np.uint64) if isinstance(x, np.ndarray) else np.array([x], dtype=np.uint64)
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x85EBCA6B)) & m
    x ^= x >> np.uint64(13)
    x = (x * np.uint64(0xC2B2AE35)) & m
    return x ^ (x >> np.uint64(16))


def random_bits(n, first, seed, step):
    """(low 16, high 16) random bits of elements first .. first + n - 1 of the state buffer at this step"""
    at = np.arange(first, first + n, dtype=np.uint64)
    key = hash32(np.array([(seed + 0x9E3779B9 * step) & 0xFFFFFFFF], dtype=np.uint64))
    r = hash32(hash32(((at >> np.uint64(32)) + key) & np.uint64(0xFFFFFFFF)) ^ (at & np.uint64(0xFFFFFFFF)))
    return (r & np.uint64(0xFFFF)).astype(np.float64), (r >> np.uint64(16)).astype(np.float64)


def grid(exp_bits):
    """magnitudes of all codes relative to the block's power of two, ascending: `exp_bits` exponent bits over 3 mantissa bits"""
    top = (1 << exp_bits) - 1
    out = []
    for code in range(1 << (exp_bits + 3)):
        e, k = code >> 3, code & 7
        out.append((1 + k / 8) * 2.0 ** (e - top) if e else k / 8 * 2.0 ** (1 - top))
    return np.array(out)


GRID_M, GRID_V = grid(4), grid(5)


def block_power(top):
    """exponent (unbiased) of the block's power of two for a largest magnitude `top`"""
    if top < 2.0 ** -126:
        return -126
    e = int(np.floor(np.log2(top)))
    return e + 1 if top > 1.875 * 2.0 ** e else e


def quantise(x, rnd, exp_bits):
    """(values, candidates below, above) of the blocks of x: each magnitude goes up with the probability that makes its mean right"""
    g = grid(exp_bits)
    out, lo_all, hi_all = (np.zeros_like(x) for _ in range(3))
    for b in range(0, len(x), BLOCK):
        a = np.abs(x[b:b + BLOCK])
        scale = 2.0 ** block_power(a.max() if len(a) else 0.0)
        i = np.clip(np.searchsorted(g, a / scale, side='right') - 1, 0, len(g) - 1)
        lo, hi = g[i] * scale, g[np.minimum(i + 1, len(g) - 1)] * scale
        up = np.where(hi > lo, (a - lo) / np.where(hi > lo, hi - lo, 1), 0.0) + rnd[b:b + BLOCK] / 65536 >= 1
        q = np.where(up, hi, lo)
        if exp_bits == 5:
            q = np.where((a > 0) & (q == 0), g[1] * scale, q)
        s = np.sign(x[b:b + BLOCK])
        out[b:b + BLOCK], lo_all[b:b + BLOCK], hi_all[b:b + BLOCK] = q * s, lo * s, hi * s
    return out, lo_all, hi_all


def decode(codes, exponents, exp_bits):
    """values of uint8 codes (m: bit 7 is the sign; v: none) with one biased exponent per block"""
    g = grid(exp_bits)
    codes = codes.astype(np.int64)
    if exp_bits == 4:
        v = g[codes & 127] * np.where(codes & 128, -1.0, 1.0)
    else:
        v = g[codes]
    e = np.repeat(exponents.astype(np.float64), BLOCK)[:len(codes)]
    return np.where(e == 255, np.nan, v * 2.0 ** (e - 127))


def coefficient(grads, max_norm):
    norm = np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads))
    return (1.0 if not max_norm else min(1.0, max_norm / (norm + 1e-6))), norm


def step(p, g, m, v, t, coef=1.0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, decay=0.01):
    """one tensor, 64-bit arrays; returns the new (p, m, v)"""
    g = g * coef
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p * (1 - lr * decay) - lr / (1 - betas[0] ** t) * m / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p, m, v
