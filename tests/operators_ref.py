"""Plain 64-bit implementations of group norm + activation, the matrix product with an epilogue, and AdamW with 8-bit
moments, written from their formulas for the tests of those kernels."""
import math

import numpy as np
import torch


def act64(u, name):
    if name == "relu":
        return torch.where(u > 0, u, torch.zeros_like(u))
    if name == "silu":
        return u * torch.sigmoid(u)
    if name == "gelu":
        return 0.5 * u * torch.special.erfc(-u / math.sqrt(2.0))
    return u


def group_norm_act64(x, G, weight, bias, eps, act):
    B, C, H, W = x.shape
    g = x.reshape(B, G, -1)
    mean = g.mean(-1, keepdim=True)
    var = ((g - mean) ** 2).mean(-1, keepdim=True)
    u = ((g - mean) / torch.sqrt(var + eps)).reshape(B, C, H, W)
    if weight is not None:
        u = u * weight[:, None, None]
    if bias is not None:
        u = u + bias[:, None, None]
    return act64(u, act)


def linear_act64(x, weight, bias, act, residual):
    u = x @ weight.t()
    if bias is not None:
        u = u + bias
    y = act64(u, act)
    return y if residual is None else y + residual


# ---------------------------------------------------------------------------------------------------------------
# AdamW8
# ---------------------------------------------------------------------------------------------------------------
def philox(n, step, seed, first=0):
    """n 32-bit words from the word `first` (a multiple of 4) on, word i from the counter (i // 4, step) under the key
    `seed`."""
    u = np.uint64
    i = np.arange((n + 3) // 4, dtype=np.uint64) + u(first // 4)
    m32 = u(0xFFFFFFFF)
    c = [i & m32, i >> u(32), np.full_like(i, step & 0xFFFFFFFF), np.full_like(i, step >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p, q = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(q >> u(32)) ^ c[1] ^ u(k0), q & m32, (p >> u(32)) ^ c[3] ^ u(k1), p & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)[:n].astype(np.int64)


def code_values(bits):
    k = np.arange(16 << bits)
    e, f = k >> bits, (k & ((1 << bits) - 1)) / (1 << bits)
    return np.where(e > 0, (1 + f) * 2.0 ** (e - 15.0), f * 2.0 ** -14)


def decode(codes, scales, signed):
    t = code_values(3 if signed else 4)
    if signed:
        t = np.concatenate([t, -t])
    f = np.where(scales == 0, 0.0, np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127)))
    return (t[codes].reshape(-1, 128) * f[:, None]).reshape(-1)


def encode(x, r16, signed):
    """float64 values -> (codes, scales): scanning the table of code values for the two neighbours of each value."""
    bits = 3 if signed else 4
    a = np.abs(x).astype(np.float32).astype(np.float64).reshape(-1, 128)
    a[a < 2.0 ** -126] = 0
    table = code_values(bits)
    codes, scales = np.zeros(a.shape, np.int64), np.zeros(len(a), np.int64)
    for b in range(len(a)):
        top = a[b].max()
        if not np.isfinite(a[b]).all():
            scales[b] = 255
            continue
        if top == 0:
            continue
        s = int(math.floor(math.log2(top))) + 127
        while top > table[-1] * 2.0 ** (s - 127):
            s += 1
        while s > 1 and top <= table[-1] * 2.0 ** (s - 1 - 127):
            s -= 1
        if s >= 255:
            scales[b] = 255
            continue
        scales[b] = s
        v = a[b] / 2.0 ** (s - 127)
        lo = np.searchsorted(table, v, side="right") - 1
        step = np.where(lo + 1 < len(table), table[np.minimum(lo + 1, len(table) - 1)] - table[lo], 1.0)
        drop = 23 - bits
        part = np.floor((v - table[lo]) / step * 2.0 ** drop)            # the dropped bits of the float
        r = (r16.reshape(-1, 128)[b] << (drop - 16)) + (1 << (drop - 17))
        q = lo + ((part + r) >= 2 ** drop)
        if not signed:
            q = np.where((a[b] > 0) & (q == 0), 1, q)
        codes[b] = q
    codes = codes.reshape(-1)
    if signed:
        codes = codes + 128 * np.signbit(x)
    return codes, scales


def adamw8_step(p, g, m, ms, v, vs, words, lr, b1, b2, eps, wd, step, coef=1.0):
    """One step in 64 bits on flat arrays padded to 128: (p, m, ms, v, vs) new."""
    g = g * coef
    m1 = b1 * decode(m, ms, True) + (1 - b1) * g
    v1 = b2 * decode(v, vs, False) + (1 - b2) * g * g
    with np.errstate(all="ignore"):
        upd = m1 / (np.sqrt(v1) / math.sqrt(1 - b2 ** step) + eps)
        p = p * (1 - lr * wd) - lr / (1 - b1 ** step) * upd
        return (p,) + encode(m1, words & 0xFFFF, True) + encode(v1, words >> 16, False)
