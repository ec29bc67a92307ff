"""Oracle of the decode operators in fewer bits (include/g2hip.h: 4-bit
weights, the 8-bit K/V cache, rules on logits), from their definitions in
numpy: what is rounded by definition is rounded here, everything else is in
64 bits."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
BLOCK, DH = 16, 64


# ------------------------------------------------------------ 4-bit weights

def bf16(x):
    """fp32 values rounded to bf16 (nearest even), as fp32."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint32) << np.uint32(16)
    return np.where(np.isnan(x), np.float32(np.nan), r.view(np.float32)).astype(np.float32)


def quantize_q4(W, group):
    """(codes [N, K], scales [N, groups] as fp32) of fp32 W."""
    W = np.asarray(W, np.float32)
    N, K = W.shape
    codes = np.zeros((N, K), np.uint8)
    scales = np.zeros((N, -(-K // group)), np.float32)
    with np.errstate(all="ignore"):
        for g in range(scales.shape[1]):
            w = W[:, g * group:(g + 1) * group]
            a = np.abs(w).max(1)
            s = bf16(a / np.float32(6))
            s[~(a <= np.float32(2.0 ** 96))] = np.nan
            scales[:, g] = s
            q = np.where(s[:, None] > 0, (w / s[:, None]).astype(np.float32), 0).astype(np.float64)
            d = np.abs(np.abs(q)[:, :, None] - LEVELS)  # exact: both are short binary fractions next to each other
            best = d.min(2, keepdims=True)
            even = np.where(d == best, np.array([0, 8, 0, 8, 0, 8, 0, 8]) + np.arange(8) / 16, 99)  # a tie: the even code
            c = even.argmin(2).astype(np.uint8)
            codes[:, g * group:(g + 1) * group] = np.where((q < 0) & (c > 0), c + 8, c)
    return codes, scales


def lay_out_q4(codes, scales, group):
    """The bytes of the two buffers, by their description in the header."""
    N, K = codes.shape
    tiles, steps, chunks, per = -(-N // 16), -(-K // 32), -(-K // 128), 128 // group
    out = np.zeros((tiles, steps * 256), np.uint8)
    sc = np.zeros((tiles, chunks, 16, per), np.uint16)
    sb = (np.asarray(scales, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    for n in range(N):
        t, row = divmod(n, 16)
        for g in range(scales.shape[1]):
            sc[t, g // per, row, g % per] = sb[n, g]
    k = np.arange(K)
    chunk, j, place, i = k // 128, k % 128 // 32, k % 32 // 8, k % 8
    r = np.minimum(4, steps - 4 * chunk)
    at = 1024 * chunk + 4 * j + i // 2
    for n in range(N):
        t, row = divmod(n, 16)
        np.bitwise_or.at(out[t], at + (16 * place + row) * 4 * r, codes[n] << (4 * (i % 2)).astype(np.uint8))
    return out.ravel(), sc.ravel()


def values_q4(codes, scales, group):
    """[N, K] fp64 values."""
    v = np.concatenate([LEVELS, -LEVELS])[codes]
    return v * np.repeat(scales.astype(np.float64), group, 1)[:, :codes.shape[1]]


def gelu(y):
    return 0.5 * y * (1 + np.tanh(0.7978845608 * (y + 0.044715 * y ** 3)))


# ------------------------------------------------------------ 8-bit cache

def to8(x):
    """(codes, scale) of one block [16, 64] of fp32."""
    x = np.asarray(x, np.float32)
    if not np.isfinite(x).all():
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    s = np.float32(np.abs(x).max() / np.float32(127))
    if s == 0:
        return np.zeros(x.shape, np.int8), s
    return np.clip(np.rint((x / s).astype(np.float32)), -127, 127).astype(np.int8), s


class Kv8:
    """One sequence: what its cache holds."""

    def __init__(self, NH):
        self.raw = np.zeros((2, 0, NH, DH), np.float32)  # every position as it was appended

    def append(self, pos, k, v):
        NH = self.raw.shape[2]
        new = np.stack([k, v]).reshape(2, -1, NH, DH)
        self.raw = np.concatenate([self.raw[:, :pos], new], 1)

    def values(self, length=None):
        """[2, length, NH, 64] fp32: whole blocks in 8 bits."""
        n = self.raw.shape[1] if length is None else length
        out = self.raw[:, :n].copy()
        for b in range(n // BLOCK):
            for i in range(2):
                for h in range(out.shape[2]):
                    c, s = to8(out[i, b * BLOCK:(b + 1) * BLOCK, h])
                    out[i, b * BLOCK:(b + 1) * BLOCK, h] = c.astype(np.float32) * s
        return out


def attend(q, kv, scale):
    """(out [NH, 64], sum of p |v| [NH, 64], the largest score's sum of |q k| [NH], spread of the scores [NH]) of q
    [NH, 64] over kv [2, T, NH, 64]: the output and what its rounding bound is made of."""
    NH = q.shape[0]
    if kv.shape[1] == 0:
        z = np.zeros((NH, DH))
        return z, z, np.zeros(NH), np.zeros(NH)
    k, v = kv.astype(np.float64)
    prod = q.astype(np.float64)[None] * k
    s = prod.sum(2) * scale
    p = np.exp(s - s.max(0))
    p /= p.sum(0)
    out = np.einsum("th,thd->hd", p, v)
    return out, np.einsum("th,thd->hd", p, np.abs(v)), np.abs(prod).sum(2).max(0) * abs(scale), s.max(0) - s.min(0)


# ------------------------------------------------------------ rules on logits

def rules(logits, ctx=None, repetition=1.0, frequency=0.0, presence=0.0, bias=(), mask=None, forbid=-1):
    """(adjusted fp32 logits, pick) of one row; ctx a list of ids, bias a list of (id, value), mask [V] of bools."""
    l = np.array(logits, np.float32)
    V = len(l)
    r, f, p = np.float32(repetition or 1.0), np.float32(frequency), np.float32(presence)
    with np.errstate(all="ignore"):
        ids, counts = np.unique([i for i in (ctx if ctx is not None else []) if 0 <= i < V], return_counts=True)
        for i, n in zip(ids.astype(int), counts):
            x = l[i] / r if l[i] > 0 else l[i] * r
            l[i] = np.float32(np.float32(x - np.float32(f * np.float32(n))) - p)
        for i, b in {int(i): np.float32(b) for i, b in bias}.items():
            if 0 <= i < V:
                l[i] = l[i] + b
    if mask is not None:
        l[~np.asarray(mask, bool)] = -np.inf
    if forbid >= 0:
        l[forbid] = -np.inf
    best, pick = -np.inf, -1
    for i in np.flatnonzero(l > -np.inf):
        if l[i] > best:
            best, pick = l[i], int(i)
    return l, pick
