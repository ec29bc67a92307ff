"""Oracle of the operators for several texts at once (include/g2hip.h: packed
prompt attention, the 4-bit K/V cache, beam search), from their definitions in
numpy: what is rounded by definition is rounded here, everything else is in 64
bits."""
import numpy as np

from oracle import lowbit

DH = 64


# ------------------------------------------------------------ attention

def attend(q, k, v, scale, seen):
    """Attention of rows q [n, NH, 64] over keys and values [m, NKV, 64], seen [n, m] saying who sees what: (out [n,
    NH, 64], sum of p |v|, the largest sum of |q k| of a row and head [n, NH]): the output and what its rounding bound
    is made of.  A row that sees nothing gives zeros."""
    n, NH, _ = q.shape
    m, NKV, _ = k.shape
    out, mass = np.zeros((n, NH, DH)), np.zeros((n, NH, DH))
    top = np.zeros((n, NH))
    some = seen.any(1)
    if not m or not some.any():
        return out, mass, top
    with np.errstate(all="ignore"):
        for h in range(NH):
            x, key, val = q[some, h].astype(np.float64), k[:, h * NKV // NH].astype(np.float64), v[:, h * NKV // NH].astype(np.float64)
            hidden = ~seen[some]
            s = x @ key.T * scale
            s[hidden] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            clean, bad = np.where(np.isfinite(val), val, 0), np.where(np.isfinite(val), 0, val)
            y = p @ clean
            for j in np.flatnonzero(bad.any(1)):  # values that are not finite count for the rows that see them
                y[~hidden[:, j]] += bad[j]
            out[some, h], mass[some, h] = y, p @ np.abs(clean)
            a = np.abs(x) @ np.abs(np.where(np.isfinite(key), key, 0)).T * abs(scale)
            a[hidden] = 0
            top[some, h] = a.max(1)
    return out, mass, top


def causal(n, m):
    """Who sees what of n rows and m keys: row i the keys j <= i + m - n."""
    return np.arange(m)[None] <= np.arange(n)[:, None] + (m - n)


# ------------------------------------------------------------ 4-bit cache

def to4(x):
    """fp32 values that rows [..., 64] stand for in 4 bits, and their codes and scales."""
    x = np.asarray(x, np.float32)
    codes, scales = lowbit.quantize_q4(x.reshape(-1, 32), 32)
    v = lowbit.values_q4(codes, scales, 32).astype(np.float32)
    return v.reshape(x.shape), codes.reshape(x.shape), scales.reshape(x.shape[:-1] + (2,))


def cache_bytes(k, v):
    """Codes and scales' bytes of one sequence's keys and values [32 tiles, NKV, 64], by the header: [NKV][tiles][2304]."""
    T, NKV, _ = k.shape
    out = np.zeros((NKV, T // 32, 2304), np.uint8)
    for i, x in enumerate((k, v)):
        _, codes, scales = to4(x)
        for p in range(T):
            for h in range(NKV):
                t, j = divmod(p, 32)
                at = (i * 32 + j) * 32
                out[h, t, at:at + 32] = codes[p, h, 0::2] | codes[p, h, 1::2] << 4
                sc = (scales[p, h].astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
                at = 2048 + (i * 32 + j) * 4
                out[h, t, at:at + 4] = sc.view(np.uint8)
    return out


# ------------------------------------------------------------ beam search

def select(logits, score, done, eos, beams, n_out):
    """(scores fp64, parents, ids, ended) [groups, n_out] of logits [groups * beams, V]."""
    rows, V = logits.shape
    l = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        top = l.max(1, keepdims=True)
        total = l - (top + np.log(np.exp(l - top).sum(1, keepdims=True))) + score.astype(np.float64)[:, None]
        total[~(total > -np.inf)] = -np.inf
        total[np.isnan(l).any(1) | np.isposinf(l).any(1)] = -np.inf
    if done is not None:
        for r in np.flatnonzero(done):
            total[r] = -np.inf
            total[r, eos] = score[r] if score[r] > -np.inf else -np.inf
    total = total.reshape(-1, beams * V)
    flat = np.argsort(-total, 1, kind="stable")[:, :n_out]
    if flat.shape[1] < n_out:
        flat = np.concatenate([flat, np.zeros((len(flat), n_out - flat.shape[1]), int)], 1)
    s = np.take_along_axis(total, flat, 1)
    s[:, beams * V:] = -np.inf
    none = ~(s > -np.inf)
    parent, ids = np.where(none, -1, flat // V), np.where(none, -1, flat % V)
    rows = np.maximum(parent, 0) + beams * np.arange(len(flat))[:, None]
    over = (ids == eos) & (eos >= 0)
    if done is not None:
        over |= np.asarray(done)[rows] != 0
    return s, parent, ids, (over & ~none).astype(np.int32)


def reorder(table, parent, new, n, beams):
    """Rows [groups * beams, stride] in their parents' order up to n (one for each group), new ints behind."""
    out = table.copy()
    for r in range(len(table)):
        g, p = r // beams, int(parent[r])
        if 0 <= p < beams:
            out[r, :n[g]] = table[g * beams + p, :n[g]]
            out[r, n[g]] = new[r]
    return out
