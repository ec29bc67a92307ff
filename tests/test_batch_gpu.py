"""The operators for several texts at once against their oracle (oracle/batch.py): packed prompt attention, the 4-bit
K/V cache and its attention, beam search; at the sizes, lengths, strides and values where they can go wrong, captured
and replayed, and together as the decoding of several prompts with beams."""
import ctypes as C

import numpy as np
import pytest

from oracle import batch
from parity import EPS32
from test_lowbit_gpu import guarded, rng, same, take, within

pytestmark = pytest.mark.gpu

H = 64
FILL = 7.0


def ints(g2, x):
    return g2.to_device(np.asarray(x, np.int32))


# ------------------------------------------------------------------ packed prompts

def prompt_bound(mass, top, T, f16, out):
    """|error| of a computed row.  A score is a sum of 64 products, each of six products of parts (a second
    part is below 2^-7 of its value, a third below 2^-15, so what they leave out is below 2 * 2^-22 + 2^-30 of it), so it goes through at most 6 * 64 + 2 roundings, each 2^-24 of the sum of |q k|; a weight's relative error is twice
    that (its own and the largest's) and 2^-21 for its exponent's product with log2 e, the exponential and the
    sum's share; the weighted sum of T keys goes through 6 T roundings and the joining of at most eight parts 16, and
    as many in the sum of the weights.  fp16: scores of exact products, a weight rounded by 2^-11, the output by 2^-11 of itself
    (or the half of fp16's smallest step)."""
    score = (386 * EPS32 + (0 if f16 else 2.0 ** -21 + 2.0 ** -30)) * top[..., None] * 2
    w = np.expm1(np.minimum(score, 1)) + 2.0 ** -21 * (1 + top[..., None]) + (12 * T + 32) * EPS32
    if f16:
        return (w + 2.0 ** -11) * mass * 1.001 + 2.0 ** -11 * np.abs(out) + 2.0 ** -25
    return w * mass + 2.0 ** -22 * np.abs(out)


class Prompts:
    """Packed buffers of sequences (rows, keys there before) and the call on them."""

    def __init__(self, seqs, NH, NKV, f16, seed=0, pad=(0, 0), gap=0):
        r = rng(len(seqs), NH, NKV, seed)
        self.seqs, self.NH, self.NKV, self.f16 = seqs, NH, NKV, f16
        self.n = [n for n, _ in seqs]
        self.m = [max(0, n + p) for n, p in seqs]
        self.qs = gap + np.concatenate([[0], np.cumsum(self.n)])
        self.ks = np.concatenate([[0], np.cumsum(self.m)])
        self.t = np.float16 if f16 else np.float32
        self.rows, self.keys = int(self.qs[-1]) + gap, int(self.ks[-1])
        self.sq, self.skv = NH * H + pad[0], NKV * H + pad[1]
        self.q = r.standard_normal((max(self.rows, 1), self.sq)).astype(self.t)
        self.k = r.standard_normal((max(self.keys, 1), self.skv)).astype(self.t)
        self.v = r.standard_normal((max(self.keys, 1), self.skv)).astype(self.t)

    def run(self, g2, scale=0.125, shift=0, so=None, lists=True):
        so = so or self.NH * H
        rows = max(self.rows, 1)

        def up(x):
            return g2.to_device(np.concatenate([np.zeros(shift, self.t), x.ravel()]))

        size = np.dtype(self.t).itemsize
        q, k, v = up(self.q), up(self.k), up(self.v)
        out = g2.to_device(np.full(rows * so + 8 + shift, FILL, self.t))
        qs, ks = (ints(g2, self.qs), ints(g2, self.ks)) if lists else (None, None)
        g2.attn_prompt(q.offset(shift * size), self.sq, k.offset(shift * size), v.offset(shift * size), self.skv, out.offset(shift * size),
                       so, g2.F16 if self.f16 else g2.F32, qs, ks, len(self.seqs), rows, self.keys, self.NH, self.NKV, scale)
        y = out.download(self.t)
        assert (y[:shift] == FILL).all() and (y[shift + rows * so:] == FILL).all(), "written past the end"
        y = y[shift:shift + rows * so].reshape(rows, so)
        assert (y[:, self.NH * H:] == FILL).all(), "written between the rows"
        return y[:, :self.NH * H].reshape(rows, self.NH, H)

    def want(self, scale=0.125):
        out = np.full((max(self.rows, 1), self.NH, H), FILL)
        bound = np.zeros(out.shape)
        for i in range(len(self.seqs)):
            a, b = slice(self.qs[i], self.qs[i + 1]), slice(self.ks[i], self.ks[i + 1])
            q = self.q[a, :self.NH * H].reshape(-1, self.NH, H)
            k, v = (x[b, :self.NKV * H].reshape(-1, self.NKV, H) for x in (self.k, self.v))
            o, mass, top = batch.attend(q, k, v, scale, batch.causal(self.n[i], self.m[i]))
            out[a], bound[a] = o, prompt_bound(mass, top, max(1, self.m[i]), self.f16, np.where(np.isfinite(o), o, 0))
        return out, bound

    def check(self, g2, **kw):
        got = self.run(g2, **kw)
        want, bound = self.want(kw.get("scale", 0.125))
        odd = ~np.isfinite(want)
        same(got[odd].astype(np.float64), want[odd], "not finite")
        within(got[~odd], want[~odd], bound[~odd] + 1e-38, str(self.seqs)[:60])
        return got


SEQS = {
    "one": [(1, 0)], "two": [(2, 0)], "tile": [(32, 0)], "below": [(31, 0)], "above": [(33, 0)], "mixed": [(17, 0), (1, 0), (0, 0), (5, 0), (70, 0)],
    "tiny": [(i % 4, 0) for i in range(150)], "empty": [(0, 0)] * 130 + [(3, 0)] + [(0, 0)] * 70 + [(2, 0)], "long": [(200, 0), (129, 0), (64, 0)],
    "more": [(1, 100), (5, 33), (40, 0), (1, 0), (31, 257), (64, 64)], "fewer": [(40, -3), (3, -5), (1, -1), (34, -33), (2, 10)],
    "context": [(1000, 0)], "halves": [(512, 0), (300, 212)],
}
HEADS = [(1, 1), (4, 4), (6, 2), (5, 1)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("name", list(SEQS))
def test_prompt(g2, name, f16):
    for NH, NKV in HEADS if name != "context" else [(2, 1)]:
        Prompts(SEQS[name], NH, NKV, f16).check(g2)


def prompt_forms():
    """(f16, sequences, NH, NKV): every form for many rows, with starts that a wave holds and with more of them."""
    r = rng(11)

    def some(n, lo, hi, past=0):
        return [(int(k), past) for k in r.integers(lo, hi, n)]

    few, more = some(24, 150, 350), some(70, 60, 120)
    return [(False, few, 12, 12), (False, more, 12, 6), (False, [(400, 0), (1, 7), (3000, 5)], 20, 4), (False, [(2100, 0)], 32, 32),
            (True, few, 8, 8), (True, more, 10, 2), (True, [(n, 5 * i) for i, (n, _) in enumerate(few)], 25, 25), (True, more, 20, 20),
            (True, [(2100, 0)], 20, 5), (True, [(2100, 0), (1, 0), (77, 900)], 12, 4), (True, some(80, 60, 90, -3), 25, 25), (True, [(1600, 0)], 12, 12)]


@pytest.mark.parametrize("case", range(len(prompt_forms())))
def test_prompt_many_rows(g2, case):
    f16, seqs, NH, NKV = prompt_forms()[case]
    Prompts(seqs, NH, NKV, f16, gap=case % 4).check(g2)


@pytest.mark.parametrize("case", range(len(prompt_forms())))
def test_prompt_many_rows_not_finite(g2, case):
    """Values that are not finite count for the rows that see them, and for no others, in the forms for many rows."""
    f16, seqs, NH, NKV = prompt_forms()[case]
    p = Prompts(seqs, NH, NKV, f16, seed=1)
    r = rng(case)
    for bad in (np.inf, np.nan, -np.inf):
        for j in r.integers(0, p.keys, 3):
            p.v[j, r.integers(0, NKV * H)] = bad
    p.check(g2)


@pytest.mark.parametrize("f16", [False, True])
def test_prompt_strides_and_addresses(g2, f16):
    """Rows apart by odd numbers of elements, buffers at any element's address, rows that are no sequence's."""
    for pad, so, shift, gap in (((1, 3), 4 * H + 5, 1, 0), ((0, 0), None, 3, 7), ((130, 2), 4 * H + 1, 0, 40)):
        p = Prompts([(33, 0), (20, 4), (5, -2)], 4, 2, f16, pad=pad, gap=gap)
        p.check(g2, shift=shift, so=so)
    p = Prompts([(45, 0)], 3, 3, f16)
    p.check(g2, lists=False)
    Prompts([(1, 60)], 3, 1, f16).check(g2, lists=False)


def test_prompt_in_rows_of_qkv(g2):
    """Queries, keys and values in the same rows, as the product of the attention's input leaves them."""
    p = Prompts([(33, 0), (80, 0)], 4, 2, False)
    row = np.concatenate([p.q, p.k, p.v], 1)
    d = g2.to_device(row)
    out, qs = guarded(g2, p.rows * 4 * H), ints(g2, p.qs)
    W = row.shape[1]
    g2.attn_prompt(d, W, d.offset(16 * H), d.offset(24 * H), W, out, 4 * H, g2.F32, qs, qs, 2, p.rows, p.rows, 4, 2, 0.125)
    want, bound = p.want()
    within(take(out, p.rows * 4 * H).reshape(want.shape), want, bound)


@pytest.mark.parametrize("f16", [False, True])
def test_prompt_scales_and_magnitudes(g2, f16):
    for scale in (1.0, 0.0, -0.125, 1e-30):
        Prompts([(70, 0), (9, 5)], 2, 1, f16, seed=1).check(g2, scale=scale)
    p = Prompts([(70, 0)], 2, 2, f16, seed=2)
    big = 2.0 ** 14 if f16 else 2.0 ** 60
    p.q, p.k, p.v = (p.q / big).astype(p.t), (p.k * p.t(big / 4)).astype(p.t), (p.v * p.t(big / 4)).astype(p.t)
    p.q = np.where(np.abs(p.q) < 2.0 ** -14, 0, p.q).astype(p.t) if f16 else p.q
    p.check(g2)
    p = Prompts([(70, 0)], 2, 2, f16, seed=3)
    if not f16:  # small values beside far larger ones: each row by its own
        p.v[::2] *= np.float32(2.0 ** 40)
        p.v[::3] *= np.float32(2.0 ** -60)
        p.k[:, ::5] *= np.float32(2.0 ** 30)
        p.q[:, ::5] *= np.float32(2.0 ** -30)
        p.check(g2)
    p = Prompts([(70, 0)], 2, 2, f16, seed=4)
    p.k = (p.k * 200).astype(p.t)  # weights of one key nearly all
    p.check(g2)


@pytest.mark.parametrize("seqs,NH", [([(70, 0), (9, 5)], 2), ([(700, 0)], 100)])
@pytest.mark.parametrize("scale", [0.0, 1e-42, -2.0 ** -140])
def test_prompt_smallest_scales(g2, seqs, NH, scale):
    """Scores near fp32's end times scales near 0 are still small: the exponent's factor, scale / log 2, is off by half
    of fp32's smallest step at most, 2^-150 of scores below 2^125, within the bound's share for the exponent."""
    p = Prompts(seqs, NH, NH, False, seed=8)
    p.q, p.k = np.clip(p.q, -4, 4) * np.float32(2.0 ** 60), np.clip(p.k, -4, 4) * np.float32(2.0 ** 54)
    p.check(g2, scale=scale)


@pytest.mark.parametrize("f16", [False, True])
def test_prompt_not_finite_in_masked_places(g2, f16):
    """Infinities and NaN in keys and values that a row does not see leave it as it is; a value counts where it is
    seen, a key makes the rows that see it NaN."""
    for seqs, at in (([(70, 0), (40, 3)], (40, 100)), ([(200, 0)], (150,)), ([(5, 0), (9, 0), (30, 0)], (4, 13))):
        for bad in (np.inf, -np.inf, np.nan):
            p = Prompts(seqs, 2, 1, f16, seed=5)
            for j in at:
                p.v[j, j % 60] = bad
                p.v[j, 63] = bad
            want = p.check(g2)
            assert not np.isfinite(want).all()
            p = Prompts(seqs, 2, 1, f16, seed=6)
            clean = p.run(g2)
            for j in at:
                p.k[j] = np.nan if np.isnan(bad) else p.k[j]
                p.k[j, 7] = bad
            got = p.run(g2)
            for i in range(len(seqs)):
                see = batch.causal(p.n[i], p.m[i])[:, [j - p.ks[i] for j in at if p.ks[i] <= j < p.ks[i + 1]]].any(1)
                rows = np.arange(p.qs[i], p.qs[i + 1])
                same(got[rows[~see]], clean[rows[~see]], "rows that do not see the key")
                if np.isnan(bad):
                    assert np.isnan(got[rows[see]]).all()


def test_prompt_lowest_and_all_equal(g2):
    """Scores that are all the type's lowest value, or all equal."""
    p = Prompts([(40, 0)], 1, 1, False, seed=7)
    p.q[:], p.k[:] = 0, 0
    p.check(g2)
    p.q[:, 0], p.k[:, 0] = np.float32(-3.4028235e38), 1  # every score -3.4e38 / 8
    got = p.run(g2)
    p.q[:] = 0
    within(got, p.want()[0], p.want()[1])


@pytest.mark.parametrize("f16", [False, True])
def test_prompt_lists_in_no_order(g2, f16):
    """Lists that are no lists of starts: nothing outside the buffers is touched, every row is one the buffer has."""
    p = Prompts([(30, 0), (30, 0), (30, 0)], 2, 1, f16)
    for lists in ([-5, 1 << 30, -(1 << 31), 60], [90, 60, 30, 0], [2147483647] * 4, [-2147483648] * 4, [10, 10, 10, 10], [0, 500, 20, 90]):
        p.qs = np.array(lists)
        p.rows = 90
        p.run(g2)
        p.qs, p.ks = np.array([0, 30, 60, 90]), np.array(lists)
        got = p.run(g2)
        assert np.isfinite(got).all()
        p.ks = np.array([0, 30, 60, 90])


# ------------------------------------------------------------------ 4-bit cache

class Cache:
    """A 4-bit cache, and what was appended to each sequence."""

    def __init__(self, g2, S, NKV, max_seq):
        self.g2, self.S, self.NKV, self.max_seq = g2, S, NKV, max_seq
        self.n = g2.kv4_bytes(S, NKV, max_seq)
        self.buf = g2.to_device(np.full(self.n + 64, 0xAB, np.uint8))
        self.raw = np.zeros((2, S, max_seq, NKV, H), np.float32)

    def append(self, lens, pos, f16=False, seed=0, pad=0, scale=1.0, lists=True):
        g2, rows = self.g2, max(1, sum(lens))
        r = rng(seed, rows, *(p & 0xFFFF for p in pos))
        x = (scale * r.standard_normal((2, rows, self.NKV * H + pad))).astype(np.float16 if f16 else np.float32)
        start = np.concatenate([[0], np.cumsum(lens)])
        self.put(x, start, pos)
        k, v = g2.to_device(x[0]), g2.to_device(x[1])
        g2.kv4_append(k, v, self.NKV * H + pad, g2.F16 if f16 else g2.F32, self.buf, ints(g2, start) if lists else None,
                      ints(g2, pos) if lists else None, 0 if lists else pos[0], self.S, rows, self.NKV, self.max_seq)
        return x

    def put(self, x, start, pos):
        for s in range(self.S):
            for i, row in enumerate(range(start[s], start[s + 1])):
                if 0 <= pos[s] + i < self.max_seq:
                    self.raw[:, s, pos[s] + i] = x[:, row, :self.NKV * H].reshape(2, self.NKV, H)

    def values(self):
        return batch.to4(self.raw)[0]

    def read(self, start, T, T_kv, lens=None, origin=None):
        g2, n = self.g2, self.S * T * self.NKV * H
        k, v = guarded(g2, n), guarded(g2, n)
        g2.kv4_read(self.buf, k, v, None if origin is None else ints(g2, origin), None if lens is None else ints(g2, lens), T_kv, start, T,
                    self.S, self.NKV, self.max_seq)
        return np.stack([take(k, n), take(v, n)]).reshape(2, self.S, T, self.NKV, H)

    def attend(self, q, scale, T_kv, lens=None, origin=None, qs=None, os=None):
        """(got, want, bound) [S, NH, 64] of queries q [S, NH, 64]."""
        g2, S, NH = self.g2, self.S, q.shape[1]
        D = NH * H
        qs, os = qs or D, os or D
        rows = np.full((S, qs), np.nan, np.float32)
        rows[:, :D] = q.reshape(S, D)
        out = guarded(g2, (S - 1) * os + D)
        work = g2.to_device(np.full(g2.kv4_work_bytes(S, NH) // 4 + 4, np.nan, np.float32))
        g2.attn_kv4(g2.to_device(rows), qs, self.buf, out, os, None if origin is None else ints(g2, origin),
                    None if lens is None else ints(g2, lens), T_kv, S, NH, self.NKV, self.max_seq, scale, work)
        flat = take(out, (S - 1) * os + D)
        flat = np.concatenate([flat, np.full(os - D, FILL, np.float32)]).reshape(S, os)
        assert (flat[:, D:] == FILL).all(), "written between the rows"
        vals, want, bound = self.values(), np.zeros((S, NH, H)), np.zeros((S, NH, H))
        for s in range(S):
            n = T_kv if lens is None else min(max(int(lens[s]), 0), T_kv)
            at = np.full(n, s) if origin is None else np.asarray(origin)[s, :n]
            ok = (at >= 0) & (at < S)
            kv = vals[:, np.where(ok, at, 0), np.arange(n)]
            want[s], mass, top = batch.attend(q[s:s + 1], kv[0], kv[1], scale, ok[None])
            bound[s] = attend_bound(mass, top, max(1, n))[0]
        return flat[:, :D].reshape(S, NH, H), want, bound


def attend_bound(mass, top, T):
    """A score: 64 products and their sum, the factors and the scale, at most 72 roundings of the sum of |q k|; weights as
    in prompt_bound; sums of T positions, each with two roundings (and those of the rescaling), and of 64 parts."""
    score = 72 * EPS32 * top[..., None] * 2
    return (np.expm1(np.minimum(score, 1)) + 2.0 ** -21 * (1 + top[..., None]) + (6 * T + 200) * EPS32) * mass + 1e-37


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,NKV,max_seq", [(1, 1, 1), (1, 3, 32), (2, 2, 33), (3, 5, 100)])
def test_kv4_append_and_read(g2, S, NKV, max_seq, f16):
    c = Cache(g2, S, NKV, max_seq)
    r = rng(S, NKV, max_seq)
    steps = [([max_seq] * S, [0] * S)]
    steps += [([int(n) for n in r.integers(0, 12, S)], [int(p) for p in r.integers(0, max_seq, S)]) for _ in range(4)]
    for i, (lens, pos) in enumerate(steps):
        if sum(lens):
            c.append(lens, pos, f16, seed=i, pad=3 * i)
        same(c.read(0, max_seq, max_seq), c.values(), f"step {i}")
    tiles = -(-max_seq // 32)
    raw = np.zeros((2, S, tiles * 32, NKV, H), np.float32)
    raw[:, :, :max_seq] = c.raw
    got = c.buf.download(np.uint8)
    assert (got[c.n:] == 0xAB).all()
    got = got[:c.n].reshape(S, NKV, tiles, 2304)
    for s in range(S):
        e = batch.cache_bytes(raw[0, s], raw[1, s])
        for p in range(max_seq):
            t, j = divmod(p, 32)
            for i in range(2):
                a, b = (32 * i + j) * 32, 2048 + (32 * i + j) * 4
                same(got[s, :, t, a:a + 32], e[:, t, a:a + 32], "codes")
                same(got[s, :, t, b:b + 4], e[:, t, b:b + 4], "scales")
    # ranges, lengths, origins
    lens = r.integers(-2, max_seq + 3, S)
    origin = r.integers(-1, S + 1, (S, max_seq))
    start = max_seq // 3
    got = c.read(start, max_seq - start, max_seq, lens, origin)
    want = np.full(got.shape, FILL, np.float32)
    for s in range(S):
        for p in range(start, min(max(int(lens[s]), 0), max_seq)):
            if 0 <= origin[s, p] < S:
                want[:, s, p - start] = c.values()[:, origin[s, p], p]
    same(got, want)


def test_kv4_append_forms(g2):
    """Rows without lists; positions outside the cache; rows before the first start and behind the last."""
    c = Cache(g2, 3, 2, 50)
    c.append([4, 4, 4], [7, 7, 7], lists=False)
    same(c.read(7, 4, 50), c.values()[:, :, 7:11])
    before = c.buf.download(np.uint8)
    c.append([3, 2, 5], [50, -2, -100], seed=3)
    same(c.buf.download(np.uint8), before)
    c.append([3, 5, 5], [48, -2, 49], seed=4)
    for s, p in ((0, 48), (0, 49), (1, 0), (1, 1), (1, 2), (2, 49)):
        same(c.read(p, 1, 50)[:, s], c.values()[:, s, p:p + 1], f"{s} {p}")
    before = c.buf.download(np.uint8)
    x = np.ones((20, 2 * H), np.float32)
    d = g2.to_device(x)
    for start in ([25, 30, 40, 50], [-9, -7, -5, 0], [20, 10, 5, 0], [2147483647] * 4, [-2147483648] * 4):
        g2.kv4_append(d, d, 2 * H, g2.F32, c.buf, ints(g2, start), ints(g2, [0, 0, 0]), 0, 3, 20, 2, 50)
        same(c.buf.download(np.uint8), before, str(start))
    g2.kv4_append(d, d, 2 * H, g2.F32, c.buf, ints(g2, [0, 1, 2, 3]), ints(g2, [2147483647, -2147483648, 2147483640]), 0, 3, 20, 2, 50)
    same(c.buf.download(np.uint8), before)


def test_kv4_many_sequences(g2):
    """More sequences than one probe of the starts sees, most of them without rows."""
    S = 300
    c = Cache(g2, S, 1, 40)
    r = rng(S)
    c.append([40] * S, [0] * S)
    lens = [int(n) for n in r.integers(0, 3, S) * (r.random(S) < 0.3)]
    c.append(lens, [int(p) for p in r.integers(0, 39, S)], seed=1)
    same(c.read(0, 40, 40), c.values())


def test_kv4_values_out_of_the_ordinary(g2):
    c = Cache(g2, 1, 1, 16)
    r = rng(2)
    x = r.standard_normal((2, 16, H)).astype(np.float32)
    x[:, 0] = 0
    x[:, 1] = -0.0
    x[:, 2] = r.integers(-24, 25, H) * 0.25
    x[:, 3] *= np.float32(2.0 ** -135)
    x[:, 4] *= np.float32(2.0 ** 90)
    x[0, 5, 3], x[1, 5, 40], x[0, 6, 33], x[1, 7, 1] = np.inf, -np.inf, np.nan, np.float32(2.0 ** 96) * np.float32(1.001)
    c.put(x, [0, 16], [0])
    g2.kv4_append(g2.to_device(x[0]), g2.to_device(x[1]), H, g2.F32, c.buf, None, None, 0, 1, 16, 1, 16)
    want = c.values()
    assert np.isnan(want).any() and np.isfinite(want[0, 0, 5, 0, 32:]).all()
    same(c.read(0, 16, 16), want)


def attention_cases():
    """(S, NH, NKV, T) on both sides of every border of a form."""
    return [(1, 1, 1, 1), (1, 1, 1, 33), (2, 4, 4, 100), (1, 2, 1, 64), (3, 6, 2, 65), (2, 4, 1, 129), (1, 5, 1, 200), (1, 7, 1, 31), (2, 16, 2, 257),
            (1, 12, 12, 701), (5, 25, 25, 300), (1, 16, 4, 3000), (1, 1, 1, 5000), (600, 1, 1, 40), (40, 16, 16, 70), (520, 2, 2, 300), (1, 9, 3, 1025),
            (8, 12, 12, 1024), (3, 2, 1, 600), (2, 6, 3, 2500), (1100, 1, 1, 200), (200, 3, 1, 70), (210, 4, 1, 900), (110, 8, 2, 800), (101, 4, 2, 100),
            (100, 4, 2, 1030), (205, 5, 1, 40), (128, 8, 2, 1100)]


ORIGINS = [(4, 4, 4, 40), (8, 12, 12, 901), (6, 8, 2, 300), (3, 5, 1, 1500), (2, 1, 1, 4000), (5, 3, 3, 200), (104, 4, 2, 100), (104, 4, 2, 900), (210, 4, 1, 70),
           (208, 4, 1, 801)]


@pytest.mark.parametrize("S,NH,NKV,T", attention_cases())
def test_attn_kv4(g2, S, NH, NKV, T):
    c = Cache(g2, S, NKV, T + 5)
    c.append([T] * S, [0] * S)
    r = rng(S, NH, T)
    q = r.standard_normal((S, NH, H)).astype(np.float32)
    got, want, bound = c.attend(q, 0.125, T)
    within(got, want, bound, "whole")
    lens = r.integers(-1, T + 3, S)
    lens[0] = 0 if S > 1 else T
    got, want, bound = c.attend(q, 0.3, T, lens, qs=NH * H + 2 * NKV * H + 1, os=NH * H + 3)
    within(got, want, bound, "ragged")
    assert S == 1 or (got[0] == 0).all()


@pytest.mark.parametrize("S,NH,NKV,T", ORIGINS)
def test_attn_kv4_origins(g2, S, NH, NKV, T):
    """Positions in other sequences' slots, and positions that are not there."""
    c = Cache(g2, S, NKV, T + 7)
    c.append([T] * S, [0] * S)
    r = rng(S, NH, T)
    q = r.standard_normal((S, NH, H)).astype(np.float32)
    for lo, hi in ((0, S), (-1, S + 1)):
        origin = r.integers(lo, hi, (S, T + 7))
        got, want, bound = c.attend(q, 0.125, T, origin=origin)
        within(got, want, bound)
    origin[0] = -1  # nothing at all
    origin[1, :T - 1] = 2147483647  # the last position alone
    origin[1, T - 1:] = 0
    got, want, bound = c.attend(q, 0.125, T, r.integers(T - 1, T + 1, S) if S > 2 else None, origin)
    within(got, want, bound)
    assert (got[0] == 0).all()


def test_attn_kv4_not_finite_in_masked_places(g2):
    """What lies behind a length, or at a position that is not there, does not matter; a NaN that is seen does."""
    S, NH, T = 2, 2, 70
    c = Cache(g2, S, 1, T)
    x = rng(5).standard_normal((2, S * T, H)).astype(np.float32)
    x[:, 50] = np.nan
    x[:, T + 10] = np.inf
    start = [0, T, 2 * T]
    c.put(x, start, [0, 0])
    g2.kv4_append(g2.to_device(x[0]), g2.to_device(x[1]), H, g2.F32, c.buf, ints(g2, start), None, 0, S, S * T, 1, T)
    q = rng(6).standard_normal((S, NH, H)).astype(np.float32)
    got, want, bound = c.attend(q, 0.125, T, [50, 10])
    within(got, want, bound)
    origin = np.tile(np.arange(S)[:, None], (1, T))
    origin[0, 50], origin[1, 10] = -1, 5
    got, want, bound = c.attend(q, 0.125, T, None, origin)
    within(got, want, bound)
    got, _, _ = c.attend(q, 0.125, T)
    assert np.isnan(got).all()


# ------------------------------------------------------------------ beam search

def select(g2, logits, score, done, eos, beams, n_out, want_done=True):
    rows, V = logits.shape
    G = rows // beams
    n = G * n_out
    ds = ints(g2, done) if done is not None else None
    os, op, oi, od = guarded(g2, n), guarded(g2, n), guarded(g2, n), guarded(g2, n)
    nw = g2.beam_work_bytes(G, beams, V, n_out)
    work = g2.to_device(np.concatenate([np.zeros(nw, np.uint8), np.full(64, 0xAB, np.uint8)]))
    g2.beam_select(g2.to_device(logits.astype(np.float32)), g2.to_device(np.asarray(score, np.float32)), ds, eos, os, op, oi,
                   od if want_done else None, G, beams, V, n_out, work)
    left = work.download(np.uint8)
    assert (left[nw:nw + 64] == 0xAB).all() and (left[:64 * G] == 0).all()
    s = take(os, n).reshape(G, n_out)
    p, i, d = (take(x, n).view(np.int32).reshape(G, n_out) for x in (op, oi, od))
    return s, p, i, d


def check_select(g2, logits, score, done, eos, beams, n_out):
    """Scores: the largest logit's distance is exact, the sum of exponentials is within 2^-20 of its value (an exponential's
    2^-22 and at most 30 roundings of the sums), the total rounded once."""
    got = select(g2, logits, score, done, eos, beams, n_out)
    want = batch.select(np.asarray(logits, np.float32), np.asarray(score, np.float32), done, eos, beams, n_out)
    for g, w, name in zip(got[1:], want[1:], ("parents", "ids", "ended")):
        same(g, w, name)
    s = want[0]
    none = ~np.isfinite(s)
    same(got[0][none], s[none].astype(np.float32))
    within(got[0][~none], s[~none], 2.0 ** -20 + 2.0 ** -24 * np.abs(s[~none]), "scores")
    return got


@pytest.mark.parametrize("G,beams,V,n_out", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 4), (1, 4, 4095, 4), (3, 5, 4096, 10), (2, 2, 4097, 2), (1, 8, 50257, 8),
                                             (5, 8, 9000, 16), (1, 32, 1000, 64), (2, 32, 5000, 32), (1, 1, 50257, 64), (40, 4, 300, 4), (1, 3, 262144, 5),
                                             (65, 16, 700, 16), (4, 8, 50257, 8), (300, 4, 1030, 3), (33, 1, 33000, 64), (600, 1, 1000, 5), (4, 6, 50257, 20),
                                             (2, 3, 260, 33), (1, 2, 520, 64), (70, 8, 29000, 9), (12, 8, 10000, 8)])
def test_select(g2, G, beams, V, n_out):
    r = rng(G, beams, V, n_out)
    logits = 3 * r.standard_normal((G * beams, V))
    score = -5 + r.standard_normal(G * beams)
    check_select(g2, logits, score, None, V - 1, beams, n_out)
    check_select(g2, logits, score, r.integers(0, 2, G * beams), int(r.integers(0, V)), beams, n_out)
    check_select(g2, logits, np.where(np.arange(G * beams) % beams, -np.inf, 0), None, -1, beams, n_out)
    check_select(g2, logits, score, np.ones(G * beams, int), 0, beams, n_out)


def test_select_ties(g2):
    """Equal sums: the lower beam, then the lower id."""
    for V in (50, 5000, 9001):
        check_select(g2, np.zeros((8, V)), np.zeros(8), None, -1, 4, 9)
        logits = np.zeros((8, V))
        logits[:, [V - 1, 7, V // 2, 3]] = 2
        check_select(g2, logits, np.zeros(8), None, 3, 4, 12)
        logits[:, 11] = -0.0
        check_select(g2, logits, np.zeros(8), np.array([0, 1, 0, 0, 1, 1, 1, 1]), 3, 4, 64)
    check_select(g2, np.zeros((1100, 1024)), np.zeros(1100), None, -1, 11, 64)  # (the wide form, more equal ones than its lists hold)
    check_select(g2, np.zeros((264, 5000)), np.zeros(264), None, -1, 8, 33)


def test_select_beside_each_other(g2):
    """Logits that differ in their last place are told apart, also where the sums in 32 bits are equal."""
    V = 3000
    logits = np.full((2, V), -3.0, np.float32)
    logits[:, 100:140] = np.float32(1) + np.arange(40, dtype=np.float32) * np.float32(2.0 ** -23)
    check_select(g2, logits, [-1000.0, -2000.0], None, -1, 2, 40)


def test_select_not_finite(g2):
    """-infinity is never chosen; a row with a NaN or +infinity goes on in no way, an ended one does."""
    r = rng(9)
    logits = r.standard_normal((6, 4500)).astype(np.float32)
    logits[0, 3], logits[1, 4400], logits[2, :] = np.nan, np.inf, -np.inf
    logits[3, 5:] = -np.inf
    score = np.array([0, 0, 0, 0, np.nan, -np.inf], np.float32)
    s, p, i, d = select(g2, logits, score, None, 2, 6, 8)
    w = batch.select(logits[3:4], score[3:4], None, 2, 1, 5)
    same(p[0], [3] * 5 + [-1] * 3)
    same(i[0, :5], w[2][0])
    assert (i[0, 5:] == -1).all() and np.isneginf(s[0, 5:]).all() and (d[0, 5:] == 0).all()
    s, p, i, d = select(g2, logits, np.zeros(6), np.array([1, 1, 0, 0, 0, 0]), 2, 6, 4)
    same(p[0, :2], [0, 1])
    same(i[0, :2], [2, 2])
    same(d[0, :2], [1, 1])
    same(s[0, :2], [0, 0])


@pytest.mark.parametrize("G,beams,T,stride", [(1, 1, 0, 1), (1, 4, 10, 11), (3, 8, 255, 300), (2, 5, 256, 257), (16, 8, 1001, 1024), (1, 32, 700, 701)])
def test_reorder(g2, G, beams, T, stride):
    R = G * beams
    r = rng(G, beams, T)
    ids, origin = r.integers(0, 50000, (R, stride)).astype(np.int32), r.integers(0, R, (R, stride + 3)).astype(np.int32)
    for lens in (None, r.integers(-2, T + 4, G)):
        n = np.full(G, T) if lens is None else np.clip(lens, 0, T)
        parent = r.integers(-1, beams + 1, R)
        new = r.integers(0, 50000, R)
        want = (batch.reorder(ids, parent, new, n, beams), batch.reorder(origin, parent, np.arange(R), n, beams))
        dp, dn, dl = ints(g2, parent), ints(g2, new), None if lens is None else ints(g2, lens)
        a, b = g2.to_device(ids), g2.to_device(origin)
        g2.beam_reorder(a, a, stride, dn, b, b, stride + 3, dp, dl, T, G, beams)
        same(a.download(np.int32).reshape(R, -1), want[0], "ids in place")
        same(b.download(np.int32).reshape(R, -1), want[1], "origins in place")
        a, b = g2.to_device(ids), g2.to_device(origin)
        oa, ob = g2.to_device(np.full(ids.shape, -9, np.int32)), g2.to_device(np.full(origin.shape, -9, np.int32))
        g2.beam_reorder(a, oa, stride, dn, b, ob, stride + 3, dp, dl, T, G, beams)
        moved = (parent >= 0) & (parent < beams)
        for out, w, src in ((oa, want[0], ids), (ob, want[1], origin)):
            e = np.full(src.shape, -9, np.int32)
            for row in np.flatnonzero(moved):
                e[row, :n[row // beams] + 1] = w[row, :n[row // beams] + 1]
            same(out.download(np.int32).reshape(R, -1), e)
        a = g2.to_device(ids)
        g2.beam_reorder(a, a, stride, dn, None, None, 0, dp, dl, T, G, beams)
        same(a.download(np.int32).reshape(R, -1), want[0], "ids alone")
        b = g2.to_device(origin)
        g2.beam_reorder(None, None, 0, None, b, b, stride + 3, dp, dl, T, G, beams)
        same(b.download(np.int32).reshape(R, -1), want[1], "origins alone")


# ------------------------------------------------------------------ together

class Search:
    """A one-layer model that decodes G prompts with beams: prompts packed, their keys and values in the first beam's
    slot, then steps of one token for every beam.  The model's products are plain numpy on downloaded rows (what is
    tested are the operators), in fp32."""

    NH, NKV, E, V = 4, 2, 256, 500

    def __init__(self, g2, lens, beams, steps, seed=3):
        r = rng(seed, len(lens), beams)
        self.g2, self.lens, self.B, self.G, self.steps = g2, lens, beams, len(lens), steps
        # (short binary fractions: rows of q, k and v come out the same however their sums are ordered, so the cache's codes do)
        self.wte = (r.integers(-4, 5, (self.V, self.E)) / 4).astype(np.float32)
        self.qkv = (r.integers(-6, 7, (self.E, (self.NH + 2 * self.NKV) * H)) / 32).astype(np.float32)
        self.proj = (r.standard_normal((self.NH * H, self.E)) * 0.3).astype(np.float32)
        self.head = (r.standard_normal((self.E, self.V)) * 0.1).astype(np.float32)
        self.prompts = [r.integers(0, self.V - 1, n) for n in lens]
        self.max_seq = max(lens) + steps + 1
        self.eos = self.V - 1

    def logits(self, x, att):
        return ((x + att.reshape(len(x), -1) @ self.proj) @ self.head).astype(np.float32)

    def run(self):
        g2, G, B, R = self.g2, self.G, self.B, self.G * self.B
        ND, KD = self.NH * H, self.NKV * H
        W = ND + 2 * KD
        start = np.concatenate([[0], np.cumsum(self.lens)])
        x = self.wte[np.concatenate(self.prompts)]
        rows = g2.to_device((x @ self.qkv).astype(np.float32))
        ds, att = ints(g2, start), guarded(g2, len(x) * ND)
        g2.attn_prompt(rows, W, rows.offset(4 * ND), rows.offset(4 * (ND + KD)), W, att, ND, g2.F32, ds, ds, G, len(x), len(x), self.NH, self.NKV, 0.125)
        # the cache has a slot for each beam; a group's prompt goes to its first
        cache = g2.to_device(np.full(g2.kv4_bytes(R, self.NKV, self.max_seq), 0xCD, np.uint8))
        of_beam = np.repeat(start[:-1], B) + np.repeat(np.diff(start), B) * (np.arange(R) % B > 0)
        g2.kv4_append(rows.offset(4 * ND), rows.offset(4 * (ND + KD)), W, g2.F32, cache, ints(g2, np.append(of_beam, start[-1])), None, 0, R,
                      len(x), self.NKV, self.max_seq)
        last = start[1:] - 1
        l = self.logits(x[last], take(att, len(x) * ND).reshape(len(x), ND)[last])
        ids = np.zeros((R, self.max_seq), np.int32)
        origin = np.repeat(np.arange(G) * B, B)[:, None] * np.ones((1, self.max_seq), np.int32)
        for g in range(G):
            ids[g * B:(g + 1) * B, :self.lens[g]] = self.prompts[g]
        dids, dorigin = g2.to_device(ids), g2.to_device(origin.astype(np.int32))
        score = g2.to_device(np.zeros(R, np.float32))
        first, work = g2.beam_work(G, 1, self.V, B), g2.beam_work(G, B, self.V, B)
        parent, nxt, done, new, ended = (ints(g2, np.zeros(R)) for _ in range(5))
        # the first choice is among one beam's continuations
        g2.beam_select(g2.to_device(l), g2.to_device(np.zeros(G, np.float32)), None, self.eos, score, parent, nxt, done, G, 1, self.V, B, first)
        n = np.array(self.lens, np.int32)
        g2.beam_reorder(dids, dids, self.max_seq, nxt, dorigin, dorigin, self.max_seq, parent, ints(g2, n), int(n.max()), G, B)
        awork = g2.to_device(np.zeros(g2.kv4_work_bytes(R, self.NH) // 4, np.float32))
        for _ in range(self.steps - 1):
            x = self.wte[nxt.download(np.int32)]
            rows = g2.to_device((x @ self.qkv).astype(np.float32))
            pos = ints(g2, np.repeat(n, B))
            g2.kv4_append(rows.offset(4 * ND), rows.offset(4 * (ND + KD)), W, g2.F32, cache, None, pos, 0, R, R, self.NKV, self.max_seq)
            n = n + 1
            att = guarded(g2, R * ND)
            g2.attn_kv4(rows, W, cache, att, ND, dorigin, ints(g2, np.repeat(n, B)), int(n.max()), R, self.NH, self.NKV, self.max_seq, 0.125, awork)
            l = self.logits(x, take(att, R * ND).reshape(R, ND))
            g2.beam_select(g2.to_device(l), score, done, self.eos, new, parent, nxt, ended, G, B, self.V, B, work)
            score, new, done, ended = new, score, ended, done
            g2.beam_reorder(dids, dids, self.max_seq, nxt, dorigin, dorigin, self.max_seq, parent, ints(g2, n), int(n.max()), G, B)
        ids = dids.download(np.int32).reshape(R, -1)
        return [[list(ids[g * B + b, self.lens[g]:n[g] + 1]) for b in range(B)] for g in range(G)], score.download(np.float32).reshape(G, B)

    def plain(self):
        """The same, a beam at a time, every beam with its whole history in 64 bits (and keys and values rounded as the
        cache holds them, but for the prompt's own attention)."""
        out, scores, gaps = [], [], []
        for p in self.prompts:
            beams = [(0.0, [], False)]
            for step in range(self.steps):
                cand = []
                for b, (s, tail, over) in enumerate(beams):
                    if over:
                        cand.append((s, b, self.eos))
                        continue
                    t = np.concatenate([p, tail]).astype(int)
                    x = self.wte[t]
                    r = (x @ self.qkv).astype(np.float32)
                    q = r[-1:, :self.NH * H].reshape(1, self.NH, H)
                    k, v = (r[:, self.NH * H + i * self.NKV * H:][:, :self.NKV * H].reshape(-1, self.NKV, H) for i in range(2))
                    if step:
                        k, v = batch.to4(k)[0], batch.to4(v)[0]
                    o, _, _ = batch.attend(q, k, v, 0.125, np.ones((1, len(t)), bool))
                    l = ((x[-1:] + o.reshape(1, -1) @ self.proj) @ self.head)[0].astype(np.float64)
                    l = s + l - (l.max() + np.log(np.exp(l - l.max()).sum()))
                    cand += [(l[i], b, i) for i in np.argsort(-l)[:self.B + 1]]
                cand.sort(key=lambda c: (-c[0], c[1], c[2]))
                gaps += [cand[i][0] - cand[i + 1][0] for i in range(min(self.B, len(cand) - 1))]
                beams = [(s, beams[b][1] + [i], beams[b][2] or i == self.eos) for s, b, i in cand[:self.B]]
            out.append([b[1] for b in beams])
            scores.append([b[0] for b in beams])
        return out, np.array(scores), min(gaps)


@pytest.mark.parametrize("lens,beams,steps", [([5, 40, 1], 4, 9), ([33, 64], 3, 12), ([17], 8, 6), ([100], 1, 5)])
def test_several_prompts_with_beams(g2, lens, beams, steps):
    s = Search(g2, lens, beams, steps)
    want, scores, gap = s.plain()
    got, got_scores = s.run()
    assert gap > 1e-4, "the oracle's own choices are too close for this test's model"
    assert [[list(map(int, b)) for b in g] for g in got] == [[list(map(int, b)) for b in g] for g in want]
    within(got_scores, scores, 1e-4 * (1 + np.abs(scores)))


def test_captured_and_replayed(g2):
    """All calls recorded into one graph and replayed with other rows, lengths, starts and beams in the buffers, eager
    calls on other buffers between the replays; every replay bit for bit as the eager calls on the same inputs."""
    from test_lowbit_gpu import _hip

    hip, stream = _hip(), g2._lib.g2_stream()
    NH, NKV, G, B, V, M = 4, 2, 2, 4, 5000, 600

    class State:
        def __init__(self):
            R = G * B
            self.rows = g2.DevBuf(4 * 100 * (NH + 2 * NKV) * H)
            self.att, self.out = g2.DevBuf(4 * 100 * NH * H), g2.DevBuf(4 * R * NH * H)
            self.start, self.row_start, self.pos, self.len = ints(g2, [0] * 4), ints(g2, [0] * (R + 1)), ints(g2, [0] * R), ints(g2, [0] * R)
            self.cache = g2.to_device(np.zeros(g2.kv4_bytes(R, NKV, M), np.uint8))
            self.work = g2.DevBuf(g2.kv4_work_bytes(R, NH))
            self.origin, self.ids = ints(g2, np.zeros((R, M))), ints(g2, np.zeros((R, M)))
            self.logits, self.score, self.done = g2.DevBuf(4 * R * V), g2.DevBuf(4 * R), ints(g2, [0] * R)
            self.new, self.parent, self.next, self.ended = (g2.DevBuf(4 * R) for _ in range(4))
            self.n, self.bwork = ints(g2, [0] * G), g2.beam_work(G, B, V, B)
            self.k, self.v = g2.to_device(np.zeros(R * M * NKV * H, np.float32)), g2.to_device(np.zeros(R * M * NKV * H, np.float32))

        def upload(self, seed):
            r, R = rng(60, seed), G * B
            self.rows.upload(r.standard_normal((100, (NH + 2 * NKV) * H)).astype(np.float32))
            cut = np.sort(r.integers(0, 101, 2))
            self.start.upload(np.array([0, *cut, 100], np.int32))
            self.row_start.upload(np.concatenate([[0], np.sort(r.integers(0, 101, R))]).astype(np.int32))
            self.pos.upload(r.integers(0, M - 100, R).astype(np.int32))
            self.len.upload(r.integers(0, M + 1, R).astype(np.int32))
            self.origin.upload(r.integers(0, R, (R, M)).astype(np.int32))
            self.ids.upload(r.integers(0, V, (R, M)).astype(np.int32))
            self.logits.upload(r.standard_normal((R, V)).astype(np.float32))
            self.score.upload(r.standard_normal(R).astype(np.float32))
            self.done.upload(r.integers(0, 2, R).astype(np.int32))
            self.n.upload(r.integers(0, M, G).astype(np.int32))

        def calls(self):
            W, R = (NH + 2 * NKV) * H, G * B
            k, v = self.rows.offset(4 * NH * H), self.rows.offset(4 * (NH + NKV) * H)
            g2.attn_prompt(self.rows, W, k, v, W, self.att, NH * H, g2.F32, self.start, self.start, 3, 100, 100, NH, NKV, 0.125)
            g2.kv4_append(k, v, W, g2.F32, self.cache, self.row_start, self.pos, 0, R, 100, NKV, M)
            g2.attn_kv4(self.rows, W, self.cache, self.out, NH * H, self.origin, self.len, M, R, NH, NKV, M, 0.125, self.work)
            g2.beam_select(self.logits, self.score, self.done, 7, self.new, self.parent, self.next, self.ended, G, B, V, B, self.bwork)
            g2.beam_reorder(self.ids, self.ids, M, self.next, self.origin, self.origin, M, self.parent, self.n, M - 1, G, B)
            g2.kv4_read(self.cache, self.k, self.v, self.origin, self.len, M, 0, M, R, NKV, M)

        def results(self):
            return [x.download(np.uint32) for x in (self.att, self.out, self.cache, self.new, self.parent, self.next, self.ended, self.ids, self.origin, self.k, self.v)]

    a, b, other = State(), State(), State()
    graph, exe = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    try:
        a.calls()
    finally:
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    try:
        for step in range(6):
            a.upload(step)
            b.upload(step)
            b.calls()
            other.upload(100 + step)
            other.calls()
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            for i, (x, y) in enumerate(zip(a.results(), b.results())):
                same(x, y, f"replay {step}, result {i}")
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
