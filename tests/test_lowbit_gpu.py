"""The decode operators in fewer bits against their oracle (oracle/lowbit.py): what is rounded by definition bit for
bit (4-bit codes and scales, cached values, adjusted logits and picks), products and attention within the rounding
bounds derived here; at the sizes, lengths, strides and values where they can go wrong; together as a decode step;
captured and replayed."""
import ctypes as C

import numpy as np
import pytest

from oracle import lowbit
from parity import EPS32

pytestmark = pytest.mark.gpu

H = 64


def rng(*key):
    return np.random.default_rng(list(key))


def same(got, want, what=""):
    """Bit for bit, but for the sign of zero and the payload of NaN."""
    np.testing.assert_array_equal(np.asarray(got), np.asarray(want), err_msg=what)


def within(got, ref, bound, what=""):
    got, ref = np.asarray(got, np.float64), np.asarray(ref)
    err = np.abs(got - ref)
    ok = bool((err <= bound).all())
    assert ok, f"{what}: {int((err > bound).sum())} of {err.size} off by up to {np.max(err / bound):.3g} bounds"


def guarded(g2, n, fill=7.0):
    """n floats with eight more behind them that nothing may write."""
    return g2.to_device(np.full(n + 8, fill, np.float32))


def take(buf, n, fill=7.0):
    a = buf.download(np.float32, n + 8)
    assert (a[n:] == fill).all(), "written past the end"
    return a[:n]


# ------------------------------------------------------------------ 4-bit weights

def packed(g2, W, group, f16=False, in_out=False):
    N, K = W.shape
    nc, ns = g2.q4_bytes(N, K, group)
    codes, scales = g2.to_device(np.full(nc + 16, 0xAB, np.uint8)), g2.to_device(np.full(ns + 16, 0xAB, np.uint8))
    src = np.ascontiguousarray(W.T if in_out else W)
    g2.quantize_q4(g2.to_device(src.astype(np.float16) if f16 else src), g2.F16 if f16 else g2.F32, in_out, codes, scales, N, K, group)
    return codes, scales


SHAPES = [(1, 1), (3, 31), (16, 32), (17, 33), (15, 127), (16, 128), (33, 129), (70, 300), (129, 1000), (64, 1600), (401, 2055)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", SHAPES)
def test_q4_layout_and_values(g2, N, K, group):
    for f16, in_out in ((False, False), (False, True), (True, False), (True, True)):
        W = (0.02 * rng(N, K, group).standard_normal((N, K))).astype(np.float32)
        W = W.astype(np.float16).astype(np.float32) if f16 else W
        codes, scales = packed(g2, W, group, f16, in_out)
        c, s = lowbit.quantize_q4(W, group)
        ec, es = lowbit.lay_out_q4(c, s, group)
        nc, ns = g2.q4_bytes(N, K, group)
        got = codes.download(np.uint8)
        assert (got[nc:] == 0xAB).all()
        same(got[:nc], ec, f"codes f16 {f16} in_out {in_out}")
        got = scales.download(np.uint8)
        assert (got[ns:] == 0xAB).all()
        same(got[:ns].view(np.uint16), es, "scales")
        for order in (False, True):
            out = guarded(g2, N * K)
            g2.dequantize_q4(codes, scales, out, order, N, K, group)
            want = lowbit.values_q4(c, s, group)
            same(take(out, N * K), (want.T if order else want).ravel().astype(np.float32), "values")


def test_q4_values_out_of_the_ordinary(g2):
    """Zeros of both signs, ties, denormals, the largest scales, groups with infinities and NaN."""
    r = rng(1)
    W = r.standard_normal((48, 160)).astype(np.float32)
    W[0] = 0
    W[1] = -0.0
    W[2, ::3] = 0
    W[3] = r.integers(-24, 25, 160) * 0.25  # many ties at scale 1
    W[3, ::32] = 6
    W[4] *= np.float32(2.0 ** -135)
    W[5] *= np.float32(1e-42)
    W[6] = r.choice(np.float32([0, 1.4e-45, -1.4e-45, 4e-45]), 160)
    W[7] *= np.float32(2.0 ** 94) / np.abs(W[7]).max()
    W[8, 5], W[9, 70], W[10, 100], W[11, 159] = np.inf, -np.inf, np.nan, np.float32(2.0 ** 96) * np.float32(1.001)
    W[12, 33] = 2.0 ** 96
    W[13:20] = r.choice(np.concatenate([lowbit.LEVELS, -lowbit.LEVELS]), (7, 160))
    for group in (32, 64, 128):
        codes, scales = packed(g2, W, group)
        c, s = lowbit.quantize_q4(W, group)
        ec, es = lowbit.lay_out_q4(c, s, group)
        same(codes.download(np.uint8)[:ec.size], ec)
        got = scales.download(np.uint16)[:es.size]
        nan = (es & 0x7FFF) > 0x7F80
        same(got[~nan], es[~nan])
        assert ((got[nan] & 0x7FFF) > 0x7F80).all()


def matvec_bound(x, v, K):
    """|error| of a computed product: each activation enters within 2^-22 of its value (and 2^-38 of the largest of
    its 128: the low half's last place), a sum of K terms goes through at most 160 roundings (128 columns, their
    groups, the parts of an operand) and one for each 128 columns more, the epilogue through 4; each 2^-24."""
    n = 164 + K / 128
    pad = -K % 128
    top = np.abs(np.pad(x, ((0, 0), (0, pad)))).reshape(x.shape[0], -1, 128).max(2).repeat(128, 1)[:, :K]
    return (n * EPS32 + 2.0 ** -22) * (np.abs(x) @ np.abs(v).T) + 2.0 ** -38 * (top @ np.abs(v).T)


def run_matvec(g2, x, codes, scales, N, K, group, bias=None, res=None, gelu=0, shift=0):
    M = x.shape[0]
    dx = g2.to_device(np.concatenate([np.zeros(shift, np.float32), x.ravel().astype(np.float32)]))
    y = guarded(g2, M * N)
    db, dr = (None if t is None else g2.to_device(t) for t in (bias, res))
    g2.matvec_q4(dx.offset(4 * shift), codes, scales, db, dr, y, M, N, K, group, gelu)
    return take(y, M * N).reshape(M, N)


# sizes on both sides of every border of a form: few and many tiles, short and long columns, whole and partial chunks
PRODUCTS = [(1, 1, 32), (5, 40, 64), (16, 128, 128), (17, 129, 32), (50, 257, 64), (100, 768, 128), (768, 768, 64), (333, 1600, 32),
            (1000, 1601, 128), (33, 6400, 64), (40, 9000, 32), (20, 1100, 128), (15, 2100, 32), (18, 2100, 128), (2563, 100, 32)]
# tiles >= 256, >= 512, >= 2048 with 8 and 16 chunks, 16 waves; every group of 32, 64, 128
LARGE = [(N, K, G) for N, K in ((4100, 160), (8200, 200), (8195, 2100), (32780, 130), (32770, 1060)) for G in (32, 64, 128)]
LARGE += [(48, 300, G) for G in (32, 64, 128)] + [(48, 2200, G) for G in (32, 64, 128)] + [(24, 1400, G) for G in (32, 64, 128)]
ROWS, LARGE_ROWS = [1, 2, 3, 7, 8, 9, 16, 21], [1, 3, 9]


def product_cases():
    return [(M, *s) for s in PRODUCTS for M in ROWS] + [(M, *s) for s in LARGE for M in LARGE_ROWS]


_weights = {}


def product_weights(g2, N, K, group):
    """(codes, scales, the values they stand for) of random weights, those of the last sizes kept."""
    if (N, K, group) not in _weights:
        _weights.clear()
        W = (0.02 * rng(N, K).standard_normal((N, K))).astype(np.float32)
        _weights[N, K, group] = (*packed(g2, W, group), lowbit.values_q4(*lowbit.quantize_q4(W, group), group))
    return _weights[N, K, group]


@pytest.mark.parametrize("N,K,group,M", [(*s, M) for s in PRODUCTS for M in ROWS] + [(*s, M) for s in LARGE for M in LARGE_ROWS])
def test_matvec_q4(g2, M, N, K, group):
    r = rng(M, N, K)
    x, bias, res = (r.standard_normal(n).astype(np.float32) for n in ((M, K), N, (M, N)))
    codes, scales, v = product_weights(g2, N, K, group)
    ref, bound = x.astype(np.float64) @ v.T, matvec_bound(x, v, K)
    tiny = 1e-37
    within(run_matvec(g2, x, codes, scales, N, K, group, shift=1), ref, bound + tiny, "plain")
    bound = bound + 4 * EPS32 * (np.abs(ref) + np.abs(bias) + np.abs(res))
    within(run_matvec(g2, x, codes, scales, N, K, group, bias, res), ref + bias + res, bound, "bias and residual")
    # GELU's slope is at most 1.13; its own formula in fp32 costs a few roundings of its terms, the largest below 1 + |y|
    y = ref + bias
    within(run_matvec(g2, x, codes, scales, N, K, group, bias, None, 1), lowbit.gelu(y), 1.13 * bound + 16 * EPS32 * (1 + np.abs(y)), "GELU")


@pytest.mark.parametrize("in_out", [False, True])
def test_q4_beyond_32_bit_offsets(g2, in_out):
    """Codes beyond 4 GB, weights and their values beyond 16 and 32: zeros but for the last five columns."""
    N, K, group, n = 4112, 2 ** 21, 32, 5
    v = (0.02 * rng(41).standard_normal((N, n))).astype(np.float16)
    tail = np.zeros((N, group), np.float32)
    tail[:, -n:] = v
    want = lowbit.values_q4(*lowbit.quantize_q4(tail, group), group)
    nc, ns = g2.q4_bytes(N, K, group)
    assert nc > 2 ** 32
    W, codes, scales = g2.DevBuf(2 * N * K), g2.DevBuf(nc), g2.DevBuf(ns)
    g2.check(g2._lib.g2_memset(W.ptr, 0, 2 * N * K))
    if in_out:
        vt = np.ascontiguousarray(v.T)
        g2.check(g2._lib.g2_upload(W.ptr + 2 * N * (K - n), vt.ctypes.data, v.nbytes))
    else:
        rows = [0, 1, 700, N - 2, N - 1]  # (a copy for each row: a few rows)
        want[[r for r in range(N) if r not in rows]] = 0
        for r in rows:
            g2.check(g2._lib.g2_upload(W.ptr + 2 * ((r + 1) * K - n), v[r].ctypes.data, 2 * n))
    g2.quantize_q4(W, g2.F16, in_out, codes, scales, N, K, group)
    del W
    out = g2.DevBuf(4 * N * K)
    g2.dequantize_q4(codes, scales, out, in_out, N, K, group)
    got = np.empty((40, N) if in_out else (2, K), np.float32)
    g2.check(g2._lib.g2_download(got.ctypes.data, out.ptr + 4 * N * K - got.nbytes, got.nbytes))
    assert (got[:-n] == 0).all() if in_out else (got[:, :-n] == 0).all()
    same(got[-n:].T if in_out else got[:, -n:], want[:, -n:] if in_out else want[-2:, -n:])
    del out
    for M in (1, 9):
        x = rng(42, M).standard_normal((M, K)).astype(np.float32)
        y = run_matvec(g2, x, codes, scales, N, K, group)
        xt = x[:, -n:].astype(np.float64)
        top = np.abs(x[:, -128:]).max(1)[:, None]
        bound = ((164 + K / 128) * EPS32 + 2.0 ** -22) * (np.abs(xt) @ np.abs(want[:, -n:]).T)
        within(y, xt @ want[:, -n:].T, bound + 2.0 ** -38 * top * np.abs(want[:, -n:]).sum(1))


def test_matvec_q4_residual_in_place(g2):
    M, N, K, group = 3, 200, 300, 64
    r = rng(2)
    W, x, res = (r.standard_normal(n).astype(np.float32) for n in ((N, K), (M, K), (M, N)))
    codes, scales = packed(g2, W, group)
    v = lowbit.values_q4(*lowbit.quantize_q4(W, group), group)
    y = g2.to_device(np.concatenate([res.ravel(), np.full(8, 7.0, np.float32)]))
    g2.matvec_q4(g2.to_device(x), codes, scales, None, y, y, M, N, K, group)
    within(take(y, M * N).reshape(M, N), x.astype(np.float64) @ v.T + res, matvec_bound(x, v, K) + 4 * EPS32 * (1 + np.abs(res)) * 40)


@pytest.mark.parametrize("M,N,K,group", [(1, 300, 256, 32), (3, 4500, 200, 64), (1, 32800, 96, 128), (9, 32800, 96, 32)])
def test_matvec_q4_bias_residual_and_gelu(g2, M, N, K, group):
    """All of the epilogue at once: GELU of the product, the bias and the residual."""
    r = rng(33, N)
    W = (0.05 * r.standard_normal((N, K))).astype(np.float32)
    x, bias, res = (r.standard_normal(n).astype(np.float32) for n in ((M, K), N, (M, N)))
    codes, scales = packed(g2, W, group)
    v = lowbit.values_q4(*lowbit.quantize_q4(W, group), group)
    y = x.astype(np.float64) @ v.T + bias + res
    bound = 1.13 * (matvec_bound(x, v, K) + 4 * EPS32 * (np.abs(y) + np.abs(bias) + np.abs(res))) + 16 * EPS32 * (1 + np.abs(y))
    within(run_matvec(g2, x, codes, scales, N, K, group, bias, res, 1), lowbit.gelu(y), bound)


@pytest.mark.parametrize("M", [1, 2, 8, 9])
def test_matvec_q4_range_of_activations(g2, M):
    """Activations of any size: every row scaled differently, columns over 30 orders of magnitude, zeros, denormals."""
    N, K, group = 60, 900, 64
    r = rng(3, M)
    W = (0.02 * r.standard_normal((N, K))).astype(np.float32)
    codes, scales = packed(g2, W, group)
    v = lowbit.values_q4(*lowbit.quantize_q4(W, group), group)
    for size in (1e-41, 1e-30, 1e-6, 70000.0, 1e20, 1e35, "columns", "chunks", "zero"):
        x = r.standard_normal((M, K))
        if size == "columns":
            x *= 10.0 ** r.uniform(-20, 10, (M, K))
        elif size == "chunks":
            x *= np.repeat(10.0 ** r.uniform(-30, 30, (M, 8)), 128, 1)[:, :K]
        else:
            x = x * (0 if size == "zero" else size) * 10.0 ** np.arange(M)[:, None]
        with np.errstate(over="ignore"):
            x = np.clip(x, -1e37, 1e37).astype(np.float32)
        ref = x.astype(np.float64) @ v.T
        # results below fp32's normal range: a last place of 2^-149 for each of their sums
        within(run_matvec(g2, x, codes, scales, N, K, group), ref, matvec_bound(x.astype(np.float64), v, K) + 64 * 2.0 ** -149, size)


@pytest.mark.parametrize("M", [1, 4])
def test_matvec_q4_infinities_and_nan(g2, M):
    """They reach the outputs that a sum over the columns gives them to, and no other row or output."""
    N, K, group = 37, 200, 32
    r = rng(4, M)
    W = r.standard_normal((N, K)).astype(np.float32)
    W[5, 10:40], W[6] = 0, 0
    x = r.standard_normal((M, K)).astype(np.float32)
    x[0, 3], x[0, 100] = np.inf, np.inf
    if M > 1:
        x[1, 150], x[2, 199] = np.nan, -np.inf
    W[9, 40] = np.nan
    codes, scales = packed(g2, W, group)
    v = lowbit.values_q4(*lowbit.quantize_q4(W, group), group)
    with np.errstate(all="ignore"):
        ref = np.array([[(x[m].astype(np.float64) * v[n]).sum() for n in range(N)] for m in range(M)])
    got = run_matvec(g2, x, codes, scales, N, K, group)
    same(np.isnan(got), np.isnan(ref))
    same(got[np.isinf(ref)], ref[np.isinf(ref)])
    f = np.isfinite(ref)
    within(got[f], ref[f], 1e-3)


# ------------------------------------------------------------------ 8-bit cache

def fresh_cache(g2, S, NH, max_seq):
    n = g2.kv8_bytes(S, NH, max_seq)
    return g2.to_device(np.full(n + 64, 0xFF, np.uint8)), n  # NaN everywhere: what is not appended must not be read


def cache_values(g2, cache, lens, S, NH, max_seq, start=0, T=None, T_kv=None):
    """[S][2][T, NH, 64] by kv8_read, rows at or behind the length as they were."""
    T = max_seq - start if T is None else T
    n = S * T * NH * H
    k, v = guarded(g2, n), guarded(g2, n)
    dl = g2.to_device(np.asarray(lens, np.int32))
    g2.kv8_read(cache, k, v, dl, max_seq if T_kv is None else T_kv, start, T, S, NH, max_seq)
    k, v = take(k, n).reshape(S, T, NH, H), take(v, n).reshape(S, T, NH, H)
    for s in range(S):
        for a in (k, v):
            assert (a[s, max(0, min(lens[s], max_seq) - start):] == 7.0).all(), "rows behind the length were written"
    return k, v


def check_cache(g2, cache, models, NH, max_seq):
    S = len(models)
    lens = [m.raw.shape[1] for m in models]
    k, v = cache_values(g2, cache, lens, S, NH, max_seq)
    for s, m in enumerate(models):
        same(k[s, :lens[s]], m.values()[0], f"keys of sequence {s}")
        same(v[s, :lens[s]], m.values()[1], f"values of sequence {s}")


@pytest.mark.parametrize("steps", [[1] * 35, [16, 16, 5], [15, 1, 1], [17, 14, 2, 30, 1], [50], [3, 40, 4]])
def test_kv8_append_in_any_steps(g2, steps):
    NH, max_seq = 3, 64
    D = NH * H
    cache, n = fresh_cache(g2, 1, NH, max_seq)
    m, p = lowbit.Kv8(NH), 0
    for i, T in enumerate(steps):
        qkv = rng(5, i).standard_normal((T, 3 * D)).astype(np.float32)
        g2.kv8_append(g2.to_device(qkv), cache, None, None, p, 1, T, NH, max_seq)
        m.append(p, qkv[:, D:2 * D], qkv[:, 2 * D:])
        p += T
        check_cache(g2, cache, [m], NH, max_seq)
    assert (cache.download(np.uint8)[n:] == 0xFF).all()


@pytest.mark.parametrize("S,NH,max_seq,T", [(1, 1, 1, 1), (2, 1, 15, 15), (3, 5, 33, 20), (4, 12, 100, 37), (2, 25, 257, 250)])
def test_kv8_ragged_batches(g2, S, NH, max_seq, T):
    """Sequences at positions of their own, counts from none to more than the rows, positions behind the cache's end."""
    D = NH * H
    cache, n = fresh_cache(g2, S, NH, max_seq)
    models = [lowbit.Kv8(NH) for _ in range(S)]
    r = rng(6, S, max_seq)
    for turn in range(4):
        pos = np.array([m.raw.shape[1] for m in models], np.int32)
        count = r.integers(-1, T + 3, S).astype(np.int32)
        if turn == 0:
            count[:] = T // 2 + 1
        qkv = r.standard_normal((S, T, 3 * D)).astype(np.float32)
        for s in range(S):
            c = int(np.clip(min(count[s], T), 0, max_seq - pos[s]))
            qkv[s, max(0, min(count[s], T)):] = np.nan  # rows behind the count are not read
            models[s].append(pos[s], qkv[s, :c, D:2 * D], qkv[s, :c, 2 * D:])
        g2.kv8_append(g2.to_device(qkv), cache, g2.to_device(pos), g2.to_device(count), 0, S, T, NH, max_seq)
        check_cache(g2, cache, models, NH, max_seq)
    before = cache.download(np.uint8)
    for bad in (-1, max_seq, -2 ** 31, 2 ** 31 - 1):  # sequences altogether outside
        g2.kv8_append(g2.to_device(qkv), cache, g2.to_device(np.full(S, bad, np.int32)), None, 0, S, T, NH, max_seq)
    after = cache.download(np.uint8)
    same(after, before)
    assert (after[n:] == 0xFF).all()


def test_kv8_cut_back_and_read_in_part(g2):
    NH, max_seq, D = 2, 80, 128
    cache, _ = fresh_cache(g2, 1, NH, max_seq)
    r = rng(7)
    m = lowbit.Kv8(NH)
    for p, T in ((0, 45), (34, 20), (48, 3), (49, 31)):  # back within the last block, to a block's begin, within one again
        qkv = r.standard_normal((T, 3 * D)).astype(np.float32)
        if p == 34:  # (a cut into the last block, which 45 positions left at 32)
            assert m.raw.shape[1] == 45
        g2.kv8_append(g2.to_device(qkv), cache, None, None, p, 1, T, NH, max_seq)
        m.append(p, qkv[:, D:2 * D], qkv[:, 2 * D:])
        check_cache(g2, cache, [m], NH, max_seq)
    full = m.values()
    for start, T in ((0, 1), (15, 2), (31, 40), (79, 1)):
        k, v = cache_values(g2, cache, [80], 1, NH, max_seq, start, T)
        same(k[0], full[0, start:start + T])
        same(v[0], full[1, start:start + T])
    k, _ = cache_values(g2, cache, [-5], 1, NH, max_seq)  # a length below 0 is 0, one above T_kv is T_kv
    k, _ = cache_values(g2, cache, [48], 1, NH, max_seq, 0, 48, 48)
    same(k[0], full[0, :48])


def test_kv8_values_out_of_the_ordinary(g2):
    """Blocks of zeros, denormals, huge and tiny values, half steps; an infinity or NaN makes its block NaN and no other."""
    NH, T, D = 1, 16 * 9, 64
    r = rng(8)
    x = r.standard_normal((T, 3 * D)).astype(np.float32)
    b = x.reshape(9, 16, 3 * D)
    b[0] = 0
    b[1] *= np.float32(1e-41)
    b[2] = r.choice(np.float32([0, 1.4e-45, -2.8e-45]), (16, 3 * D))
    b[3] *= np.float32(1e38) / np.abs(b[3]).max()
    b[4] = r.integers(-254, 255, (16, 3 * D)) * 0.5
    b[4, 0] = 127
    b[5, 3, 70], b[6, 5, 140], b[7, 0, 90] = np.inf, np.nan, -np.inf
    cache, _ = fresh_cache(g2, 1, NH, T)
    g2.kv8_append(g2.to_device(x), cache, None, None, 0, 1, T, NH, T)
    m = lowbit.Kv8(NH)
    m.append(0, x[:, D:2 * D], x[:, 2 * D:])
    k, v = cache_values(g2, cache, [T], 1, NH, T)
    same(k[0], m.values()[0])
    same(v[0], m.values()[1])
    assert np.isnan(k[0, 80:96]).all() and np.isnan(v[0, 96:112]).all() and np.isfinite(v[0, 80:96]).all()


# ------------------------------------------------------------------ attention

def attend_bound(q, kv, scale, T):
    """A score's error: 2^-24 of the sum of its 64 products' magnitudes for each of their 64 sums and of 8 more steps
    (scales, the exponent's argument), and of its distance from the maximum for the exponent's own rounding; it moves
    a weight by as much, the normalised output by twice that; sums over positions (a quarter of T in a chain, 200 for
    the joining of parts) round each time, numerator and denominator."""
    out, pv, mag, spread = lowbit.attend(q, kv, scale)
    d = EPS32 * (72 * mag + 8 * spread + 8)
    return out, pv * (2 * np.expm1(d) + 2 * EPS32 * (T / 4 + 200))[:, None] + 1e-37


def run_attend(g2, q, cache, lens, T_kv, S, NH, max_seq, scale, q_stride=None, out_stride=None, shift=0):
    D = NH * H
    q_stride, out_stride = q_stride or D, out_stride or D
    buf = np.full(shift + S * q_stride, np.nan, np.float32)
    for s in range(S):
        buf[shift + s * q_stride:shift + s * q_stride + D] = q[s].ravel()
    n = (S - 1) * out_stride + D
    out = g2.to_device(np.full(shift + n + 8, 7.0, np.float32))
    work = g2.to_device(np.full(g2.kv8_work_bytes(S, NH) // 4 + 8, np.nan, np.float32))
    dq, dl = g2.to_device(buf), None if lens is None else g2.to_device(np.asarray(lens, np.int32))
    g2.attn_kv8(dq.offset(4 * shift), q_stride, cache, out.offset(4 * shift), out_stride, dl, T_kv, S, NH, max_seq, scale, work)
    got = out.download(np.float32)
    assert (got[:shift] == 7.0).all() and (got[shift + n:] == 7.0).all()
    got = got[shift:shift + n]
    for s in range(S - 1):
        assert (got[s * out_stride + D:(s + 1) * out_stride] == 7.0).all(), "written between the rows"
    assert np.isnan(work.download(np.float32)[-8:]).all()
    return np.stack([got[s * out_stride:s * out_stride + D].reshape(NH, H) for s in range(S)])


def filled_cache(g2, S, NH, max_seq, lens, seed, size=1.0):
    cache, _ = fresh_cache(g2, S, NH, max_seq)
    D, T = NH * H, max(max(lens), 1)
    qkv = (size * rng(seed).standard_normal((S, T, 3 * D))).astype(np.float32)
    g2.kv8_append(g2.to_device(qkv), cache, g2.to_device(np.zeros(S, np.int32)), g2.to_device(np.asarray(lens, np.int32)), 0, S, T, NH,
                  max_seq)
    models = []
    for s in range(S):
        models.append(lowbit.Kv8(NH))
        models[s].append(0, qkv[s, :lens[s], D:2 * D], qkv[s, :lens[s], 2 * D:])
    return cache, models


LENGTHS = [(1, 2100), (12, 1024), (25, 1100), (3, 1003), (20, 14000)]
BATCHES = [(1, 2, 40, [1]), (4, 3, 64, [0, 1, 15, 64]), (7, 12, 130, [17, 16, 33, 0, 129, 130, 31]), (3, 25, 700, [699, 5, 345]),
           (40, 4, 90, [(37 * i) % 91 for i in range(40)]), (2, 1, 3000, [2999, 1500]), (70, 12, 50, [(11 * i) % 51 for i in range(70)]),
           (45, 12, 128, [(29 * i) % 129 for i in range(45)]), (5, 3, 1500, [1490, 1499, 0, 1, 700])]


def attention_cases():
    """(sequences x heads, bound of the lengths) of the tests below."""
    return [(NH, top) for NH, top in LENGTHS] + [(NH, 64) for NH, _ in LENGTHS] + [(S * NH, m) for S, NH, m, _ in BATCHES]


@pytest.mark.parametrize("NH,max_seq", LENGTHS)
def test_attend_lengths(g2, NH, max_seq):
    top = max_seq
    cache, (m,) = filled_cache(g2, 1, NH, max_seq, [top], NH)
    q = 2 * rng(9, NH).standard_normal((1, NH, H)).astype(np.float32)
    full = m.values()
    # whole blocks are the same at any length; a length inside a block would need its fp32 rows, so lengths are whole
    # blocks and the whole cache
    for T in [0, 16, 32, 48, 64, 80, 128, 256, 272, 512, 640, 1008, 1024, 1040, 2096, 5008, 13984, top]:
        if T > top or (T % 16 and T != top):
            continue
        got = run_attend(g2, q, cache, None, T, 1, NH, max_seq, 0.125)
        ref, bound = attend_bound(q[0], full[:, :T], 0.125, T)
        within(got[0], ref, bound, f"length {T}")


@pytest.mark.parametrize("S,NH,max_seq,lens", BATCHES)
def test_attend_batches(g2, S, NH, max_seq, lens):
    cache, models = filled_cache(g2, S, NH, max_seq, lens, 10)
    q = rng(11, S).standard_normal((S, NH, H)).astype(np.float32)
    D = NH * H
    for q_stride, out_stride, shift in ((D, D, 0), (3 * D, D + 5, 1)):
        got = run_attend(g2, q, cache, lens, max_seq, S, NH, max_seq, 0.125, q_stride, out_stride, shift)
        for s in range(S):
            ref, bound = attend_bound(q[s], models[s].values(), 0.125, lens[s])
            within(got[s], ref, bound, f"sequence {s} of length {lens[s]}")
    # lengths above T_kv are T_kv, below 0 are 0 (T_kv whole blocks: see above)
    cut = max(lens) // 16 * 16
    if cut:
        got = run_attend(g2, q, cache, [10 ** 9 if n >= cut else -3 for n in lens], cut, S, NH, max_seq, 0.125)
        for s in range(S):
            if lens[s] >= cut:
                ref, bound = attend_bound(q[s], models[s].values()[:, :cut], 0.125, cut)
                within(got[s], ref, bound)
            else:
                assert (got[s] == 0).all()


@pytest.mark.parametrize("scale,size", [(0.125, 30.0), (-0.125, 1.0), (0.0, 1.0), (1e-3, 1e3), (1.0, 1e-20), (1e-20, 1e10)])
def test_attend_scores_of_any_size(g2, scale, size):
    """One key that takes all the weight, equal weights, negative scales, values of other magnitudes."""
    S, NH, max_seq, lens = 2, 3, 200, [200, 77]
    cache, models = filled_cache(g2, S, NH, max_seq, lens, 12, size)
    q = rng(13).standard_normal((S, NH, H)).astype(np.float32)
    got = run_attend(g2, q, cache, lens, max_seq, S, NH, max_seq, scale)
    for s in range(S):
        ref, bound = attend_bound(q[s], models[s].values(), float(np.float32(scale)), lens[s])
        within(got[s], ref, bound, f"sequence {s}")


def test_attend_infinities_and_nan(g2):
    """A NaN or infinite query, a block of NaN: their heads are NaN, the others as before."""
    NH, max_seq, T = 4, 64, 50
    D = NH * H
    cache, (m,) = filled_cache(g2, 1, NH, max_seq, [T], 14)
    q = rng(15).standard_normal((1, NH, H)).astype(np.float32)
    q[0, 1, 5], q[0, 2, 9] = np.nan, np.inf
    got = run_attend(g2, q, cache, None, T, 1, NH, max_seq, 0.125)
    assert np.isnan(got[0, 1:3]).all()
    qkv = np.ones((1, 3 * D), np.float32)
    qkv[0, D + 3 * H] = np.inf  # a key of head 3, still in the incomplete block
    g2.kv8_append(g2.to_device(qkv), cache, None, None, T, 1, 1, NH, max_seq)
    got = run_attend(g2, q, cache, None, T + 1, 1, NH, max_seq, 0.125)
    m.append(T, qkv[:, D:2 * D], qkv[:, 2 * D:])
    ref, bound = attend_bound(q[0], np.nan_to_num(m.values(), posinf=1.0), 0.125, T + 1)
    within(got[0, 0], ref[0], bound[0])
    if q[0, 3, 0] > 0:
        assert np.isnan(got[0, 3]).all()  # infinite score: inf - inf
    assert not np.isfinite(got[0, 3]).all() or q[0, 3, 0] < 0
    qkv = np.ones((13, 3 * D), np.float32)  # the block fills: its keys of head 3 are NaN altogether, no other head's
    g2.kv8_append(g2.to_device(qkv), cache, None, None, T + 1, 1, 13, NH, max_seq)
    got = run_attend(g2, q, cache, None, 64, 1, NH, max_seq, 0.125)
    m.append(T + 1, qkv[:, D:2 * D], qkv[:, 2 * D:])
    ref, bound = attend_bound(q[0], np.nan_to_num(m.values(), nan=1.0), 0.125, 64)
    within(got[0, 0], ref[0], bound[0])
    assert np.isnan(got[0, 1:]).all()


def test_attend_beyond_32_bit_offsets(g2):
    """A cache whose last head's codes lie beyond 4 GB: zeros but for its last positions."""
    NH, max_seq = 17, 2 ** 21
    D = NH * H
    n = g2.kv8_bytes(1, NH, max_seq)
    assert n > 2 ** 32
    cache = g2.DevBuf(n)
    g2.check(g2._lib.g2_memset(cache.ptr, 0, n))
    T, start = 37, max_seq - 48
    qkv = rng(16).standard_normal((T, 3 * D)).astype(np.float32)
    g2.kv8_append(g2.to_device(qkv), cache, None, None, start, 1, T, NH, max_seq)
    m = lowbit.Kv8(NH)
    m.append(0, qkv[:, D:2 * D], qkv[:, 2 * D:])
    k, v = cache_values(g2, cache, [start + T], 1, NH, max_seq, start, 48)
    vals = m.values()
    same(k[0, :T], vals[0])
    same(v[0, :T], vals[1])
    q = 8 * rng(17).standard_normal((1, NH, H)).astype(np.float32)
    got = run_attend(g2, q, cache, None, start + T, 1, NH, max_seq, 0.125)
    s = np.einsum("hd,thd->ht", q[0].astype(np.float64), vals[0].astype(np.float64)) * 0.125
    e = np.exp(s)
    den = start + e.sum(1)
    ref = np.einsum("ht,thd->hd", e, vals[1].astype(np.float64)) / den[:, None]
    mag = np.einsum("hd,thd->ht", np.abs(q[0]), np.abs(vals[0])).max(1) * 0.125
    pv = np.einsum("ht,thd->hd", e, np.abs(vals[1])) / den[:, None]
    d = EPS32 * (80 * mag + 8)
    within(got[0], ref, pv * (2 * np.expm1(d) + 2 * EPS32 * (max_seq / 64 + 400))[:, None])


# ------------------------------------------------------------------ rules on logits

def run_rules(g2, l, pick=True, out=True, in_place=False, **kw):
    R, V = l.shape
    dl = guarded(g2, R * V)
    l = np.ascontiguousarray(l)
    g2.check(g2._lib.g2_upload(dl.ptr, l.ctypes.data, l.nbytes))
    do = dl if in_place else guarded(g2, R * V) if out else None
    dp = g2.to_device(np.full(R + 4, 77, np.int32)) if pick else None
    work = g2.to_device(np.zeros(g2.logits_work_bytes(R) + 8, np.uint8)) if pick else None
    dev = {k: g2.to_device(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    g2.apply_logit_rules(dl, do, dp, R, V, g2.logit_rules(**dev), work)
    ids = None
    if pick:
        ids = dp.download(np.int32)
        assert (ids[R:] == 77).all()
        ids = ids[:R]
        assert (work.download(np.uint8) == 0).all()  # left as it has to be for the next call
    return (take(do, R * V).reshape(R, V) if do is not None else None), ids


def bits(allowed, stride):
    R, V = allowed.shape
    m = np.zeros((R, stride), np.uint32)
    for v in range(V):
        m[:, v // 32] |= allowed[:, v].astype(np.uint32) << np.uint32(v % 32)
    return m


@pytest.mark.parametrize("R,V", [(1, 1), (1, 31), (2, 33), (3, 1000), (2, 1025), (5, 4097), (1, 50257), (9, 50257), (2, 65537), (1, 262144)])
def test_rules(g2, R, V):
    r = rng(18, R, V)
    for turn in range(3):
        l = (4 * r.standard_normal((R, V))).astype(np.float32)
        l[:, r.integers(0, V, 5)] = l.max()  # equal ones
        n, nb = int(r.integers(1, 300)), int(r.integers(1, 60))
        ctx = (V * r.random((R, n)) ** 3).astype(np.int32)
        ctx[r.random((R, n)) < 0.05] = r.choice([-1, V, -2 ** 31, 2 ** 31 - 1])
        lens = r.integers(-1, n + 2, R).astype(np.int32)
        bid = r.integers(-2, V + 2, nb).astype(np.int32)
        bid[nb // 2:] = bid[:nb - nb // 2]  # ids twice
        bias = (3 * r.standard_normal(nb)).astype(np.float32)
        stride = (V + 31) // 32 + turn
        allowed = r.random((R, V)) < (0.5 if turn else 0.02)
        rep, freq, pres = [(1.3, 0.25, 0.5), (1.0, -0.7, 0.1), (0.8, 0.0, -2.0)][turn]
        forbid = int(r.integers(0, V)) if turn else -1
        shared = turn == 2
        kw = dict(ctx=ctx, ctx_len=lens if turn != 1 else None, max_ctx=n, repetition=rep, frequency=freq, presence=pres, bias_id=bid,
                  bias=bias, n_bias=nb, mask=bits(allowed, stride), mask_stride=0 if shared else stride, forbid=forbid)
        want = [lowbit.rules(l[i], ctx[i, :max(0, min(lens[i], n))] if turn != 1 else ctx[i], rep, freq, pres, zip(bid, bias),
                             allowed[0 if shared else i], forbid) for i in range(R)]
        got, ids = run_rules(g2, l, **kw)
        same(got, [w[0] for w in want])
        same(ids, [w[1] for w in want])
        got, ids = run_rules(g2, l, in_place=True, **kw)
        same(got, [w[0] for w in want])
        same(ids, [w[1] for w in want])
        same(run_rules(g2, l, out=False, **kw)[1], ids)
        same(run_rules(g2, l, pick=False, **kw)[0], [w[0] for w in want])


def test_rules_one_at_a_time(g2):
    R, V = 2, 3000
    r = rng(19)
    l = r.standard_normal((R, V)).astype(np.float32)
    l[0, :10] = [np.inf, -np.inf, np.nan, 0.0, -0.0, 1e38, -1e38, 1e-44, 3.0, 3.0]
    ctx = np.tile(np.arange(12, dtype=np.int32), (R, 3))
    for kw, ref in ((dict(), dict()), (dict(forbid=0), dict(forbid=0)), (dict(ctx=ctx, max_ctx=36, repetition=2.0), dict(repetition=2.0)),
                    (dict(ctx=ctx, max_ctx=36, repetition=0.0), dict()), (dict(ctx=ctx, max_ctx=36, frequency=1e38), dict(frequency=1e38)),
                    (dict(ctx=ctx, max_ctx=36, presence=0.1), dict(presence=0.1)), (dict(ctx=ctx, max_ctx=0, presence=0.1), dict())):
        got, ids = run_rules(g2, l, **kw)
        want = [lowbit.rules(l[i], ctx[i] if kw.get("max_ctx") else None, **ref) for i in range(R)]
        same(got, [w[0] for w in want])
        same(ids, [w[1] for w in want])


def test_rules_that_leave_nothing(g2):
    """A mask of zeros, logits of -infinity or NaN alone: pick -1; a NaN is never picked."""
    l = rng(20).standard_normal((4, 2000)).astype(np.float32)
    l[1], l[2] = -np.inf, np.nan
    l[3] = np.nan
    l[3, 1999] = -3e38
    none = np.zeros((4, 63), np.uint32)
    out, ids = run_rules(g2, l, mask=none, mask_stride=63)
    assert (ids == -1).all() and (out == -np.inf).all()
    same(run_rules(g2, l)[1], [int(l[0].argmax()), -1, -1, 1999])
    same(run_rules(g2, l, out=False, forbid=1999)[1][1:], [-1, -1, -1])


def test_calls_give_the_same_bits_again(g2):
    """No result depends on an order of atomics or on what an earlier call left: calls of other sizes between, the same
    workspaces."""
    S, NH, max_seq, V = 3, 5, 3000, 50257
    lens = [3000, 17, 1600]
    cache, _ = filled_cache(g2, S, NH, max_seq, lens, 30)
    small, _ = filled_cache(g2, 2, 3, 2000, [2000, 1999], 31)
    r = rng(32)
    q = g2.to_device(r.standard_normal((S, NH * H)).astype(np.float32))
    dl, work = g2.to_device(np.asarray(lens, np.int32)), g2.DevBuf(g2.kv8_work_bytes(S, NH))
    out = g2.DevBuf(4 * S * NH * H)
    logits = g2.to_device(r.standard_normal((30, V)).astype(np.float32))
    ctx = g2.to_device(r.integers(0, 300, (30, 500)).astype(np.int32))
    lwork, lo, pick = g2.logits_work(30), g2.DevBuf(120 * V), g2.DevBuf(120)
    rules = g2.logit_rules(ctx=ctx, max_ctx=500, repetition=1.3, presence=0.1)
    first = None
    for turn in range(6):
        g2.attn_kv8(q, NH * H, cache, out, NH * H, dl, max_seq, S, NH, max_seq, 0.125, work)
        g2.apply_logit_rules(logits, lo, pick, 30, V, rules, lwork)
        got = [b.download(np.float32) for b in (out, lo)] + [pick.download(np.int32)]
        first = first or got
        for a, b in zip(got, first):
            same(a.view(np.uint32), b.view(np.uint32))
        g2.attn_kv8(q, 192, small, out, 192, None, 1999 - turn, 2, 3, 2000, 0.3, work)
        g2.apply_logit_rules(logits, lo, pick, 3 + turn, 2000 * (turn + 1), rules, lwork)


# ------------------------------------------------------------------ together

class Step:
    """A decode step of a small GPT-2 over these operators and the ones beside them: 4-bit matrices, 8-bit cache, the
    token chosen on the device; for S sequences at once."""

    def __init__(self, g2, S, NH=2, L=2, V=700, max_seq=64, seed=21):
        r = rng(seed)
        E = NH * H
        self.g2, self.S, self.NH, self.L, self.V, self.E, self.F, self.max_seq = g2, S, NH, L, V, E, 4 * E, max_seq
        mats = lambda n, k, g: (0.06 * r.standard_normal((n, k))).astype(np.float32)  # noqa: E731
        vec = lambda n, m, s: (m + s * r.standard_normal(n)).astype(np.float32)  # noqa: E731
        self.groups = {"qkv": 32, "proj": 64, "fc": 64, "fc2": 128, "head": 32}
        sizes = {"qkv": (3 * E, E), "proj": (E, E), "fc": (4 * E, E), "fc2": (E, 4 * E)}
        self.layers = []
        for _ in range(L):
            w = {n: mats(*sizes[n], self.groups[n]) for n in sizes}
            b = {n: vec(sizes[n][0], 0, 0.05) for n in sizes}
            ln = [vec(E, 1, 0.1), vec(E, 0, 0.1), vec(E, 1, 0.1), vec(E, 0, 0.1)]
            self.layers.append((w, b, ln))
        self.head = mats(V, E, 32)
        self.wte, self.wpe = vec((V, E), 0, 0.5), vec((1024, E), 0, 0.2)
        self.lnf = [vec(E, 1, 0.1), vec(E, 0, 0.1)]
        # device copies
        self.d = []
        for w, b, ln in self.layers:
            self.d.append(({n: packed(g2, w[n], self.groups[n], in_out=n in ("fc", "qkv")) for n in w}, {n: g2.to_device(b[n]) for n in b},
                           [g2.to_device(x) for x in ln], g2.DevBuf(g2.kv8_bytes(S, NH, max_seq))))
        self.dhead = packed(g2, self.head, 32)
        self.dwte, self.dwpe, self.dlnf = g2.to_device(self.wte), g2.to_device(self.wpe), [g2.to_device(x) for x in self.lnf]
        f = lambda n: g2.DevBuf(4 * n)  # noqa: E731
        self.x, self.n, self.qkv, self.att, self.h = f(S * E), f(S * E), f(S * 3 * E), f(S * E), f(S * 4 * E)
        self.logits, self.out, self.pick = f(S * V), f(S * V), f(S)
        self.work, self.lwork = g2.DevBuf(g2.kv8_work_bytes(S, NH)), g2.logits_work(S)
        self.ids, self.pos, self.len = g2.DevBuf(4 * S), g2.DevBuf(4 * S), g2.DevBuf(4 * S)
        self.ctx, self.ctx_len = g2.DevBuf(4 * S * max_seq), g2.DevBuf(4 * S)

    def upload(self, ids, pos, ctx):
        i32 = lambda a: np.asarray(a, np.int32)  # noqa: E731
        self.ids.upload(i32(ids)), self.pos.upload(i32(pos)), self.len.upload(i32(pos) + 1)
        pad = np.zeros((self.S, self.max_seq), np.int32)
        for s, c in enumerate(ctx):
            pad[s, :len(c)] = c
        self.ctx.upload(pad), self.ctx_len.upload(i32([len(c) for c in ctx]))

    def calls(self, start):
        """The launches of one step, all sequences' embeddings at position `start`."""
        g2, S, E, NH, L = self.g2, self.S, self.E, self.NH, self.L
        for s in range(S):  # (the embedding takes one run of positions)
            g2.embed(self.dwte, self.dwpe, self.x.offset(4 * s * E), E, 1, start, self.ids.offset(4 * s))

        def mat(x, name, layer, y, n, k, res=None, gelu=0):
            codes, scales = self.d[layer][0][name]
            g2.matvec_q4(x, codes, scales, self.d[layer][1][name], res, y, S, n, k, self.groups[name], gelu)

        for i, (_, _, ln, cache) in enumerate(self.d):
            g2.layernorm(self.x, self.n, ln[0], ln[1], E, S)
            mat(self.n, "qkv", i, self.qkv, 3 * E, E)
            g2.kv8_append(self.qkv, cache, self.pos, None, 0, S, 1, NH, self.max_seq)
            g2.attn_kv8(self.qkv, 3 * E, cache, self.att, E, self.len, self.max_seq, S, NH, self.max_seq, 0.125, self.work)
            mat(self.att, "proj", i, self.x, E, E, self.x)
            g2.layernorm(self.x, self.n, ln[2], ln[3], E, S)
            mat(self.n, "fc", i, self.h, 4 * E, E, None, 1)
            mat(self.h, "fc2", i, self.x, E, 4 * E, self.x)
        g2.layernorm(self.x, self.n, self.dlnf[0], self.dlnf[1], E, S)
        g2.matvec_q4(self.n, *self.dhead, None, None, self.logits, S, self.V, E, 32)
        g2.apply_logit_rules(self.logits, self.out, self.pick, S, self.V,
                             g2.logit_rules(ctx=self.ctx, ctx_len=self.ctx_len, max_ctx=self.max_seq, repetition=1.2, presence=0.3, forbid=3),
                             self.lwork)

    def reference(self):
        """A function of (ids, pos) that runs one step of every sequence in 64 bits, keeping its caches."""
        S, E, NH = self.S, self.E, self.NH
        val = [{n: lowbit.values_q4(*lowbit.quantize_q4(w[n], self.groups[n]), self.groups[n]) for n in w} for w, _, _ in self.layers]
        head = lowbit.values_q4(*lowbit.quantize_q4(self.head, 32), 32)
        caches = [[lowbit.Kv8(NH) for _ in range(S)] for _ in range(self.L)]

        def ln(x, g, b):
            m = x.mean()
            return (x - m) / np.sqrt(((x - m) ** 2).mean() + 1e-5) * g + b

        def step(ids, pos):
            out = []
            for s in range(S):
                x = self.wte[ids[s]].astype(np.float64) + self.wpe[pos[s]]
                for i, (_, b, g) in enumerate(self.layers):
                    qkv = val[i]["qkv"] @ ln(x, g[0], g[1]) + b["qkv"]
                    c = caches[i][s]
                    c.append(pos[s], qkv[None, E:2 * E].astype(np.float32), qkv[None, 2 * E:].astype(np.float32))
                    a = lowbit.attend(qkv[:E].reshape(NH, H), c.values(), 0.125)[0].ravel()
                    x = x + val[i]["proj"] @ a + b["proj"]
                    h = lowbit.gelu(val[i]["fc"] @ ln(x, g[2], g[3]) + b["fc"])
                    x = x + val[i]["fc2"] @ h + b["fc2"]
                out.append(head @ ln(x, *self.lnf))
            return np.array(out)

        return step


def test_decode_steps_together(g2):
    """Two sequences decoded for 40 tokens (over two block ends) against the same in 64 bits.  The caches' codes are
    chosen from keys that differ in their last places, so a code may fall on the other side of a border: one step of
    1/127 of a block's largest value in one of thousands of values; logits of size 5 then agree to 1e-2, others to
    1e-4 (about 20 roundings of 2^-24 per operator and 15 operators a layer, times the size of a logit, is 1e-4)."""
    S = 2
    t = Step(g2, S)
    ref = t.reference()
    ids, ctx = [5, 11], [[5], [11]]
    worst, far = 0.0, 0
    for pos in range(40):
        t.upload(ids, [pos] * S, ctx)
        t.calls(pos)
        got = t.logits.download(np.float32).reshape(S, t.V)
        want = ref(ids, [pos] * S)
        err = np.abs(got - want).max()
        worst, far = max(worst, err), far + (err > 1e-4)
        assert err < 1e-2, f"position {pos}: logits differ by {err:.2e}"
        picks = t.pick.download(np.int32)
        out = t.out.download(np.float32).reshape(S, t.V)
        for s in range(S):
            l, p = lowbit.rules(got[s], ctx[s], 1.2, 0.0, 0.3, forbid=3)
            same(out[s], l)
            assert picks[s] == p
            ids[s] = int(p)
            ctx[s].append(int(p))
    print(f"\n[lowbit] 40 steps, logits differ by at most {worst:.2e}, {far} steps above 1e-4", flush=True)


def _hip():
    hip = C.CDLL("libamdhip64.so")
    vp = C.c_void_p
    hip.hipStreamBeginCapture.argtypes = [vp, C.c_int]
    hip.hipStreamEndCapture.argtypes = [vp, C.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [C.POINTER(vp), vp, vp, vp, C.c_size_t]
    hip.hipGraphLaunch.argtypes = [vp, vp]
    hip.hipStreamSynchronize.argtypes = [vp]
    hip.hipGraphExecDestroy.argtypes = [vp]
    hip.hipGraphDestroy.argtypes = [vp]
    return hip


def test_captured_step_replayed(g2):
    """One step recorded into a graph on the library's stream and replayed for other tokens and positions (both are
    device arrays), with eager steps of other buffers between; every replay against the eager result, bit for bit.
    (The embedding's position is an argument, so the graph keeps the recorded one; the eager step takes the same.)"""
    hip = _hip()
    stream = g2._lib.g2_stream()
    a, b, other = Step(g2, 2), Step(g2, 2), Step(g2, 3, seed=22)
    graph, exe = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    try:
        a.calls(4)
    finally:
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    try:
        ids, ctx = [7, 8], [[7], [8, 1]]
        for pos in range(20):
            p = [pos, pos // 2]
            for t in (a, b):
                t.upload(ids, p, ctx)
            b.calls(4)
            other.upload([1, 2, 3], [pos] * 3, [[1], [2], [3]])
            other.calls(pos)
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            same(a.out.download(np.float32), b.out.download(np.float32), f"replay {pos}")
            same(a.pick.download(np.int32), b.pick.download(np.int32))
            ids = b.pick.download(np.int32).tolist()
            for s in range(2):
                ctx[s] = (ctx[s] + [ids[s]])[-60:]
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
