"""What the header allows of the decode operators in fewer bits beyond test_lowbit_gpu.py's calls: cutting a sequence
back from a block that is full; activations beside far larger ones."""
import numpy as np
import pytest

import test_lowbit_gpu as base
from oracle import lowbit
from parity import EPS32

pytestmark = pytest.mark.gpu

H = base.H


# ------------------------------------------------------------------ 8-bit cache: cutting back

def appended(g2, cache, m, p, T, NH, max_seq, key):
    """T rows at position p, to the cache and to its model."""
    D = NH * H
    qkv = base.rng(50, key, p, T).standard_normal((T, 3 * D)).astype(np.float32)
    g2.kv8_append(g2.to_device(qkv), cache, None, None, p, 1, T, NH, max_seq)
    m.append(p, qkv[:, D:2 * D], qkv[:, 2 * D:])


def check_attention(g2, cache, m, NH, max_seq):
    T = m.raw.shape[1]
    q = base.rng(51, T).standard_normal((1, NH, H)).astype(np.float32)
    got = base.run_attend(g2, q, cache, None, T, 1, NH, max_seq, 0.125)
    ref, bound = base.attend_bound(q[0], m.values(), 0.125, T)
    base.within(got[0], ref, bound, f"length {T}")


# lengths of whole blocks reached in one call, in several, row by row, from a block's middle, up to the cache's end
FULL = [[48], [32, 16], [16] * 3, [1] * 48, [40, 8], [33, 15], [5, 43], [31, 17], [47, 1], [3, 20, 25], [64], [60, 4]]


@pytest.mark.parametrize("steps", FULL, ids=lambda s: "-".join(map(str, s)) if len(s) < 9 else f"{len(s)}x{s[0]}")
def test_kv8_cut_back_from_a_full_block(g2, steps):
    """A sequence whose last block is full, cut back to every length in it: read, attended and appended to from there."""
    NH, max_seq = 3, 64
    top = sum(steps)
    for cut in range(top - 15, top):
        cache, n = base.fresh_cache(g2, 1, NH, max_seq)
        m, p = lowbit.Kv8(NH), 0
        for T in steps:
            appended(g2, cache, m, p, T, NH, max_seq, 0)
            p += T
        m.raw = m.raw[:, :cut]
        base.check_cache(g2, cache, [m], NH, max_seq)
        check_attention(g2, cache, m, NH, max_seq)
        for T in (top - cut, 0 if top == max_seq else 7):  # to the same end again, and into a block behind it
            if T:
                appended(g2, cache, m, m.raw.shape[1], T, NH, max_seq, 1)
                base.check_cache(g2, cache, [m], NH, max_seq)
        assert (cache.download(np.uint8)[n:] == 0xFF).all()


def test_kv8_cut_back_of_a_batch(g2):
    """Sequences of their own lengths, all of whole blocks, one token taken back from each and another one put there, on
    device positions and counts; a second cut into the same block."""
    S, NH, max_seq = 5, 2, 100
    D, lens = NH * H, [16, 96, 48, 32, 80]
    cache, models = base.filled_cache(g2, S, NH, max_seq, lens, 52)
    for back in (1, 3):
        for m in models:
            m.raw = m.raw[:, :m.raw.shape[1] - back]
        base.check_cache(g2, cache, models, NH, max_seq)
        pos = np.array([m.raw.shape[1] for m in models], np.int32)
        qkv = base.rng(53, back).standard_normal((S, back, 3 * D)).astype(np.float32)
        g2.kv8_append(g2.to_device(qkv), cache, g2.to_device(pos), None, 0, S, back, NH, max_seq)
        for s, m in enumerate(models):
            m.append(pos[s], qkv[s, :, D:2 * D], qkv[s, :, 2 * D:])
        base.check_cache(g2, cache, models, NH, max_seq)


def test_kv8_cut_back_from_an_end_inside_a_block(g2):
    """A cache of 41 positions that is full: its last block never fills, rows behind the end are left out."""
    NH, max_seq = 2, 41
    cache, n = base.fresh_cache(g2, 1, NH, max_seq)
    m = lowbit.Kv8(NH)
    appended(g2, cache, m, 0, 30, NH, max_seq, 2)
    D = NH * H
    qkv = base.rng(54).standard_normal((20, 3 * D)).astype(np.float32)
    g2.kv8_append(g2.to_device(qkv), cache, g2.to_device(np.array([30], np.int32)), None, 0, 1, 20, NH, max_seq)
    m.append(30, qkv[:11, D:2 * D], qkv[:11, 2 * D:])
    for cut in (41, 40, 33, 32):
        m.raw = m.raw[:, :cut]
        base.check_cache(g2, cache, [m], NH, max_seq)
    assert (cache.download(np.uint8)[n:] == 0xFF).all()


# ------------------------------------------------------------------ 4-bit weights: activations of unlike sizes

# every form of a product, each with groups of 32, 64 and 128
OUTLIERS = [(M, N, K, (32, 64, 128)[(i + j) % 3]) for i in range(3)
            for j, (M, N, K) in enumerate([(1, 100, 768), (1, 48, 2200), (1, 32780, 130), (1, 32770, 1060), (3, 100, 768), (9, 24, 1400),
                                           (8, 4100, 160), (2, 8200, 200), (9, 32780, 130), (3, 32770, 1060), (9, 8195, 2100)])]


def strict_bound(x, v, K):
    """|error| of a computed product: each activation enters within 2^-22 of its own value, whatever stands beside it;
    a sum of K terms goes through at most 160 roundings (128 columns, their groups, the parts of an operand), 4 more
    and one for each 128 columns; a product below fp32's normal range is off by half its last place."""
    return ((164 + K / 128) * EPS32 + 2.0 ** -22) * (np.abs(x) @ np.abs(v).T) + (K + 64) * 2.0 ** -149


@pytest.mark.parametrize("M,N,K,group", OUTLIERS)
def test_matvec_q4_activations_beside_larger_ones(g2, M, N, K, group):
    """Large activations whose weights are 0 (a quarter of the columns) leave the others their own accuracy."""
    r = base.rng(55, M, N, K)
    W = (0.02 * r.standard_normal((N, K))).astype(np.float32)
    zero = r.random(K) < 0.25
    zero[::128] = True
    W[:, zero] = 0
    W[::2] *= r.random((len(W[::2]), K)) < 0.2  # (rows with few weights, so that no large term hides the others)
    codes, scales = base.packed(g2, W, group)
    out = g2.DevBuf(4 * N * K)
    g2.dequantize_q4(codes, scales, out, False, N, K, group)
    v = out.download(np.float32).reshape(N, K)  # (bit for bit the oracle's: test_q4_layout_and_values)
    assert (v[:, zero] == 0).all()
    pick = slice(None) if N < 9000 else r.choice(N, 4000, False)  # rows of the result that are compared
    v = v[pick].astype(np.float64)
    for size in (2.0 ** 17, 2.0 ** 20, 1e7, 2.0 ** 30, 2.0 ** 40, 2.0 ** 100, "mixed", "spread"):
        x = r.standard_normal((M, K))
        big = r.standard_normal((M, K))
        if size == "mixed":  # every row and column its own
            big *= 2.0 ** r.uniform(-10, 100, (M, K))
        elif size == "spread":  # all columns, down to the smallest numbers
            big *= 2.0 ** r.uniform(-140, 120, (M, K))
            x *= 2.0 ** r.uniform(-140, -40, (M, K))
        else:
            big *= size * (r.random((M, K)) < 0.1)
            big[:, ::128] = size
        x = np.where(zero, big, x).astype(np.float32)
        got = base.run_matvec(g2, x, codes, scales, N, K, group)[:, pick]
        x = x.astype(np.float64)
        base.within(got, x @ v.T, strict_bound(x, v, K), f"beside {size}")


# ------------------------------------------------------------------ rules on logits

@pytest.mark.parametrize("penalty", [1.0, 1.3, 3.0])
def test_rules_pick_as_the_host_sampler(g2, penalty):
    """The device's choice is g2_sample_greedy's on a model's logits: with and without a penalty, the end of text
    forbidden or not, ids twice in the context and outside the vocabulary."""
    cfg = g2.make_config(1, 128, 2)
    w = g2.synth_weights(cfg, 5)
    w["wte"] = w["wte"].copy()
    w["wte"][g2.EOS] *= 40  # (often the greatest logit, so that forbidding it matters)
    m = g2.Model.from_host(cfg, w, g2.F32, g2.PATH_FUSED)
    V = cfg.vocab_size
    r = base.rng(60)
    for turn in range(4):
        prompt = r.integers(0, V, 20 + turn).astype(np.int32)
        m.prefill(prompt)
        logits = m.logits()
        top = np.argsort(logits)[::-1][:4 * turn]  # so that the penalty changes the choice
        ctx = np.concatenate([prompt, prompt[:3], top, [-1, V]]).astype(np.int32)
        for forbid in (False, True):
            _, ids = base.run_rules(g2, logits[None], ctx=ctx, max_ctx=len(ctx), repetition=penalty, forbid=g2.EOS if forbid else -1)
            assert ids[0] == m.sample_greedy(ctx, forbid, penalty)


# the wide form (more than 1024 narrow slices in all): several slices to a row and one, the last of one id and of nearly all
WIDE = [(21, 50257), (5, 262144), (130, 8193), (1030, 37), (520, 1025), (200, 8191)]


@pytest.mark.parametrize("R,V", WIDE)
def test_rules_wide(g2, R, V):
    """test_rules' cases on more rows: all rules at once against the oracle, in place, the choice and the logits alone."""
    base.test_rules(g2, R, V)


@pytest.mark.parametrize("R,V", [(2, 50257), (30, 50257), (130, 8193)])
def test_rules_ties_across_slices(g2, R, V):
    """Equal logits on both sides of the slices' borders: the lowest id that is allowed, of 0 and -0 too."""
    edges = sorted({i for i in (1023, 1024, 8191, 8192, 16384, V - 1) if i < V})
    for value in (7.0, 0.0):
        l = -np.abs(base.rng(61, R).standard_normal((R, V))).astype(np.float32) - 1
        l[:, edges] = value
        l[:, edges[::2]] = -value if value == 0 else value
        for n in range(len(edges)):  # the first n of them not allowed
            allowed = np.ones((1, V), bool)
            allowed[0, edges[:n]] = False
            mask = base.bits(allowed, (V + 31) // 32)
            assert (base.run_rules(g2, l, mask=mask)[1] == edges[n]).all()
        assert (base.run_rules(g2, l, forbid=edges[0], out=False)[1] == edges[1]).all()
