"""The operators for several texts at once where their arithmetic or their index ranges end, and as they are used with others."""
import numpy as np
import pytest

from oracle import batch
from parity import EPS32
from test_batch_gpu import H, Cache, Prompts, attend_bound, ints, prompt_bound, select
from test_batch_parts import NORM16, NORM32, off
from test_lowbit_gpu import guarded, rng, same, take, within

pytestmark = pytest.mark.gpu

# 700 rows of so many heads are each of the forms: 32 queries to a work-group, 128, 128 in two groups of waves
FORMS = [(False, 2), (False, 100), (True, 2), (True, 180), (True, 100)]


@pytest.mark.parametrize("f16,NH", FORMS)
@pytest.mark.parametrize("e,unit", [(10, 4), (13, 4), (16, 8), (20, 4), (23, 16), (24, 4), (25, 4), (26, 8), (27, 16), (28, 32), (29, 64), (30, 128)])
def test_prompt_scores_far_from_zero(g2, f16, NH, e, unit):
    """Scores 2^e + r unit with small whole r, exact in fp32 whatever the order of their sums, whose largest grows along
    the keys by a step at a time.  Only differences of scores count: they are exact, too, so a weight's error is that of
    its exponent (a product of at most 2^7 that is rounded twice, 2^-17), of the exponential and the sums, and, where the
    largest score is below 2^10 in powers of two, two roundings of it, 2^-15 each."""
    p = Prompts([(700, 0)], NH, NH, f16, seed=20)
    j = np.arange(700)
    r = j // 100 + (j // 32) % 3
    p.q[:], p.k[:] = 0, 0
    p.q[:, 0::H], p.k[:, 0::H] = 2.0 ** ((e + 1) // 2), 2.0 ** (e // 2)
    p.q[:, 1::H], p.k[:, 1::H] = 8, (r * unit / 8)[:, None]
    p.v[::3, 0::5] = 0
    s = p.q[0, 0] * np.float64(p.k[:, 0]) + p.q[0, 1] * np.float64(p.k[:, 1])
    assert (s.astype(np.float32) == s).all() and (s == 2.0 ** e + r * unit).all()
    got, want = p.run(g2), np.empty((700, NH, H))
    q, k, v = (x.reshape(700, NH, H) for x in (p.q, p.k, p.v))
    want, mass, _ = batch.attend(q, k, v, 0.125, batch.causal(700, 700))
    bound = (2.0 ** -17 + 2.0 ** -14 + (12 * 700 + 32) * EPS32) * mass
    if f16:
        bound = bound + 2.0 ** -11 * mass * 1.001 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    within(got, want, bound)


@pytest.mark.parametrize("seqs", [[(17, 0)], [(700, 0)], [(300, 0), (1000, 0), (64, 200), (1, 0)], [(9, 30)] * 80])
@pytest.mark.parametrize("f16,NH,NKV", [(False, 2, 2), (False, 6, 2), (False, 100, 100), (False, 120, 60), (True, 4, 2), (True, 180, 180), (True, 100, 100)])
def test_prompt_norms(g2, seqs, f16, NH, NKV):
    """The error of all outputs together and of each head's: test_batch_parts.py has the limits' reasons."""
    p = Prompts(seqs, NH, NKV, f16, seed=24)
    got, want = p.run(g2), p.want()[0]
    limit = NORM16 if f16 else NORM32
    assert off(got, want) < limit
    assert max(off(got[:, h], want[:, h]) for h in range(NH)) < limit


@pytest.mark.parametrize("f16,NH", FORMS)
def test_prompt_values_not_finite_before_far_larger_scores(g2, f16, NH):
    """A value that is not finite counts in the rows that see it also where later keys' scores are so much larger that its
    weight is 0 in 32 bits: a weight is never 0 by the formula."""
    for down in (1, -1):
        p = Prompts([(700, 0)], NH, NH, f16, seed=21)
        p.q[:], p.k[:] = 0, 0
        p.q[:, 0::H], p.k[:, 0::H] = 32, (64 * (np.arange(700) // 100))[:, None] * down
        for j, bad, d in ((5, np.inf, 3), (130, -np.inf, 7), (250, np.nan, 9), (10, np.inf, 11), (420, -np.inf, 11), (333, np.inf, 62), (699, np.inf, 20)):
            p.v[j, d::H] = bad
        p.check(g2)


def test_prompt_smallest_f16_numbers(g2):
    """Numbers below 2^-14 (fp16's subnormal ones) as queries, keys and values: products are exact as any others."""
    for NH in (2, 100, 180):
        p = Prompts([(700, 0)], NH, NH, True, seed=22)
        small, large = np.float32(2.0 ** -17), np.float32(2.0 ** 14)
        q, k = p.q.astype(np.float32).clip(-3.9, 3.9), p.k.astype(np.float32).clip(-3.9, 3.9)
        p.q, p.k = (q * small).astype(p.t), (k * large).astype(p.t)
        p.v[:, 0::2] = (p.v[:, 0::2].astype(np.float32) * np.float32(2.0 ** -18)).astype(p.t)
        assert (p.q != 0).mean() > 0.99
        p.check(g2, scale=0.5)
        p.q, p.k = (q * large).astype(p.t), (k * small).astype(p.t)
        p.check(g2, scale=0.5)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,rows,NH,NKV,past", [(64, 1, 4, 4, 700), (64, 40, 6, 2, 300), (100, 5, 5, 1, 129), (500, 3, 2, 2, 40), (70, 300, 25, 5, 17)])
def test_prompt_many_sequences_behind_earlier_keys(g2, f16, S, rows, NH, NKV, past):
    """64 sequences and more, whose tiles are cut from all rows, with keys that were there before."""
    r = rng(S, rows)
    Prompts([(int(n), int(m)) for n, m in zip(r.integers(min(rows, 2) - 1, rows + 1, S), r.integers(past - 10, past + 1, S))], NH, NKV, f16, gap=S % 3).check(g2)


@pytest.mark.parametrize("f16,NH", [(False, 1), (False, 32), (True, 1), (True, 64), (True, 20)])
@pytest.mark.parametrize("seqs", [[(2100, -2100)], [(2100, -2050)], [(700, -700), (1300, -1290), (100, 0)], [(33, -33)] * 70 + [(5, 200)]])
def test_prompt_tiles_that_see_no_key(g2, f16, NH, seqs):
    """Whole tiles whose rows come before the first key, in every form: zeros."""
    p = Prompts(seqs, NH, NH, f16, seed=23)
    got, blind = p.check(g2), [r for i, (n, _) in enumerate(seqs) for r in range(p.qs[i], p.qs[i] + n - p.m[i])]
    assert len(blind) >= 1990 and (got[blind] == 0).all()


def close_beams(V, G, spread, seed):
    """Logits of G groups of two beams, and scores that leave the beams' best sums apart by some 1e-8 to 1e-6, far below
    what an fp32 sum of the exponentials tells apart."""
    r = rng(V, G, seed)
    logits = (spread * r.standard_normal((2 * G, V))).astype(np.float32)
    l = logits.astype(np.float64)
    top = l.max(1)
    lse = top + np.log(np.exp(l - top[:, None]).sum(1))
    best = top - lse
    gap = r.choice([-1, 1], G) * 10.0 ** r.uniform(-8, -6, G)
    score = np.zeros(2 * G, np.float32)
    score[1::2] = (best[0::2] - best[1::2] + gap).astype(np.float32)
    gap = (score + best).reshape(G, 2)
    return logits, score, np.abs(gap[:, 0] - gap[:, 1]).min()


@pytest.mark.parametrize("V,G,spread,seed", [(50257, 2, 4, 0), (50257, 32, 4, 1), (50257, 64, 4, 2), (5000, 100, 1, 3), (262144, 4, 0.1, 4), (700, 200, 2, 5)])
def test_select_between_close_beams(g2, V, G, spread, seed):
    """Continuations of different beams are compared in 64 bits as those of one beam are."""
    logits, score, gap = close_beams(V, G, spread, seed)
    assert gap > 1e-11, "the 64-bit oracle's own choice is not certain"
    want = batch.select(logits, score, None, -1, 2, 4)
    got = select(g2, logits, score, None, -1, 2, 4)
    for g, w, name in zip(got[1:3], want[1:3], ("parents", "ids")):
        same(g, w, name)


def chosen(g2, logits, score, done, eos, beams, n_out):
    want = batch.select(logits, score, done, eos, beams, n_out)
    for _ in range(2):
        got = select(g2, logits, score, done, eos, beams, n_out)
        for g, w, name in zip(got[1:], want[1:], ("parents", "ids", "ended")):
            same(g, w, name)
    return want


def test_select_close_beams_of_equal_ones(g2):
    """Close beams where more continuations are equal than the lists hold, and close ended beams."""
    for V, G in ((5000, 8), (1024, 40)):
        r = rng(V)
        logits = np.repeat(r.uniform(-3, 3, 2 * G).astype(np.float32), V).reshape(2 * G, V)
        score = np.zeros(2 * G, np.float32)
        score[r.integers(0, 2, G) + 2 * np.arange(G)] = 10.0 ** r.uniform(-8, -6, G)
        chosen(g2, logits, score, None, -1, 2, 9)
    logits, score, _ = close_beams(3000, 50, 3, 6)
    l = logits.astype(np.float64)
    lse = l.max(1) + np.log(np.exp(l - l.max(1, keepdims=True)).sum(1))
    score[1::2] = (lse - l.max(1))[1::2].astype(np.float32)  # the beam's best sum: 0 and a rounding
    score[0::2] = rng(7).uniform(-3e-7, 3e-7, 50).astype(np.float32)
    total = score[1::2] + (l.max(1) - lse)[1::2]
    assert np.abs(total - score[0::2]).min() > 1e-10
    want = chosen(g2, logits, score, np.tile([1, 0], 50), 5, 2, 3)
    assert 5 < (want[1][:, 0] == 0).sum() < 45


@pytest.mark.parametrize("beams,n_out,V", [(32, 64, 1500), (8, 8, 50257), (5, 40, 300)])
def test_select_chains_of_close_beams(g2, beams, n_out, V):
    """Every beam close to the next one, in each of the groups."""
    G, r = 3, rng(beams, n_out)
    logits = (2 * r.standard_normal((G * beams, V))).astype(np.float32)
    l = logits.astype(np.float64)
    best = -np.log(np.exp(l - l.max(1, keepdims=True)).sum(1))
    score = (-best + 3e-7 * r.permuted(np.tile(np.arange(beams), (G, 1)), axis=1).ravel()).astype(np.float32)
    total = np.sort((score + best).reshape(G, beams), 1)
    assert np.diff(total, axis=1).min() > 1e-12
    chosen(g2, logits, score, None, 7, beams, n_out)


# ------------------------------------------------------------------ as they are used

@pytest.mark.parametrize("lens,new", [([33, 5, 64], [7, 40, 1]), ([10] * 40, [3] * 40), ([0, 90], [20, 2])])
def test_second_turn_over_the_cache(g2, lens, new):
    """Texts of different lengths go on: their new rows are appended to the 4-bit cache, all positions read back, [S][T],
    and the packed new rows see their own; what lies between a text's last position and the next text's first belongs to
    sequences without rows."""
    S, NH, NKV, M = len(lens), 4, 2, 128
    KD = NKV * H
    c = Cache(g2, S, NKV, M)
    c.append(lens, [0] * S)
    x = c.append(new, lens, seed=1)
    total = np.add(lens, new)
    T = int(total.max())
    k, v = guarded(g2, S * T * KD, 0.0), guarded(g2, S * T * KD, 0.0)
    g2.kv4_read(c.buf, k, v, None, ints(g2, total), M, 0, T, S, NKV, M)
    rows = np.concatenate([[0], np.cumsum(new)])
    qs = np.concatenate([[0], np.repeat(rows[1:], 2)])  # 0, r1, r1, r2, r2, ...: every second one has no rows
    ks = np.append(np.stack([T * np.arange(S), T * np.arange(S) + total], 1).ravel(), S * T)
    q = rng(3, S).standard_normal((rows[-1], NH * H)).astype(np.float32)
    out = guarded(g2, q.size)
    g2.attn_prompt(g2.to_device(q), NH * H, k, v, KD, out, NH * H, g2.F32, ints(g2, qs), ints(g2, ks), 2 * S, int(rows[-1]), S * T, NH, NKV, 0.125)
    got, vals = take(out, q.size).reshape(-1, NH, H), c.values()
    for s in range(S):
        a = slice(rows[s], rows[s + 1])
        want, mass, top = batch.attend(q[a].reshape(-1, NH, H), vals[0, s, :total[s]], vals[1, s, :total[s]], 0.125, batch.causal(new[s], total[s]))
        within(got[a], want, prompt_bound(mass, top, T, False, want), f"text {s}")
