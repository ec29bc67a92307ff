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


class Layer:
    """A model of one layer whose embedding, norms, products and sums are the framework's own operators."""

    NH, NKV, E, V = 4, 2, 256, 500
    W = (NH + 2 * NKV) * H

    def __init__(self, g2, max_seq):
        r = rng(77, max_seq)
        self.g2 = g2
        self.h = {n: (s * r.standard_normal(shape)).astype(np.float32) for n, s, shape in (
            ("wte", 1, (self.V, self.E)), ("wpe", 0.3, (max_seq, self.E)), ("g1", 1, self.E), ("b1", 0.1, self.E), ("g2", 1, self.E), ("b2", 0.1, self.E),
            ("wqkv", 0.1, (self.E, self.W)), ("bqkv", 0.1, self.W), ("wo", 0.1, (self.E, self.E)), ("bo", 0.1, self.E), ("head", 0.2, (self.E, self.V)))}
        self.d = {n: g2.to_device(x) for n, x in self.h.items()}

    def qkv(self, ids, runs):
        """(x, qkv) of tokens on the device: runs of (first row, rows, first position)."""
        g2, d = self.g2, self.d
        n = sum(r[1] for r in runs)
        x, y, rows = (guarded(g2, n * w) for w in (self.E, self.E, self.W))
        for row, count, pos in runs:
            g2.embed(d["wte"], d["wpe"], x.offset(4 * row * self.E), self.E, count, pos, ids.offset(4 * row))
        g2.layernorm(x, y, d["g1"], d["b1"], self.E, n)
        g2.matmul(y, d["wqkv"], d["bqkv"], rows, n, self.W, self.E)
        return x, rows, n

    def logits(self, x, att, n, at):
        """Logits [len(at), V] of the rows `at`, on the device."""
        g2, d = self.g2, self.d
        y, z, out = guarded(g2, n * self.E), guarded(g2, n * self.E), guarded(g2, len(at) * self.V)
        g2.matmul(att, d["wo"], d["bo"], y, n, self.E, self.E)
        g2.add(y, x, n * self.E)
        g2.layernorm(y, z, d["g2"], d["b2"], self.E, n)
        for i, row in enumerate(at):
            g2.matmul(z.offset(4 * int(row) * self.E), d["head"], None, out.offset(4 * i * self.V), 1, self.V, self.E)
        return out

    def check(self, ids, pos, x, rows, att, l, at):
        """Each product's and norm's rows against 64 bits, from the tokens and the attention's rows: sums of 256 in fp32, 2^-16
        of the sum of magnitudes each, and three of them, one behind the other, through norms that keep the size."""
        h, n = {k: v.astype(np.float64) for k, v in self.h.items()}, len(ids)

        def norm(y, g, b):
            y = y - y.mean(1, keepdims=True)
            return y / np.sqrt((y * y).mean(1, keepdims=True) + 1e-5) * h[g] + h[b]

        e = h["wte"][ids] + h["wpe"][pos]
        within(take(x, n * self.E).reshape(n, -1), e, 2.0 ** -23 * (1 + np.abs(e)))
        y = norm(e, "g1", "b1")
        within(take(rows, n * self.W).reshape(n, -1), y @ h["wqkv"] + h["bqkv"], 2.0 ** -14 * (1 + np.abs(y) @ np.abs(h["wqkv"])), "qkv")
        z = norm(e + att.reshape(n, -1) @ h["wo"] + h["bo"], "g2", "b2")[at]
        within(take(l, len(at) * self.V).reshape(len(at), -1), z @ h["head"], 2.0 ** -13 * (1 + np.abs(z) @ np.abs(h["head"])), "logits")


@pytest.mark.parametrize("lens,B,steps", [([5, 40, 1], 4, 6), ([70], 8, 5), ([12] * 9, 2, 4)])
def test_beams_between_the_frameworks_own_operators(g2, lens, B, steps):
    """Prompts packed, then steps of all beams: embedding, norms and products by the framework's operators, keys and values
    to the 4-bit cache, attention through the beams' table, selection, tables moved; every call against the oracle on what
    the device had before it, and the tables at the end against the choices followed by hand."""
    G, M = len(lens), max(lens) + steps
    R, m = G * B, Layer(g2, M)
    r = rng(5, G, B)
    prompts = [r.integers(0, m.V, n) for n in lens]
    flat, start = np.concatenate(prompts), np.concatenate([[0], np.cumsum(lens)])
    pos = np.concatenate([np.arange(n) for n in lens])
    ND, KD, W = m.NH * H, m.NKV * H, m.W
    x, rows, n = m.qkv(ints(g2, flat), [(int(start[g]), lens[g], 0) for g in range(G)])
    att = guarded(g2, n * ND)
    ds = ints(g2, start)
    g2.attn_prompt(rows, W, rows.offset(4 * ND), rows.offset(4 * (ND + KD)), W, att, ND, g2.F32, ds, ds, G, n, n, m.NH, m.NKV, 0.125)
    got, qkv = take(att, n * ND).reshape(n, m.NH, H), take(rows, n * W).reshape(n, W)
    q, k, v = qkv[:, :ND].reshape(n, m.NH, H), qkv[:, ND:ND + KD].reshape(n, m.NKV, H), qkv[:, ND + KD:].reshape(n, m.NKV, H)
    for g in range(G):
        a = slice(start[g], start[g + 1])
        want, mass, top = batch.attend(q[a], k[a], v[a], 0.125, batch.causal(lens[g], lens[g]))
        within(got[a], want, prompt_bound(mass, top, lens[g], False, want), f"prompt {g}")
    cache = g2.to_device(np.full(g2.kv4_bytes(R, m.NKV, M), 0xCD, np.uint8))
    held = np.zeros((2, R, M, m.NKV, H), np.float32)  # what the cache was given
    for g in range(G):
        held[:, g * B, :lens[g]] = k[start[g]:start[g + 1]], v[start[g]:start[g + 1]]
    of_beam = np.repeat(start[:-1], B) + np.repeat(lens, B) * (np.arange(R) % B > 0)
    g2.kv4_append(rows.offset(4 * ND), rows.offset(4 * (ND + KD)), W, g2.F32, cache, ints(g2, np.append(of_beam, n)), None, 0, R, n, m.NKV, M)
    at = start[1:] - 1
    l = m.logits(x, att, n, at)
    m.check(flat, pos, x, rows, got, l, at)
    ids, origin = np.zeros((R, M), np.int32), np.repeat(np.arange(G) * B, B)[:, None].astype(np.int32) * np.ones((1, M), np.int32)
    for g in range(G):
        ids[g * B:(g + 1) * B, :lens[g]] = prompts[g]
    dids, dorigin = g2.to_device(ids), g2.to_device(origin)
    score, done, eos = np.zeros(R, np.float32), np.zeros(R, np.int32), m.V - 1
    dscore, ddone, dnew, dended, parent, nxt = (g2.to_device(np.zeros(R, t)) for t in (np.float32, np.int32, np.float32, np.int32, np.int32, np.int32))
    works = g2.beam_work(G, 1, m.V, B), g2.beam_work(G, B, m.V, B)
    awork, length = g2.to_device(np.zeros(g2.kv4_work_bytes(R, m.NH) // 4, np.float32)), np.array(lens)
    for step in range(steps):
        beams = B if step else 1
        old = (np.zeros(G, np.float32), None) if not step else (score, done)
        want = batch.select(take(l, G * beams * m.V).reshape(-1, m.V), old[0], old[1], eos, beams, B)
        g2.beam_select(l, dscore if step else g2.to_device(old[0]), ddone if step else None, eos, dnew, parent, nxt, dended, G, beams, m.V, B, works[step > 0])
        score, done = dnew.download(np.float32), dended.download(np.int32)
        hp, hn = parent.download(np.int32), nxt.download(np.int32)
        for name, a, b in (("parents", hp, want[1]), ("ids", hn, want[2]), ("ended", done, want[3])):
            same(a.reshape(G, B), b, f"{name} of step {step}")
        within(score.reshape(G, B), want[0], 2.0 ** -20 + 2.0 ** -23 * np.abs(want[0]))
        g2.beam_reorder(dids, dids, M, nxt, dorigin, dorigin, M, parent, ints(g2, length), int(length.max()), G, B)
        ids, origin = batch.reorder(ids, hp, hn, length, B), batch.reorder(origin, hp, np.arange(R), length, B)
        same(dids.download(np.int32).reshape(R, M), ids)
        same(dorigin.download(np.int32).reshape(R, M), origin)
        dscore, dnew, ddone, dended = dnew, dscore, dended, ddone
        if step == steps - 1:
            break
        p = np.repeat(length, B)
        x, rows, _ = m.qkv(nxt, [(b, 1, int(p[b])) for b in range(R)])
        g2.kv4_append(rows.offset(4 * ND), rows.offset(4 * (ND + KD)), W, g2.F32, cache, None, ints(g2, p), 0, R, R, m.NKV, M)
        qkv = take(rows, R * W).reshape(R, W)
        held[:, np.arange(R), p] = qkv[:, ND:ND + KD].reshape(R, m.NKV, H), qkv[:, ND + KD:].reshape(R, m.NKV, H)
        length = length + 1
        att = guarded(g2, R * ND)
        g2.attn_kv4(rows, W, cache, att, ND, dorigin, ints(g2, np.repeat(length, B)), M, R, m.NH, m.NKV, M, 0.125, awork)
        got, vals = take(att, R * ND).reshape(R, m.NH, H), batch.to4(held)[0]
        for b in range(R):
            t = np.arange(length[b // B])
            kv = vals[:, origin[b, t], t]
            want, mass, top = batch.attend(qkv[b:b + 1, :ND].reshape(1, m.NH, H), kv[0], kv[1], 0.125, np.ones((1, len(t)), bool))
            within(got[b:b + 1], want, attend_bound(mass, top, len(t)), f"beam {b}, step {step}")
        l = m.logits(x, att, R, np.arange(R))
        m.check(hn, p, x, rows, got, l, np.arange(R))
