"""What the header allows of the decode operators in fewer bits beyond test_lowbit_gpu.py's calls: cutting a sequence
back from a block that is full."""
import numpy as np
import pytest

import test_lowbit_gpu as base
from oracle import lowbit

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
