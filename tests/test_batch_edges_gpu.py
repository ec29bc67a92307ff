"""The operators for several texts at once where their arithmetic or their index ranges end."""
import numpy as np
import pytest

from oracle import batch
from parity import EPS32
from test_batch_gpu import H, Prompts
from test_lowbit_gpu import within

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


@pytest.mark.parametrize("f16,NH", [(False, 1), (False, 32), (True, 1), (True, 64), (True, 20)])
@pytest.mark.parametrize("seqs", [[(2100, -2100)], [(2100, -2050)], [(700, -700), (1300, -1290), (100, 0)], [(33, -33)] * 70 + [(5, 200)]])
def test_prompt_tiles_that_see_no_key(g2, f16, NH, seqs):
    """Whole tiles whose rows come before the first key, in every form: zeros."""
    p = Prompts(seqs, NH, NH, f16, seed=23)
    got, blind = p.check(g2), [r for i, (n, _) in enumerate(seqs) for r in range(p.qs[i], p.qs[i] + n - p.m[i])]
    assert len(blind) >= 1990 and (got[blind] == 0).all()
