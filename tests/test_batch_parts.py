"""How near the results of packed prompts have to come to 64 bits as a whole, and that a part or a product left out would be
noticed: the mistakes are made in a copy of the arithmetic on the CPU.

The bounds of single outputs are for the worst case, whose roundings all point one way; a lost part of every operand stays
below them.  The 2-norm of a call's error does not have that room.  For rows N(0, 1), a scale of 1/8 and up to 1000 keys, in
roundings of fp32, which are off by 2^-24 / sqrt 3 of what is rounded in the mean square:
  a score: 24 matrix instructions' sums of at most sqrt 64 in the mean square, twice that for what an instruction rounds
  inside: 2 sqrt(24) 8 / (8 sqrt 3) 2^-24 = 3.4e-7; products left out (a second part times a third, twice, 64 dims): 0.8e-7;
  exponent and exponential: 1.5e-7.  These are errors relative to a weight, and the error of the output's sum relative to
  the sum is as large in the mean square.
  the weighted sum: 6 * 1000 / 16 = 375 sums, of half the last one's square on average: sqrt(375 / 2) 2^-24 / sqrt 3 = 4.7e-7
Together 6.1e-7, and 2^-20 = 9.5e-7 allowed.  fp16: the weights' rounding and the outputs', 2^-11 / sqrt 3 each of values that
are 1.4 times a binade's end on average: sqrt 2 * 2^-11 / (sqrt 3 * 1.4) = 2.8e-4, and 2^-11 = 4.9e-4 allowed."""
import numpy as np
import pytest

NORM32, NORM16 = 2.0 ** -20, 2.0 ** -11


def off(got, want):
    """The 2-norm of the error beside the result's."""
    return float(np.linalg.norm(np.asarray(got, np.float64) - want) / np.linalg.norm(want))


def bf16(x):
    """x rounded to bf16, ties to even, as fp32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return (((u + 0x7FFF + (u >> 16 & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


def parts(x):
    """The three bf16 parts: the first cut off, the others rounded."""
    x = np.asarray(x, np.float32)
    a = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
    b = bf16(x - a)
    return a, b, bf16(x - a - b)


SIX = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]


def product(x, y, pairs):
    px, py = parts(x), parts(y)
    return sum(px[i].astype(np.float64) @ py[j].astype(np.float64) for i, j in pairs)


def attention(q, k, v, scores=SIX, values=SIX):
    """Causal attention with the products of parts that are given, sums in 64 bits."""
    s = product(q, k.T.copy(), scores) / 8
    s[np.triu_indices(len(q), 1)] = -np.inf
    p = np.exp(s - s.max(1, keepdims=True))
    return product(p.astype(np.float32), v, values) / p.sum(1, keepdims=True)


@pytest.mark.parametrize("n", [17, 300, 1000])
def test_a_lost_part_would_be_noticed(n):
    r = np.random.default_rng(n)
    q, k, v = r.standard_normal((3, n, 64)).astype(np.float32)
    s = q.astype(np.float64) @ k.astype(np.float64).T / 8
    s[np.triu_indices(n, 1)] = -np.inf
    p = np.exp(s - s.max(1, keepdims=True))
    want = p @ v.astype(np.float64) / p.sum(1, keepdims=True)
    assert off(attention(q, k, v), want) < NORM32 / 3
    mistakes = [[x for x in SIX if x != lost] for lost in SIX[1:]]  # a product left out
    mistakes += [[x for x in SIX if x[side] != part] for side in (0, 1) for part in (1, 2)]  # a part of one operand
    mistakes += [[x for x in SIX if 2 not in x], [(1, 1) if x == (0, 2) else x for x in SIX], [(0, 0), (0, 1), (1, 0), (1, 1), (1, 2), (2, 1)]]
    for pairs in mistakes:
        assert off(attention(q, k, v, scores=pairs), want) > 2 * NORM32, ("scores", pairs)
        assert off(attention(q, k, v, values=pairs), want) > 2 * NORM32, ("values", pairs)


def test_weights_of_fewer_bits_would_be_noticed():
    """fp16 rows: weights rounded to fp16 stay within the limit, weights rounded to bf16 do not."""
    r = np.random.default_rng(1)
    q, k, v = r.standard_normal((3, 500, 64)).astype(np.float16).astype(np.float64)
    s = q @ k.T / 8
    s[np.triu_indices(500, 1)] = -np.inf
    p = np.exp(s - s.max(1, keepdims=True))
    want = p @ v / p.sum(1, keepdims=True)
    for rounded, ok in ((p.astype(np.float16).astype(np.float64), True), (bf16(p).astype(np.float64), False)):
        got = (rounded @ v / p.sum(1, keepdims=True)).astype(np.float16)
        assert (off(got, want) < NORM16) == ok
