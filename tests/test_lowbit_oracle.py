"""The oracle of the low-bit operators against closed forms, and the calls'
refusals: every wrong call is an error code before any device is asked for
(no GPU here: a right call answers G2_E_STATE)."""
import ctypes as C

import numpy as np
import pytest

import g2hip
from oracle import lowbit


def test_codes_are_the_nearest_values_and_ties_go_to_even_codes():
    # scale 1 exactly (largest magnitude 6): the values themselves, the borders between them, and both sides
    up = lowbit.LEVELS
    mid = (up[1:] + up[:-1]) / 2
    row = np.concatenate([up, mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                          np.nextafter(mid.astype(np.float32), np.float32(9))]).astype(np.float32)
    W = np.zeros((2, 32), np.float32)
    W[0, :len(row)], W[1, :len(row)] = row, -row
    c, s = lowbit.quantize_q4(W, 32)
    assert (s == 1).all()
    tie = [i if i % 2 == 0 else i + 1 for i in range(7)]
    want = list(range(8)) + tie + list(range(7)) + list(range(1, 8))
    np.testing.assert_array_equal(c[0, :len(row)], want)
    np.testing.assert_array_equal(c[1, :len(row)], [w + 8 if w else 0 for w in want])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 1), (17, 31), (16, 128), (33, 300)])
def test_layout_holds_every_code_once(N, K, group):
    codes = np.random.default_rng(N + K).integers(1, 16, (N, K)).astype(np.uint8)
    sc = np.ones((N, -(-K // group)), np.float32)
    a, b = lowbit.lay_out_q4(codes, sc, group)
    nc, ns = g2hip.q4_bytes(N, K, group)
    assert a.nbytes == nc and b.nbytes == ns
    assert (a & 15 > 0).sum() + (a >> 4 > 0).sum() == N * K and (b > 0).sum() == sc.size


def test_weights_of_a_group_without_finite_values_read_back_as_nan():
    W = np.ones((4, 64), np.float32)
    W[0, 3], W[1, 40], W[2, 0] = np.inf, np.nan, 2.0 ** 97
    v = lowbit.values_q4(*lowbit.quantize_q4(W, 32), 32)
    assert np.isnan(v[0, :32]).all() and np.isnan(v[1, 32:]).all() and np.isnan(v[2, :32]).all()
    assert (v[0, 32:] == v[3, 0]).all() and np.isfinite(v[3]).all()


def test_cache_does_not_depend_on_how_it_was_filled():
    r = np.random.default_rng(0)
    k, v = r.standard_normal((2, 50, 2 * 64)).astype(np.float32)
    a, b = lowbit.Kv8(2), lowbit.Kv8(2)
    a.append(0, k, v)
    for p in range(50):
        b.append(p, k[p:p + 1], v[p:p + 1])
    np.testing.assert_array_equal(a.values(), b.values())
    # eight bits: at most half a step of the block's largest value
    err = np.abs(a.values()[0].reshape(50, -1) - k)
    assert (err[48:] == 0).all() and (err[:48] <= np.abs(k).max() / 127 * 0.5001).all()


def test_rules_by_hand():
    l, pick = lowbit.rules([2.0, -1.0, 4.0, 4.0], ctx=[2, 2, 1, 9, -3], repetition=2.0, frequency=0.5, presence=0.25)
    np.testing.assert_array_equal(l, np.float32([2.0, -2.75, 0.75, 4.0]))
    assert pick == 3
    assert lowbit.rules([1.0, 5.0, 5.0], forbid=1)[1] == 2
    assert lowbit.rules([1.0, 5.0, 5.0])[1] == 1  # the lowest of equal ones
    assert lowbit.rules([1.0, 5.0], mask=[False, False])[1] == -1
    assert lowbit.rules([np.nan, -9.0])[1] == 1
    assert lowbit.rules([0.0, 0.0], bias=[(0, 3.0), (0, -3.0), (7, 9.0)])[1] == 1  # an id's later entry counts


# ------------------------------------------------------------------ refusals

P = 1 << 20  # an address that no call may look at


def rc(fn, *args):
    code = getattr(g2hip._lib, fn)(*args)
    if code < 0:
        assert g2hip.last_error()
    return code


def checked(fn, good, bad):
    """good: a right call's arguments; bad: {index: (wrong value, code)} lists."""
    assert rc(fn, *good) == g2hip.G2_E_STATE, g2hip.last_error()
    for i, value, code in bad:
        args = list(good)
        for at, v in zip(i if isinstance(i, tuple) else (i,), value if isinstance(i, tuple) else (value,)):
            args[at] = v
        assert rc(fn, *args) == code, (fn, i, value, g2hip.last_error())


ARG, LIMIT = g2hip.G2_E_ARG, g2hip.G2_E_LIMIT
A, B, D, E, F = (P * i for i in (64, 128, 192, 256, 320))


@pytest.fixture(autouse=True)
def no_device():
    """These calls must not reach a device: the library is not initialised."""
    if g2hip._lib.g2_stream():
        pytest.skip("the library is initialised in this process")


def test_sizes():
    assert g2hip.q4_bytes(16, 32, 32) == (256, 128) and g2hip.q4_bytes(17, 33, 64) == (2 * 512, 2 * 64)
    for N, K, G in ((0, 1, 32), (1, 0, 32), (1, 1 << 25, 32), (1, 1, 48), (1, 1, 0)):
        assert g2hip.q4_bytes(N, K, G)[1] == 0
    assert g2hip.q4_bytes(-1, 5, 32)[0] == 0
    assert g2hip.kv8_bytes(1, 1, 16) == 2048 + 256 + 8192 and g2hip.kv8_bytes(1, 1, 17) == 4096 + 256 + 8192
    for S, H, n in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1025, 1), (1 << 23, 1, 1), (1, 1, (1 << 24) + 1)):
        assert g2hip.kv8_bytes(S, H, n) == 0
    assert g2hip.kv8_bytes(1 << 10, 1 << 10, 1 << 24) > 1 << 50  # in 64 bits
    assert g2hip.kv8_work_bytes(2, 3) > 0 and g2hip.kv8_work_bytes(0, 3) == 0
    assert g2hip.logits_work_bytes(1) > 0 and g2hip.logits_work_bytes(0) == 0 and g2hip.logits_work_bytes((1 << 16) + 1) == 0


def test_q4_refusals():
    checked("g2_quantize_q4", (A, 0, 0, B, D, 100, 100, 32),
            [(0, None, ARG), (3, None, ARG), (4, None, ARG), (1, 2, ARG), (5, 0, ARG), (6, -4, ARG), (7, 16, ARG), (7, 0, ARG),
             (5, (1 << 24) + 1, LIMIT), (3, B + 8, ARG), (4, D + 4, ARG), (3, A, ARG), (4, A + 16, ARG), (4, B, ARG)])
    checked("g2_dequantize_q4", (A, B, D, 1, 100, 100, 128),
            [(0, None, ARG), (1, None, ARG), (2, None, ARG), (4, 0, ARG), (5, 0, ARG), (6, 100, ARG), (0, A + 4, ARG), (2, A + 4, ARG), (2, B, ARG)])
    checked("g2_matvec_q4", (A, B, D, None, None, E, 2, 100, 100, 64, 0),
            [(0, None, ARG), (1, None, ARG), (2, None, ARG), (5, None, ARG), (6, 0, ARG), (7, 0, ARG), (8, 0, ARG), (9, 96, ARG),
             (6, 65536, LIMIT), (8, (1 << 24) + 1, LIMIT), (1, B + 1, ARG), (2, D + 2, ARG), (5, A + 4, ARG), (5, B, ARG), (5, D, ARG),
             (3, E + 4, ARG), (4, E + 4, ARG)])
    assert rc("g2_matvec_q4", A, B, D, F, E, E, 2, 100, 100, 64, 1) == g2hip.G2_E_STATE  # residual in place


def test_kv8_refusals():
    checked("g2_kv8_append", (A, B, None, None, 3, 2, 4, 12, 64),
            [(0, None, ARG), (1, None, ARG), (1, B + 4, ARG), (4, -1, ARG), (4, 61, ARG), (5, 0, ARG), (6, 0, ARG), (6, 65, ARG),
             (7, 0, ARG), (7, 1025, LIMIT), (8, 0, ARG), (8, (1 << 24) + 1, LIMIT), (0, B + 64, ARG), (2, B + 16, ARG), (3, B, ARG)])
    checked("g2_kv8_read", (A, B, D, None, 60, 8, 50, 2, 12, 64),
            [(0, None, ARG), (1, None, ARG), (2, None, ARG), (4, 65, ARG), (4, -1, ARG), (5, -1, ARG), (5, 15, ARG), (6, 0, ARG), (7, 0, ARG),
             (8, 0, ARG), (9, 0, ARG), (1, A, ARG), (2, B, ARG), (0, A + 8, ARG), (3, B, ARG), (3, D + 8, ARG)])
    checked("g2_attn_kv8", (A, 3 * 768, B, D, 768, None, 60, 2, 12, 64, C.c_float(0.125), E),
            [(0, None, ARG), (2, None, ARG), (3, None, ARG), (11, None, ARG), (1, 767, ARG), (4, 767, ARG), (6, 65, ARG), (6, -1, ARG),
             (7, 0, ARG), (8, 0, ARG), (9, 0, ARG), (8, 2000, LIMIT), (2, B + 8, ARG), (3, A + 4, ARG), (3, B, ARG), (3, E, ARG), (11, A, ARG),
             (11, B, ARG), (5, D, ARG), (5, E, ARG)])
    # one sequence: its strides do not matter
    assert rc("g2_attn_kv8", A, 0, B, D, 0, None, 60, 1, 12, 64, C.c_float(0.125), E) == g2hip.G2_E_STATE


def test_logit_rule_refusals():
    def call(logits=A, out=B, pick=D, rows=2, V=100, work=E, **kw):
        return rc("g2_apply_logit_rules", logits, out, pick, rows, V, C.byref(g2hip.logit_rules(**kw)), work)

    ok = g2hip.G2_E_STATE
    assert call() == ok and call(out=A) == ok and call(out=None) == ok and call(pick=None, work=None) == ok
    assert call(repetition=0.0) == ok and call(ctx=F, max_ctx=5) == ok and call(mask=F, mask_stride=0) == ok
    assert call(ctx=F, max_ctx=0) == ok and call(forbid=99) == ok
    for kw in (dict(logits=None), dict(out=None, pick=None), dict(rows=0), dict(V=0), dict(work=None), dict(work=E + 4), dict(out=A + 4),
               dict(max_ctx=-1), dict(max_ctx=3), dict(n_bias=2), dict(n_bias=2, bias=F), dict(n_bias=2, bias_id=F), dict(n_bias=-1),
               dict(repetition=-1.0), dict(repetition=float("nan")), dict(repetition=float("inf")), dict(frequency=float("inf")),
               dict(presence=float("nan")), dict(mask=F, mask_stride=3), dict(mask=F, mask_stride=-1), dict(forbid=100), dict(forbid=-2),
               dict(pick=A), dict(work=A), dict(work=B), dict(pick=B + 8), dict(work=D), dict(ctx=B, max_ctx=4), dict(mask=B, mask_stride=4),
               dict(ctx=D, max_ctx=4), dict(ctx=E, max_ctx=4), dict(bias=B, bias_id=F, n_bias=1)):
        assert call(**kw) == ARG, kw
    assert call(V=262145) == LIMIT and call(rows=65537) == LIMIT
    assert rc("g2_apply_logit_rules", A, B, D, 1, 10, None, E) == ARG
