"""What the operators for several texts at once refuse, without a GPU: addresses are numbers, and each call either names
its mistake or asks for the runtime."""
import re

import pytest

import g2hip

A = [(i + 1) << 36 for i in range(14)]  # buffers far apart
ARG, LIMIT, STATE = g2hip.G2_E_ARG, g2hip.G2_E_LIMIT, g2hip.G2_E_STATE


def code(fn, args):
    with pytest.raises(g2hip.G2Error) as e:
        fn(*args)
    return e.value.code


def refused(fn, good, cases):
    """`good` is a dict of arguments in order that only lacks the runtime; each case changes some of them."""
    if code(fn, good.values()) != STATE:
        raise AssertionError(g2hip.last_error())
    for want, change in cases:
        args = {**good, **change}
        assert len(args) == len(good), change
        assert code(fn, args.values()) == want, (change, g2hip.last_error())
        assert re.match(r"g2_", g2hip.last_error())


@pytest.fixture(autouse=True, scope="module")
def no_runtime():
    if g2hip._lib.g2_stream():
        pytest.skip("the runtime is up")


def test_prompt():
    good = dict(q=A[0], q_stride=768, k=A[1], v=A[2], kv_stride=256, out=A[3], out_stride=512, dtype=0, q_start=A[4], k_start=A[5], n_seq=3,
                q_rows=100, k_rows=120, n_head=8, n_kv=4, scale=0.125)
    same_rows = dict(k=A[0] + 4 * 512, v=A[0] + 4 * 640, kv_stride=768, k_start=A[4], k_rows=100)  # (a row of qkv; one list)
    assert code(g2hip.attn_prompt, {**good, **same_rows}.values()) == STATE
    assert code(g2hip.attn_prompt, {**good, "n_seq": 1, "q_start": None, "k_start": None}.values()) == STATE
    assert code(g2hip.attn_prompt, {**good, "k_rows": 0}.values()) == STATE
    assert code(g2hip.attn_prompt, {**good, "q_rows": 1, "q_stride": 0, "out_stride": 0}.values()) == STATE
    out_end = A[3] + 4 * (99 * 512 + 512)
    refused(g2hip.attn_prompt, good, [
        (ARG, dict(q=None)), (ARG, dict(k=None)), (ARG, dict(v=None)), (ARG, dict(out=None)), (ARG, dict(dtype=2)), (ARG, dict(dtype=-1)),
        (ARG, dict(n_head=0)), (ARG, dict(n_kv=0)), (ARG, dict(n_kv=3)), (ARG, dict(n_head=-8, n_kv=-4)), (LIMIT, dict(n_head=1032, q_stride=1 << 20, out_stride=1 << 20)),
        (ARG, dict(n_seq=0)), (ARG, dict(q_rows=0)), (ARG, dict(k_rows=-1)), (ARG, dict(q_start=None)), (ARG, dict(k_start=None)),
        (ARG, dict(q_stride=511)), (ARG, dict(out_stride=511)), (ARG, dict(kv_stride=255)),
        (LIMIT, dict(q_rows=(1 << 24) + 1)), (LIMIT, dict(k_rows=(1 << 24) + 1)), (LIMIT, dict(q_stride=(1 << 24) + 1)), (LIMIT, dict(out_stride=(1 << 24) + 1)),
        (LIMIT, dict(kv_stride=(1 << 24) + 1)), (LIMIT, dict(n_seq=(1 << 20) + 1)),
        (LIMIT, dict(q_rows=1 << 24, n_head=1024, q_stride=1 << 16, out_stride=1 << 16, q=1 << 50, out=1 << 55)),
        (ARG, dict(scale=float("nan"))), (ARG, dict(scale=float("inf"))), (ARG, dict(q=A[0] + 2)), (ARG, dict(v=A[2] + 1)), (ARG, dict(dtype=1, out=A[3] + 1)),
        (ARG, dict(q=A[3])), (ARG, dict(q=out_end - 4)), (ARG, dict(k=A[3] - 4 * (119 * 256 + 256) + 4)), (ARG, dict(v=out_end - 4)),
        (ARG, dict(q_start=out_end - 4)), (ARG, dict(k_start=A[3] - 12)),
    ])


def test_kv4_append():
    good = dict(k=A[0], v=A[1], stride=256, dtype=0, cache=A[2], row_start=A[3], pos=A[4], start=0, n_seq=3, rows=100, n_kv=4, max_seq=1024)
    assert code(g2hip.kv4_append, {**good, "row_start": None, "pos": None, "rows": 99, "start": 1023}.values()) == STATE
    size = g2hip.kv4_bytes(3, 4, 1024)
    refused(g2hip.kv4_append, good, [
        (ARG, dict(k=None)), (ARG, dict(v=None)), (ARG, dict(cache=None)), (ARG, dict(dtype=3)), (ARG, dict(n_seq=0)), (ARG, dict(n_kv=0)),
        (ARG, dict(max_seq=0)), (ARG, dict(rows=0)), (ARG, dict(stride=255)), (ARG, dict(row_start=None)), (ARG, dict(pos=None, start=-1)),
        (ARG, dict(pos=None, start=1024)), (ARG, dict(cache=A[2] + 8)), (ARG, dict(k=A[0] + 2)), (ARG, dict(dtype=1, v=A[1] + 1)),
        (LIMIT, dict(n_kv=1025, stride=1 << 20)), (LIMIT, dict(max_seq=(1 << 24) + 1)), (LIMIT, dict(n_seq=1 << 21)), (LIMIT, dict(rows=(1 << 24) + 1)),
        (LIMIT, dict(stride=(1 << 24) + 1)), (LIMIT, dict(rows=1 << 24, n_kv=1024, stride=1 << 16, k=1 << 50, v=1 << 55)),
        (ARG, dict(k=A[2] + size - 4)), (ARG, dict(v=A[2])), (ARG, dict(row_start=A[2] + size - 16)), (ARG, dict(pos=A[2] + 100)),
    ])


def test_kv4_read():
    good = dict(cache=A[0], k=A[1], v=A[2], origin=A[3], lens=A[4], T_kv=1024, start=10, T=1000, n_seq=3, n_kv=4, max_seq=1024)
    n = 4 * 3 * 1000 * 256
    refused(g2hip.kv4_read, good, [
        (ARG, dict(cache=None)), (ARG, dict(k=None)), (ARG, dict(v=None)), (ARG, dict(T_kv=-1)), (ARG, dict(T_kv=1025)), (ARG, dict(start=-1)), (ARG, dict(T=0)),
        (ARG, dict(start=25)), (ARG, dict(cache=A[0] + 4)), (LIMIT, dict(n_seq=1 << 21)), (ARG, dict(v=A[1] + n - 4)), (ARG, dict(k=A[0])),
        (ARG, dict(origin=A[1] + n - 4)), (ARG, dict(lens=A[2])), (ARG, dict(k=A[1] + 2)), (ARG, dict(v=A[2] + 1)),
    ])


def test_attn_kv4():
    good = dict(q=A[0], q_stride=768, cache=A[1], out=A[2], out_stride=512, origin=A[3], lens=A[4], T_kv=1000, n_seq=3, n_head=8, n_kv=4, max_seq=1024,
                scale=0.125, work=A[5])
    assert code(g2hip.attn_kv4, {**good, "origin": None, "lens": None, "T_kv": 0}.values()) == STATE
    nw = g2hip.kv4_work_bytes(3, 8)
    assert nw == 3 * 8 * 32 * 66 * 4
    refused(g2hip.attn_kv4, good, [
        (ARG, dict(q=None)), (ARG, dict(cache=None)), (ARG, dict(out=None)), (ARG, dict(work=None)), (ARG, dict(n_kv=3)), (ARG, dict(n_head=0)),
        (ARG, dict(T_kv=-1)), (ARG, dict(T_kv=1025)), (ARG, dict(q_stride=511)), (ARG, dict(out_stride=511)), (ARG, dict(scale=float("inf"))),
        (ARG, dict(q=A[0] + 2)), (ARG, dict(work=A[5] + 1)), (ARG, dict(out=A[2] + 3)),
        (LIMIT, dict(n_head=2048, q_stride=1 << 20, out_stride=1 << 20)), (LIMIT, dict(n_seq=1 << 20, q_stride=1 << 10, out_stride=1 << 10)),
        (LIMIT, dict(max_seq=1 << 25)), (ARG, dict(out=A[0])), (ARG, dict(out=A[1] + 64)), (ARG, dict(work=A[2] + 4 * (2 * 512 + 511))), (ARG, dict(work=A[0] + 64)),
        (ARG, dict(work=A[1] - nw + 4)), (ARG, dict(lens=A[2])), (ARG, dict(lens=A[5] + nw - 4)), (ARG, dict(origin=A[2] - 4)), (ARG, dict(origin=A[5])),
    ])
    assert g2hip.kv4_bytes(0, 1, 1) == g2hip.kv4_bytes(1, 1025, 1) == g2hip.kv4_work_bytes(1, 0) == g2hip.kv4_work_bytes(1 << 22, 2) == 0


def test_beam_select():
    good = dict(logits=A[0], score=A[1], done=A[2], eos=99, out_score=A[3], out_parent=A[4], out_id=A[5], out_done=A[6], groups=3, beams=4, V=100,
                n_out=4, work=A[7])
    assert code(g2hip.beam_select, {**good, "done": None, "out_done": None, "eos": -1}.values()) == STATE
    nw = g2hip.beam_work_bytes(3, 4, 100, 4)
    refused(g2hip.beam_select, good, [(ARG, {k: None}) for k in ("logits", "score", "out_score", "out_parent", "out_id", "work")] + [
        (ARG, dict(groups=0)), (ARG, dict(beams=0)), (ARG, dict(V=0)), (ARG, dict(n_out=0)), (LIMIT, dict(beams=33)), (LIMIT, dict(n_out=65)),
        (LIMIT, dict(V=(1 << 18) + 1)), (LIMIT, dict(groups=(1 << 14) + 1)), (ARG, dict(eos=100)), (ARG, dict(eos=-2)), (ARG, dict(eos=-1)), (ARG, dict(work=A[7] + 4)),
        (ARG, dict(out_score=A[1])), (ARG, dict(out_parent=A[2] + 44)), (ARG, dict(out_id=A[0] + 4 * 1200 - 4)), (ARG, dict(out_done=A[2])), (ARG, dict(out_id=A[4])),
        (ARG, dict(out_done=A[3] + 44)), (ARG, dict(work=A[0])), (ARG, dict(out_parent=A[7] + nw - 4)),
        (ARG, dict(logits=A[0] + 2)), (ARG, dict(score=A[1] + 1)), (ARG, dict(out_score=A[3] + 2)),
    ])
    assert g2hip.beam_work_bytes(1, 33, 10, 1) == g2hip.beam_work_bytes(1, 1, 10, 65) == g2hip.beam_work_bytes(0, 1, 1, 1) == 0


def test_beam_reorder():
    good = dict(ids=A[0], ids_out=A[1], ids_stride=1024, next_ids=A[2], origin=A[3], origin_out=A[4], origin_stride=1025, parent=A[5], lens=A[6], T=1000,
                groups=3, beams=4)
    for change in (dict(ids_out=A[0], origin_out=A[3]), dict(lens=None), dict(ids=None, ids_out=None, next_ids=None), dict(origin=None, origin_out=None),
                   dict(T=0), dict(T=1023)):
        assert code(g2hip.beam_reorder, {**good, **change}.values()) == STATE
    refused(g2hip.beam_reorder, good, [
        (ARG, dict(parent=None)), (ARG, dict(ids=None)), (ARG, dict(ids_out=None)), (ARG, dict(next_ids=None)), (ARG, dict(origin=None)), (ARG, dict(origin_out=None)),
        (ARG, dict(ids=None, ids_out=None, origin=None, origin_out=None)), (ARG, dict(groups=0)), (ARG, dict(beams=0)), (LIMIT, dict(beams=33)),
        (LIMIT, dict(groups=1 << 15)), (ARG, dict(T=-1)), (ARG, dict(T=1024)), (ARG, dict(ids_stride=1000)), (ARG, dict(origin_stride=0)),
        (LIMIT, dict(T=1 << 24, ids_stride=1 << 25, origin_stride=1 << 25)), (ARG, dict(ids_out=A[0] + 4)), (ARG, dict(origin_out=A[3] - 4)),
        (ARG, dict(origin_out=A[1] + 400)), (ARG, dict(origin=A[1])), (ARG, dict(origin_out=A[0])), (ARG, dict(parent=A[1] + 4)), (ARG, dict(lens=A[4])), (ARG, dict(next_ids=A[1])),
    ])
