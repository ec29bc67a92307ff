"""Calls of the operators for several texts at once that are refused because a kernel would read something else than it was
given, without a GPU (addresses are numbers)."""
import pytest

import g2hip
from test_batch_contract import A, ARG, STATE, code, no_runtime  # noqa: F401 (the fixture skips where the runtime is up)

CALLS = {
    "attn_prompt": (dict(q=A[0], q_stride=768, k=A[1], v=A[2], kv_stride=256, out=A[3], out_stride=512, dtype=0, q_start=A[4], k_start=A[5], n_seq=3,
                         q_rows=100, k_rows=120, n_head=8, n_kv=4, scale=0.125), ["q_start", "k_start"]),
    "kv4_append": (dict(k=A[0], v=A[1], stride=256, dtype=0, cache=A[2], row_start=A[3], pos=A[4], start=0, n_seq=3, rows=100, n_kv=4, max_seq=1024),
                   ["row_start", "pos"]),
    "kv4_read": (dict(cache=A[0], k=A[1], v=A[2], origin=A[3], lens=A[4], T_kv=1024, start=10, T=1000, n_seq=3, n_kv=4, max_seq=1024), ["origin", "lens"]),
    "attn_kv4": (dict(q=A[0], q_stride=768, cache=A[1], out=A[2], out_stride=512, origin=A[3], lens=A[4], T_kv=1000, n_seq=3, n_head=8, n_kv=4,
                      max_seq=1024, scale=0.125, work=A[5]), ["origin", "lens"]),
    "beam_select": (dict(logits=A[0], score=A[1], done=A[2], eos=99, out_score=A[3], out_parent=A[4], out_id=A[5], out_done=A[6], groups=3, beams=4,
                         V=100, n_out=4, work=A[7]), ["done", "out_parent", "out_id", "out_done"]),
    "beam_reorder": (dict(ids=A[0], ids_out=A[1], ids_stride=1024, next_ids=A[2], origin=A[3], origin_out=A[4], origin_stride=1025, parent=A[5],
                          lens=A[6], T=1000, groups=3, beams=4), ["ids", "ids_out", "next_ids", "origin", "origin_out", "parent", "lens"]),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_ints_at_ints_addresses(name):
    """Scalar loads drop an address's last two bits."""
    good, ints = CALLS[name]
    fn = getattr(g2hip, name)
    assert code(fn, good.values()) == STATE
    for arg in ints:
        for off in (1, 2, 3):
            assert code(fn, {**good, arg: good[arg] + off}.values()) == ARG, (arg, off)
            assert "int's address" in g2hip.last_error()


@pytest.mark.parametrize("name", ["attn_prompt", "attn_kv4"])
def test_scales_whose_unit_overflows(name):
    """Scores are taken in units of log 2: scale / log 2 has to be finite, or a score of 0 becomes NaN."""
    good, _ = CALLS[name]
    fn = getattr(g2hip, name)
    for scale in (2.0 ** 127, -(2.0 ** 127), 0.0):
        assert code(fn, {**good, "scale": scale}.values()) == STATE
    for scale in (1.0001 * 2.0 ** 127, -3e38, float("-inf"), float("nan")):
        assert code(fn, {**good, "scale": scale}.values()) == ARG
