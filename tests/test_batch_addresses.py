"""CPU check of the index arithmetic of the operators for several texts at once and of the host's choice of forms.

tests/native/batch_addr.cpp compiles the kernels' own index functions (csrc/g2_batch_plan.h) with g++ and walks the
cache's tiles, the pieces of work, the search of a row's sequence (in lists of starts, and in lists in no order, whose
probes have to stay inside) and the keys that a row sees; a planted mistake must be caught.  No GPU is involved."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import g2hip
import test_batch_gpu as gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "gpt2-opencl-1.1_amd", "csrc")


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("batch") / "batch_addr")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I" + CSRC, "-o", out, os.path.join(ROOT, "tests", "native", "batch_addr.cpp")],
                   check=True)

    def run(*args):
        return subprocess.run([out, *map(str, args)], capture_output=True, text=True).stdout.strip()

    return run


@pytest.mark.parametrize("S,NKV,max_seq", [(1, 1, 1), (1, 3, 32), (2, 5, 33), (3, 25, 1000), (7, 12, 1024)])
def test_cache(walk, S, NKV, max_seq):
    assert walk("cache", S, NKV, max_seq) == "ok"
    assert g2hip.kv4_bytes(S, NKV, max_seq) == S * NKV * -(-max_seq // 32) * 2304
    assert walk("cache", S, NKV, max_seq, 1) != "ok"


@pytest.mark.parametrize("NKV", [1, 2, 4, 5, 7, 8, 9, 12, 16, 20, 25, 40, 1023])
def test_items(walk, NKV):
    for tiles in (1, 2, 7, 8, 9, 63, 250):
        assert walk("items", NKV, tiles) == "ok"


@pytest.mark.parametrize("n", [2, 3, 63, 64, 65, 66, 128, 129, 1000, 4096, 4097, 5000])
def test_search(walk, n):
    assert walk("search", n, n) == "ok"


def test_rows(walk):
    for seed in range(3):
        assert walk("rows", seed) == "ok"


def beam_form(rows, V):
    fn = g2hip._lib.g2i_beam_form
    fn.argtypes = [C.c_int, C.c_int, C.POINTER(C.c_int)]
    slices = C.c_int()
    return fn(rows, V, C.byref(slices)), slices.value


def test_beam_workspace(walk):
    for G, B, V, n in ((1, 1, 1, 1), (1, 4, 50257, 4), (16, 8, 50257, 8), (3, 7, 4097, 64), (2048, 32, 262144, 64)):
        times, slices = beam_form(G * B, V)
        assert (slices - 1) * 4096 * times < V <= slices * 4096 * times and slices <= 64
        assert walk("beams", G, G * B, slices, n) == "ok"
        assert g2hip.beam_work_bytes(G, B, V, n) == 64 * G + G * B * slices * 8 * (1 + n)
        assert G * B * slices * 1024 < 2 ** 32


def test_every_form_of_the_selection_is_tested():
    cases = [m for m in gpu.test_select.pytestmark if m.name == "parametrize"][0].args[1]
    seen = {(beam_form(G * B, V)[0], beam_form(G * B, V)[1] > 1) for G, B, V, _ in cases}
    assert len(seen) == 6


def prompt_form(f16, q_rows, k_rows, S, NH, NKV):
    fn = g2hip._lib.g2i_prompt_form
    fn.argtypes = [C.c_int] * 6 + [C.POINTER(C.c_long)]
    tiles = C.c_long()
    return fn(int(f16), q_rows, k_rows, S, NH, NKV, C.byref(tiles)), tiles.value


def test_prompt_tiles_cover_the_rows():
    for f16 in (False, True):
        for S in (1, 2, 63, 64, 500):
            for rows in (1, 31, 32, 33, 600, 5000, 100000):
                for NH, NKV in ((1, 1), (12, 12), (16, 4), (25, 5), (7, 1)):
                    form, tiles = prompt_form(f16, rows, rows, S, NH, NKV)
                    size, group = 32 if form == 0 else 128, NH // NKV
                    assert tiles >= -(-rows * group // size)
                    if 1 < S < 64:  # (sequences' own tiles: the most is one that is not full for each)
                        lens = [rows // S + (i < rows % S) for i in range(S)]
                        assert tiles >= sum(-(-n * group // size) for n in lens)


def test_every_form_of_the_prompts_is_tested():
    cases = [(f16, seqs, NH, NKV) for f16, seqs, NH, NKV in gpu.prompt_forms()]
    cases += [(f16, s, NH, NKV) for f16 in (False, True) for s in gpu.SEQS.values() for NH, NKV in gpu.HEADS]
    seen = set()
    for f16, seqs, NH, NKV in cases:
        n, m = sum(n for n, _ in seqs), sum(max(0, n + p) for n, p in seqs)
        seen.add((f16, prompt_form(f16, max(n, 1), m, len(seqs), NH, NKV)[0], min(len(seqs), 64) // 32))
    for f16, form in ((False, 0), (False, 1), (True, 0), (True, 1), (True, 2)):
        assert {k for g, f, k in seen if (g, f) == (f16, form)} >= {0, 2}, (f16, form, seen)


def kv4_form(S, NH, NKV, T):
    fn = g2hip._lib.g2i_kv4_form
    fn.argtypes = [C.c_int] * 4 + [C.POINTER(C.c_int)] * 4
    heads, chunks, span, waves = C.c_int(), C.c_int(), C.c_int(), C.c_int()
    splits = fn(S, NH, NKV, T, C.byref(heads), C.byref(chunks), C.byref(span), C.byref(waves))
    return splits, heads.value, chunks.value, span.value, waves.value


def test_attention_parts():
    for NKV in (1, 2, 3, 5, 12, 25, 512):
        for group in (1, 2, 3, 4, 5, 7, 8, 9, 16, 25):
            for S in (1, 3, 48, 1000):
                for T in (0, 1, 31, 32, 33, 256, 257, 700, 1024, 5000, 50001, 1 << 24):
                    splits, heads, chunks, span, waves = kv4_form(S, NKV * group, NKV, T)
                    tiles = max(1, -(-T // 32))
                    assert 1 <= splits <= 32 and (splits - 1) * span < tiles <= splits * span
                    assert 1 <= heads <= 4 and (chunks - 1) * heads < group <= chunks * heads
                    assert waves in (1, 4, 8) and (waves > 1 or heads == 1) and S * NKV * chunks * splits * 64 * waves < 2 ** 32


def test_every_form_of_the_attention_is_tested():
    got = {(f[0] > 1, f[1] if f[1] < 3 else 4, f[4]) for f in (kv4_form(*c) for c in gpu.attention_cases())}
    assert {f[1:] for f in got} == {(1, 1), (1, 4), (1, 8), (2, 4), (2, 8), (4, 4), (4, 8)} and {f[0] for f in got} == {False, True}
    through = {(f[1] if f[1] < 3 else 4, f[4]) for f in (kv4_form(*c) for c in gpu.ORIGINS)}
    assert through == {f[1:] for f in got}
