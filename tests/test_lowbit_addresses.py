"""CPU check of the low-bit operators' index arithmetic and of the host's choice of forms.

tests/native/lowbit_addr.cpp compiles the kernels' own index functions (csrc/g2_lowbit_plan.h) with g++ and walks
every lane of every chunk of laid-out weights (16-byte reads inside the buffer, every word found where its lane has
it, each one lane's), the parts of a cache buffer, the waves of an append and the blocks of a head as its waves take
them; planted mistakes must be caught.  The forms that g2i_q4_form and g2i_kv8_form choose are covered by the sizes of
test_lowbit_gpu.py.  No GPU is involved."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

import g2hip
import test_lowbit_gpu as gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "gpt2-opencl-1.1_amd", "csrc")


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("lowbit") / "lowbit_addr")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I" + CSRC, "-o", out,
                    os.path.join(ROOT, "tests", "native", "lowbit_addr.cpp")], check=True)

    def run(*args):
        r = subprocess.run([out, *map(str, args)], capture_output=True, text=True)
        return r.stdout.strip()

    return run


@pytest.mark.parametrize("K", [1, 31, 32, 33, 64, 65, 96, 97, 128, 129, 160, 192, 200, 255, 256, 257, 768, 1600, 1633, 6400])
def test_weights(walk, K):
    for N in (1, 16, 17, 100):
        assert walk("weights", N, K) == "ok"


@pytest.mark.parametrize("K", [32, 64, 96, 160])
def test_planted_mistakes_in_reading_weights(walk, K):
    assert walk("weights", 16, K, 1) != "ok"  # lanes read past a short chunk's end
    assert walk("weights", 16, K, 2) != "ok"  # words that moved are not moved back


@pytest.mark.parametrize("S,NH,max_seq", [(1, 1, 1), (1, 1, 16), (3, 5, 17), (2, 25, 1000), (7, 12, 1024)])
def test_cache(walk, S, NH, max_seq):
    assert walk("cache", S, NH, max_seq) == "ok"


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 250, 1001])
def test_append(walk, T):
    for S, NH in ((1, 1), (1, 12), (3, 25), (5, 7)):
        assert walk("append", S, NH, T) == "ok"


def kv8_form(heads, T_kv):
    fn = g2hip._lib.g2i_kv8_form
    fn.argtypes = [C.c_long, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int)]
    span, waves = C.c_int(), C.c_int()
    splits = fn(heads, T_kv, C.byref(span), C.byref(waves))
    return splits, span.value, waves.value


@pytest.mark.parametrize("heads", [1, 3, 12, 25, 100, 255, 256, 512, 3000])
def test_attention_parts(walk, heads):
    for T in (0, 1, 15, 16, 17, 64, 65, 128, 129, 512, 513, 1008, 1023, 1024, 1025, 1040, 1300, 2048, 4001, 8192, 50001):
        splits, span, waves = kv8_form(heads, T)
        blocks = max(1, -(-T // 16))
        assert 1 <= splits <= 32 and waves in (1, 4, 8) and heads * splits <= max(heads, 512) and (splits - 1) * span < blocks
        for n in sorted({0, 1, T // 2, max(0, T - 1), T, T // 16 * 16}):
            if n <= T:
                assert walk("attend", blocks, span, splits, waves, n) == "ok", (heads, T, n)


def test_planted_mistakes_in_taking_blocks(walk):
    assert walk("attend", 64, 64, 1, 8, 1001, 1) != "ok"
    assert walk("attend", 64, 16, 4, 4, 1001, 1) != "ok"
    assert walk("attend", 64, 64, 1, 4, 1001, 2) != "ok"  # the last block is a wave's that is not there


def q4_form(M, N, K):
    fn = g2hip._lib.g2i_q4_form
    fn.argtypes = [C.c_int, C.c_int, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_uint)]
    waves, wgs = C.c_int(), C.c_uint()
    return fn(M, N, K, C.byref(waves), C.byref(wgs)), waves.value, wgs.value


def kernels():
    """Names of the 4-bit products' kernels for groups of 32, by the position in the kernel table."""
    text = open(os.path.join(CSRC, "g2_internal.h")).read()
    return {f"{'h' if m[0] else ''}{m[1]}_{m[2]}_{m[3]}" for m in re.findall(r"G2_Q4MV(H?)_LIST\(X, (\d+), (\d+), (\d+)\)", text)
            if m[1].isdigit()}


def test_every_form_of_a_product_is_tested():
    forms = {q4_form(M, N, K)[0] for M, N, K, _ in gpu.product_cases()}
    assert len(forms) == len(kernels()), (sorted(forms), kernels())
    seen = {(q4_form(M, N, K)[0], G) for M, N, K, G in gpu.product_cases()}
    assert len(seen) == 3 * len(forms)  # each with every group


def test_products_launch_within_limits():
    for M in (1, 2, 8, 65535):
        for N in (1, 16, 17, 2048, 4095, 8192, 32768, 50257, 1 << 24):
            for K in (1, 128, 1024, 1025, 2048, 2049, 4096, 4097, 1 << 24):
                _, waves, wgs = q4_form(M, N, K)
                assert 1 <= wgs and wgs * waves * 64 < 2 ** 32 and wgs <= -(-N // 16)


def test_every_form_of_the_attention_is_tested():
    got = {(kv8_form(h, T)[0] > 1, kv8_form(h, T)[2]) for h, T in gpu.attention_cases()}
    assert got >= {(False, 1), (False, 4), (False, 8), (True, 4), (True, 8)}
