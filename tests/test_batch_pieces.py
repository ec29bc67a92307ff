"""CPU check of the pieces of keys of a tile of 128 queries (tests/native/batch_pieces.cpp): every key in one piece, as many
turns for both groups of waves, none where no row of the tile sees a key, and no int that overflows on the way."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("pieces") / "batch_pieces")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "gpt2-opencl-1.1_amd", "csrc"), "-o", out, os.path.join(ROOT, "tests", "native", "batch_pieces.cpp")], check=True)
    return lambda *args: subprocess.run([out, *map(str, args)], capture_output=True, text=True)


@pytest.mark.parametrize("seed", range(3))
def test_pieces(walk, seed):
    r = walk(seed)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_pieces_of_no_keys_unguarded(walk):
    """Without the guard the walk ends: the ints overflow."""
    r = walk(0, "mistake")
    assert r.returncode != 0 or r.stdout.strip() != "ok"
