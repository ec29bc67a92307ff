"""The built code object's matrix instructions and who reads their results.

A vector instruction that reads a matrix instruction's result too soon reads what was there before: the compiler puts
the wait there, and within a block it does.  Behind a branch it once did not (the sum of a product's two parts, moved
into the block after an `if` that followed the products: one of 25 chunk lengths and groups gave wrong sums).  This
test walks the disassembly of the library's own kernels, along branches too, from every matrix instruction to the
first reader of its result: at least 8 wait states for the 16x16x32 products of 16-bit values, which is what the
compiler leaves within a block, 4 for any."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HSACO = os.path.join(ROOT, "gpt2-opencl-1.1_amd", "build", "g2_kernels.hsaco")
LLVM = "/opt/rocm/llvm/bin"


def need(name):
    return 8 if re.match(r"v_mfma_f32_16x16x32_(f16|bf16)", name) else 4


def registers(text):
    out = set()
    for a, b, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out |= {int(one)} if one else set(range(int(a), int(b) + 1))
    return out


def parse(text):
    """{kernel: [(address, name, operands, branch target or None)]}"""
    kernels, cur = {}, None
    for line in text.splitlines():
        m = re.match(r"^[0-9a-f]+ <(\w+)>:", line)
        if m:
            cur = kernels.setdefault(m[1], [])
            continue
        m = re.match(r"^\s+(\w+)\s*([^/]*)//\s*([0-9A-F]+):[^<]*(?:<\w+\+0x([0-9a-f]+)>)?", line)
        if m and cur is not None:
            cur.append((int(m[3], 16), m[1], m[2].strip(), int(m[4], 16) if m[4] else None))
    return kernels


def early_readers(ins):
    base = ins[0][0]
    at = {a - base: i for i, (a, *_) in enumerate(ins)}
    found = []
    for i, (_, name, ops, _) in enumerate(ins):
        if not name.startswith("v_mfma"):
            continue
        walk, seen = [(i + 1, 0, frozenset(registers(ops.split(",")[0])))], set()
        while walk:
            j, waited, live = walk.pop()
            if j >= len(ins) or waited >= need(name) or not live or (j, waited) in seen:
                continue
            seen.add((j, waited))
            _, other, o, target = ins[j]
            if other == "s_endpgm":
                continue
            if other == "s_nop":
                walk.append((j + 1, waited + 1 + int(o, 0), live))
                continue
            if other == "s_branch" or other.startswith("s_cbranch"):
                if target in at:
                    walk.append((at[target], waited + 1, live))
                if other != "s_branch":
                    walk.append((j + 1, waited + 1, live))
                continue
            parts = o.split(",")
            stores = other.startswith(("global_store", "buffer_store", "ds_write", "ds_bpermute", "v_cmp"))
            reads = registers(o if stores or other.startswith(("v_fmac", "v_permlane")) else ",".join(parts[1:]))
            if not other.startswith("v_mfma") and other.startswith(("v_", "ds_", "global_", "buffer_")) and reads & live:
                found.append((name, ops, other, o, waited))
                continue
            writes = registers(parts[0]) if other.startswith("v_") else set()
            walk.append((j + 1, waited + 1, live - writes))
    return found


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HSACO) or not shutil.which(f"{LLVM}/llvm-objdump") or not shutil.which(f"{LLVM}/clang-offload-bundler"):
        pytest.skip("no built code object or no disassembler")
    out = str(tmp_path_factory.mktemp("waits") / "kernels.o")
    subprocess.run([f"{LLVM}/clang-offload-bundler", "--type=o", "--unbundle", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                    f"--input={HSACO}", f"--output={out}"], check=True)
    text = subprocess.run([f"{LLVM}/llvm-objdump", "-d", out], capture_output=True, text=True, check=True).stdout
    return parse(text)


def test_no_result_is_read_too_soon(kernels):
    products = {k: sum(n.startswith("v_mfma") for _, n, _, _ in v) for k, v in kernels.items()}
    assert sum(products.values()) > 1000 and sum(bool(n) for n in products.values()) > 50
    bad = {k: early_readers(v)[:2] for k, v in kernels.items() if products[k] and early_readers(v)}
    assert not bad, bad


def test_the_walk_sees_a_reader_behind_a_branch():
    text = """0000000000001000 <k>:
\tv_mfma_f32_16x16x32_f16 v[10:13], v[22:25], v[10:13], v[38:41]// 000000001000: D3D40826
\ts_cbranch_vccnz 2                                          // 000000001008: BF870002 <k+0x14>
\ts_nop 7                                                    // 00000000100C: BF800007
\tv_mov_b32_e32 v1, v2                                       // 000000001010: 7E020302
\tv_add_f32_e32 v3, v10, v11                                 // 000000001014: 0206170A
\ts_endpgm                                                   // 000000001018: BF810000
"""
    ins = parse(text)["k"]
    assert len(early_readers(ins)) == 1 and early_readers(ins)[0][4] == 1
    assert not early_readers([i for i in ins if i[1] != "s_cbranch_vccnz"])
