"""No instruction of the paged attention reads a matrix product's result before it is there: the hardware does not hold a vector
instruction back, the compiler counts the wait, and where a branch lies between the two it has been seen to count one way only.
Checked over the assembly that the library's own source compiles to, along every way from a product.  CPU only."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "peregrine_amd", "csrc")
# Wait states from a product to a vector, LDS or memory instruction that reads its result: four more than its passes (4 and 8 of them).
NEED = {"16x16x64_i8": 8, "16x16x32_f16": 8, "32x32x16_f16": 12}


def registers(text):
    out = set()
    for a, b in re.findall(r"v\[(\d+):(\d+)\]", text):
        out |= set(range(int(a), int(b) + 1))
    return out | {int(a) for a in re.findall(r"\bv(\d+)\b", text)}


def reads(op, rest):
    """The vector registers that an instruction reads; a product's addend is forwarded to it and does not count."""
    parts = [p.strip() for p in re.split(r",(?![^\[]*\])", rest)]
    if op.startswith("v_mfma"):
        return registers(",".join(parts[1:3]))
    if op.startswith(("ds_write", "global_store", "buffer_store", "scratch_store")):
        return registers(rest)
    if op.startswith(("v_", "ds_", "global_", "buffer_", "scratch_")):
        got = registers(",".join(parts[1:]))
        return got | (registers(parts[0]) if re.search("fmac|swap|dot", op) else set())
    return set()


def early_readers(body):
    """(product, reader, wait states between) of a function's assembly, branches followed."""
    lines = [x for x in (x.split(";")[0].strip() for x in body.split("\n")) if x and not (x.startswith(".") and not x.startswith(".LBB"))]
    labels = {x[:-1]: i for i, x in enumerate(lines) if x.endswith(":")}
    found = []
    for start, product in enumerate(lines):
        m = re.match(r"v_mfma_\w+?_(\d+x\d+x\d+_\w+)\s+(\S+),", product)
        if not m:
            continue
        need, result = NEED[m.group(1)], registers(m.group(2))
        ways, seen = [(start + 1, 0)], {}
        while ways:
            at, waited = ways.pop()
            while at < len(lines) and waited < need and seen.get(at, need) > waited:
                seen[at] = waited
                line = lines[at]
                at += 1
                if line.endswith(":"):
                    continue
                op = line.split()[0]
                if reads(op, line[len(op):]) & result:
                    found.append((product, line, waited))
                    break
                if op == "s_endpgm":
                    break
                if op == "s_branch":
                    at, waited = labels[line.split()[1]], waited + 1
                    continue
                if op.startswith("s_cbranch"):
                    ways.append((labels[line.split()[1]], waited + 1))
                nop = re.match(r"s_nop (\w+)", line)
                waited += int(nop.group(1), 0) + 1 if nop else 1
    return found


def test_the_check_sees_a_reader_behind_a_branch():
    product = "v_mfma_i32_16x16x64_i8 v[0:3], v[8:11], v[12:15], v[0:3]\n"
    assert early_readers(product + "v_add_f32_e32 v20, v21, v2\ns_endpgm")
    assert not early_readers(product + "s_nop 7\nv_add_f32_e32 v20, v21, v2\ns_endpgm")
    assert not early_readers(product + "v_mfma_i32_16x16x64_i8 v[0:3], v[16:19], v[12:15], v[0:3]\ns_nop 7\nv_add_f32_e32 v20, v21, v2\ns_endpgm")
    around = product + "s_cbranch_vccz .LBB0_2\ns_nop 7\n.LBB0_2:\nv_add_f32_e32 v20, v21, v2\ns_endpgm"
    assert [f[2] for f in early_readers(around)] == [1]                   # (the other way has waited)
    back = ".LBB0_1:\nv_mul_f32_e32 v5, v4, v2\n" + product + "v_mov_b32_e32 v6, v7\ns_cbranch_scc1 .LBB0_1\ns_nop 7\nds_write_b32 v9, v3\ns_endpgm"
    assert [f[1].split()[0] for f in early_readers(back)] == ["v_mul_f32_e32"]


@pytest.mark.skipif(not (shutil.which("make") and (os.path.exists("/opt/rocm/bin/hipcc") or shutil.which("hipcc"))), reason="needs hipcc")
def test_paged_attention_waits_for_its_products():
    target = "../../build/csrc/pg_kv4_attn.s"
    subprocess.run(["make", "-C", CSRC, target], check=True, capture_output=True, timeout=600)
    with open(os.path.join(CSRC, target)) as f:
        text = f.read()
    functions = re.findall(r"\n(_ZN\S*kv4_\S*):\s*; @(.*?)\.Lfunc_end", text, re.S)
    products = sum(body.count("v_mfma_") for _, body in functions)
    assert len(functions) > 40 and products == text.count("v_mfma_") > 1000
    for name, body in functions:
        assert not early_readers(body), name
