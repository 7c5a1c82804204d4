"""Static check of the gfx950 code: no vector or memory instruction touches the
registers of a matrix instruction's result too soon after it, on any path.

The hardware does not wait for a matrix instruction's result (other than as the C
operand of another one): the code has to keep NEED wait states before reading or
overwriting it. The compiler counts them along the paths that lead to the reader,
but visits every block once, by the first path it meets: where a branch skips a
block between the two, it can count the longer path only. A reader then gets the old
value of the result's first register, now and then (seen as wrong, nondeterministic
outputs). Kernels keep such branches out; this scan follows every path."""
import os
import re
import subprocess

import pytest

from test_store_hazards import CSRC, HIPCC, ROOT

# Wait states of a result by its passes of four cycles: passes + 3, one more from four
# passes on (the counts the compiler keeps in straight-line code).
NEED = {"16x16x32_f16": 8, "16x16x32_bf16": 8, "16x16x64_i8": 8, "16x16x32_i8": 8,
        "16x16x16_bf16": 8, "16x16x16_f16": 8, "32x32x16_f16": 12, "32x32x16_bf16": 12,
        "32x32x32_i8": 12, "32x32x8_f16": 12, "32x32x8_bf16": 12, "16x16x4_f32": 12,
        "32x32x2_f32": 20}
_MFMA = re.compile(r"^v_mfma_[a-z0-9]+_(\d+x\d+x\d+_[a-z0-9]+?)(?:_1k)?$")
_REG = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")


def _regs(text):
    out = set()
    for kind, one, lo, hi in _REG.findall(text):
        if one:
            out.add(kind + one)
        else:
            out |= {kind + str(i) for i in range(int(lo), int(hi) + 1)}
    return out


def _parse(asm_text):
    """Functions as (instructions, labels): (op, operand text), label -> index."""
    funcs, code, labels = [], [], {}
    for line in asm_text.split("\n"):
        t = line.split(";")[0].strip()
        if not t:
            continue
        if t.endswith(":"):
            if t.startswith("_Z") or not t.startswith("."):
                code, labels = [], {}
                funcs.append((code, labels))
            labels[t[:-1]] = len(code)
        elif not t.startswith("."):
            op, _, rest = t.partition(" ")
            op, _, rest2 = op.partition("\t")
            code.append((op, (rest2 + " " + rest).strip()))
    return funcs


def scan(asm_text, need=NEED):
    """(matrix instruction, reader, wait states) of every path that is too short."""
    bad = []
    for code, labels in _parse(asm_text):
        for i, (op, rest) in enumerate(code):
            m = _MFMA.match(op)
            if not m:
                continue
            want = need[m.group(1)]
            dst = _regs(rest.split(",")[0])
            todo, seen = [(i + 1, 0, frozenset(dst))], {}
            while todo:
                at, waits, regs = todo.pop()
                while at < len(code) and waits < want and regs:
                    if seen.get((at, regs), want) <= waits:
                        break
                    seen[(at, regs)] = waits
                    o, r = code[at]
                    if o.startswith(("s_endpgm", "s_setpc")):
                        break
                    if o == "s_branch":
                        at, waits = labels.get(r, len(code)), waits + 1
                        continue
                    if o.startswith("s_cbranch"):
                        todo.append((labels.get(r, len(code)), waits + 1, regs))
                    elif o == "s_nop":
                        waits += int(r, 0)
                    elif _MFMA.match(o):
                        d, a, b, _c = [_regs(x) for x in r.split(",")[:4]]
                        if (a | b) & regs:
                            bad.append((f"{op} {rest}", f"{o} {r}", waits))
                        regs = regs - d  # the later one's own path counts from there
                    elif o.startswith(("v_", "ds_", "buffer_", "global_", "flat_", "scratch_")):
                        if _regs(r) & regs:
                            bad.append((f"{op} {rest}", f"{o} {r}", waits))
                            break
                    at, waits = at + 1, waits + 1
    return bad


# A matrix instruction reads its C operand late: a vector instruction may write over it
# (where it is not the result's own registers) only so many wait states later. Written
# out by hand the compiler does not see such an instruction as one. By the passes, as
# NEED: one less than those.
KEEP = {form: n - 5 for form, n in NEED.items()}


def scan_c(asm_text):
    """(matrix instruction, writer, wait states) where C is written over too soon, in a
    straight line from the instruction."""
    bad = []
    for code, _ in _parse(asm_text):
        for i, (op, rest) in enumerate(code):
            m = _MFMA.match(op)
            if not m:
                continue
            ops = rest.split(",")
            regs = _regs(ops[3]) - _regs(ops[0]) if len(ops) > 3 else set()
            want = KEEP[m.group(1)]
            waits = 0
            for o, r in code[i + 1:i + 1 + want]:
                if waits >= want or not regs:
                    break
                if o == "s_nop":
                    waits += int(r, 0)
                elif o.startswith("v_") and not _MFMA.match(o) and _regs(r.split(",")[0]) & regs:
                    bad.append((f"{op} {rest}", f"{o} {r}", waits))
                waits += 1
    return bad


@pytest.mark.slow
@pytest.mark.parametrize("src", ["sdq_gemm.hip", "sdq_glue.hip", "sdq_sdpa.hip", "sdq_w4.hip",
                                 "sdq_kv_attn.hip"])
def test_results_are_waited_for_on_every_path(tmp_path, src):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = tmp_path / (src + ".s")
    r = subprocess.run(
        [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off",
         "-fno-gpu-flush-denormals-to-zero", "-fhip-fp32-correctly-rounded-divide-sqrt",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-I" + os.path.join(ROOT, "include"), "--cuda-device-only", "-S", os.path.join(CSRC, src),
         "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    assert "v_mfma_" in text
    bad = scan(text)
    assert not bad, f"{len(bad)} results touched too soon:\n" + "\n".join(
        f"{a}  ->  {b}  ({n} wait states)" for a, b, n in bad[:10])
    bad = scan_c(text)
    assert not bad, f"{len(bad)} C operands written over too soon:\n" + "\n".join(
        f"{a}  ->  {b}  ({n} wait states)" for a, b, n in bad[:10])


def test_scan_sees_a_c_operand_written_over():
    asm = """
kernel:
    v_mfma_f32_16x16x32_f16 v[22:25], v[22:25], v[52:55], v[48:51]
    s_nop 1
    v_fma_mix_f32 v50, v60, -1.0, v61 op_sel_hi:[1,0,0]
    s_endpgm
"""
    assert [n for _, _, n in scan_c(asm)] == [2]
    assert not scan_c(asm.replace("s_nop 1", "s_nop 2"))
    assert not scan_c(asm.replace("v50", "v52"))


def test_scan_follows_the_shorter_path():
    asm = """
kernel:
    v_mfma_f32_16x16x32_f16 v[22:25], v[22:25], v[52:55], v[48:51]
    s_cbranch_scc1 .L1
    global_load_dwordx4 v[2:5], v[26:27], off
    s_nop 7
.L1:
    s_waitcnt lgkmcnt(0)
    s_nop 0
    v_fmac_f32_e32 v59, v22, v18
    s_endpgm
"""
    assert [n for _, _, n in scan(asm)] == [3]
    assert not scan(asm.replace("s_nop 0", "s_nop 5"))
    assert scan(asm.replace("s_nop 0", "s_nop 4"))
    # as another matrix instruction's C operand no wait is needed, as its A or B it is
    other = asm.replace("v_fmac_f32_e32 v59, v22, v18",
                        "v_mfma_f32_16x16x32_f16 v[22:25], v[6:9], v[10:13], v[22:25]")
    assert not scan(other)
    assert scan(other.replace("v[6:9]", "v[22:25]"))
    # an overwritten register is the later instruction's
    assert not scan(asm.replace("s_waitcnt lgkmcnt(0)",
                                "v_mfma_f32_16x16x32_f16 v[22:25], v[6:9], v[10:13], 0\n    s_nop 7"))
    # a store of the result, and a write over it
    assert scan(asm.replace("v_fmac_f32_e32 v59, v22, v18", "global_store_dwordx4 v[0:1], v[22:25], off"))
    assert scan(asm.replace("v_fmac_f32_e32 v59, v22, v18", "v_mov_b32_e32 v25, 0"))
