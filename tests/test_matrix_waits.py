"""No built kernel reads the result of a matrix instruction before it is there.

The hardware does not hold back a vector instruction that reads a result which the
matrix cores are still working on: the compiler counts the wait states between them.  It
can miss some where a branch lies between, and then the last products are missing from
what is read, now and then.  So every path from every matrix instruction is followed here,
in the disassembly of the library's own kernels, until the wait is over."""
import glob
import os
import re
import shutil
import subprocess

import pytest

import edgecore_amd as ec

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"

# wait states (an instruction is one, s_nop n is n + 1) from an instruction to a reader of its
# result: 4 more than its passes of 4 cycles, 2 more for fp32's own
STATES = {"f32_32x32x16_f16": 12, "f32_16x16x32_f16": 8, "f32_16x16x32_bf16": 8, "i32_16x16x64_i8": 8, "f32_16x16x4_f32": 10,
          "f32_16x16x1_4b_f32": 10}


def registers(op):
    m = re.match(r"[-|]*([av])(\d+)", op)
    if m:
        return {m[1] + m[2]}
    m = re.match(r"[-|]*([av])\[(\d+):(\d+)\]", op)
    return {m[1] + str(i) for i in range(int(m[2]), int(m[3]) + 1)} if m else set()


def kernels(text):
    """{name: [(address, instruction, operands)]}; a branch's operand is its target's address."""
    label = {m[2]: int(m[1], 16) for m in re.finditer(r"(?m)^([0-9a-f]+) <(\w+)>:", text)}
    out, code = {}, None
    for line in text.splitlines():
        m = re.match(r"[0-9a-f]+ <(_Z\w+)>:", line)  # (others are labels inside a kernel)
        if m:
            code = out[m[1]] = []
        m = re.match(r"\s+([a-z]\w+)\s*(.*?)\s*// ([0-9A-F]+): ", line)
        if not m or code is None:
            continue
        at, ops = int(m[3], 16), [x.strip() for x in re.split(r",(?![^\[]*\])", m[2])]
        if m[1].startswith(("s_branch", "s_cbranch")):
            to = ops[0]
            ops = [at + 4 + 4 * (int(to) - (int(to) >> 15 << 16)) if to.isdigit() else label[to]]
        code.append((at, m[1], ops))
    return out


def too_soon(code):
    """(matrix instruction, reader, states between them) of a kernel."""
    index = {at: i for i, (at, _, _) in enumerate(code)}
    bad = []
    for i, (_, op, ops) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        need = STATES[op[len("v_mfma_"):]]  # (an unknown one: its passes belong in the table)
        paths, seen = [(i + 1, 0, frozenset(registers(ops[0])))], set()
        while paths:
            j, states, live = paths.pop()
            while states < need and live and j < len(code) and (j, states, live) not in seen:
                seen.add((j, states, live))
                _, o, args = code[j]
                if o == "s_endpgm":
                    break
                states += int(args[0], 0) + 1 if o == "s_nop" else 1
                if o == "s_branch":
                    j = index[args[0]]
                    continue
                if o.startswith("s_cbranch"):
                    paths.append((index[args[0]], states, live))
                elif o.startswith("v_mfma"):
                    # into the same registers it may follow at once; as a factor it may not
                    if any(registers(a) & live for a in args[1:3]):
                        bad.append((op, o, states - 1))
                    live -= registers(args[0])
                elif o[0] in "vgdbf" or o.startswith("scratch"):
                    if any(registers(a) & live for a in args):
                        bad.append((op, f"{o} {args}", states - 1))
                        break
                j += 1
    return bad


def test_scan():
    """The scan itself, on lines as the disassembler writes them."""
    lines = ["0000000000001000 <_Zk>:",
             "\tv_mfma_f32_32x32x16_f16 v[2:17], v[20:23], v[24:27], v[2:17] // 000000001000: D3D40002 040A3114",
             "\ts_cbranch_vccz 2 // 000000001008: BF860002 <_Zk+0x14>", "\ts_nop 11 // 00000000100C: BF80000B",
             "\tv_add_f32_e32 v1, v2, v3 // 000000001010: 02020702", "\ts_endpgm // 000000001014: BF810000"]

    def states():
        return [b[2] for b in too_soon(kernels("\n".join(lines))["_Zk"])]

    assert states() == []
    lines[2] = lines[2].replace("vccz 2", "vccz 1")
    assert states() == [1]
    lines[2], lines[3] = "\ts_nop 5 // 000000001008: BF800005", lines[3].replace("nop 11", "nop 4")
    assert states() == [11]
    lines[3] = lines[3].replace("nop 4", "nop 5")
    assert states() == []


def test_results_are_waited_for(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    shutil.copy(ec.LIB_PATH, tmp_path / "l.so")
    subprocess.run([OBJDUMP, "--offloading", "l.so"], cwd=tmp_path, check=True, capture_output=True)
    bad, n = [], 0
    for f in sorted(glob.glob(str(tmp_path / "*amdgcn*gfx950*"))):
        text = subprocess.run([OBJDUMP, "-d", f], check=True, capture_output=True, text=True).stdout
        for name, code in kernels(text).items():
            n += any(o.startswith("v_mfma") for _, o, _ in code)
            bad += [(name, *b) for b in too_soon(code)]
    assert n > 100 and not bad, (n, bad[:5])
