"""Wait states around the matrix instructions of the model's unit (hip_model.hip with the serving operators), in the
gfx950 code of the built library.  The hardware does not hold a vector instruction back until a matrix instruction has
read its accumulator or written its result: instructions between them, or s_nop, have to.  The compiler sees to it
wherever it knows both, which it does not inside inline assembly."""
import collections
import os
import re
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
OBJ = os.path.join(os.path.dirname(HERE), "_build", "hip_model.o")
sys.path.insert(0, os.path.join(HERE, "hostcheck"))

# least wait states (instructions in between; s_nop N is N + 1) that the compiler leaves around these instructions
# where it made both sides, of this unit's kernels without inline assembly: v_mfma_f32_16x16x32_bf16
LEAST = {"accumulator read, then written": 3, "result written, then written or read": 8, "operand written, then read": 2}


def regs(op):
    m = re.fullmatch(r"-?\|?v(\d+)\|?|-?v\[(\d+):(\d+)\]|sext\(v(\d+)\)", op)
    if not m:
        return range(0)
    one = m[1] or m[4]
    return range(int(one), int(one) + 1) if one else range(int(m[2]), int(m[3]) + 1)


def waits(lines, matrix="v_mfma_f32_16x16x32_bf16"):
    """{dependence: fewest wait states} of one kernel's listing, along its lines"""
    least = dict.fromkeys(LEAST, 99)
    now = 0
    read_c, result, vector = {}, {}, {}                  # register -> when the instruction was issued

    def see(what, table, r):
        if r in table:
            least[what] = min(least[what], now - table[r] - 1)

    for line in lines:
        text = line.split("//")[0].split("<")[0].strip()
        name, _, rest = text.partition(" ")
        if name == "s_nop":
            now += int(rest, 0) + 1
            continue
        if name in ("s_branch", "s_endpgm", "s_setpc_b64"):    # what follows comes from elsewhere
            read_c, result, vector = {}, {}, {}
            continue
        now += 1
        if not name.startswith("v_"):
            if name.startswith(("global_load", "buffer_load", "ds_read")):   # the loads' own counters order these
                for r in regs(rest.split(",")[0].strip()):
                    vector.pop(r, None)
            continue
        ops = [o.strip().split(" ")[0] for o in rest.split(",")]
        if name.startswith("v_mfma"):
            for r in (r for o in ops[1:3] for r in regs(o)):
                see("operand written, then read", vector, r)
            if name == matrix:
                for r in regs(ops[3]):
                    read_c[r] = now
                for r in regs(ops[0]):
                    result[r] = now
            else:
                for r in regs(ops[0]):
                    result.pop(r, None)
            for r in regs(ops[0]):
                vector.pop(r, None)
            continue
        both = name.startswith("v_permlane") or name.startswith("v_swap")
        for i, o in enumerate(ops):
            for r in regs(o):
                see("result written, then written or read", result, r)
                if i == 0 or (both and i == 1):
                    see("accumulator read, then written", read_c, r)
                    read_c.pop(r, None)
                    vector[r] = now
        for r in regs(ops[0]):
            result.pop(r, None)
    return least


def kernels(tmp):
    import kernel_args
    list(kernel_args.kernels_of(OBJ, tmp))
    text = subprocess.run([f"{kernel_args.LLVM}/llvm-objdump", "-d", "--no-show-raw-insn", os.path.join(tmp, "hip_model.o.co")],
                          check=True, capture_output=True, text=True).stdout
    out, name = collections.OrderedDict(), None
    for line in text.splitlines():
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            name = m[1]
            out[name] = []
        elif name and line.startswith("\t"):
            out[name].append(line)
    return out


def test_the_scan_counts_as_the_table_says():
    listing = ["v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[4:7]", "v_add_f32_e32 v20, v21, v22",
               "v_mov_b32_e32 v5, v20", "s_nop 3", "v_mul_f32_e32 v30, v1, v31", "v_mov_b32_e32 v12, 0",
               "v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], 0"]
    assert waits(listing) == {"accumulator read, then written": 1, "result written, then written or read": 6,
                              "operand written, then read": 0}


@pytest.mark.skipif(not os.path.exists(OBJ) or not os.path.exists("/opt/rocm/llvm/bin/llvm-objdump"),
                    reason="the library is not built here")
def test_vector_instructions_wait_for_matrix_instructions(tmp_path):
    found = {n: waits(t) for n, t in kernels(str(tmp_path)).items() if any("v_mfma_f32_16x16x32_bf16" in x for x in t)}
    assert len(found) >= 28, len(found)
    short = {n: {k: v for k, v in w.items() if v < LEAST[k]} for n, w in found.items()}
    short = {n: w for n, w in short.items() if w}
    assert not short, "\n".join(f"{n}: {w}" for n, w in short.items())
