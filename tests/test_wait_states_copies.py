"""Copies from memory into LDS, in the assembly that the library's own flags give:
what the hardware does not hold back by itself is waited for.

  - between a scalar write of M0, which holds the place in LDS, and the copy that
    goes by it: one wait state;
  - between a vector instruction's write of a scalar register (v_readfirstlane_b32,
    a comparison) and a memory instruction that takes its address from it: five.

The compiler puts these where it emits both instructions itself, and does not look
into an asm string.  `early_copies` follows every way out of every write."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from fable5_llm_amd import build
from wait_states import functions

MEMORY = ("global_", "buffer_", "flat_", "scratch_")


def _scalars(operand):
    if operand in ("vcc", "m0"):
        return {"vcc_lo", "vcc_hi"} if operand == "vcc" else {"m0"}
    m = re.match(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return {f"s{i}" for i in range(int(m[1]), int(m[2]) + 1)}
    return {operand} if re.match(r"(s\d+|vcc_lo|vcc_hi)$", operand) else set()


def _into_lds(op, line):
    return op.startswith("global_load_lds") or (op.startswith("buffer_load") and
                                                re.search(r"\blds\b", line))


def _written(op, operands, line):
    """(scalar registers that an instruction writes, wait states they need)."""
    if not operands:
        return set(), 0
    if op.startswith("s_") and not op.startswith(("s_cmp", "s_bitcmp", "s_nop", "s_wait")):
        return _scalars(operands[0]), 1
    if op.startswith(("v_readfirstlane", "v_readlane", "v_cmp")):
        return _scalars(operands[0]), 5
    if "_co_" in op or op.startswith("v_div_scale"):
        return _scalars(operands[1]), 5
    return set(), 0


def early_copies(text):
    """(number of copies into LDS, ["function: write | use"]) of an assembly file."""
    found, copies = [], 0
    for name, body in functions(text).items():
        labels = {b[1][0]: i for i, b in enumerate(body) if b[0] == "label"}
        copies += sum(bool(_into_lds(op, line)) for op, _, line in body)
        for i, (op, operands, line) in enumerate(body):
            regs, need = _written(op, operands, line)
            if need == 1:
                regs &= {"m0"}
            if not regs:
                continue
            best, todo = {}, [(i + 1, 0)]
            while todo:
                j, passed = todo.pop()
                while j < len(body) and passed < need and best.get(j, need) > passed:
                    best[j] = passed
                    o, args, code = body[j]
                    j += 1
                    if o == "label":
                        continue
                    if o == "s_endpgm":
                        break
                    if need == 1:
                        if _into_lds(o, code):
                            found.append(f"{name}: {line} | {code}")
                    elif o.startswith(MEMORY) and regs & set().union(
                            *(_scalars(a.split()[0]) for a in args if a)):
                        found.append(f"{name}: {line} | {code}")
                    if o.startswith("s_") and regs <= _written(o, args, code)[0]:
                        break                       # written again, by a scalar instruction
                    passed += int(args[0], 0) + 1 if o == "s_nop" else 1
                    if o == "s_branch":
                        j = labels[args[0]]
                    elif o.startswith("s_cbranch"):
                        todo.append((labels[args[0]], passed))
    return copies, sorted(set(found))


SAMPLE = """_Zk:
	v_readfirstlane_b32 s5, v1
	s_mov_b32 m0, s4
	s_cbranch_scc1 .LBB0_2
	%s
.LBB0_2:
	%s
	global_load_lds_dwordx4 v0, s[4:5]
	s_endpgm
.Lfunc_end0:
"""


@pytest.mark.parametrize("first,then,uses", [
    ("s_nop 0", "s_nop 2", 0), ("s_nop 3", "s_nop 1", 1), ("s_nop 0", "s_mov_b32 m0, s3", 2),
    ("s_mov_b32 m0, s3", "s_mov_b32 s5, s7", 0), ("s_mov_b32 s5, 0", "s_nop 1", 1)])
def test_the_search(first, then, uses):
    copies, found = early_copies(SAMPLE % (first, then))
    assert copies == 1 and len(found) == uses, found


def test_the_search_behind_the_write():
    text = "_Zk:\n\ts_mov_b32 m0, s4\n\t%sglobal_load_lds_dwordx4 v0, s[4:5]\n\ts_endpgm\n.Lfunc_end0:\n"
    assert early_copies(text % "")[1] and not early_copies(text % "s_nop 0\n\t")[1]


@pytest.mark.parametrize("source,least", [("w4a8_chunk.hip", 150), ("w4a8_stream.hip", 16),
                                          ("w4a8_mfma.hip", 1)])
def test_the_kernels(tmp_path, source, least):
    out = os.path.join(tmp_path, source + ".s")
    subprocess.run([build.hipcc()] + build.flags() + ["-S", "--cuda-device-only", "-o", out,
                                                       os.path.join(build.CSRC, source)],
                   check=True, capture_output=True)
    with open(out) as f:
        copies, found = early_copies(f.read())
    assert copies >= least and not found, (copies, len(found), found[:5])


def test_no_other_source_copies_into_lds():
    sources = [s for s in build.SOURCES
               if re.search(r"load_lds|lds_dword", open(os.path.join(build.CSRC, s)).read())]
    headers = [h for h in os.listdir(build.CSRC) if h.endswith(".h") and
               re.search(r"load_lds|lds_dword", open(os.path.join(build.CSRC, h)).read())]
    assert set(sources) == {"w4a8_stream.hip", "w4a8_mfma.hip"}
    assert headers == ["w4a8_mfma_ops.h"]          # of w4a8_chunk.hip
