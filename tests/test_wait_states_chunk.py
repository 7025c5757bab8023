"""No kernel of the attention of several tokens uses a matrix product's result
before it is there (wait_states.py), in the assembly that the library's own flags
give; behind its 32 x 32 products the compiler leaves 12 states."""
import os
import subprocess

import wait_states
from fable5_llm_amd import build


def test_the_kernels(tmp_path, monkeypatch):
    for op in ("v_mfma_f32_32x32x16_bf16", "v_mfma_f32_32x32x16_f16"):
        monkeypatch.setitem(wait_states.STATES, op, 12)
    out = os.path.join(tmp_path, "chunk.s")
    subprocess.run([build.hipcc()] + build.flags() + ["-S", "--cuda-device-only", "-o", out,
                                                       os.path.join(build.CSRC, "w4a8_chunk.hip")],
                   check=True, capture_output=True)
    with open(out) as f:
        products, found = wait_states.early_uses(f.read())
    assert products > 100 and not found, found
