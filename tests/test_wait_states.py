"""No kernel uses a matrix product's result before it is there (wait_states.py), in
the assembly that the library's own flags give; and the search finds such a use."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

from fable5_llm_amd import build
from wait_states import early_uses

SAMPLE = """_Zk:
	v_mfma_f32_16x16x32_bf16 v[4:7], v[8:11], v[12:15], v[4:7]
	v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[16:19], v[0:3]
	s_cbranch_vccz .LBB0_2
.LBB0_1:
	%s
	v_cvt_pk_bf16_f32 v20, v4, v5
	s_endpgm
.LBB0_2:
	s_nop 7
	s_branch .LBB0_1
.Lfunc_end0:
"""


def test_the_search():
    assert early_uses(SAMPLE % "s_nop 0")[1]           # 3 states on the short way
    assert early_uses(SAMPLE % "s_nop 4")[1]           # 7
    assert early_uses(SAMPLE % "s_nop 5") == (2, [])   # 8
    assert early_uses(SAMPLE % "v_mfma_f32_16x16x32_bf16 v[20:23], v[4:7], v[8:11], 0")[1]


def test_the_kernels(tmp_path):
    def check(source):
        out = os.path.join(tmp_path, source + ".s")
        subprocess.run([build.hipcc()] + build.flags() + ["-S", "--cuda-device-only", "-o", out,
                                                           os.path.join(build.CSRC, source)],
                       check=True, capture_output=True)
        with open(out) as f:
            return early_uses(f.read())
    sources = [s for s in build.SOURCES
               if "builtin_amdgcn_mfma" in open(os.path.join(build.CSRC, s)).read()]
    with ThreadPoolExecutor() as pool:
        got = dict(zip(sources, pool.map(check, sources)))
    assert set(got) == {"w4a8_mfma.hip", "w4a8_attend.hip", "w4a8_delta.hip"}
    assert all(n > 100 and not found for n, found in got.values()), got
