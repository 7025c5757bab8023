"""The mixers' checks of arguments on a machine without a GPU: the C ABI on
the stand-in HIP runtime (each refused call launches nothing), the Python
layer's own, and the page model that the GPU tests compare with."""
import random

import pytest
import torch

import fake_hip
from page_model import Pages, Refused


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    return fake_hip.build(tmp_path_factory.mktemp("hip"))


@pytest.mark.parametrize("check", ["cache", "lists", "append", "attend", "delta", "launches"])
def test_abi(runtime, check):
    assert fake_hip.run(runtime, "mixers_check.py", check) == "ok"


class Ctx:
    h, device = None, 0


def test_python_layer_takes_device_tensors_only():
    from fable5_llm_amd import mixers as M
    with pytest.raises(ValueError, match="device tensor"):
        M._act(torch.zeros(2, 4, 64), Ctx, "q", (2, 4, 64))
    with pytest.raises(ValueError, match="device tensor"):
        M._list(torch.zeros(2, dtype=torch.int32), Ctx, "seqs")
    with pytest.raises(ValueError, match="device tensor"):
        M.PagedKV(Ctx, *(torch.zeros(1),) * 4)


def test_page_model_keeps_what_sequences_read():
    rng = random.Random(4)
    m, want = Pages(60, 12, 9, 16), {}
    for step in range(400):
        op = rng.choice(["extend", "extend", "fork", "free", "compact"])
        try:
            if op == "extend":
                s, c = rng.randrange(12), rng.randrange(40)
                m.extend([s], [c])
                for t in range(m.lens[s] - c, m.lens[s]):
                    m.write(s, t, (step, t))
                want[s] = want.get(s, []) + [(step, t) for t in range(m.lens[s] - c, m.lens[s])]
            elif op == "fork":
                p, c = rng.sample(range(12), 2)
                m.fork([p], [c])
                want[c] = list(want.get(p, []))
            elif op == "free":
                s = rng.randrange(12)
                m.free([s])
                want[s] = []
            else:
                m.compact()
                used = sum(r > 0 for r in m.refs)
                assert all(m.refs[:used]) and not any(m.refs[used:])
        except Refused:
            pass
        held = [m.tables[s][j] for s in range(12) for j in range(m.held(m.lens[s]))]
        assert [held.count(p) for p in range(60)] == m.refs
        assert all(m.read(s) == want.get(s, []) for s in range(12))
