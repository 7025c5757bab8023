"""A plan one of whose words is nothing that a map leaves there: its unit is left out
and the next sync reports it; the other units' tokens get their attention."""
import pytest
import torch

from test_gpu_attend import make
from test_gpu_chunk import mapped, random_q, run

pytestmark = pytest.mark.gpu
UNIT, WORDS = 16, 8                    # the plan's words before its units, and of one


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("word,value", [
    (0, 5), (1, -1), (1, 40), (2, -3), (2, 1000), (3, -1), (3, 1 << 30), (4, -64), (4, 1),
    (5, -1), (5, -(1 << 31)), (5, 1 << 30), (6, 1 << 20)], ids=str)
def test_a_word_that_no_map_writes(engine, dtype, word, value):
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [100, 90], 1, 64, 16, dtype)
    q = random_q(gen, 40, 2, 64, dtype)
    m = mapped(engine, kv, [0, 1], [20, 20], 2)
    want = run(engine, kv, 0, q, m)
    plan = m.plan.view(torch.int32)
    assert plan[0] == 2
    unit = plan[UNIT:UNIT + WORDS].tolist()
    assert unit[2] == 20                 # a whole row's tokens
    plan[UNIT + word] = value
    out = torch.full_like(q, 7)
    with pytest.raises(AssertionError):
        run(engine, kv, 0, q, m, out=out)
    mine = slice(unit[1], unit[1] + 20)
    other = slice(20, 40) if unit[1] == 0 else slice(0, 20)
    assert (out[mine] == 7).all() and torch.equal(out[other], want[other])
