"""The integration text's program of a prompt's step runs behind that of the mixers."""
import math

import pytest
import torch

from test_integration_text import programs


@pytest.mark.gpu
def test_the_prompt_program_runs():
    env = {}
    exec(next(t for t in programs() if "PagedKV.empty" in t), env)
    exec(next(t for t in programs() if "attend_chunk_async" in t), env)
    kv, maps = env["kv"], env["maps"]
    assert [kv.lens.tolist()[s] for s in (10, 11)] == [30, 17]
    assert maps.cu.tolist() == [0, 30, 47, 47]
    assert maps.pos.tolist() == [*range(30), *range(17), -1]
    assert maps.seqs.tolist() == [10] * 30 + [11] * 17 + [-1]
    assert (env["out"] == 0).all() and (env["turned"] == 0).all()
    # 1,000 equal logits: the sum is exact; its logarithm to the base 2 (an ulp), ln 2's
    # and the product's rounding are at most 2^-21 each of a value below 8
    want = torch.full((48,), -math.log(1000))
    assert torch.allclose(env["logp"].cpu(), want, rtol=0, atol=4 * 2.0 ** -21)
    assert env["best"].tolist() == [[0, 1, 2, 3, 4]] * 48
    env["ctx"].close()
