"""Log probabilities of hundreds of rows of a large vocabulary, where the rule for a
full chip limits the workgroups of a row (16 a compute unit over the rows, rounded up)
and a wavefront takes several blocks: test_gpu_logprobs.py's check, eight rows at a
time, with the logits that a lane adds up counted by that rule."""
import types

import pytest
import torch

from test_gpu_attend import DEV
from test_gpu_logprobs import TYPES, UNIT, check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(300, 100003), (509, 248320), (1501, 50257)])
def test_rows_whose_workgroups_are_few(engine, dtype, rows, vocab):
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, vocab, generator=gen, device=DEV) * 3.0
    x = (x * 2 ** 18).to(torch.int32) if dtype == torch.int32 else x.to(dtype)
    ids = torch.randint(0, vocab, (rows,), generator=gen, device=DEV).int()
    got = run(engine, x, ids, 5, UNIT[dtype])
    blocks, splits = (vocab + 7 + 1023) // 1024, -(-16 * engine.num_cu // rows)
    assert splits < blocks // 4                           # the rule, not the blocks, limits them
    for at in (0, rows // 2, rows - 8):
        mine = slice(at, at + 8)
        # what check takes as eight workgroups a compute unit over eight rows
        check(types.SimpleNamespace(num_cu=splits), x[mine], ids[mine], 5, UNIT[dtype],
              got=[t[mine] for t in got])
