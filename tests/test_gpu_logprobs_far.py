"""Log probabilities where scale * logits is far from 0 (a temperature near 0, or
logits with a large sum in common): weights go by differences to the largest logit,
whatever its size.  Against the definition in 64 bits, with test_gpu_logprobs.py's
tolerances."""
import pytest
import torch

from test_gpu_attend import ints
from test_gpu_logprobs import TYPES, check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [700, 5003, 40000])
@pytest.mark.parametrize("scale", [1e5, 1e7, 3e8, 1e9, 1e12, 1e20, 1e30])
def test_temperatures_near_zero(engine, dtype, vocab, scale):
    gen = torch.Generator().manual_seed(vocab)
    x = logits(gen, 4, vocab, dtype)
    x[1, :] = x[1, 0]                                # all equal
    x[2, vocab // 2] = x[2].max()                    # two of the largest
    if dtype == torch.int32:
        x, scale = x >> 9, scale * 2.0 ** -9
    check(engine, x, ints([0, 5, vocab // 2, vocab - 1]), 9, scale)


@pytest.mark.parametrize("common", [2.0 ** 22, -2.0 ** 22, 2.0 ** 27])
def test_a_large_sum_in_common(engine, common):
    # float32 logits common + j step, exact; probabilities are those of j step
    gen = torch.Generator().manual_seed(3)
    step = 0.5 if abs(common) < 2.0 ** 24 else 16.0
    x = (common + torch.randint(0, 40, (3, 30000), generator=gen) * step).cuda()
    check(engine, x, ints([0, 100, 29999]), 12, 1.0 / step)
    check(engine, x, ints([0, 100, 29999]), 12, 2.0 ** 8)
