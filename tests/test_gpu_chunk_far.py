"""Attention of several new tokens whose scores are large and near each other: weights
go by the differences of scores, whatever their size.

Scores here are sums of few products that 32 bits hold exactly, and so are their
differences.  A weight's exponent, at most 16, is then off by 2^-19 (two roundings and
the scale's), the weight by less than that and 4 last bits, and a quotient of two sums of
weights by 2^-18; where weights and outputs are rounded to the cache's type, half a step u of it for
either: |out - want| <= A (u + 2^-18) + u |want|, with A = sum p |v| / sum p."""
import math

import pytest
import torch

from test_gpu_attend import DEV, U, make
from test_gpu_chunk import TYPES, mapped, run
from test_gpu_chunk_plan import UNIT, WORDS

pytestmark = pytest.mark.gpu
DIMS, KEYS = [64, 128, 256], 3000


def scored(engine, dtype, dim, heads, big, scores):
    """A cache of KEYS random values whose keys score 0, but for big + d at key t for
    each {t: d} in scores; and the query's first elements."""
    gen = torch.Generator().manual_seed(dim)
    kv = make(engine, gen, [KEYS], heads, dim, 32, dtype)
    for page in kv.tables[0, :-(-KEYS // 32)].tolist():
        kv.pool[page, 0, 0] = 0.0
    for t, d in scores.items():
        page = int(kv.tables[0, t // 32])
        kv.pool[page, 0, 0, :, t % 32, 0] = big / 1024.0
        kv.pool[page, 0, 0, :, t % 32, 1] = d
    return kv


def queries(tokens, heads, dim, dtype):
    q = torch.zeros(tokens, heads, dim, dtype=dtype, device=DEV)
    q[..., 0], q[..., 1] = 1024.0, 1.0
    return q


def near(kv, got, scores):
    w = torch.tensor([math.exp(d - max(scores.values())) for d in scores.values()],
                     dtype=torch.float64)
    v = torch.stack([kv.pool[int(kv.tables[0, t // 32]), 0, 1, :, t % 32] for t in scores]) \
        .double().cpu()                                   # [keys, heads, dim]
    p = (w / w.sum())[:, None, None]
    want, A = (p * v).sum(0), (p * v.abs()).sum(0)
    u = U[kv.pool.dtype]
    tol = A * ((u if u > 2.0 ** -20 else 0.0) + 2.0 ** -18) + u * want.abs()
    off = ((got.double().cpu() - want).abs() / tol).max()
    assert off <= 1, float(off)


def units(m):
    plan = m.plan.view(torch.int32)
    return plan[UNIT:UNIT + WORDS * int(plan[0])].view(-1, WORDS).tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("big", [2.0 ** 10, 2.0 ** 16, 2.0 ** 19, 2.0 ** 22])
def test_equal_scores_in_two_parts(engine, dtype, dim, big):
    # the first part's maximum stays at a lesser score that came a turn before; the
    # second's is the score itself
    q = queries(3, 2, dim, dtype)
    kv = scored(engine, dtype, dim, 2, big, {})
    m = mapped(engine, kv, [0], [3], 2)
    parts = sorted({(u[4], u[5]) for u in units(m) if u[2]})
    assert len(parts) > 2
    (_, end), (start, _) = parts[:2]
    scores = {2: -0.5 if dtype == torch.float16 else -5.0, end - 1: 0.0, start: 0.0}
    kv = scored(engine, dtype, dim, 2, big, scores)
    m = mapped(engine, kv, [0], [3], 2)
    for got in run(engine, kv, 0, q, m, scale=1.0):
        near(kv, got, scores)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("big", [2.0 ** 10, 2.0 ** 16, 2.0 ** 19, 2.0 ** 21])
def test_the_maximum_moves_between_equal_scores(engine, dtype, dim, big):
    # in turns one after another: a lesser score, one that does not move the maximum,
    # one that does, and one equal to the second
    below, above = (-0.5, 0.25) if dtype == torch.float16 else (-5.5, 0.25)
    scores = {10: below, 74: 0.0, 138: above, 202: 0.0}
    kv = scored(engine, dtype, dim, 8, big, scores)
    q = queries(2048, 8, dim, dtype)
    m = mapped(engine, kv, [0], [2048], 8)
    assert min(u[5] for u in units(m) if u[2] and u[4] == 0) > 202
    out = run(engine, kv, 0, q, m, scale=1.0)
    near(kv, out[0], scores)
    assert torch.equal(out, out[:1].expand_as(out))
