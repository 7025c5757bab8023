"""Attention of several new tokens over values that are infinite: sum p v / sum p is
that infinity for each query that sees it, whichever turn of the kernel or part of the
keys it lies in and however far the maximum rises behind it; no other element and no
other query changes a bit.  A query's weights are powers of e that 32 bits hold, but
where a test says so."""
import math

import pytest
import torch

from test_gpu_attend import DEV, make
from test_gpu_chunk import TYPES, mapped, random_q, run
from test_gpu_chunk_plan import UNIT, WORDS

pytestmark = pytest.mark.gpu
DIMS, SIGNS, COLUMN = [64, 128, 256], [1, -1], 3


def put(kv, which, key, column, value, seq=0, head=slice(None)):
    page = int(kv.tables[seq, key // kv.page_tokens])
    kv.pool[page, 0, which, head, key % kv.page_tokens, column] = value


def check(got, want, seen, sign):
    """Column COLUMN of the queries `seen` (of every head) that infinity, int16 at its
    end; all else as in want."""
    end = sign * math.inf
    if got.dtype == torch.int16:
        end = 32767 if sign > 0 else -32768
    assert (got[seen][..., COLUMN] == end).all()
    want = want.clone()
    want[seen, :, COLUMN] = end
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("sign", SIGNS)
@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("key", [0, 5, 31, 40, 70])
def test_in_a_prompts_first_turns(engine, dtype, dim, sign, whole, key):
    gen = torch.Generator().manual_seed(dim + key)
    kv = make(engine, gen, [150, 20], 2, dim, 16, dtype)
    q = random_q(gen, 170, 4, dim, dtype)
    m = mapped(engine, kv, [1, 0], [20, 150], 4)
    out = [torch.full_like(q, 7, dtype=torch.int16 if whole else dtype) for _ in range(2)]
    frac = dict(out_frac=10) if whole else {}
    want = run(engine, kv, 0, q, m, out=out[0], **frac)
    put(kv, 1, key, COLUMN, sign * math.inf)
    got = run(engine, kv, 0, q, m, out=out[1], **frac)
    check(got, want, slice(20 + key, None), sign)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("sign", SIGNS)
@pytest.mark.parametrize("which", ["first", "inner", "last"])
def test_in_a_parts_first_turn(engine, dtype, dim, sign, which):
    gen = torch.Generator().manual_seed(dim)
    kv = make(engine, gen, [3000], 2, dim, 32, dtype)
    q = random_q(gen, 20, 4, dim, dtype)
    m = mapped(engine, kv, [0], [20], 4)
    plan = m.plan.view(torch.int32)
    units = plan[UNIT:UNIT + WORDS * int(plan[0])].view(-1, WORDS).tolist()
    starts = sorted({u[4] for u in units if u[2]})
    assert len(starts) > 2
    key = starts[{"first": 0, "inner": 1, "last": -1}[which]] + 2
    want = run(engine, kv, 0, q, m)
    put(kv, 1, key, COLUMN, sign * math.inf)
    check(run(engine, kv, 0, q, m), want, slice(max(key - 2980, 0), None), sign)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("sign", SIGNS)
def test_the_maximum_rises_far_behind_it(engine, dtype, dim, sign):
    # a score of 400 behind scores of 0: what came before weighs e^-400, which 32 bits
    # do not hold, and an infinity is still one; in a turn that hides keys (the first
    # queries) and in one that hides none (the last)
    gen = torch.Generator().manual_seed(dim)
    kv = make(engine, gen, [700], 1, dim, 16, dtype)
    for j, page in enumerate(kv.tables[0, :44].tolist()):
        kv.pool[page, 0, 0] = 0.0
    put(kv, 0, 100, 0, 400.0)
    q = random_q(gen, 700, 1, dim, dtype)
    q[..., 0] = 1.0
    m = mapped(engine, kv, [0], [700], 1)
    want = run(engine, kv, 0, q, m, scale=1.0)
    put(kv, 1, 5, COLUMN, sign * math.inf)
    check(run(engine, kv, 0, q, m, scale=1.0), want, slice(5, None), sign)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("sign", SIGNS)
@pytest.mark.parametrize("key", [0, 1])
def test_another_parts_maximum_is_far_above(engine, dtype, dim, sign, key):
    # the part with the infinity before the one with a score of 400, and behind it
    gen = torch.Generator().manual_seed(dim)
    kv = make(engine, gen, [3000], 1, dim, 32, dtype)
    for page in kv.tables[0, :94].tolist():
        kv.pool[page, 0, 0] = 0.0
    at = [70, 2700]
    put(kv, 0, at[1 - key], 0, 400.0)
    q = random_q(gen, 9, 3, dim, dtype)
    q[..., 0] = 1.0
    m = mapped(engine, kv, [0], [9], 3)
    assert int(m.plan.view(torch.int32)[1]) > 0              # parts to be joined
    want = run(engine, kv, 0, q, m, scale=1.0)
    put(kv, 1, at[key], COLUMN, sign * math.inf)
    check(run(engine, kv, 0, q, m, scale=1.0), want, slice(0, None), sign)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_both_infinities_and_a_nan(engine, dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    kv = make(engine, gen, [150], 1, dim, 16, dtype)
    q = random_q(gen, 150, 2, dim, dtype)
    m = mapped(engine, kv, [0], [150], 2)
    want = run(engine, kv, 0, q, m)
    put(kv, 1, 10, COLUMN, math.inf)
    put(kv, 1, 20, COLUMN, -math.inf)
    put(kv, 1, 30, COLUMN + 1, math.nan)
    got = run(engine, kv, 0, q, m)
    assert (got[10:20, :, COLUMN] == math.inf).all()
    assert torch.isnan(got[20:, :, COLUMN]).all() and torch.isnan(got[30:, :, COLUMN + 1]).all()
    keep = torch.ones_like(want, dtype=torch.bool)
    keep[10:, :, COLUMN] = keep[30:, :, COLUMN + 1] = False
    assert torch.equal(got[keep], want[keep])
