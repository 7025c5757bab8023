"""Plans: the rows with the longest units come first, each unit once; and a plan one of
whose words is nothing that a map leaves there: its unit is left out
and the next sync reports it; the other units' tokens get their attention."""
import pytest
import torch

from test_gpu_attend import make
from test_gpu_chunk import check, mapped, random_q, run

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


@pytest.mark.parametrize("rows", [1, 2, 65, 127, 128, 129])
def test_units_in_order(engine, rows):
    # one query head a key-value head: 128 tokens a unit, and with 16 heads 32 units of
    # 256 compute units' work fill the chip, so that these are more
    gen = torch.Generator().manual_seed(rows)
    count = [1 + (7 * i) % 3 for i in range(rows)]
    if rows < 65:
        count = [128 * 40 + 1] * rows
    lens = [c + (37 * i) % 101 for i, c in enumerate(count)]
    kv = make(engine, gen, lens, 16, 64, 16, torch.bfloat16)
    seqs, total = list(range(rows)), sum(count)
    m = mapped(engine, kv, seqs, count, 16)
    plan = m.plan.view(torch.int32)
    n = int(plan[0])
    units = plan[UNIT:UNIT + WORDS * n].view(n, WORDS).tolist()
    split = -(-2 * torch.cuda.get_device_properties(0).multi_processor_count // 16)
    assert n > split
    starts = torch.tensor([0] + count).cumsum(0).tolist()
    seen = {}                            # (row, first token): its keys, in the plan's order
    for seq, tok, ntok, pos0, k0, k1, _, _ in units:
        assert pos0 == lens[seq] - count[seq] + tok - starts[seq]
        if ntok:
            assert tok + ntok <= starts[seq + 1]
            seen.setdefault((seq, tok, ntok), []).append((k0, k1))
    for (seq, tok, ntok), keys in seen.items():
        end = lens[seq] - count[seq] + tok - starts[seq] + ntok
        assert sorted(keys)[0][0] == 0 and sorted(keys)[-1][1] == end
        assert all(a[1] == b[0] for a, b in zip(sorted(keys), sorted(keys)[1:]))
    assert sum(k[2] for k in seen) == total
    order = [lens[u[0]] for u in units]  # none is split for want of keys: a unit's are a row's
    if 65 <= rows <= 128:
        assert order == sorted(order, reverse=True)
    if rows == 129:
        assert [u[0] for u in units] == seqs
    if rows >= 65:
        q = random_q(gen, total, 16, 64, torch.bfloat16)
        check(kv, 0, q, seqs, count, run(engine, kv, 0, q, m))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("counts,lens", [((5, 1, 3, 2), (200, 3000, 1500, 31)),
                                         ((1, 200, 0, 3), (129, 333, 50, 4000))], ids=str)
def test_rows_in_parts_and_in_order(engine, counts, lens, dtype):
    # 32 units fill the chip; the long rows' parts come to more with the short rows
    gen = torch.Generator().manual_seed(len(lens))
    kv = make(engine, gen, list(lens), 16, 64, 16, dtype)
    m = mapped(engine, kv, [0, 1, 2, 3], list(counts), 16)
    plan = m.plan.view(torch.int32)
    assert plan[0] > -(-2 * torch.cuda.get_device_properties(0).multi_processor_count // 16)
    assert plan[1] >= 2                  # rows whose parts are joined
    q = random_q(gen, sum(counts), 16, 64, dtype)
    out = run(engine, kv, 0, q, m)
    check(kv, 0, q, [0, 1, 2, 3], counts, out)
    assert torch.equal(out, run(engine, kv, 0, q, m))
