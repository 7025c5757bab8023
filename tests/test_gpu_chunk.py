"""Attention of several new tokens of each sequence (PagedKV.map_async,
attend_chunk_async) against its definition in 64 bits, and where the tokens lie
against a loop over them.

The tolerance, per output, in half steps u of the cache's type (bfloat16 2^-8,
float16 2^-11, float32 2^-24), with A = sum p |v| / sum p, X the largest
sum |q k| scale of a token's scores and V the largest |v|:

    u A              the weights p rounded for the second product (float32: none)
  + u |out|          the output (int16: half of one step instead)
  + 2^-38 n V        float16: weights, held 2^13 as large as their maximum or
                     more, end at 2^-24; half of that
  + 2^-24 A (X (D + 4) + n + 16)   scores summed in float32 and scaled (an error
                     d of a score is a factor e^d of its weight), exponentials
                     within 4 of their last bits twice, sums of n weights
"""
import math
import random

import pytest
import torch

from fable5_llm_amd.engine import PagedKV
from test_gpu_attend import DEV, U, ints, make, rows_of

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def mapped(engine, kv, seqs, counts, q_heads, tokens=None):
    m = kv.chunk_maps(len(seqs), sum(max(c, 0) for c in counts) if tokens is None else tokens,
                      q_heads)
    for t in (m.cu, m.seqs, m.pos, m.slots, m.plan):
        t.fill_(77)
    s, c = ints(seqs), ints(counts)
    torch.cuda.synchronize()
    kv.map_async(s, c, m)
    engine.sync()
    return m


def run(engine, kv, layer, q, m, out=None, **kw):
    out = torch.full_like(q, 7) if out is None else out
    ws = kv.attend_chunk_workspace(m)
    ws.fill_(0xFF)                                        # NaNs, if anything is read unwritten
    torch.cuda.synchronize()
    kv.attend_chunk_async(layer, q, out, m, ws, **kw)
    engine.sync()
    return out


def check(kv, layer, q, seqs, counts, got, scale=None, out_unit=None):
    """got within the tolerance of the definition, token by token; those of no
    row as they were (7)."""
    dim, dtype = kv.head_dim, kv.pool.dtype
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    q, out = q.double().cpu(), got.double().cpu() * (out_unit or 1.0)
    u, low = U[dtype], 2.0 ** -38 if dtype == torch.float16 else 0.0
    lens, per, t = kv.lens.tolist(), q.shape[1] // kv.kv_heads, 0
    for i, (s, c) in enumerate(zip(seqs, counts)):
        mine, x = out[t:t + c].transpose(0, 1), q[t:t + c].transpose(0, 1)
        t += c
        if s < 0 or c == 0:
            assert not mine.any(), i
            continue
        n = lens[s]
        k, v = (r.repeat_interleave(per, 0) for r in rows_of(kv, layer, s, n))
        late = torch.arange(n) > n - c + torch.arange(c)[:, None]
        sc = (x @ k.transpose(1, 2).contiguous() * scale).masked_fill(late, -math.inf)
        X = (x.abs() @ k.abs().transpose(1, 2).contiguous()) * abs(scale)
        X = torch.where(torch.isfinite(X), X, 0.0).amax(-1, keepdim=True)
        p = torch.softmax(sc, -1)
        want, A = p @ v, p @ v.abs()
        tol = 2.0 ** -24 * A * (X * (dim + 4) + n + 16) + low * n * v.abs().max() + \
            (u * A if u > 2.0 ** -20 else 0.0)
        if out_unit is None:
            tol = tol + u * want.abs()
        else:
            tol = tol + 0.5 * out_unit
            want = want.clamp(-32768 * out_unit, 32767 * out_unit)
        off = (mine - want).abs() / tol
        assert not torch.isnan(mine).any(), (i, s, c, n)
        assert off.max() <= 1, (i, s, c, n, float(off.max()))
    assert (got[t:] == 7).all()


def random_q(gen, tokens, heads, dim, dtype):
    return torch.randn(tokens, heads, dim, generator=gen).to(DEV).to(dtype)


ROWS = [(1, 1), (1, 15), (16, 16), (17, 33), (2, 64), (65, 65), (0, 9), (31, 129), (64, 200),
        (130, 160), (3, 700), (100, 100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,group,page", [
    (64, 3, 1, 16), (64, 1, 16, 64), (128, 2, 4, 16), (128, 1, 17, 32), (128, 2, 7, 128),
    (256, 1, 4, 16), (256, 2, 3, 64), (256, 1, 40, 32), (64, 1, 130, 16)])
def test_lengths(engine, dtype, dim, heads, group, page):
    gen = torch.Generator().manual_seed(dim * heads + group)
    lens = [n for _, n in ROWS]
    kv = make(engine, gen, lens, heads, dim, page, dtype)
    order = random.Random(group).sample(range(len(ROWS)), len(ROWS))
    seqs, counts = order[:6] + [-1] + order[6:], [ROWS[i][0] for i in order]
    counts = counts[:6] + [9] + counts[6:]
    q = random_q(gen, sum(counts) + 3, heads * group, dim, dtype)
    m = mapped(engine, kv, seqs, counts, heads * group, tokens=sum(counts) + 3)
    check(kv, 0, q, seqs, counts, run(engine, kv, 0, q, m))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", [[(1, 5000)], [(40, 3333), (7, 513), (1, 512), (90, 90)],
                                   [(600, 2100)], [(5, 9000), (5, 64), (200, 1500)]])
def test_keys_in_parts(engine, dtype, dim, shape):
    # few tokens, long contexts: a tile's keys in parts, joined
    gen = torch.Generator().manual_seed(dim)
    kv = make(engine, gen, [n for _, n in shape], 2, dim, 32, dtype, layers=2)
    counts, seqs = [c for c, _ in shape], list(range(len(shape)))
    q = random_q(gen, sum(counts), 6, dim, dtype)
    m = mapped(engine, kv, seqs, counts, 6)
    got = run(engine, kv, 1, q, m)
    check(kv, 1, q, seqs, counts, got)
    assert torch.equal(got, run(engine, kv, 1, q, m))     # the same from run to run


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_int16_out_with_strides(engine, cache, dim):
    gen = torch.Generator().manual_seed(11)
    rows = [(1, 1), (20, 200), (70, 77), (33, 2000)]
    kv = make(engine, gen, [n for _, n in rows], 2, dim, 16, cache)
    counts = [c for c, _ in rows]
    q = random_q(gen, sum(counts), 16, 2 * dim, cache)[:, ::2, :dim]
    m = mapped(engine, kv, [0, 1, 2, 3], counts, 8)
    out = torch.zeros(sum(counts), 16, dim, dtype=torch.int16, device=DEV)
    run(engine, kv, 0, q, m, out=out[:, ::2], out_frac=12)
    check(kv, 0, q, [0, 1, 2, 3], counts, out[:, ::2], out_unit=2.0 ** -12)
    assert not out[:, 1::2].any()
    run(engine, kv, 0, q, m, out=out[:, 1::2], out_frac=15)     # saturates
    check(kv, 0, q, [0, 1, 2, 3], counts, out[:, 1::2], out_unit=2.0 ** -15)
    assert int(out.max()) == 32767 and int(out.min()) == -32768


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-3, 0.7])
def test_scales(engine, dtype, dim, scale):
    gen = torch.Generator().manual_seed(4)
    kv = make(engine, gen, [150, 40], 1, dim, 16, dtype)
    q = random_q(gen, 90, 3, dim, dtype)
    m = mapped(engine, kv, [1, 0], [10, 80], 3)
    check(kv, 0, q, [1, 0], [10, 80], run(engine, kv, 0, q, m, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", [0, 1])
def test_no_later_token_reaches_an_earlier_one(engine, dtype, dim, bad, which):
    # an infinity or a NaN in a key or value of a late token: the tokens before
    # it are what they are without it, to the bit; the others are no numbers
    # (a key: of q's sign, +infinity and NaN; -infinity weighs nothing)
    gen = torch.Generator().manual_seed(7)
    kv = make(engine, gen, [230], 2, dim, 16, dtype)
    q = random_q(gen, 150, 4, dim, dtype)
    q[..., 3] = q[..., 3].abs() + 0.25
    m = mapped(engine, kv, [0], [150], 4)
    want = run(engine, kv, 0, q, m)
    at = 187                                              # the token 107 of the chunk
    kv.pool[kv.tables[0, at // 16], 0, which, 1, at % 16, 3] = bad
    got = run(engine, kv, 0, q, m)
    assert torch.equal(got[:107], want[:107])
    assert torch.equal(got[:, :2], want[:, :2])           # another head's
    seen = got[107:, 2:].float()
    if which == 0 and bad == -math.inf:
        check(kv, 0, q, [0], [150], got)
    elif which == 0:
        assert torch.isnan(seen).all()
    else:
        assert not torch.isfinite(seen[..., 3]).any()
        seen[..., 3] = 0
        assert torch.isfinite(seen).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 256])
def test_scores_far_apart_and_many_small_weights(engine, dtype, dim):
    # weights that underflow against the running maximum, whichever comes first;
    # then one token that weighs 1 and 4096 of 2^-25 each
    gen = torch.Generator().manual_seed(5)
    for big in (60.0, -60.0):
        kv = make(engine, gen, [400], 1, dim, 16, dtype)
        kv.pool[kv.tables[0, 200 // 16], 0, 0, :, 200 % 16] *= big
        q = random_q(gen, 300, 4, dim, dtype) * 3
        m = mapped(engine, kv, [0], [300], 4)
        check(kv, 0, q, [0], [300], run(engine, kv, 0, q, m))
    N = 4096
    kv = make(engine, gen, [N + 1], 1, dim, 16, dtype, fill=torch.zeros_like)
    for p in kv.tables[0, :-(-(N + 1) // 16)].tolist():
        kv.pool[p, 0, 1] = 1024.0
    first = int(kv.tables[0, 0])
    kv.pool[first, 0, 0, 0, 0, 0] = 25.0
    kv.pool[first, 0, 1, 0, 0] = 0.0
    q = torch.zeros(3, 2, dim, dtype=dtype, device=DEV)
    q[..., 0] = 1
    m = mapped(engine, kv, [0], [3], 2)
    kw = dict(scale=math.log(2.0))
    check(kv, 0, q, [0], [3], run(engine, kv, 0, q, m, **kw), **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [600.0, 1100.0, 1.2e4, 6e4])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_millions(engine, dtype, dim, size, sign):
    # scores of 2^k for whole k, exact in float32 as equal products; the largest
    # weighs 1, those 64 and more below it nothing, whatever their size
    kv = make(engine, torch.Generator().manual_seed(3), [700, 200], 1, dim, 16, dtype)
    near = 2.0 ** math.floor(math.log2(size))
    for s, n in ((0, 700), (1, 200)):
        for j, page in enumerate(kv.tables[s, :-(-n // 16)].tolist()):
            kv.pool[page, 0, 0] = sign * near * (1.0 if sign < 0 else 0.5)
            if j == 5:
                kv.pool[page, 0, 0, :, 3] = sign * near * (0.5 if sign < 0 else 1.0)
    q = torch.full((50, 2, dim), near, device=DEV).to(dtype)
    m = mapped(engine, kv, [0, 1], [30, 20], 2)
    out = run(engine, kv, 0, q, m, scale=1.0)
    for s, rows in ((0, out[:30]), (1, out[30:])):
        want = kv.pool[kv.tables[s, 5], 0, 1, :, 3]
        # one weight: p v / p, each of them rounded
        assert torch.allclose(rows.double(), want.double().expand(rows.shape),
                              rtol=2 * U[dtype] if dtype != torch.float32 else 2.0 ** -22, atol=0)


def test_rows_without_a_finite_score(engine):
    for dtype in TYPES:
        gen = torch.Generator().manual_seed(6)
        kv = make(engine, gen, [40, 33], 1, 64, 16, dtype)
        for t in range(33):
            kv.pool[kv.tables[1, t // 16], 0, 0, 0, t % 16] = -math.inf
        q = torch.rand(20, 2, 64, generator=gen).to(DEV).to(dtype) + 0.25
        m = mapped(engine, kv, [1, 0], [12, 8], 2)
        out = run(engine, kv, 0, q, m)
        assert not out[:12].any()
        check(kv, 0, q[12:], [0], [8], out[12:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [-1, 10 ** 9])
def test_a_table_that_names_no_page(engine, dtype, page):
    gen = torch.Generator().manual_seed(8)
    kv = make(engine, gen, [300, 100], 2, 64, 16, dtype)
    q = random_q(gen, 60, 4, 64, dtype)
    m = mapped(engine, kv, [0, 1], [40, 20], 4)
    want = run(engine, kv, 0, q, m)
    kv.tables[0, 3] = page
    out, ws = torch.zeros_like(q), kv.attend_chunk_workspace(m)
    torch.cuda.synchronize()
    kv.attend_chunk_async(0, q, out, m, ws)
    with pytest.raises(AssertionError, match="outside the cache"):
        engine.sync()
    assert torch.equal(out[40:], want[40:]) and torch.isfinite(out.float()).all()


def test_pages_past_32_bit_offsets(engine):
    # a pool of 4.6 GB: byte offsets over 2^32, element offsets over 2^31
    kv = PagedKV.empty(engine, 70000, 1, 2, 128, 64, 2, 40, torch.bfloat16)
    gen = torch.Generator().manual_seed(2)
    n = 40 * 128 - 5
    pages = torch.cat([torch.arange(69960, 69999), torch.tensor([1])])
    x = torch.randn(40, 1, 2, 2, 128, 64, generator=gen).to(torch.bfloat16)
    kv.pool[pages.to(DEV)] = x.to(DEV)
    kv.tables[1, :40] = pages.to(torch.int32).to(DEV)
    kv.lens[1] = n
    q = random_q(gen, 9, 4, 64, torch.bfloat16)
    m = mapped(engine, kv, [1], [9], 4)
    check(kv, 0, q, [1], [9], run(engine, kv, 0, q, m))
    assert int(m.slots[0]) == 1 * 128 + (n - 9) % 128 and int(m.slots.max()) < 70000 * 128


def test_a_captured_step_serves_a_cache_that_grows(engine):
    # extend, map, append and attend of a step, captured once: replayed with
    # other counts, between eager steps
    gen = torch.Generator().manual_seed(12)
    kv = PagedKV.empty(engine, 300, 1, 2, 16, 64, 4, 100, torch.float16)
    T, rows = 40, 3
    seqs, counts = ints([2, 0, -1]), ints([0, 0, 0])
    m, q = kv.chunk_maps(rows, T, 8), random_q(gen, T, 8, 64, torch.float16)
    k, v = (random_q(gen, T, 2, 64, torch.float16) for _ in range(2))
    out, ws = torch.full_like(q, 7), kv.attend_chunk_workspace(m)

    def step():
        kv.extend_async(seqs, counts)
        kv.map_async(seqs, counts, m)
        kv.append_async(0, k, v, m.seqs, m.pos)
        kv.attend_chunk_async(0, q, out, m, ws)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=side):
            engine.set_stream(side)
            step()
    finally:
        engine.set_stream(None)
    for i, c in enumerate([(20, 9, 3), (1, 1, 1), (0, 30, 0), (17, 16, 2), (1, 0, 0), (3, 4, 5)]):
        counts.copy_(ints(c))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen))
        out.fill_(7)
        torch.cuda.synchronize()
        if i % 2:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        engine.sync()
        check(kv, 0, q, [2, 0, -1], c, out)


# ------------------------------------------------------------------- maps
def want_maps(kv, seqs, counts, tokens):
    lens, tables, page = kv.lens.tolist(), kv.tables.tolist(), kv.page_tokens
    cu, out = [0], []
    for s, c in zip(seqs, counts):
        c = max(c, 0)
        fine = 0 <= s < len(lens) and c <= lens[s]
        for j in range(c):
            p = lens[s] - c + j if fine else -1
            out.append((s, p, tables[s][p // page] * page + p % page) if fine else (-1, -1, -1))
        cu.append(cu[-1] + c)
    return cu, out + [(-1, -1, -1)] * (tokens - len(out))


def same(m, cu, out):
    assert m.cu.tolist() == cu
    assert list(zip(m.seqs.tolist(), m.pos.tolist(), m.slots.tolist())) == out


@pytest.mark.parametrize("rows,most,spare", [(0, 1, 0), (0, 1, 5), (1, 1, 0), (1, 700, 3),
                                             (7, 60, 1), (61, 1, 0), (1024, 3, 2), (1025, 4, 0),
                                             (3000, 40, 700)])
def test_maps(engine, rows, most, spare):
    rng = random.Random(rows + most)
    n = max(rows, 2)
    lens = [rng.randrange(1, 90) for _ in range(n)]
    lens[0] = 900
    kv = PagedKV.empty(engine, 6 * n + 60, 1, 1, 16, 64, n, 60, torch.float32)
    held = [-(-x // 16) for x in lens]
    pages = rng.sample(range(6 * n + 60), sum(held))
    table, at = torch.full((n, 60), -1, dtype=torch.int32), 0
    for s in range(n):
        table[s, :held[s]] = torch.tensor(pages[at:at + held[s]])
        at += held[s]
    kv.tables.copy_(table)
    kv.lens.copy_(ints(lens))
    seqs = rng.sample(range(n), rows) if rows != 1 else [0]
    seqs = [s if rng.random() < 0.9 or rows == 1 else -1 for s in seqs]
    counts = [min(rng.randint(0, most) if most > 1 else 1, lens[s] if s >= 0 else 9) for s in seqs]
    tokens = sum(counts) + spare
    m = mapped(engine, kv, seqs, counts, 4, tokens=tokens)
    same(m, *want_maps(kv, seqs, counts, tokens))


def test_maps_report_what_is_wrong(engine):
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [40, 8], 1, 64, 16, torch.float32)
    for seqs, counts in (([0, 1], [3, 9]), ([0, 2], [3, 2]), ([1, 0], [-1, 5])):
        m = kv.chunk_maps(2, 20, 2)
        s, c = ints(seqs), ints(counts)
        torch.cuda.synchronize()
        kv.map_async(s, c, m)
        with pytest.raises(AssertionError, match="outside the cache"):
            engine.sync()
        same(m, *want_maps(kv, seqs, counts, 20))
        q = random_q(gen, 20, 2, 64, torch.float32)
        out = run(engine, kv, 0, q, m)                    # the other row is served
        good = [i if 0 <= i < 2 and 0 <= n <= [40, 8][i] else -1 for i, n in zip(seqs, counts)]
        check(kv, 0, q, good, [max(n, 0) for n in counts], out)
    m, s, c = kv.chunk_maps(2, 20, 2), ints([0, 1]), ints([15, 6])      # more than 20
    torch.cuda.synchronize()
    kv.map_async(s, c, m)
    with pytest.raises(AssertionError, match="outside the cache"):
        engine.sync()
    same(m, [0, 0, 0], [(-1, -1, -1)] * 20)
    assert (run(engine, kv, 0, random_q(gen, 20, 2, 64, torch.float32), m) == 7).all()


def test_maps_behind_a_refused_extend_name_nothing(engine):
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [40, 8], 1, 64, 16, torch.float32, spare=0)
    m, s, c = kv.chunk_maps(2, 400, 2), ints([0, 1]), ints([1, 60])
    two = ints([1, 2])
    torch.cuda.synchronize()
    kv.extend_async(s, c)
    kv.map_async(s, two, m)
    with pytest.raises(AssertionError, match="too few free pages"):
        engine.sync()
    same(m, [0, 0, 0], [(-1, -1, -1)] * 400)


def test_a_plan_that_was_not_made_here(engine):
    # never mapped, or another step's: what does not fit is left out
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [40, 8], 1, 64, 16, torch.float32)
    m, q = kv.chunk_maps(2, 20, 2), random_q(gen, 20, 2, 64, torch.float32)
    for fill in (0, 0xFF):
        m.plan.fill_(fill)
        assert (run(engine, kv, 0, q, m) == 7).all()


def test_no_tokens_and_wrong_tensors(engine):
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [40], 2, 64, 16, torch.bfloat16)
    other = make(engine, gen, [40], 2, 64, 16, torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    m = mapped(engine, kv, [0], [3], 4)
    ws, f = kv.attend_chunk_workspace(m), kv.attend_chunk_async
    none = mapped(engine, kv, [], [], 4, tokens=0)
    f(0, q[:0], q[:0], none, ws)
    engine.sync()
    out = torch.empty_like(q)
    for call in (lambda: f(0, q.half(), out.half(), m, ws), lambda: f(0, q, out.half(), m, ws),
                 lambda: f(0, q, out.float(), m, ws), lambda: f(0, q.short(), out, m, ws),
                 lambda: f(0, q[:, :2], out[:, :2], m, ws), lambda: f(0, q[:2], out[:2], m, ws),
                 lambda: f(1, q, out, m, ws), lambda: f(-1, q, out, m, ws),
                 lambda: f(0, q.cpu(), out, m, ws), lambda: f(0, q, out, m, ws.cpu()),
                 lambda: f(0, q, out, None, ws), lambda: other.attend_chunk_async(0, q, out, m, ws),
                 lambda: f(0, q, out.short(), m, ws, out_frac=32),
                 lambda: kv.chunk_maps(1, 3, 3), lambda: kv.chunk_maps(-1, 3, 4),
                 lambda: kv.chunk_maps(1, (1 << 20) + 1, 4),
                 lambda: kv.map_async(ints([0, 0]), ints([1, 1]), m),
                 lambda: kv.map_async(ints([0]), ints([1, 1]), m),
                 lambda: kv.map_async(ints([0]).long(), ints([1]), m),
                 lambda: other.map_async(ints([0]), ints([1]), m)):
        with pytest.raises(ValueError):
            call()
    big = PagedKV.empty(engine, 600, 1, 2, 16, 64, 1, 500, torch.bfloat16)
    m = big.chunk_maps(1, 3, 4)
    with pytest.raises(ValueError, match="workspace"):
        big.attend_chunk_async(0, q, out, m, torch.zeros(16, dtype=torch.uint8, device=DEV))
    engine.sync()
