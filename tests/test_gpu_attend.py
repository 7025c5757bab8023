"""Attention of one token per row over a paged cache (PagedKV.attend_async)
against its definition in 64 bits.

The tolerance, per output, in half steps u of the type the values are rounded
to (bfloat16 2^-8, float16 2^-11, float32 2^-24), with A = sum p |v| / sum p and
X the largest sum |q k| scale of a row's scores:

    u A              the weights p rounded for the second product (float32:
                     none; int16 calls: as two values, u^2)
  + u |out|          the output (int16: half of one step instead)
  + 2^-24 A (X (D + 4) + n + 16)   scores summed in float32 and scaled (an error
                     d of a score is a factor e^d of its weight), exponentials
                     within 4 of their last bits twice, sums of n weights
"""
import math

import numpy as np
import pytest
import torch

from fable5_llm_amd.engine import PagedKV

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make(engine, gen, lens, heads, dim, page, dtype, layers=1, spare=3, fill=None):
    """A cache of random rows, its sequences' pages scattered; what no sequence
    holds is NaN."""
    held = [-(-n // page) for n in lens]
    pages = sum(held) + spare
    kv = PagedKV.empty(engine, pages, layers, heads, page, dim, len(lens), max(max(held), 1) + 2,
                       dtype)
    order = torch.randperm(pages, generator=gen)
    kv.pool.fill_(float("nan"))
    at = 0
    for s, n in enumerate(lens):
        mine = order[at:at + held[s]].to(DEV)
        at += held[s]
        kv.tables[s, :held[s]] = mine.to(torch.int32)
        kv.refs[mine] = 1
        for j, p in enumerate(mine.tolist()):
            used = min(page, n - j * page)
            x = torch.randn(layers, 2, heads, used, dim, generator=gen)
            kv.pool[p, :, :, :, :used] = (x if fill is None else fill(x)).to(DEV).to(dtype)
    kv.lens.copy_(ints(lens))
    torch.cuda.synchronize()
    return kv


def rows_of(kv, layer, s, n):
    """Keys and values [heads, n, dim] of a sequence in 64 bits, on the host."""
    pages = kv.tables[s, :-(-n // kv.page_tokens)].long()
    x = kv.pool[pages, layer].double().cpu()              # [pages, 2, heads, page, dim]
    x = x.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
    return x[0], x[1]


def check(kv, layer, q, seqs, got, upto=None, scale=None, unit=1.0, out_unit=None):
    """got within the tolerance of the definition, row by row."""
    dim = kv.head_dim
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    q, out = q.double().cpu() * unit, got.double().cpu() * (out_unit or 1.0)
    u = U[kv.pool.dtype]
    lens = kv.lens.tolist()
    per = q.shape[1] // kv.kv_heads
    for i, s in enumerate(seqs):
        n = 0 if s < 0 else lens[s] if upto is None else max(0, min(lens[s], upto[i]))
        if n == 0:
            assert torch.equal(out[i], torch.zeros_like(out[i])), i
            continue
        k, v = (x.repeat_interleave(per, 0) for x in rows_of(kv, layer, s, n))
        sc = (k @ q[i][:, :, None])[:, :, 0] * scale
        X = (k.abs() @ q[i].abs()[:, :, None]).amax().item() * scale
        p = torch.softmax(sc, -1)[:, None]
        want, A = (p @ v)[:, 0], (p @ v.abs())[:, 0]
        tol = 2.0 ** -24 * A * (X * (dim + 4) + n + 16)
        if out_unit is None:
            tol = tol + u * want.abs() + (u * A if u > 2.0 ** -20 else 0.0)
        else:
            tol = tol + 0.5 * out_unit + (u * u * A if u > 2.0 ** -20 else 0.0)
            want = want.clamp(-32768 * out_unit, 32767 * out_unit)
        off = (out[i] - want).abs() / tol
        assert not torch.isnan(out[i]).any(), (i, s, n)
        assert off.max() <= 1, (i, s, n, float(off.max()))


def run(engine, kv, layer, q, seqs, upto=None, **kw):
    out = torch.full_like(q, 7)
    ws = kv.attend_workspace(q.shape[0], q.shape[1])
    ws.fill_(0xFF)                                        # NaNs, if anything is read unwritten
    sq, up = ints(seqs), None if upto is None else ints(upto)
    torch.cuda.synchronize()
    kv.attend_async(layer, q, sq, out, ws, upto=up, **kw)
    engine.sync()
    return out


LENS = [1, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 160, 300]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,heads,group,page", [
    (64, 3, 1, 16), (64, 1, 16, 64), (128, 2, 4, 16), (128, 1, 17, 32), (128, 2, 7, 128),
    (256, 1, 4, 16), (256, 2, 3, 64), (256, 1, 40, 32)])
def test_lengths(engine, dtype, dim, heads, group, page):
    gen = torch.Generator().manual_seed(dim * heads + group)
    kv = make(engine, gen, LENS, heads, dim, page, dtype)
    q = torch.randn(len(LENS) + 1, heads * group, dim, generator=gen).to(DEV).to(dtype)
    seqs = list(reversed(range(len(LENS)))) + [-1]
    check(kv, 0, q, seqs, run(engine, kv, 0, q, seqs))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n", [(1, 5000), (3, 2111), (1, 130), (70, 700)])
def test_split_rows(engine, dtype, rows, n):
    # few rows: split over workgroups and joined, the last split short
    gen = torch.Generator().manual_seed(n)
    lens = [max(0, n - 97 * i) for i in range(rows)]
    kv = make(engine, gen, lens, 2, 128, 32, dtype, layers=2)
    q = torch.randn(rows, 8, 128, generator=gen).to(DEV).to(dtype)
    got = run(engine, kv, 1, q, list(range(rows)))
    check(kv, 1, q, list(range(rows)), got)
    again = run(engine, kv, 1, q, list(range(rows)))
    assert torch.equal(got, again)                        # the same from run to run


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_several_new_tokens_of_a_sequence(engine, dtype):
    # rows of one sequence with lengths of their own, as a verification's tokens
    gen = torch.Generator().manual_seed(3)
    kv = make(engine, gen, [140, 20], 2, 64, 16, dtype)
    upto = [136, 137, 138, 139, 140, 141, 0, -5, 20, 900]
    seqs = [0] * 8 + [1, 1]
    q = torch.randn(10, 4, 64, generator=gen).to(DEV).to(dtype)
    check(kv, 0, q, seqs, run(engine, kv, 0, q, seqs, upto=upto), upto=upto)


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 256])
def test_int16_rows_with_strides(engine, cache, dim):
    # q as a projection leaves it, each head's gate beside it; out into every
    # other head of a wider row
    gen = torch.Generator().manual_seed(11)
    lens = [1, 200, 77, 2000]
    kv = make(engine, gen, lens, 2, dim, 16, cache)
    wide = torch.randint(-32768, 32768, (4, 8, 2 * dim), generator=gen, dtype=torch.int32) \
        .to(torch.int16).to(DEV)
    wide[0] = 32767
    wide[1, 0] = -32768
    q = wide[:, :, :dim]
    out = torch.zeros(4, 16, dim, dtype=torch.int16, device=DEV)
    ws, sq = kv.attend_workspace(4, 8), ints([3, 1, 2, 0])
    torch.cuda.synchronize()
    kv.attend_async(0, q, sq, out[:, ::2], ws, frac=13, out_frac=12)
    engine.sync()
    check(kv, 0, q, [3, 1, 2, 0], out[:, ::2], unit=2.0 ** -13, out_unit=2.0 ** -12)
    assert not out[:, 1::2].any()
    big = run(engine, kv, 0, q, [3, 1, 2, 0], frac=13, out_frac=15)    # saturates
    check(kv, 0, q, [3, 1, 2, 0], big, unit=2.0 ** -13, out_unit=2.0 ** -15)
    assert int(big.max()) == 32767 and int(big.min()) == -32768


def test_scores_far_apart(engine):
    # weights that underflow against the running maximum, whichever comes first,
    # and scores that are all far below zero
    gen = torch.Generator().manual_seed(5)
    for order in (1, -1):
        kv = make(engine, gen, [400], 1, 64, 16, torch.float32)
        at = kv.tables[0, 200 // 16]
        kv.pool[at, 0, 0, :, 200 % 16] *= 60.0 * order
        q = torch.randn(1, 4, 64, generator=gen).to(DEV) * 3
        check(kv, 0, q, [0], run(engine, kv, 0, q, [0]))
    kv = make(engine, gen, [300], 1, 64, 16, torch.float32, fill=lambda x: x.abs())
    q = -torch.rand(1, 4, 64, generator=gen).to(DEV) * 1e4
    check(kv, 0, q, [0], run(engine, kv, 0, q, [0]))


@pytest.mark.parametrize("int16", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_many_small_weights(engine, dtype, int16):
    # weights of 2^-25 of the largest, which carries no value: they are not lost.
    # out = N 2^-25 V / (1 + N 2^-25); scores of 0 and 25 log 2 are off by 2^-24
    # of 25 at most.  int16 out: N 2^-25 V = 0.125, at a step of 2^-15
    N, V = (4096, 1024.0) if int16 else (4096, 1.0)
    kv = make(engine, torch.Generator().manual_seed(1), [N + 1], 1, 64, 16, dtype,
              fill=torch.zeros_like)
    first = int(kv.tables[0, 0])
    for p in kv.tables[0, :-(-(N + 1) // 16)].tolist():
        kv.pool[p, 0, 1] = V
    kv.pool[first, 0, 0, 0, 0, 0] = 25.0
    kv.pool[first, 0, 1, 0, 0] = 0.0
    q = torch.zeros(1, 2, 64, dtype=torch.int16 if int16 else dtype, device=DEV)
    q[..., 0] = 1
    check(kv, 0, q, [0], run(engine, kv, 0, q, [0], scale=math.log(2.0),
                             **(dict(out_frac=15) if int16 else {})),
          scale=math.log(2.0), **(dict(out_unit=2.0 ** -15) if int16 else {}))


def test_infinite_scores(engine):
    # a key that scores -infinity weighs nothing; a row of such keys gets zeros;
    # +infinity and NaN make the row NaN, and no other row
    gen = torch.Generator().manual_seed(6)
    kv = make(engine, gen, [40, 33, 20, 50], 1, 64, 16, torch.float32)
    kv.pool[kv.tables[0, 1], 0, 0, 0, 3] = -float("inf")
    for t in range(33):
        kv.pool[kv.tables[1, t // 16], 0, 0, 0, t % 16] = -float("inf")
    kv.pool[kv.tables[2, 0], 0, 0, 0, 7, 0] = float("nan")
    q = torch.rand(4, 2, 64, generator=gen).to(DEV) + 0.1
    out = run(engine, kv, 0, q, [0, 1, 2, 3])
    k, v = rows_of(kv, 0, 0, 40)
    p = torch.softmax((k[0] @ q[0].double().cpu().T).T / 8, -1)
    assert p[0, 19] == 0
    assert torch.allclose(out[0].double().cpu(), p @ v[0], rtol=1e-5, atol=1e-6)
    assert not out[1].any()
    assert torch.isnan(out[2]).all()
    check(kv, 0, q[3:], [3], out[3:])


@pytest.mark.parametrize("page", [-1, 10 ** 9])
def test_a_table_that_names_no_page(engine, page):
    gen = torch.Generator().manual_seed(8)
    kv = make(engine, gen, [300, 100], 2, 64, 16, torch.bfloat16)
    q = torch.randn(2, 4, 64, generator=gen).to(DEV).to(torch.bfloat16)
    want = run(engine, kv, 0, q, [0, 1])
    keep = int(kv.tables[0, 3])
    kv.tables[0, 3] = page
    out, ws, sq = torch.zeros_like(q), kv.attend_workspace(2, 4), ints([0, 1])
    torch.cuda.synchronize()
    kv.attend_async(0, q, sq, out, ws)
    with pytest.raises(AssertionError, match="outside the cache"):
        engine.sync()
    assert torch.equal(out[1], want[1]) and torch.isfinite(out[0].float()).all()
    kv.tables[0, 3] = keep
    sq = ints([0, 2])                                     # nor a sequence of the cache's
    torch.cuda.synchronize()
    kv.attend_async(0, q, sq, out, ws)
    with pytest.raises(AssertionError, match="outside the cache"):
        engine.sync()
    assert torch.equal(out[0], want[0]) and not out[1].any()


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
    q = torch.randn(1, 4, 64, generator=gen).to(DEV).to(torch.bfloat16)
    check(kv, 0, q, [1], run(engine, kv, 0, q, [1]))


def test_two_graphs_with_workspaces_of_their_own(engine):
    gen = torch.Generator().manual_seed(12)
    kv = make(engine, gen, [3000, 2500], 2, 128, 32, torch.float16)
    qs = [torch.randn(2, 8, 128, generator=gen).to(DEV).half() for _ in range(2)]
    want = [run(engine, kv, 0, q, [0, 1]) for q in qs]
    sq = ints([0, 1])
    graphs, outs, streams, keep = [], [], [], []
    for q in qs:
        out, ws = torch.zeros_like(q), kv.attend_workspace(2, 8)
        side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        try:
            with torch.cuda.graph(g, stream=side):
                engine.set_stream(side)
                kv.attend_async(0, q, sq, out, ws)
        finally:
            engine.set_stream(None)
        graphs.append(g), outs.append(out), streams.append(side), keep.append(ws)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        assert torch.equal(run(engine, kv, 0, qs[0], [0, 1]), want[0])


def test_no_rows_and_wrong_tensors(engine):
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [40], 2, 64, 16, torch.bfloat16)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV)
    ws, one = kv.attend_workspace(1, 4), ints([0])
    kv.attend_async(0, q[:0], one[:0], q[:0], ws)
    f = kv.attend_async
    for call in (lambda: f(0, q.half(), one, q.half(), ws), lambda: f(0, q, one, q.half(), ws),
                 lambda: f(0, q[:, :3], one, q[:, :3], ws), lambda: f(1, q, one, q, ws),
                 lambda: f(0, q, ints([0, 0]), q, ws), lambda: f(0, q, one, q, ws.cpu()),
                 lambda: f(0, q, one, q, ws, upto=ints([1, 2])),
                 lambda: f(0, q.cpu(), one, q, ws), lambda: f(0, q, one, q[:, :2], ws),
                 lambda: f(0, torch.zeros_like(q).transpose(1, 2).contiguous().transpose(1, 2),
                           one, q, ws),
                 lambda: kv.attend_workspace(1, 3), lambda: f(0, q, one, q, ws, frac=99)):
        with pytest.raises(ValueError):
            call()
    big = PagedKV.empty(engine, 600, 1, 2, 16, 64, 1, 500, torch.bfloat16)
    with pytest.raises(ValueError, match="workspace"):
        big.attend_async(0, q, one, q, torch.zeros(16, dtype=torch.uint8, device=DEV))
    engine.sync()
