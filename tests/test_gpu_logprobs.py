"""Log probabilities, entropy and best alternatives of rows of logits
(Context.logprobs_async) against the definition in 64 bits; indices exactly.

Tolerances in units of 2^-24, with d = y - max y (nats), p the probabilities, E
their mean, N the logits that one lane adds up one after another and 24 for the
sums' joining:

    a difference d is off by 3 |d| (two roundings and the scale's), so a weight
    by 3 |d| + 2 of itself, and Z by D = 3 E|d| + N + 2;
    log Z by D + 4 log Z + 4;      log p = d - log Z by that + 3 |d| + 2 |log p|;
    sum d p by (D + N + 4) E|d| + 3 E d^2 + 2 E|d|, and the entropy by both
"""
import math
import random

import pytest
import torch

from test_gpu_attend import DEV, ints

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.int32]
STEP = 2.0 ** -24


def run(engine, x, ids, k, scale=1.0, entropy=True):
    rows = x.shape[0]
    logp, ent = (torch.full((rows,), 9.0, device=DEV) for _ in range(2))
    tl = torch.full((rows, k), 9.0, device=DEV)
    ti = torch.full((rows, k), -9, dtype=torch.int32, device=DEV)
    ws = engine.logprobs_workspace(rows, x.shape[1])
    ws.fill_(0xFF)                                        # NaNs, if anything is read unwritten
    torch.cuda.synchronize()
    engine.logprobs_async(x, ids, None if ids is None else logp, ws, entropy=ent if entropy else None,
                          top_logp=tl if k else None, top_ids=ti if k else None, scale=scale)
    engine.sync()
    return logp, ent, tl, ti


def check(engine, x, ids, k, scale=1.0, got=None):
    rows, vocab = x.shape
    logp, ent, tl, ti = (t.cpu() for t in (got or run(engine, x, ids, k, scale)))
    blocks = (vocab + 7 + 1023) // 1024
    splits = min(-(-8 * engine.num_cu // rows), -(-blocks // 4))
    N = 16 * -(--(-blocks // splits) // 4) + 24
    x = x.cpu()
    best = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(ti.long(), best)
    y = x.double() * scale
    lp = torch.log_softmax(y, -1)
    d = y - y.amax(-1, keepdim=True)
    p, dd = lp.exp(), torch.where(torch.isfinite(d), d, 0.0)
    e1, e2 = (p * dd.abs()).sum(-1), (p * dd * dd).sum(-1)
    logZ = torch.log(torch.exp(d).sum(-1))
    D = 3 * e1 + N + 2
    zt = D + 4 * logZ + 4

    def near(got, want, dw, zt):
        tol = STEP * (zt + 3 * dw.abs() + 2 * want.abs())
        off = (got.double() - want).abs() / tol
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        assert not (off[torch.isfinite(want)] > 1).any(), float(off.max())

    near(tl, lp.gather(1, best), d.gather(1, best), zt[:, None])
    if ids is not None:
        at = ids.cpu().long().clamp(min=0)[:, None]
        want = torch.where(ids.cpu() < 0, 0.0, lp.gather(1, at)[:, 0])
        dw = torch.where(ids.cpu() < 0, 0.0, d.gather(1, at)[:, 0])
        near(logp, want, torch.where(torch.isfinite(dw), dw, 0.0), zt)
    want = -(p * torch.where(p > 0, lp, 0.0)).sum(-1)
    tol = STEP * (zt + (D + N + 4) * e1 + 3 * e2 + 2 * e1 + 2 * want.abs())
    assert ((ent.double() - want).abs() <= tol).all(), float(((ent - want).abs() / tol).max())


def logits(gen, rows, vocab, dtype, spread=3.0):
    x = torch.randn(rows, vocab, generator=gen) * spread
    if dtype == torch.int32:
        return (x * 2 ** 18).to(torch.int32).to(DEV)
    return x.to(dtype).to(DEV)


UNIT = {t: 2.0 ** -18 if t == torch.int32 else 0.7 for t in TYPES}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k", [
    (1, 1, 1), (3, 2, 2), (2, 31, 20), (5, 32, 32), (2, 33, 32), (1, 255, 0), (3, 1017, 5),
    (2, 1023, 32), (2, 1024, 32), (3, 1025, 7), (70, 2049, 1), (2, 31 * 1024 + 5, 32),
    (2, 33 * 1024, 32), (5, 50257, 20), (1, 248320, 32), (40, 100003, 5), (2500, 1500, 3)])
def test_sizes(engine, dtype, rows, vocab, k):
    gen = torch.Generator().manual_seed(vocab)
    x = logits(gen, rows, vocab, dtype)
    ids = torch.randint(0, vocab, (rows,), generator=gen).int()
    ids[0] = vocab - 1
    if rows > 2:
        ids[rows // 2] = -1
    check(engine, x, ids.to(DEV), k, UNIT[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1024 * 1024 - 3, 1100003, 4200001])
def test_more_blocks_than_are_ranked_at_once(engine, dtype, vocab):
    # over 1,024 blocks of 1,024 logits, and over 4,096; among 7 values in a
    # second row, so that blocks' maxima are equal everywhere
    gen = torch.Generator().manual_seed(vocab)
    x = logits(gen, 2, vocab, dtype)
    x[1] = torch.randint(0, 7, (vocab,), generator=gen).to(DEV).to(dtype)
    for k in (1, 32):
        check(engine, x, ints([vocab - 1, 5]), k, 1e-6 if dtype == torch.int32 else 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_at_any_place(engine, dtype):
    # rows that begin at every element of 16 bytes, apart by odd strides
    gen = torch.Generator().manual_seed(4)
    flat = logits(gen, 1, 40000, dtype)[0]
    for off in range(16 // dtype.itemsize):
        for vocab, stride in ((3001, 3001), (4000, 4003), (1000, 1111)):
            x = flat[off:].as_strided((7, vocab), (stride, 1), off)
            check(engine, x, ints([0, 1, 2, vocab - 1, 5, 6, 7]), 9, UNIT[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["equal", "two", "few", "falling", "rising", "ends", "crowded"])
def test_equal_logits_go_by_index(engine, dtype, kind):
    rng, gen, V = random.Random(kind), torch.Generator().manual_seed(1), 70007
    x = torch.zeros(3, V)
    if kind == "two":
        x[:] = torch.randint(0, 2, (3, V), generator=gen).float()
    elif kind == "few":
        for r in range(3):
            for _ in range(20):
                x[r, rng.randrange(V)] = 4.0
    elif kind == "falling":
        x[:] = -(torch.arange(V) // 64).float() / 8
    elif kind == "rising":
        x[:] = (torch.arange(V) // 64).float() / 8
    elif kind == "ends":
        x[:, -1], x[:, 0], x[:, 1023:1026] = 2.0, 2.0, 2.0
    elif kind == "crowded":                                # 2,000 equals in two blocks
        x[:, 5000:7000], x[:, 60000] = 3.0, 5.0
    x = (x * 8).to(torch.int32).to(DEV) if dtype == torch.int32 else x.to(dtype).to(DEV)
    ids = ints([0, V - 1, 1024])
    for k in (1, 31, 32):
        check(engine, x, ids, k, 0.125 if dtype == torch.int32 else 1.0)


@pytest.mark.parametrize("dtype", TYPES[:3])
def test_zeros_of_either_sign_are_equal(engine, dtype):
    x = torch.zeros(2, 5000, device=DEV, dtype=dtype)
    x[0, ::3] = -0.0
    x[1, 100:200] = -0.0
    check(engine, x, ints([3, 1]), 32)


@pytest.mark.parametrize("dtype", TYPES[:3])
@pytest.mark.parametrize("vocab", [300, 5000, 70000])
def test_tokens_ruled_out(engine, dtype, vocab):
    # -infinity in most places, or all but one, or all
    gen = torch.Generator().manual_seed(7)
    x = logits(gen, 4, vocab, dtype)
    x[0, 1:] = -math.inf
    x[1, ::2] = -math.inf
    x[2, :vocab - 3] = -math.inf
    check(engine, x[:3], ints([0, 2, vocab - 1]), 20)
    x[3] = -math.inf
    logp, ent, tl, ti = run(engine, x, ints([0, 2, 1, 5]), 20)
    assert logp[3] == -math.inf and ent[3] == 0 and (tl[3] == -math.inf).all()
    assert ti[3].tolist() == list(range(20))


@pytest.mark.parametrize("dtype", TYPES[:3])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_row_without_numbers_spoils_no_other(engine, dtype, bad):
    gen = torch.Generator().manual_seed(8)
    x = logits(gen, 3, 9000, dtype)
    want = run(engine, x, ints([1, 2, 3]), 8)
    x[1, 4321] = bad
    got = run(engine, x, ints([1, 2, 3]), 8)
    for g, w in zip(got, want):
        assert torch.equal(g[::2], w[::2])
    assert torch.isnan(got[1][1]) and not torch.isfinite(got[2][1]).any()
    assert ((got[3][1] >= 0) & (got[3][1] < 9000)).all() and not torch.isfinite(got[0][1])


@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_a_row_of_nans_has_indices(engine, vocab):
    x = torch.full((2, vocab), math.nan, device=DEV)
    x[1, 3] = 1.0
    logp, ent, tl, ti = run(engine, x, ints([0, 3]), 32)
    assert torch.isnan(logp).all() and torch.isnan(ent).all() and torch.isnan(tl).all()
    assert ((ti >= 0) & (ti < vocab)).all()


def test_extremes(engine):
    # differences past 32 bits of whole numbers, and of floats; tiny scales
    x = torch.zeros(4, 3000, dtype=torch.int32, device=DEV)
    x[0, 5], x[0, 6] = 2 ** 31 - 1, -2 ** 31
    x[1] = -2 ** 31
    x[2] = torch.arange(3000, device=DEV).int() * 1000003
    x[3] = 2 ** 31 - 1
    ids = ints([6, 1, 2, 3])
    check(engine, x, ids, 32, 2.0 ** -28)
    got = run(engine, x, ids, 3, 1.0)
    assert got[0][0] == -4294967295.0 and got[1][0] == 0 and got[3][0].tolist() == [5, 0, 1]
    f = torch.zeros(2, 3000, device=DEV)
    f[0, 7], f[0, 8], f[1] = 3e38, -3e38, -3e38
    got = run(engine, f, ints([7, 1]), 2)
    assert got[0][0] == 0 and got[1][0] == 0 and got[3][0].tolist() == [7, 0]
    assert abs(float(got[1][1]) - math.log(3000)) < 1e-5
    check(engine, torch.randn(2, 4000, generator=torch.Generator().manual_seed(1)).to(DEV),
          ints([0, 1]), 4, 1e-6)


def test_ids_outside_the_vocabulary(engine):
    gen = torch.Generator().manual_seed(2)
    x = logits(gen, 3, 500, torch.float32)
    logp, ws = torch.full((3,), 9.0, device=DEV), engine.logprobs_workspace(3, 500)
    ids = ints([7, 500, 2 ** 31 - 1])
    torch.cuda.synchronize()
    engine.logprobs_async(x, ids, logp, ws)
    with pytest.raises(AssertionError, match="outside the vocabulary"):
        engine.sync()
    assert logp[1:].tolist() == [0, 0]
    assert abs(float(logp[0]) - float(torch.log_softmax(x[0].double(), -1)[7])) < 1e-5
    engine.sync()


def test_parts_of_the_call_and_wrong_tensors(engine):
    gen = torch.Generator().manual_seed(2)
    x = logits(gen, 3, 500, torch.bfloat16)
    ids, logp = ints([1, 2, 3]), torch.zeros(3, device=DEV)
    want = run(engine, x, ids, 4)
    ws = engine.logprobs_workspace(3, 500)
    engine.logprobs_async(x, ids, logp, ws)
    engine.sync()
    assert torch.equal(logp, want[0])
    assert torch.equal(run(engine, x, None, 0)[1], want[1])
    assert torch.equal(run(engine, x, None, 4, entropy=False)[3], want[3])
    f = engine.logprobs_async
    f(x[:0], ids[:0], logp[:0], ws)
    tl, ti = torch.zeros(3, 4, device=DEV), torch.zeros(3, 4, dtype=torch.int32, device=DEV)
    for call in (lambda: f(x.cpu(), ids, logp, ws), lambda: f(x.double(), ids, logp, ws),
                 lambda: f(x.short(), ids, logp, ws), lambda: f(x.t(), ids, logp, ws),
                 lambda: f(x, ids[:2], logp, ws), lambda: f(x, ids.long(), logp, ws),
                 lambda: f(x, ids, None, ws), lambda: f(x, None, logp, ws),
                 lambda: f(x, ids, logp.half(), ws), lambda: f(x, ids, logp, ws.cpu()),
                 lambda: f(x, ids, logp, ws[:59]), lambda: f(x, ids, logp, ws, scale=0.0),
                 lambda: f(x, ids, logp, ws, scale=-1.0), lambda: f(x, ids, logp, ws, scale=math.inf),
                 lambda: f(x, ids, logp, ws, scale=math.nan),
                 lambda: f(x, ids, logp, ws, entropy=logp[:2]),
                 lambda: f(x, ids, logp, ws, top_logp=tl), lambda: f(x, ids, logp, ws, top_ids=ti),
                 lambda: f(x, ids, logp, ws, top_logp=tl, top_ids=ti[:, :3]),
                 lambda: f(x, ids, logp, ws, top_logp=tl, top_ids=ti.long()),
                 lambda: f(x[:, :3], ids, logp, ws, top_logp=tl, top_ids=ti),
                 lambda: f(x, ids, logp, ws, top_logp=torch.zeros(3, 33, device=DEV),
                           top_ids=torch.zeros(3, 33, dtype=torch.int32, device=DEV)),
                 lambda: engine.logprobs_workspace(3, 0),
                 lambda: engine.logprobs_workspace(3, (1 << 24) + 1)):
        with pytest.raises(ValueError):
            call()
    engine.sync()


def test_two_graphs_with_workspaces_of_their_own(engine):
    gen = torch.Generator().manual_seed(12)
    xs = [logits(gen, 2, 40000, torch.float16) for _ in range(2)]
    ids = ints([5, 39999])
    want = [run(engine, x, ids, 8) for x in xs]
    graphs, outs, streams, keep = [], [], [], []
    for x in xs:
        out = [torch.zeros_like(t) for t in want[0]]
        ws, side, g = engine.logprobs_workspace(2, 40000), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        try:
            with torch.cuda.graph(g, stream=side):
                engine.set_stream(side)
                engine.logprobs_async(x, ids, out[0], ws, entropy=out[1], top_logp=out[2],
                                      top_ids=out[3])
        finally:
            engine.set_stream(None)
        graphs.append(g), outs.append(out), streams.append(side), keep.append(ws)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert torch.equal(run(engine, xs[0], ids, 8)[0], want[0][0])
