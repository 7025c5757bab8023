"""Heads normalised and rotated to their tokens' positions (Context.rotary_async,
PagedKV.append_rotary_async) against the definition in 64 bits.

The tolerance, per output, for a pair (a, b) after the norm, with u half a step
of the outputs' type (bfloat16 2^-8, float16 2^-11, float32 2^-24):

    u |out|                    the output (int16: half of one step instead;
                               float16: 2^-25 more, half its smallest step)
  + 2^-24 A (|a| + |b|) (8 + N)   cosine and sine within 4 of their last bits, the
                               amplitude A, a product and a sum; a norm: N = D / 2
                               + 4, the sum of D squares, its root, two products
"""
import math

import pytest
import torch

from fable5_llm_amd.engine import PagedKV
from fable5_llm_amd.mixers import rotary_frequencies
from test_gpu_attend import DEV, U, ints, make

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-5


def turned(x, pos, freq, layout, amplitude, norm):
    """(want, slack) of x [tokens, heads, dim] in 64 bits on the host."""
    x, rot, d = x.double().cpu(), 2 * freq.shape[0], x.shape[-1]
    n = 0.0
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * norm.double().cpu()
        n = d / 2 + 4
    t = pos.double().cpu()[:, None, None] * freq.double().cpu()
    i = torch.arange(rot // 2)
    ia, ib = (i, i + rot // 2) if layout == "halves" else (2 * i, 2 * i + 1)
    y, slack = x.clone(), 2.0 ** -24 * x.abs() * n
    a, b, c, s = x[..., ia], x[..., ib], t.cos() * amplitude, t.sin() * amplitude
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    slack[..., ia] = slack[..., ib] = 2.0 ** -24 * abs(amplitude) * (a.abs() + b.abs()) * (8 + n)
    return y, slack


def near(got, want, out_unit=None):
    want, slack = want
    if out_unit is None:
        tol = slack + U[got.dtype] * want.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    else:
        tol, want = slack + 0.5 * out_unit, want.clamp(-32768 * out_unit, 32767 * out_unit)
    off = (got.double().cpu() * (out_unit or 1.0) - want).abs()
    assert (off <= tol).all(), float((off / tol).nan_to_num(math.inf).max())


def inputs(gen, tokens, heads, dim, dtype):
    if dtype == torch.int16:
        return torch.randint(-20000, 20000, (tokens, heads, dim), generator=gen).short().to(DEV)
    return torch.randn(tokens, heads, dim, generator=gen).to(DEV).to(dtype)


def frequencies(rot, **kw):
    f, amplitude = rotary_frequencies(rot, **kw)
    return f.to(DEV), amplitude


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dim,rot,hq,hk", [(256, 64, 16, 4), (64, 64, 3, 1), (128, 112, 5, 5),
                                           (80, 32, 7, 1), (16, 16, 1, 1), (208, 0, 2, 3)])
@pytest.mark.parametrize("tokens", [1, 33, 700])
@pytest.mark.parametrize("types", [(t, t) for t in TYPES] + [(torch.int16, t) for t in
                                                             TYPES + [torch.int16]])
def test_rotary(engine, layout, dim, rot, hq, hk, tokens, types):
    gen = torch.Generator().manual_seed(dim + tokens)
    q, k = (inputs(gen, tokens, h, dim, types[0]) for h in (hq, hk))
    pos = torch.randint(0, 5000, (tokens,), generator=gen, dtype=torch.int32)
    pos[0] = 0
    if tokens > 1:
        pos[tokens // 2] = -1                              # a padded token
    freq, _ = frequencies(max(rot, 2))
    freq, norm = freq[:rot // 2], (1 + 0.3 * torch.randn(dim, generator=gen)).to(DEV)
    q_out, k_out = (torch.full(x.shape, 9, dtype=types[1], device=DEV) for x in (q, k))
    i16 = types[0] == torch.int16
    kw = dict(frac=12, out_frac=11) if i16 else {}
    dpos = pos.to(DEV)
    torch.cuda.synchronize()
    engine.rotary_async(q, k, dpos, freq, q_out, k_out, layout=layout, amplitude=1.25,
                        q_norm=norm, eps=EPS, **kw)
    engine.sync()
    live = pos >= 0
    for x, out, w in ((q, q_out, norm), (k, k_out, None)):
        x = x.double() * 2.0 ** -12 if i16 else x
        want = [y[live] for y in turned(x, pos, freq, layout, 1.25, w)]
        near(out.cpu()[live], want, 2.0 ** -11 if types[1] == torch.int16 else None)
        assert (out.cpu()[~live] == 9).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_in_place_with_strides_and_one_tensor_alone(engine, dtype, layout):
    gen = torch.Generator().manual_seed(3)
    wide = inputs(gen, 300, 12, 256, dtype)
    kept, pos = wide.clone(), torch.arange(300, dtype=torch.int32, device=DEV) * 7
    freq, _ = frequencies(96)
    q, k = wide[:, 1:9, 128:], wide[:, 9:, :128]
    torch.cuda.synchronize()
    engine.rotary_async(q, k, pos, freq, q, k, layout=layout)
    engine.sync()
    for x, y in ((q, kept[:, 1:9, 128:]), (k, kept[:, 9:, :128])):
        near(x, turned(y, pos, freq, layout, 1.0, None))
    assert torch.equal(wide[:, 0], kept[:, 0]) and torch.equal(wide[:, 1:9, :128], kept[:, 1:9, :128])
    out = torch.zeros_like(kept)
    for args in ((kept, None, pos, freq, out, None), (None, kept, pos, freq, None, out)):
        out.zero_()
        torch.cuda.synchronize()
        engine.rotary_async(*args, layout=layout)
        engine.sync()
        near(out, turned(kept, pos, freq, layout, 1.0, None))


def test_far_positions_keep_their_angle(engine):
    gen = torch.Generator().manual_seed(5)
    pos = torch.tensor([0, 1, 4095, 131071, 1000003, 2 ** 24 + 1, 2 ** 30 + 7, 2 ** 31 - 1],
                       dtype=torch.int32, device=DEV)
    q = inputs(gen, 8, 4, 128, torch.float32)
    for kw in (dict(), dict(base=1e6), dict(stretch="positions", factor=8.0),
               dict(stretch="base", factor=4.0),
               dict(stretch="parts", factor=16.0, trained=4096)):
        freq, amplitude = frequencies(128, **kw)
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        engine.rotary_async(q, None, pos, freq, out, None, amplitude=amplitude)
        engine.sync()
        near(out, turned(q, pos, freq, "halves", amplitude, None))


def test_every_quarter_of_a_turn(engine):
    # angles at and beside the quarters, by frequencies of exact fractions of 2 pi
    n = 64
    freq = torch.arange(n, dtype=torch.float64, device=DEV) * (2 * math.pi / n)
    q = torch.ones(41, 1, 2 * n, device=DEV)
    q[..., n:] = 0
    pos, out = torch.arange(41, dtype=torch.int32, device=DEV), torch.zeros_like(q)
    torch.cuda.synchronize()
    engine.rotary_async(q, None, pos, freq, out, None)
    engine.sync()
    near(out, turned(q, pos, freq, "halves", 1.0, None))


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("int16", [False, True])
@pytest.mark.parametrize("dim,heads,hq,page", [(64, 1, 3, 16), (128, 2, 14, 64), (256, 4, 16, 16)])
@pytest.mark.parametrize("counts", [(1, 0, 1), (40, 7, 400)])
def test_append(engine, cache, int16, dim, heads, hq, page, counts):
    # what is written: the slots of the new tokens in one layer, nothing else
    gen = torch.Generator().manual_seed(dim)
    lens = [70, 40, 410]
    kv = make(engine, gen, lens, heads, dim, page, cache, layers=2)
    kv.pool.nan_to_num_(5.0)
    before = kv.pool.clone()
    tokens = sum(counts) + 2 + 3
    m = kv.chunk_maps(4, tokens, hq)
    s, c = ints([2, -1, 0, 1]), ints([counts[2], 2, counts[0], counts[1]])
    dtype = torch.int16 if int16 else cache
    q, k, v = (inputs(gen, tokens, h, dim, dtype) for h in (hq, heads, heads))
    norms = [(1 + 0.3 * torch.randn(dim, generator=gen)).to(DEV) for _ in range(2)]
    q_out = torch.full(q.shape, 9, dtype=cache, device=DEV)
    freq, _ = frequencies(dim // 2)
    torch.cuda.synchronize()
    kv.map_async(s, c, m)
    kv.append_rotary_async(1, q, k, v, m.pos, m.slots, freq, q_out, q_norm=norms[0],
                           k_norm=norms[1], eps=EPS, frac=12 if int16 else 0)
    engine.sync()
    pos, slots = m.pos.cpu(), m.slots.cpu()
    live = pos >= 0
    assert int(live.sum()) == sum(counts)
    unit = 2.0 ** -12 if int16 else 1.0
    near(q_out.cpu()[live], [y[live] for y in turned(q.double() * unit, pos, freq, "halves", 1.0,
                                                     norms[0])])
    assert (q_out.cpu()[~live] == 9).all()
    at, place = (slots[live] // page).to(DEV), (slots[live] % page).to(DEV)
    got = kv.pool[at, 1, 0, :, place]
    near(got.cpu(), [y[live] for y in turned(k.double() * unit, pos, freq, "halves", 1.0, norms[1])])
    want = (v.double() * unit).to(cache)
    assert torch.equal(kv.pool[at, 1, 1, :, place], want[live.to(DEV)])
    after = kv.pool.clone()
    after[at, 1, :, :, place] = before[at, 1, :, :, place]
    assert torch.equal(after, before)


def test_append_like_append(engine):
    # without frequencies and norms, the rows that append_async writes
    gen = torch.Generator().manual_seed(9)
    pools = []
    for rotary in (False, True):
        kv = make(engine, torch.Generator().manual_seed(2), [33, 90], 2, 64, 16, torch.bfloat16)
        kv.pool.nan_to_num_(0.0)
        k, v = (inputs(torch.Generator().manual_seed(s), 50, 2, 64, torch.bfloat16) for s in (1, 2))
        m, s, c = kv.chunk_maps(2, 50, 2), ints([1, 0]), ints([40, 10])
        q, freq = torch.zeros_like(k), torch.zeros(0, dtype=torch.float64, device=DEV)
        torch.cuda.synchronize()
        kv.map_async(s, c, m)
        if rotary:
            kv.append_rotary_async(0, q, k, v, m.pos, m.slots, freq, q)
        else:
            kv.append_async(0, k, v, m.seqs, m.pos)
        engine.sync()
        pools.append(kv.pool)
    assert torch.equal(*pools) and gen is not None


def test_slots_outside_the_pool_and_a_stopped_cache(engine):
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [40, 8], 1, 64, 16, torch.float32, spare=0)
    kv.pool.nan_to_num_(5.0)
    before = kv.pool.clone()
    q, k, v = (inputs(gen, 2, 1, 64, torch.float32) for _ in range(3))
    freq, _ = frequencies(64)
    pos = ints([3, 4])
    slots = torch.tensor([4 * 16, 1 << 40], device=DEV)
    torch.cuda.synchronize()
    kv.append_rotary_async(0, q, k, v, pos, slots, freq, q)
    with pytest.raises(AssertionError, match="outside the cache"):
        engine.sync()
    assert torch.equal(kv.pool, before)
    s, c, slots = ints([0, 1]), ints([1, 60]), torch.tensor([1, 2], device=DEV)
    torch.cuda.synchronize()
    kv.extend_async(s, c)                                  # refused: no pages left
    kv.append_rotary_async(0, q, k, v, pos, slots, freq, q)
    with pytest.raises(AssertionError, match="too few free pages"):
        engine.sync()
    assert torch.equal(kv.pool, before)
    kv.append_rotary_async(0, q, k, v, pos, slots, freq, q)
    engine.sync()
    assert not torch.equal(kv.pool, before)


def test_wrong_tensors(engine):
    gen = torch.Generator().manual_seed(1)
    kv = make(engine, gen, [40], 2, 64, 16, torch.bfloat16)
    q, k = (torch.zeros(3, h, 64, dtype=torch.bfloat16, device=DEV) for h in (4, 2))
    pos, freq, f = ints([0, 1, 2]), frequencies(64)[0], engine.rotary_async
    slots, g = torch.zeros(3, dtype=torch.int64, device=DEV), kv.append_rotary_async
    norm = torch.ones(64, device=DEV)
    f(q[:0], None, pos[:0], freq, q[:0], None)
    for call in (lambda: f(q.cpu(), k, pos, freq, q, k), lambda: f(None, None, pos, freq, None, None),
                 lambda: f(q, k, pos, freq, None, k), lambda: f(None, k, pos, freq, None, None),
                 lambda: f(q, k, pos, freq, q, None), lambda: f(q, k, pos[:2], freq, q, k), lambda: f(q, k, pos.long(), freq, q, k),
                 lambda: f(q, k, pos, freq.float(), q, k), lambda: f(q, k, pos, freq[:7], q, k),
                 lambda: f(q, k, pos, frequencies(80)[0], q, k),
                 lambda: f(q, k.half(), pos, freq, q, k.half()),
                 lambda: f(q, k, pos, freq, q.float(), k.float()),
                 lambda: f(q, k, pos, freq, q, q), lambda: f(q, k[:2], pos, freq, q, k[:2]),
                 lambda: f(q, k, pos, freq, q, k, layout="both"),
                 lambda: f(q, k, pos, freq, q, k, q_norm=norm[:32]),
                 lambda: f(q, k, pos, freq, q, k, k_norm=norm.half()),
                 lambda: f(q[..., :24], None, pos, freq[:8], q[..., :24], None),
                 lambda: f(q, k, pos, freq, q, k, eps=-1.0),
                 lambda: f(q, k, pos, freq, q, k, amplitude=math.nan),
                 lambda: f(q.short(), k.short(), pos, freq, q, k, frac=32),
                 lambda: g(0, q, k, k, pos, slots.int(), freq, q),
                 lambda: g(0, q, k, k, pos, slots[:2], freq, q),
                 lambda: g(1, q, k, k, pos, slots, freq, q),
                 lambda: g(0, q, q, q, pos, slots, freq, q),
                 lambda: g(0, q, k, k[..., :32], pos, slots, freq, q),
                 lambda: g(0, q.half(), k.half(), k.half(), pos, slots, freq, q),
                 lambda: g(0, q.short(), k.short(), k.short(), pos, slots, freq, q.short()),
                 lambda: g(0, q, k, k, pos, slots, freq, None),
                 lambda: g(0, None, k, k, pos, slots, freq, None)):
        with pytest.raises(ValueError):
            call()
    engine.sync()


def test_two_streams_graphs_of_an_append(engine):
    # one captured launch, replayed with other positions and slots
    gen = torch.Generator().manual_seed(6)
    kv = PagedKV.empty(engine, 20, 1, 2, 16, 64, 2, 8, torch.float16)
    q, k, v = (inputs(gen, 5, h, 64, torch.float16) for h in (4, 2, 2))
    pos, slots = ints([0] * 5), torch.full((5,), -1, device=DEV)
    freq, out = frequencies(64)[0], torch.zeros_like(q)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=side):
            engine.set_stream(side)
            kv.append_rotary_async(0, q, k, v, pos, slots, freq, out)
    finally:
        engine.set_stream(None)
    for i in range(4):
        pos.copy_(ints([3 * i, -1, i, 70, 9]))
        slots.copy_(torch.tensor([i, 5, 20 + i, -1, 319 - i]))
        q.copy_(torch.randn(q.shape, generator=gen))
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, slack = turned(q, pos, freq, "halves", 1.0, None)
        live = torch.tensor([0, 2, 4])
        near(out.cpu()[live], [want[live], slack[live]])
        assert (out[[1, 3]] == 9).all()
        assert torch.equal(kv.pool[(320 - i - 1) // 16, 0, 1, :, (319 - i) % 16], v[4])
