"""Forms of the mixers' kernels beside those of their own files: int16 attention at
heads of 128, int16 prompts at key heads of 64, appended rows of more vectors than
a wavefront's first turn takes, a prompt of many chunks, a captured step of enough
rows that their slots are checked by a kernel of their own."""
import numpy as np
import pytest
import torch

import test_gpu_attend as A
import test_gpu_delta as D
from fable5_llm_amd.engine import PagedKV

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ints = A.ints


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,group", [(2, 4), (1, 17)])
def test_int16_attention_at_heads_of_128(engine, cache, heads, group):
    gen = torch.Generator().manual_seed(13)
    lens = [1, 200, 77, 2000, 0]
    kv = A.make(engine, gen, lens, heads, 128, 16, cache)
    q = torch.randint(-32768, 32768, (5, heads * group, 128), generator=gen, dtype=torch.int32)
    q = q.to(torch.int16).to(DEV)
    seqs = [3, 1, 4, 2, 0]
    out = A.run(engine, kv, 0, q, seqs, frac=13, out_frac=12)
    A.check(kv, 0, q, seqs, out, unit=2.0 ** -13, out_unit=2.0 ** -12)


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 80), (128, 32)])
@pytest.mark.parametrize("fresh", [False, True])
def test_int16_prompts(engine, dk, dv, fresh):
    gen = torch.Generator().manual_seed(dk + dv)
    lens = [70, 1, 0, 64, 130]
    cu = D.spans_of(lens)
    d = D.inputs(gen, cu[-1] + 3, 2, 4, dk, dv, torch.int16, len(lens))
    slots = [4, 0, 2, 1, 3]
    out = torch.full_like(d["v"], 9)
    want = D.recurrence(d, list(zip(cu[:-1], cu[1:])), slots, unit=2.0 ** -12, fresh=fresh)
    ws = engine.delta_chunk_workspace(cu[-1] + 3, len(lens), 4, hk=2, dk=dk, dtype=torch.int16)
    c, sl = ints(cu), ints(slots)
    ws.fill_(0xFF)
    torch.cuda.synchronize()
    engine.delta_chunk_async(**d, out=out, cu=c, ws=ws, slots=sl, fresh=fresh, frac=12, out_frac=14)
    engine.sync()
    assert (out[cu[-1]:] == 9).all()
    D.check(out[:cu[-1]], d["state"], (want[0][:cu[-1]], want[1], want[2][:cu[-1]], want[3]),
            out_unit=2.0 ** -14)


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,dim", [(8, 256), (5, 128), (9, 64), (1, 64)])
def test_append_of_wide_rows(engine, cache, heads, dim):
    rng = np.random.default_rng(heads)
    n = 7
    kv = PagedKV.empty(engine, 12, 2, heads, 16, dim, 3, 4, cache)
    own = torch.from_numpy(rng.normal(0, 1, (2, n, heads, dim))).to(DEV).to(cache)
    i16 = torch.from_numpy(rng.integers(-32768, 32768, (2, n, heads, dim)).astype(np.int16)).to(DEV)
    seqs, pos = [2, 0, -1, 0, 1, 2, 2], [17, 3, 0, 16, 63, 0, 39]
    args = ints([0, 1, 2]), ints([20, 64, 40]), ints(seqs), ints(pos)
    torch.cuda.synchronize()
    kv.extend_async(args[0], args[1])
    kv.append_async(1, own[0], own[1], args[2], args[3])
    kv.append_async(0, i16[0], i16[1], args[2], args[3], frac=9)
    engine.sync()
    want = torch.zeros_like(kv.pool)
    for i, (s, p) in enumerate(zip(seqs, pos)):
        if s >= 0:
            page = int(kv.tables[s, p // 16])
            want[page, 1, :, :, p % 16] = own[:, i]
            want[page, 0, :, :, p % 16] = (i16[:, i].double() / 512).to(cache)
    assert torch.equal(kv.pool, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_prompt_of_many_chunks(engine, dtype):
    gen = torch.Generator().manual_seed(40)
    lens = [4100, 130, 2048]
    cu = D.spans_of(lens)
    d = D.inputs(gen, cu[-1], 1, 2, 128, 32, dtype, 3)
    want = D.recurrence(d, list(zip(cu[:-1], cu[1:])), [0, 1, 2])
    out, ws, c = torch.zeros_like(d["v"]), engine.delta_chunk_workspace(cu[-1], 3, 2, hk=1), ints(cu)
    ws.fill_(0xFF)
    torch.cuda.synchronize()
    engine.delta_chunk_async(**d, out=out, cu=c, ws=ws)
    engine.sync()
    D.check(out, d["state"], want)


def test_a_captured_token_of_many_rows(engine):
    rows = 17000
    gen = torch.Generator().manual_seed(41)
    d = D.inputs(gen, rows, 1, 4, 64, 64, torch.bfloat16, rows)
    sl = torch.randperm(rows, generator=gen).to(torch.int32).to(DEV)
    first, out = d["state"].clone(), torch.zeros_like(d["v"])
    torch.cuda.synchronize()
    engine.delta_step_async(**d, out=out, slots=sl)
    engine.sync()
    want = out.clone(), d["state"].clone()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(g, stream=side):
            engine.set_stream(side)
            engine.delta_step_async(**d, out=out, slots=sl)
    finally:
        engine.set_stream(None)
    for i in range(3):
        d["state"].copy_(first)
        out.fill_(i)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(d["state"], want[1])
    engine.sync()
