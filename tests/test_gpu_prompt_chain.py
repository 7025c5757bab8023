"""A prompt's chunks and then single tokens through an attention layer, on the
device: reserve, maps, heads' norms and positions with the append, attention of
the new tokens, and what the head's logits say about them; int16 in, as sites
write it, int16 out, as they read it.  Each operator against its definition on its
own input; eagerly, and as one captured step replayed with other counts; and the
single-token attention on the same cache and queries."""
import math

import numpy as np
import pytest
import torch

from fable5_llm_amd.engine import PagedKV
from fable5_llm_amd.mixers import rotary_frequencies
from oracle import law
from test_gpu_attend import DEV, check as check_single, ints
from test_gpu_chunk import check as check_chunk
from test_gpu_logprobs import check as check_logprobs
from test_gpu_rotary import EPS, near, turned
from tests.helpers import rand_w4_m

pytestmark = pytest.mark.gpu
HQ, HKV, D, T, ROWS, V, FRAC, OUT = 8, 2, 64, 48, 3, 1000, 12, 13


def test_prompts_then_tokens(engine):
    rng, gen = np.random.default_rng(7), torch.Generator().manual_seed(7)
    kv = PagedKV.empty(engine, 40, 2, HKV, 16, D, 4, 12, torch.bfloat16)
    w4, m = rand_w4_m(rng, V, HQ * D)
    img, _ = law.pack_ddr_rows(w4, m)
    head = engine.upload(img, V, HQ * D, law.sh_for_k(HQ * D))
    i16 = dict(dtype=torch.int16, device=DEV)
    q, k, v = (torch.zeros(T, h, D, **i16) for h in (HQ, HKV, HKV))
    q_out = torch.zeros(T, HQ, D, dtype=torch.bfloat16, device=DEV)
    att, x8 = torch.zeros(T, HQ, D, **i16), torch.zeros(T, HQ * D, dtype=torch.int8, device=DEV)
    y32 = torch.zeros(T, V, dtype=torch.int32, device=DEV)
    seqs, counts, ids = ints([2, 0, -1]), ints([0] * ROWS), ints([0] * T)
    maps = kv.chunk_maps(ROWS, T, HQ)
    ws, lws = kv.attend_chunk_workspace(maps), engine.logprobs_workspace(T, V)
    freq = rotary_frequencies(32)[0].to(DEV)
    norms = [(1 + 0.2 * torch.randn(D, generator=gen)).to(DEV) for _ in range(2)]
    logp, ent = (torch.zeros(T, device=DEV) for _ in range(2))
    tl, ti = torch.zeros(T, 5, device=DEV), torch.zeros(T, 5, dtype=torch.int32, device=DEV)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    scale = 2.0 ** -16
    torch.cuda.synchronize()

    def step():
        kv.extend_async(seqs, counts)
        kv.map_async(seqs, counts, maps)
        kv.append_rotary_async(1, q, k, v, maps.pos, maps.slots, freq, q_out, q_norm=norms[0],
                               k_norm=norms[1], eps=EPS, frac=FRAC)
        kv.attend_chunk_async(1, q_out, att, maps, ws, out_frac=OUT)
        x8.copy_(att.view(T, -1) >> 8)
        engine.matmul_async(head, x8, y32)
        engine.logprobs_async(y32, ids, logp, lws, entropy=ent, top_logp=tl, top_ids=ti,
                              scale=scale)

    def fill(c):
        for t in (q, k, v):
            t.copy_(torch.randint(-9000, 9000, t.shape, generator=gen))
        counts.copy_(ints(c))
        ids.copy_(torch.randint(0, V, (T,), generator=gen))
        att.fill_(7)
        q_out.zero_()
        torch.cuda.synchronize()

    def check(c):
        live = maps.pos.cpu() >= 0
        assert int(live.sum()) == c[0] + c[1]
        for x, y, w in ((q, q_out.cpu()[live], norms[0]), (k, None, norms[1])):
            want = [z[live] for z in turned(x.double() * 2.0 ** -FRAC, maps.pos, freq, "halves", 1.0, w)]
            if y is None:
                s = maps.slots.cpu()[live].to(DEV)
                y = kv.pool[s // 16, 1, 0, :, s % 16].cpu()
                got = kv.pool[s // 16, 1, 1, :, s % 16]
                assert torch.equal(got, (v.double() * 2.0 ** -FRAC).bfloat16()[live.to(DEV)])
            near(y, want)
        total = sum(c)
        assert (att[total:] == 7).all()
        check_chunk(kv, 1, q_out[:total], seqs.tolist(), c, att[:total], out_unit=2.0 ** -OUT)
        assert torch.equal(x8, (att.view(T, -1) >> 8).to(torch.int8))
        rows = [0, T - 1]
        for r in rows:
            assert np.array_equal(y32[r].cpu().numpy(), law.matvec_y32(
                w4, m, law.sh_for_k(HQ * D), x8[r].cpu().numpy()))
        check_logprobs(engine, y32, ids, 5, scale, (logp, ent, tl, ti))

    engine.set_stream(side)
    try:
        for c in ([20, 7, 2], [9, 33, 0]):                # eagerly
            fill(c)
            with torch.cuda.stream(side):
                step()
            engine.sync()
            check(c)
        with torch.cuda.graph(graph, stream=side):
            step()
        for c in ([1, 1, 1], [17, 0, 5], [1, 1, 0], [1, 1, 0]):
            fill(c)
            graph.replay()
            torch.cuda.synchronize()
            engine.sync()
            check(c)
    finally:
        engine.set_stream(None)
    # the last step's tokens, one a row, by the single-token attention
    rows = kv.attend_workspace(2, HQ)
    out, two = torch.zeros(2, HQ, D, **i16), ints([2, 0])
    one = torch.zeros(2, HQ, D, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    kv.attend_async(1, q_out[:2], two, one, rows)
    engine.sync()
    check_single(kv, 1, q_out[:2], [2, 0], one)
    near_chunk = att[:2].double().cpu() * 2.0 ** -OUT
    # bfloat16 of either: half a step of it, and of the weights (2^-8 of |v| at most)
    V_max = float(kv.pool[:, 1, 1].abs().max())
    assert (near_chunk - one.double().cpu()).abs().max() <= 3 * 2.0 ** -8 * V_max + 2.0 ** -OUT
    assert kv.lens.tolist() == [20 + 9 + 1 + 17 + 1 + 1 if s == 2 else 7 + 33 + 1 + 0 + 1 + 1
                                if s == 0 else 0 for s in range(4)]
    assert out.shape == one.shape and math.isfinite(V_max)
