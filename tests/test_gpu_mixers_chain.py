"""A decoder's layers at one token a step, on the device from site to site: a
DeltaNet layer (ln1 site -> gated delta rule -> out site) and an attention layer
(ln1 site -> new token into the cache -> attention -> o_proj site), int16
between them as the engine's sites write and read it.  Every site exactly the
oracle's on its own input, every mixer within half a step of its int16 output
of the 64-bit definition on its own input; eagerly, and as one captured step
replayed token after token."""
import math

import numpy as np
import pytest
import torch

from fable5_llm_amd import _native as N
from fable5_llm_amd.engine import PagedKV
from oracle import law
from tests.helpers import activation_x16, norm_weight_q14, rand_w4_m

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E_SCALE, RS_F, QKV_F, DN_F, ATTN_F = -3, 7, 8, 11, 13
H, HK, HV, DK, DV = 512, 2, 4, 64, 64            # hidden size, DeltaNet heads
HQ, HKV, D, PAGE = 8, 2, 64, 16                  # attention heads


class Mat:
    def __init__(self, engine, rng, rows, K, in_f, out_f):
        self.w4, self.m = rand_w4_m(rng, rows, K)
        self.sh = law.sh_for_k(K)
        self.p0 = (15 - E_SCALE - self.sh) + in_f - out_f
        img, _ = law.pack_ddr_rows(self.w4, self.m)
        self.dev = engine.upload(img, rows, K, self.sh)
        self.out = torch.zeros(rows, dtype=torch.int16, device=DEV)

    def want(self, x16):
        x8, e = law.dyn_quant_i8(x16)
        return law.movy(law.matvec_y32(self.w4, self.m, self.sh, x8), self.p0 - e,
                        law.MOVY_INT16)


def near(got, want, frac, slack):
    """int16 outputs within half a step and what their inputs' 32-bit sums allow."""
    assert (np.abs(got.astype(np.int32)) < 32767).mean() > 0.9 and (got != 0).mean() > 0.5
    want = np.clip(want, -32768 * 2.0 ** -frac, 32767 * 2.0 ** -frac)
    off = np.abs(got.astype(np.float64) * 2.0 ** -frac - want)
    assert off.max() <= 0.5 * 2.0 ** -frac + slack, off.max()


def test_layers_token_by_token(engine):
    rng = np.random.default_rng(31)
    dev = dict(device=DEV)
    qkv = Mat(engine, rng, 2 * HK * DK + HV * DV, H, RS_F, RS_F)
    out = Mat(engine, rng, H, HV * DV, DN_F, RS_F)
    # an eighth of what these weights give: values within out's 13 fraction bits
    wq, wk, wv = (Mat(engine, rng, n, H, RS_F, QKV_F - 3) for n in (HQ * D, HKV * D, HKV * D))
    wo = Mat(engine, rng, H, HQ * D, ATTN_F, RS_F)
    norms = [norm_weight_q14(rng, H) for _ in range(2)]
    dnorms = [torch.from_numpy(n).to(DEV) for n in norms]
    x = torch.zeros(H, dtype=torch.int16, **dev)
    g, beta = torch.zeros(1, HV, **dev), torch.zeros(1, HV, **dev)
    state = torch.zeros(2, HV, DK, DV, **dev)
    slot = torch.tensor([1], dtype=torch.int32, **dev)
    mid = torch.zeros(1, HV, DV, dtype=torch.int16, **dev)
    kv = PagedKV.empty(engine, 8, 2, HKV, PAGE, D, 3, 4, torch.bfloat16)
    seq = torch.tensor([2], dtype=torch.int32, **dev)
    one = torch.ones(1, dtype=torch.int32, **dev)
    att = torch.zeros(1, HQ, D, dtype=torch.int16, **dev)
    ws = kv.attend_workspace(1, HQ)
    heads = qkv.out.view(1, -1)
    q = heads[:, :HK * DK].unflatten(1, (HK, DK))
    k = heads[:, HK * DK:2 * HK * DK].unflatten(1, (HK, DK))
    v = heads[:, 2 * HK * DK:].unflatten(1, (HV, DV))
    I16, RMS, DQ = N.EPI_MOVY_I16, N.PRO_RMSNORM_DYNQ8, N.PRO_DYNQ8
    torch.cuda.synchronize()

    def step():
        engine.site_async([qkv.dev], [I16], [qkv.p0], [qkv.out], x, prologue=RMS,
                          norm_w=dnorms[0], in_f=RS_F, one_plus=True)
        engine.delta_step_async(q, k, v, g, beta, state, mid, slots=slot, frac=RS_F,
                                out_frac=DN_F)
        engine.site_async([out.dev], [I16], [out.p0], [out.out], mid.view(-1), prologue=DQ)
        engine.site_async([wq.dev, wk.dev, wv.dev], [I16] * 3, [wq.p0, wk.p0, wv.p0],
                          [wq.out, wk.out, wv.out], out.out, prologue=RMS, norm_w=dnorms[1],
                          in_f=RS_F, one_plus=True)
        kv.extend_async(seq, one)
        kv.append_async(1, wk.out.view(1, HKV, D), wv.out.view(1, HKV, D), seq, frac=QKV_F)
        kv.attend_async(1, wq.out.view(1, HQ, D), seq, att, ws, frac=QKV_F, out_frac=ATTN_F)
        engine.site_async([wo.dev], [I16], [wo.p0], [wo.out], att.view(-1), prologue=DQ)

    S = np.zeros((HV, DK, DV))
    keys, values = [], []

    def check(x16, gt, bt):
        nonlocal S
        xn = law.rmsnorm_fx(x16, norms[0], RS_F, True)
        y = qkv.out.cpu().numpy()
        assert np.array_equal(y, qkv.want(xn.astype(np.int16)))
        f = y.astype(np.float64) * 2.0 ** -RS_F
        qq, kk = (a.reshape(HK, DK) for a in (f[:HK * DK], f[HK * DK:2 * HK * DK]))
        vv = f[2 * HK * DK:].reshape(HV, DV)
        qq, kk = (np.repeat(a / np.sqrt((a * a).sum(-1, keepdims=True) + 1e-6), HV // HK, 0)
                  for a in (qq, kk))
        S = S * np.exp(gt)[:, None, None]
        u = bt[:, None] * (vv - np.einsum("hk,hkv->hv", kk, S))
        S = S + kk[:, :, None] * u[:, None]
        want = np.einsum("hk,hkv->hv", qq, S) / math.sqrt(DK)
        m = mid.cpu().numpy()[0]
        near(m, want, DN_F, 1e-5 * np.abs(S).max())
        assert np.array_equal(out.out.cpu().numpy(), out.want(m.reshape(-1)))
        xn = law.rmsnorm_fx(out.out.cpu().numpy(), norms[1], RS_F, True).astype(np.int16)
        for w in (wq, wk, wv):
            assert np.array_equal(w.out.cpu().numpy(), w.want(xn))
        bf = lambda w: (w.out.double() * 2.0 ** -QKV_F).bfloat16().double().cpu().numpy() \
            .reshape(HKV, D)                          # noqa: E731
        keys.append(bf(wk)), values.append(bf(wv))
        K, V = (np.repeat(np.stack(a, 1), HQ // HKV, 0) for a in (keys, values))
        qa = wq.out.cpu().numpy().astype(np.float64).reshape(HQ, D) * 2.0 ** -QKV_F
        s = np.einsum("hd,htd->ht", qa, K) / math.sqrt(D)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        # weights as two bfloat16 values (2^-16), scores summed in float32
        X = np.einsum("hd,htd->ht", np.abs(qa), np.abs(K)).max() / math.sqrt(D)
        A = np.einsum("ht,htd->hd", p, np.abs(V)).max()
        a16 = att.cpu().numpy()[0]
        near(a16, np.einsum("ht,htd->hd", p, V), ATTN_F,
             A * (2.0 ** -16 + 2.0 ** -24 * (X * (D + 4) + len(keys) + 16)))
        assert np.array_equal(wo.out.cpu().numpy(), wo.want(a16.reshape(-1)))

    def token():
        x16 = activation_x16(rng, H)
        gt, bt = -np.exp(rng.normal(-2, 1, HV)), 1 / (1 + np.exp(-rng.normal(0, 1, HV)))
        x.copy_(torch.from_numpy(x16))
        g.copy_(torch.from_numpy(gt[None]))
        beta.copy_(torch.from_numpy(bt[None]))
        torch.cuda.synchronize()
        return x16, g.double().cpu().numpy()[0], beta.double().cpu().numpy()[0]

    for _ in range(3):
        t = token()
        step()
        engine.sync()
        check(*t)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            engine.set_stream(side)
            step()
    finally:
        engine.set_stream(None)
    for i in range(20):                               # past a page's end
        t = token()
        graph.replay() if i % 4 else step()           # with eager steps between
        torch.cuda.synchronize()
        engine.sync()
        check(*t)
    assert kv.lens.tolist() == [0, 0, 23] and int(kv.refs.sum()) == 2
