"""The gated delta rule (Context.delta_step_async, delta_chunk_async) against
its recurrence in 64 bits, token by token.

The tolerance: a rounding of 2^-24 per operation, taken as independent, over
the T tokens behind a value and the dk terms of its dot products; the map of
one token does not grow an error (|e^g (I - beta k k^T)| <= 1 for unit keys).
So a state is off by at most 8 sqrt(T + dk) 2^-24 M, M the largest state of
the row so far, and an output by that (q is a unit vector and the scale 1 /
sqrt(dk)) plus half a step of its type; int16 outputs by half a step of theirs.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def inputs(gen, tokens, hk, hv, dk, dv, dtype, slots, frac=12):
    def act(*shape):
        x = torch.randn(*shape, generator=gen)
        if dtype == torch.int16:
            x = (x * 2 ** frac).round().clamp(-32768, 32767)
        return x.to(dtype).to(DEV)
    g = -torch.exp(torch.randn(tokens, hv, generator=gen) * 1.5 - 3.0)
    return dict(q=act(tokens, hk, dk), k=act(tokens, hk, dk), v=act(tokens, hv, dv),
                g=g.to(DEV), beta=torch.sigmoid(torch.randn(tokens, hv, generator=gen)).to(DEV),
                state=(torch.randn(slots, hv, dk, dv, generator=gen) * 0.3).to(DEV))


def recurrence(d, spans, slots, unit=1.0, norm=True, scale=None, eps=1e-6, fresh=False):
    """(out, state, error scale of a token's out, of a slot's state) in 64
    bits; rows without a slot get zeros."""
    q, k, v = (d[n].double().cpu() * unit for n in "qkv")
    g, beta = d["g"].double().cpu(), d["beta"].double().cpu()
    state = d["state"].double().cpu().clone()
    dk, per = q.shape[2], v.shape[1] // q.shape[1]
    if norm:
        q, k = (x / (x.square().sum(-1, keepdim=True) + eps).sqrt() for x in (q, k))
    q, k = (x.repeat_interleave(per, 1) for x in (q, k))
    out = torch.zeros_like(v)
    tol_o, tol_s = torch.zeros(v.shape[0]), torch.zeros(state.shape[0])
    scale = 1.0 / math.sqrt(dk) if scale is None else scale
    for (t0, t1), slot in zip(spans, slots):
        if slot < 0:
            continue
        S = torch.zeros_like(state[slot]) if fresh else state[slot]
        M = S.abs().max().item()
        for n, t in enumerate(range(t0, t1)):
            S = S * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (k[t][:, None] @ S)[:, 0])
            S = S + k[t][:, :, None] * u[:, None]
            out[t] = (q[t][:, None] @ S)[:, 0] * scale
            M = max(M, S.abs().max().item())
            tol_o[t] = 8 * math.sqrt(n + 1 + dk) * 2.0 ** -24 * M
        state[slot] = S
        tol_s[slot] = 8 * math.sqrt(t1 - t0 + dk) * 2.0 ** -24 * M
    return out, state, tol_o, tol_s


def check(out, state, want, out_unit=None):
    w_out, w_state, tol_o, tol_s = want
    got = out.double().cpu() * (out_unit or 1.0)
    tol = tol_o[:, None, None].double()
    if out_unit is None:
        tol = tol + U[out.dtype] * w_out.abs()
    else:
        tol = tol + 0.5 * out_unit
        w_out = w_out.clamp(-32768 * out_unit, 32767 * out_unit)
    off = (got - w_out).abs() - tol
    assert not torch.isnan(got).any() and off.max() <= 0, float(off.max())
    off = (state.double().cpu() - w_state).abs() - tol_s[:, None, None, None]
    assert off.max() <= 0, float(off.max())


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hk,hv,dk,dv", [
    (1, 1, 1, 64, 16), (1, 16, 32, 128, 128), (7, 2, 6, 128, 80), (33, 1, 3, 64, 256),
    (5, 4, 4, 64, 48), (300, 1, 1, 64, 16)])
def test_step(engine, dtype, rows, hk, hv, dk, dv):
    gen = torch.Generator().manual_seed(rows + dv)
    d = inputs(gen, rows, hk, hv, dk, dv, dtype, rows + 2)
    slots = torch.randperm(rows + 2, generator=gen)[:rows].tolist()
    if rows > 2:
        slots[1] = -1                                     # a padded row
    out, sl = torch.full_like(d["v"], 3), ints(slots)
    for _ in range(3):
        want = recurrence(d, [(i, i + 1) for i in range(rows)], slots)
        torch.cuda.synchronize()
        engine.delta_step_async(**d, out=out, slots=sl)
        engine.sync()
        check(out, d["state"], want)


def spans_of(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,hk,hv,dk,dv", [
    ([1], 1, 1, 64, 16), ([64], 1, 2, 64, 64), ([63, 65, 0, 1, 128], 2, 2, 128, 32),
    ([0, 200], 1, 3, 128, 128), ([300], 2, 4, 128, 80), ([129, 7, 64, 2], 1, 2, 64, 256),
    ([70, 40], 1, 6, 128, 16), ([5] * 40, 1, 1, 64, 16),
    # a key head's six value heads in one workgroup, in shares of two, and in
    # shares of which the last ones are empty
    ([1] * 520, 1, 6, 64, 16), ([3] * 130, 1, 6, 64, 16), ([2] * 100, 1, 6, 128, 16)])
def test_chunk(engine, dtype, lens, hk, hv, dk, dv):
    gen = torch.Generator().manual_seed(sum(lens) + dv)
    cu = spans_of(lens)
    rows, tokens = len(lens), cu[-1] + 5                  # five tokens behind the last row
    d = inputs(gen, tokens, hk, hv, dk, dv, dtype, rows + 1)
    slots = torch.randperm(rows + 1, generator=gen)[:rows].tolist()
    spans = list(zip(cu[:-1], cu[1:]))
    for fresh in (False, True):
        want = recurrence(d, spans, slots, fresh=fresh)
        out = torch.full_like(d["v"], 3)
        ws, c, sl = engine.delta_chunk_workspace(tokens, rows, hv), ints(cu), ints(slots)
        ws.fill_(0xFF)
        torch.cuda.synchronize()
        engine.delta_chunk_async(**d, out=out, cu=c, ws=ws, slots=sl, fresh=fresh)
        engine.sync()
        assert (out[cu[-1]:] == 3).all()                  # left as they were
        want[0][cu[-1]:] = 3
        check(out, d["state"], want)


@pytest.mark.parametrize("kind", ["step", "chunk"])
def test_int16(engine, kind):
    gen = torch.Generator().manual_seed(21)
    lens = [1] * 4 if kind == "step" else [70, 1, 130]
    cu = spans_of(lens)
    d = inputs(gen, cu[-1], 2, 4, 128, 128, torch.int16, len(lens))
    d["q"][0] = 32767
    d["k"][0, 0] = -32768
    out = torch.zeros_like(d["v"])
    want = recurrence(d, list(zip(cu[:-1], cu[1:])), list(range(len(lens))), unit=2.0 ** -12)
    ws, c = engine.delta_chunk_workspace(cu[-1], len(lens), 4), ints(cu)
    torch.cuda.synchronize()
    if kind == "step":
        engine.delta_step_async(**d, out=out, frac=12, out_frac=15)
    else:
        engine.delta_chunk_async(**d, out=out, cu=c, ws=ws, frac=12, out_frac=15)
    engine.sync()
    check(out, d["state"], want, out_unit=2.0 ** -15)


@pytest.mark.parametrize("kind", ["step", "chunk"])
def test_strided_rows_without_norms(engine, kind):
    # q, k and v side by side in one row of a projection; keys of norm 1 given
    gen = torch.Generator().manual_seed(22)
    lens = [1] * 3 if kind == "step" else [90, 33]
    cu, hk, hv, dk, dv = spans_of(lens), 2, 4, 64, 128
    T = cu[-1]
    row = torch.randn(T, 2 * hk * dk + hv * dv, generator=gen).to(DEV)
    q = row[:, :hk * dk].unflatten(1, (hk, dk))
    k = row[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk))
    k /= k.square().sum(-1, keepdim=True).sqrt()
    v = row[:, 2 * hk * dk:].unflatten(1, (hv, dv))
    d = inputs(gen, T, hk, hv, dk, dv, torch.float32, len(lens))
    d.update(q=q, k=k, v=v)
    d["q"] /= q.square().sum(-1, keepdim=True).sqrt()
    gb = torch.stack([d["g"], d["beta"]], 1)
    d["g"], d["beta"] = gb[:, 0], gb[:, 1]
    wide = torch.zeros(T, 2 * hv, dv, device=DEV)
    want = recurrence(d, list(zip(cu[:-1], cu[1:])), list(range(len(lens))), norm=False,
                      scale=0.125)
    ws, c = engine.delta_chunk_workspace(T, len(lens), hv), ints(cu)
    torch.cuda.synchronize()
    if kind == "step":
        engine.delta_step_async(**d, out=wide[:, ::2], norm=False, scale=0.125)
    else:
        engine.delta_chunk_async(**d, out=wide[:, ::2], cu=c, ws=ws, norm=False, scale=0.125)
    engine.sync()
    check(wide[:, ::2], d["state"], want)
    assert not wide[:, 1::2].any()


@pytest.mark.parametrize("kind", ["step", "chunk"])
def test_decays_from_none_to_all(engine, kind):
    # no decay, a decay that clears the state (down to -infinity) in the middle
    # of a chunk and at its edges, beta 0 and 1, keys and queries of zeros
    gen = torch.Generator().manual_seed(23)
    lens = [1] * 6 if kind == "step" else [200]
    cu = spans_of(lens)
    T = cu[-1]
    d = inputs(gen, T, 1, 2, 64, 64, torch.float32, len(lens))
    d["g"][:] = 0
    for t, x in zip((0, 1, 3, 63, 64, 100, 127, 150, 199), (-1e4, -30.0, -1e30, -float("inf"),
                                                          -90.0, -float("inf"), -200.0, -88.0,
                                                          -5.0)):
        if t < T:
            d["g"][t] = x
    d["beta"][::3] = 1.0
    d["beta"][1::3] = 0.0
    d["k"][min(5, T - 1)] = 0
    d["q"][min(4, T - 1)] = 0
    out = torch.zeros_like(d["v"])
    want = recurrence(d, list(zip(cu[:-1], cu[1:])), list(range(len(lens))))
    ws, c = engine.delta_chunk_workspace(T, len(lens), 2), ints(cu)
    torch.cuda.synchronize()
    if kind == "step":
        engine.delta_step_async(**d, out=out)
    else:
        engine.delta_chunk_async(**d, out=out, cu=c, ws=ws)
    engine.sync()
    check(out, d["state"], want)


@pytest.mark.parametrize("kind", ["step", "chunk"])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta"])
def test_nan_stays_in_its_row(engine, kind, name):
    # and reaches what depends on it: a token's outputs from there on
    gen = torch.Generator().manual_seed(30)
    lens = [1, 1] if kind == "step" else [100, 130]
    cu = spans_of(lens)
    d = inputs(gen, cu[-1], 1, 2, 64, 64, torch.float32, 2)
    bad = 0 if kind == "step" else 70
    want = recurrence(d, list(zip(cu[:-1], cu[1:])), [0, 1])
    d[name][bad] = float("nan")
    out, ws, c = torch.zeros_like(d["v"]), engine.delta_chunk_workspace(cu[-1], 2, 2), ints(cu)
    torch.cuda.synchronize()
    if kind == "step":
        engine.delta_step_async(**d, out=out)
    else:
        engine.delta_chunk_async(**d, out=out, cu=c, ws=ws)
    engine.sync()
    assert torch.isnan(out[bad]).all()
    assert name == "q" or torch.isnan(d["state"][0]).all()
    # the chunks before it, and the other row
    fine = [t for t in range(cu[-1]) if t >= cu[1] or t < bad // 64 * 64]
    off = (out[fine].double().cpu() - want[0][fine]).abs()
    assert (off <= want[2][fine][:, None, None] + 2.0 ** -24 * want[0][fine].abs()).all()
    assert torch.isfinite(d["state"][1]).all()


def test_values_far_from_one(engine):
    # states and values of 1e6 and 1e-6: nothing is scaled to a narrower range
    for size in (1e6, 1e-6):
        gen = torch.Generator().manual_seed(24)
        d = inputs(gen, 150, 1, 2, 128, 64, torch.float32, 1)
        d["v"] *= size
        d["state"] *= size
        d["k"] *= 1e3
        d["q"] *= 1e3
        out, ws, c = torch.zeros_like(d["v"]), engine.delta_chunk_workspace(150, 1, 2), ints([0, 150])
        want = recurrence(d, [(0, 150)], [0])
        torch.cuda.synchronize()
        engine.delta_chunk_async(**d, out=out, cu=c, ws=ws)
        engine.sync()
        check(out, d["state"], want)


def test_prompt_then_steps(engine):
    # a prompt's chunks, then single tokens, equal the recurrence throughout
    gen = torch.Generator().manual_seed(25)
    d = inputs(gen, 140, 2, 4, 64, 64, torch.bfloat16, 1)
    want = recurrence(d, [(0, 140)], [0], fresh=True)
    out, ws, c = torch.zeros_like(d["v"]), engine.delta_chunk_workspace(130, 1, 4), ints([0, 130])
    head = {n: (x if n == "state" else x[:130]) for n, x in d.items()}
    torch.cuda.synchronize()
    engine.delta_chunk_async(**head, out=out[:130], cu=c, ws=ws, fresh=True)
    for t in range(130, 140):
        one = {n: (x if n == "state" else x[t:t + 1]) for n, x in d.items()}
        engine.delta_step_async(**one, out=out[t:t + 1])
    engine.sync()
    check(out, d["state"], want)


@pytest.mark.parametrize("kind", ["step", "chunk"])
@pytest.mark.parametrize("slots", [[2, 0, 2], [0, 3, 1], [0, 2 ** 31 - 1, 2]])
def test_bad_slots_are_reported(engine, kind, slots):
    gen = torch.Generator().manual_seed(26)
    lens = [1, 1, 1] if kind == "step" else [40, 70, 5]
    cu = spans_of(lens)
    d = inputs(gen, cu[-1], 1, 2, 64, 32, torch.float32, 3)
    good = [s if s < 3 and s not in slots[:i] else -1 for i, s in enumerate(slots)]
    want = recurrence(d, list(zip(cu[:-1], cu[1:])), good)
    out, ws = torch.ones_like(d["v"]), engine.delta_chunk_workspace(cu[-1], 3, 2)
    sl, c = ints(slots), ints(cu)
    torch.cuda.synchronize()
    if kind == "step":
        engine.delta_step_async(**d, out=out, slots=sl)
    else:
        engine.delta_chunk_async(**d, out=out, cu=c, ws=ws, slots=sl)
    with pytest.raises(AssertionError, match="state slot"):
        engine.sync()
    check(out, d["state"], want)


@pytest.mark.parametrize("cu", [[0, 50, 40, 90], [0, 30, 60, 120], [-4, 30, 60, 90],
                                [0, 2 ** 31 - 1, 60, 90]])
def test_bad_bounds_are_reported(engine, cu):
    gen = torch.Generator().manual_seed(27)
    d = inputs(gen, 100, 1, 1, 64, 16, torch.float32, 3)
    state = d["state"].clone()
    out, ws, c = torch.ones_like(d["v"]), engine.delta_chunk_workspace(100, 3, 1), ints(cu)
    torch.cuda.synchronize()
    engine.delta_chunk_async(**d, out=out, cu=c, ws=ws)
    with pytest.raises(AssertionError, match="bounds"):
        engine.sync()
    assert (out == 1).all() and torch.equal(d["state"], state)   # nothing was run


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_contexts_at_once(engine, dtype):
    # prompts and single tokens on two streams, each with states and workspace
    # of its own: what each gives alone, bit for bit
    from fable5_llm_amd.engine import Context
    gen = torch.Generator().manual_seed(31)
    cu = spans_of([200, 333, 64])
    jobs = []
    with Context(0) as other:
        for ctx in (engine, other):
            d = inputs(gen, cu[-1], 2, 4, 128, 128, dtype, 3)
            one = {n: (x if n == "state" else x[:3]) for n, x in d.items()}
            jobs.append((ctx, d, one, torch.zeros_like(d["v"]), torch.zeros_like(one["v"]),
                         ctx.delta_chunk_workspace(cu[-1], 3, 4), ints(cu), d["state"].clone()))

        def work(ctx, d, one, out, o1, ws, c, first):
            ctx.delta_chunk_async(**d, out=out, cu=c, ws=ws)
            ctx.delta_step_async(**one, out=o1)

        torch.cuda.synchronize()
        want = []
        for job in jobs:
            for _ in range(4):
                work(*job)
            job[0].sync()
            want.append([x.clone() for x in (job[3], job[4], job[1]["state"])])
            job[1]["state"].copy_(job[-1])
        torch.cuda.synchronize()
        for _ in range(4):
            for job in jobs:
                work(*job)
        for job, w in zip(jobs, want):
            job[0].sync()
            assert all(torch.equal(a, b) for a, b in zip((job[3], job[4], job[1]["state"]), w))


def test_captured_step_replays(engine):
    gen = torch.Generator().manual_seed(28)
    d = inputs(gen, 70, 2, 4, 128, 128, torch.bfloat16, 2)
    first = d["state"].clone()
    out, o1 = torch.zeros_like(d["v"]), torch.zeros_like(d["v"][:2])
    ws, c, sl = engine.delta_chunk_workspace(70, 2, 4), ints([0, 33, 70]), ints([1, 0])
    one = {n: (x if n == "state" else x[:2]) for n, x in d.items()}
    torch.cuda.synchronize()

    def work():
        engine.delta_chunk_async(**d, out=out, cu=c, ws=ws, slots=sl)
        engine.delta_step_async(**one, out=o1, slots=sl)

    work()
    engine.sync()
    want = [t.clone() for t in (out, o1, d["state"])]
    d["state"].copy_(first)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(g, stream=side):
            engine.set_stream(side)
            work()
    finally:
        engine.set_stream(None)
    for _ in range(3):
        d["state"].copy_(first)
        out.zero_()
        o1.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, o1, d["state"]), want))


def test_wrong_tensors_are_refused(engine):
    gen = torch.Generator().manual_seed(29)
    d = inputs(gen, 3, 1, 2, 64, 32, torch.float32, 3)
    out, ws, c = torch.zeros_like(d["v"]), engine.delta_chunk_workspace(3, 1, 2), ints([0, 3])
    for kw in (dict(q=d["q"].half()), dict(k=d["k"][:, :, :32]), dict(v=d["v"][:2]),
               dict(g=d["g"].double()), dict(beta=d["beta"][:, :1]), dict(state=d["state"].half()),
               dict(state=d["state"].transpose(2, 3)), dict(out=out.half()), dict(q=d["q"].cpu()),
               dict(slots=ints([0, 1])), dict(slots=ints([0, 1, 2]).long()),
               dict(state=d["state"][:2]), dict(frac=77), dict(q=d["q"][0], k=d["k"][0])):
        with pytest.raises(ValueError):
            engine.delta_step_async(**{**d, "out": out, **kw})
            print("not refused:", kw.keys())
    for kw in (dict(cu=c.long()), dict(cu=c[:0]), dict(cu=ints([[0, 3]])), dict(cu=c.cpu()),
               dict(slots=ints([0, 1]))):
        with pytest.raises((ValueError, IndexError)):
            engine.delta_chunk_async(**{**d, "out": out, "cu": c, "ws": ws, **kw})
    engine.sync()
