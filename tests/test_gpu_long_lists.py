"""Lists of many entries: right, and in a time that grows with the list and not
with its square (the bounds stand a factor of 4 from the one and at least as much
from the other)."""
import pytest
import torch

from fable5_llm_amd.engine import PagedKV

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def seconds(engine, call, restore):
    """The fastest of a few calls, alone on the GPU."""
    best = float("inf")
    side = torch.cuda.Stream()
    engine.set_stream(side)
    try:
        for _ in range(4):
            restore()
            torch.cuda.synchronize()
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            with torch.cuda.stream(side):
                a.record()
                call()
                b.record()
            engine.sync()
            best = min(best, a.elapsed_time(b) * 1e-3)
    finally:
        engine.set_stream(None)
    return best


def test_free(engine):
    times = {}
    for n in (1 << 16, 1 << 20):
        half = n // 2                                     # each listed twice, at random places
        kv = PagedKV.empty(engine, half, 1, 1, 16, 64, half, 1, torch.bfloat16)
        gen = torch.Generator().manual_seed(n)
        order = torch.randperm(n, generator=gen)
        seqs = (order % half).to(torch.int32).to(DEV)
        table = torch.randperm(half, generator=gen).to(torch.int32).to(DEV)[:, None]

        def restore():
            kv.tables.copy_(table)
            kv.lens.fill_(7)
            kv.refs.fill_(1)

        times[n] = seconds(engine, lambda: kv.free_async(seqs), restore)
        assert not kv.lens.any() and not kv.refs.any()
    assert times[1 << 20] < 64 * times[1 << 16], times


def prompts(gen, lens, dtype, dk=64, dv=16, slots=None):
    """A call's arguments, one head, and its workspace's stand-ins."""
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32)
    T, rows = int(cu[-1]), len(lens)
    x = dict(q=torch.randn(T, 1, dk, generator=gen), k=torch.randn(T, 1, dk, generator=gen),
             v=torch.randn(T, 1, dv, generator=gen))
    d = {n: t.to(dtype).to(DEV) for n, t in x.items()}
    d["g"] = -torch.rand(T, 1, generator=gen).to(DEV)
    d["beta"] = torch.rand(T, 1, generator=gen).to(DEV)
    d["state"] = torch.randn(slots or rows, 1, dk, dv, generator=gen).to(DEV)
    return d, cu.to(DEV)


def token(d, S, t):
    """One token t[i] of each row through its state S[i], in 64 bits."""
    q, k, v = (d[n][t, 0].double() for n in "qkv")
    q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    S = S * d["g"][t, 0].double().exp()[:, None, None]
    u = d["beta"][t, 0].double()[:, None] * (v - (k[:, :, None] * S).sum(1))
    S = S + k[:, :, None] * u[:, None]
    return S, (q[:, :, None] * S).sum(1) / 8


@pytest.mark.parametrize("rows", [255, 256, 257, 700, 70001])
def test_prompts_of_many_rows(engine, rows):
    # rows of no, one or two tokens: a chunk's row is found among all of them.
    # Two tokens of 64 terms: 8 sqrt(66) 2^-24 of the largest state, 8
    gen = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, 3, (rows,), generator=gen)
    d, cu = prompts(gen, lens, torch.float32)
    slots = torch.randperm(rows, generator=gen)
    slots[rows // 3] = -1
    first = d["state"][:, 0].double()
    T = int(cu[-1])
    out = torch.full_like(d["v"], 3)
    ws, sl = engine.delta_chunk_workspace(T, rows, 1, hk=1, dk=64), slots.to(torch.int32).to(DEV)
    ws.fill_(0xFF)
    torch.cuda.synchronize()
    engine.delta_chunk_async(**d, out=out, cu=cu, ws=ws, slots=sl)
    engine.sync()
    want, w_out = first.clone(), torch.zeros_like(out, dtype=torch.float64)
    start = cu[:-1].long().cpu()
    for n in (1, 2):
        at = torch.nonzero((lens >= n) & (slots >= 0))[:, 0]
        t, s = (start[at] + n - 1).to(DEV), slots[at].to(DEV)
        want[s], w_out[t, 0] = token(d, want[s], t)
    assert want.abs().max() < 8
    tol = 8 * 66 ** 0.5 * 2.0 ** -24 * 8
    assert (d["state"][:, 0].double() - want).abs().max() <= tol
    assert (out.double() - w_out).abs().max() <= tol


@pytest.mark.parametrize("at", [0, 300, 69999])
def test_a_bad_bound_among_many(engine, at):
    gen = torch.Generator().manual_seed(1)
    rows = 70000
    d, cu = prompts(gen, torch.ones(rows, dtype=torch.int64), torch.bfloat16)
    cu[at + 1] = cu[at] - 1 if at else -1
    first = d["state"].clone()
    out, ws = torch.ones_like(d["v"]), engine.delta_chunk_workspace(rows, rows, 1, hk=1, dk=64)
    torch.cuda.synchronize()
    engine.delta_chunk_async(**d, out=out, cu=cu, ws=ws)
    with pytest.raises(AssertionError, match="bounds"):
        engine.sync()
    assert (out == 1).all() and torch.equal(d["state"], first)


def test_a_slot_named_by_far_rows(engine):
    gen = torch.Generator().manual_seed(2)
    rows, again = 70000, [(600, 69990), (0, 255), (0, 256), (255, 257)]
    d, cu = prompts(gen, torch.ones(rows, dtype=torch.int64), torch.float32)
    slots = torch.randperm(rows, generator=gen)
    free = slots[[b for _, b in again]].to(DEV)          # of the later rows: left alone
    for a, b in again:
        slots[b] = slots[a]
    first = d["state"].clone()
    out = torch.full_like(d["v"], 3)
    ws, sl = engine.delta_chunk_workspace(rows, rows, 1, hk=1, dk=64), slots.to(torch.int32).to(DEV)
    torch.cuda.synchronize()
    engine.delta_chunk_async(**d, out=out, cu=cu, ws=ws, slots=sl)
    with pytest.raises(AssertionError, match="state slot"):
        engine.sync()
    assert torch.equal(d["state"][free], first[free])
    later = torch.tensor([b for _, b in again], device=DEV)
    assert not out[later].any()
    out[later] = 3
    at = torch.tensor([600, 0], device=DEV)              # the first ones that name theirs
    S, o = token(d, first[slots[at.cpu()].to(DEV), 0].double(), at)
    tol = 8 * 66 ** 0.5 * 2.0 ** -24 * 8
    assert (d["state"][slots[at.cpu()].to(DEV), 0].double() - S).abs().max() <= tol
    assert (out[at, 0].double() - o).abs().max() <= tol
    assert (out != 0).any(2).all()


def test_prompts_in_proportion(engine):
    times = {}
    for rows in (1 << 13, 1 << 18):
        gen = torch.Generator().manual_seed(3)
        d, cu = prompts(gen, torch.ones(rows, dtype=torch.int64), torch.bfloat16)
        out, ws = torch.ones_like(d["v"]), engine.delta_chunk_workspace(rows, rows, 1, hk=1, dk=64,
                                                                        dtype=torch.bfloat16)
        sl = torch.randperm(rows, generator=gen).to(torch.int32).to(DEV)
        times[rows] = seconds(engine, lambda: engine.delta_chunk_async(
            **d, out=out, cu=cu, ws=ws, slots=sl), lambda: None)
        del ws
        torch.cuda.empty_cache()
    print(times)
    assert times[1 << 18] < 4 * 32 * times[1 << 13], times


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,dv", [(16383, 256), (16400, 256), (33000, 80), (70001, 16)])
def test_a_token_of_many_rows(engine, dtype, rows, dv):
    # slots in any order, padded rows, rows that name an earlier one's slot or none
    # of the states, near and far; out in every other head of a wider row.  One
    # token of 64 terms: 8 sqrt(65) 2^-24 of the largest state, 8, and half a step
    gen = torch.Generator().manual_seed(rows)
    d, _ = prompts(gen, torch.ones(rows, dtype=torch.int64), dtype, dv=dv)
    slots = torch.randperm(rows, generator=gen)
    slots[[5, 300, rows - 2]] = -1
    slots[rows - 1] = slots[3]
    slots[256], slots[513], slots[1] = slots[255], slots[2], slots[0]
    slots[700] = rows
    good = slots.clone()
    good[[rows - 1, 256, 513, 1, 700]] = -1
    first = d["state"].clone()
    wide = torch.full((rows, 2, dv), 3.0, device=DEV).to(dtype)
    sl = slots.to(torch.int32).to(DEV)
    torch.cuda.synchronize()
    engine.delta_step_async(**d, out=wide[:, 1:], slots=sl)
    with pytest.raises(AssertionError, match="state slot"):
        engine.sync()
    at = torch.nonzero(good >= 0)[:, 0].to(DEV)
    s = good[good >= 0].to(DEV)
    want, w_out = first[:, 0].double(), torch.zeros(rows, dv, device=DEV, dtype=torch.float64)
    want[s], w_out[at] = token(d, want[s], at)
    assert want.abs().max() < 8
    tol = 8 * 65 ** 0.5 * 2.0 ** -24 * 8
    assert (d["state"][:, 0].double() - want).abs().max() <= tol
    half = torch.finfo(dtype).eps / 2
    assert ((wide[:, 1].double() - w_out).abs() <= tol + half * w_out.abs()).all()
    assert (wide[:, 0] == 3).all()


def test_tokens_in_proportion(engine):
    # 2^20 rows of four heads: the states alone against the states and the slots
    # (8.5 ms against 33 where the slots are checked once, 567 where each row's
    # workgroups look through the rows before: 16 times stands between)
    rows, hv = 1 << 20, 4
    gen = torch.Generator(device=DEV).manual_seed(3)
    act = lambda *shape: torch.randn(*shape, generator=gen, device=DEV).bfloat16()   # noqa: E731
    d = dict(q=act(rows, 1, 64), k=act(rows, 1, 64), v=act(rows, hv, 16),
             g=-torch.rand(rows, hv, generator=gen, device=DEV),
             beta=torch.rand(rows, hv, generator=gen, device=DEV),
             state=torch.randn(rows, hv, 64, 16, generator=gen, device=DEV))
    out = torch.zeros_like(d["v"])
    sl = torch.randperm(rows, generator=gen, device=DEV).to(torch.int32)
    alone, checked = (seconds(engine, lambda: engine.delta_step_async(**d, out=out, slots=s),
                              lambda: None) for s in (None, sl))
    assert checked < 16 * alone, (alone, checked)
