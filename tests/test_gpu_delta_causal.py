"""An infinity or a NaN among a prompt's inputs reaches no token before it, no other
row, head or (from v) column: all of these bit for bit as without it, wherever in a
chunk of 64 it stands; from its token on, its head's outputs and state are NaN."""
import pytest
import torch

import test_gpu_delta as D
from test_gpu_delta import DEV, ints

pytestmark = pytest.mark.gpu
LENS = [100, 150]


def run(engine, d, ws, c, fresh=False):
    out = torch.full_like(d["v"], 7)
    e = {n: t.clone() for n, t in d.items()}
    torch.cuda.synchronize()
    engine.delta_chunk_async(**e, out=out, cu=c, ws=ws, fresh=fresh)
    engine.sync()
    return out, e["state"]


@pytest.mark.parametrize("dtype,dk", [(torch.float32, 64), (torch.bfloat16, 64), (torch.float16, 64),
                                      (torch.float32, 128), (torch.bfloat16, 128),
                                      (torch.float16, 128)])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta"])
def test_nothing_reaches_an_earlier_token(engine, dtype, dk, name):
    gen = torch.Generator().manual_seed(50)
    cu = D.spans_of(LENS)
    hk, hv, dv = 2, 4, 32
    d = D.inputs(gen, cu[-1], hk, hv, dk, dv, dtype, 2)
    ws, c = engine.delta_chunk_workspace(cu[-1], 2, hv), ints(cu)
    ws.fill_(0xFF)
    out, state = run(engine, d, ws, c)
    assert torch.isfinite(out).all() and torch.isfinite(state).all()
    for n, at in enumerate([0, 1, 15, 16, 31, 32, 45, 47, 48, 63, 64, 95, 99]):
        value = [float("nan"), float("inf"), -float("inf")][n % 3]
        if name == "g" and value < 0:
            value = float("inf")                        # a g of -infinity clears the state
        t, head = cu[1] * (n % 2) + at, n % (hk if name in "qk" else hv)
        bad = {k: x.clone() for k, x in d.items()}
        if name in "qk":
            bad[name][t, head, n % dk] = value
            mine = [h for h in range(hv) if h // (hv // hk) == head]
        else:
            mine = [head]
            if name == "v":
                bad[name][t, head, 5] = value
            else:
                bad[name][t, head] = value
        got, after = run(engine, bad, ws, c)
        row = n % 2
        hit = torch.zeros_like(out, dtype=torch.bool)   # what may not be as before
        hit_s = torch.zeros_like(state, dtype=torch.bool)
        cols = slice(5, 6) if name == "v" else slice(None)
        for h in mine:
            hit[t:(t + 1 if name == "q" else cu[row + 1]), h, cols] = True
            if name != "q":
                hit_s[row, h, :, cols] = True
        assert torch.equal(torch.where(hit, 0, got), torch.where(hit, 0, out)), (n, at)
        assert torch.equal(torch.where(hit_s, 0, after), torch.where(hit_s, 0, state)), (n, at)
        assert not torch.isfinite(got[hit]).any() and torch.isnan(after[hit_s]).all(), (n, at)


def test_several_in_a_chunk(engine):
    # each column and head from its own first one on; a row whose every token is
    # one; the chunk's last tokens; and the next call on the same workspace clean
    gen = torch.Generator().manual_seed(51)
    cu = D.spans_of(LENS)
    d = D.inputs(gen, cu[-1], 1, 2, 64, 32, torch.float32, 2)
    ws, c = engine.delta_chunk_workspace(cu[-1], 2, 2), ints(cu)
    out, state = run(engine, d, ws, c)
    bad = {k: x.clone() for k, x in d.items()}
    first = torch.full((2, 32), LENS[0])
    for col, t in ((0, 99), (1, 64), (2, 63), (3, 20), (3, 10), (4, 70), (4, 71), (31, 0)):
        bad["v"][t, 0, col] = float("nan")
        first[0, col] = min(int(first[0, col]), t)
    bad["beta"][80, 1] = float("inf")
    bad["g"][37, 1] = float("nan")
    first[1] = 37
    bad["v"][cu[1]:] = float("inf")
    got, after = run(engine, bad, ws, c)
    at = torch.arange(LENS[0])[:, None, None].to(DEV)
    hit = torch.cat([at >= first.to(DEV), torch.ones(LENS[1], 2, 32, dtype=torch.bool, device=DEV)])
    assert torch.equal(torch.where(hit, 0, got), torch.where(hit, 0, out))
    assert torch.isnan(got[hit]).all()
    gone = torch.stack([(first < LENS[0]).to(DEV), torch.ones(2, 32, dtype=torch.bool, device=DEV)])
    gone = gone[:, :, None].expand_as(state)
    assert torch.equal(torch.where(gone, 0, after), torch.where(gone, 0, state))
    assert torch.isnan(after[gone]).all()
    again, s2 = run(engine, d, ws, c)
    assert torch.equal(again, out) and torch.equal(s2, state)


def test_a_state_that_is_not_finite(engine):
    # reaches its own columns alone; a fresh prompt does not read it
    gen = torch.Generator().manual_seed(52)
    cu = D.spans_of(LENS)
    d = D.inputs(gen, cu[-1], 1, 2, 128, 32, torch.bfloat16, 2)
    ws, c = engine.delta_chunk_workspace(cu[-1], 2, 2), ints(cu)
    out, state = run(engine, d, ws, c)
    fresh = run(engine, d, ws, c, fresh=True)
    d["state"][1, 0, 77, 3] = float("nan")
    got, after = run(engine, d, ws, c)
    assert torch.isnan(got[cu[1]:, 0, 3]).all() and torch.isnan(after[1, 0, :, 3]).all()
    got[cu[1]:, 0, 3], out[cu[1]:, 0, 3], after[1, 0, :, 3], state[1, 0, :, 3] = 0, 0, 0, 0
    assert torch.equal(got, out) and torch.equal(after, state)
    assert all(torch.equal(a, b) for a, b in zip(run(engine, d, ws, c, fresh=True), fresh))
