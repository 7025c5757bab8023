"""What stands between the sites of a decode step, as cases that can be timed
and checked: the mixers of the 9B shape's layers and the state they keep.

Kinds of case, and what each stands for:

  attend   one `PagedKV.attend_async`: a layer's attention of one new token per
           row over a paged key-value cache
  append   one `PagedKV.append_async`: a layer's keys and values of new tokens
           written into their pages
  branch   `PagedKV.fork_async` then `PagedKV.free_async`: children that share
           their parents' pages (a beam's continuations, a speculative branch)
           and are dropped again
  compact  `PagedKV.compact_async`: a pool's used pages moved to its start
  step     one `Context.delta_step_async`: a layer's gated delta rule for one
           token of each sequence
  chunk    one `Context.delta_chunk_async`: the same for the tokens of whole
           prompts

With `own` false the same results come from elementary torch operations in 32
bits.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6                           # of the delta rule's norms of q and k


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one sequence of the 9B shape's attention layers (16 query heads of 256,
        # 4 key-value heads) at the reference's context of 511
        dict(name="attend_one", kind="attend", dtype="bf16", rows=1, hq=16, hkv=4, d=256,
             page=16, max_len=511, ragged=False),
        # a serving batch of uneven lengths, one row of it still empty
        dict(name="attend_batch", kind="attend", dtype="f16", rows=48, hq=32, hkv=8, d=128,
             page=32, max_len=4099, ragged=True),
        # a cache in full precision, every query head with its own keys
        dict(name="attend_f32", kind="attend", dtype="f32", rows=7, hq=8, hkv=8, d=64,
             page=16, max_len=2000, ragged=True),
        # two long contexts, where few rows have to fill the chip
        dict(name="attend_long", kind="attend", dtype="bf16", rows=2, hq=16, hkv=4, d=256,
             page=64, max_len=131072, ragged=False),
        # a decode batch's new token, and a prompt's tokens of several sequences
        dict(name="append_decode", kind="append", dtype="bf16", rows=61, tokens=61, hkv=4, d=256,
             page=16, max_len=900),
        dict(name="append_prompt", kind="append", dtype="f16", rows=5, tokens=16381, hkv=8,
             d=128, page=32, max_len=6000),
        # eight beams with four continuations each, all 8 layers of the 9B shape
        dict(name="branch_beams", kind="branch", dtype="bf16", layers=8, hkv=4, d=256, page=16,
             rows=8, children=32, max_len=1500),
        # a pool of 1 GiB three fifths of which are in use, scattered
        dict(name="compact_pool", kind="compact", dtype="bf16", layers=8, hkv=4, d=256, page=16,
             rows=24, pages=2048, max_len=1600),
        # one sequence, and a batch, through a DeltaNet layer of the 9B shape
        dict(name="step_one", kind="step", dtype="bf16", rows=1, hk=16, hv=32, dk=128, dv=128),
        dict(name="step_batch", kind="step", dtype="f16", rows=125, hk=16, hv=32, dk=128,
             dv=128),
        # prompts of uneven lengths in full precision; one long prompt
        dict(name="chunk_ragged", kind="chunk", dtype="f32", rows=6, tokens=1531, hk=4, hv=8,
             dk=64, dv=128),
        dict(name="chunk_long", kind="chunk", dtype="bf16", rows=1, tokens=8192, hk=16, hv=32,
             dk=128, dv=128),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "branch", "compact", "step",
                       "step", "chunk", "chunk"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    page = rng.choice([16, 32, 64])
    if kind == "attend":
        hkv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        hq = hkv * rng.choice([1, 2, 3, 4, 7, 8, 16])
        rows = _log(rng, 1, 200)
        most = (1 << 28) // (rows * hkv * d)     # keys of a cache of at most 1 GiB
        return dict(kind=kind, dtype=dtype, rows=rows, hq=hq, hkv=hkv, d=d, page=page,
                    max_len=_log(rng, 1, max(1, min(131072, most // 2))),
                    ragged=rng.random() < 0.7)
    if kind == "append":
        rows = _log(rng, 1, 64)
        return dict(kind=kind, dtype=dtype, rows=rows, tokens=_log(rng, rows, 16000),
                    hkv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128, 256]), page=page,
                    max_len=16100 // rows + _log(rng, 1, 900))
    if kind == "branch":
        rows = _log(rng, 1, 16)
        return dict(kind=kind, dtype=dtype, layers=_log(rng, 1, 8), hkv=rng.choice([1, 2, 4]),
                    d=rng.choice([64, 128, 256]), page=page, rows=rows,
                    children=_log(rng, 1, 32), max_len=_log(rng, 1, 1500))
    if kind == "compact":
        rows, pages = _log(rng, 1, 40), _log(rng, 40, 700)
        return dict(kind=kind, dtype=dtype, layers=_log(rng, 1, 4), hkv=rng.choice([1, 2, 4]),
                    d=rng.choice([64, 128, 256]), page=page, rows=rows, pages=pages,
                    max_len=page * max(1, pages * 3 // 4 // rows))
    hk = rng.choice([1, 2, 4, 8, 16])
    hv, dk = hk * rng.choice([1, 2, 3]), rng.choice([64, 128])
    dv = rng.choice([64, 128, 16 * rng.randint(1, 8)])
    if kind == "step":
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 80), hk=hk, hv=hv, dk=dk, dv=dv)
    rows = _log(rng, 1, 20)
    return dict(kind=kind, dtype=dtype, rows=rows, tokens=_log(rng, rows, 5000), hk=min(hk, 8),
                hv=min(hk, 8) * (hv // hk), dk=dk, dv=dv)


def _lens(case):
    """Tokens of each sequence (a case's lengths are part of it, not of the seed)."""
    rows, top = case["rows"], case["max_len"]
    rng = random.Random("%d of at most %d" % (rows, top))
    if case["kind"] == "attend" and not case["ragged"]:
        return [top - (i * 37) % max(1, min(top, 1000)) for i in range(rows)]
    lens = [_log(rng, 1, top) for _ in range(rows)]
    if case["kind"] == "compact":     # a pool in use to about three fifths
        lens = [max(1, top - rng.randrange(1 + top // 2)) for _ in range(rows)]
    if case["kind"] == "attend" and rows >= 8:
        lens[rows // 2] = 0
    lens[0] = top
    return lens


def _spans(case):
    """Tokens of each prompt: `tokens` split at random places, none empty."""
    rng = random.Random("%d of %d" % (case["rows"], case["tokens"]))
    cuts = sorted(rng.sample(range(1, case["tokens"]), case["rows"] - 1)) \
        if case["rows"] > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "attend":
        n, hq, d = sum(_lens(case)), case["hq"], case["d"]
        return {"bytes": (2 * n * case["hkv"] + 2 * case["rows"] * hq) * d * e,
                "flops": 4 * n * hq * d}
    if kind == "append":
        return {"bytes": 4 * case["tokens"] * case["hkv"] * case["d"] * e, "flops": 0}
    if kind in ("branch", "compact"):
        lens, page = _lens(case), case["page"]
        token = 2 * case["layers"] * case["hkv"] * case["d"] * e
        if kind == "branch":
            lens = [lens[i % case["rows"]] for i in range(case["children"])]
            return {"bytes": sum(2 * (n % page) * token + 8 * -(-n // page) for n in lens),
                    "flops": 0}
        used = sum(-(-n // page) for n in lens)
        moved = used * (case["pages"] - used) / case["pages"]     # in the mean
        return {"bytes": 2 * moved * page * token + 8 * used, "flops": 0}
    state = case["rows"] * case["hv"] * case["dk"] * case["dv"]
    tokens = case["rows"] if kind == "step" else case["tokens"]
    io = tokens * (2 * case["hk"] * case["dk"] + 2 * case["hv"] * case["dv"]) * e
    return {"bytes": 8 * state + io + 8 * tokens * case["hv"],
            "flops": 8 * tokens * case["hv"] * case["dk"] * case["dv"]}


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", dtype=dtype, generator=gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(case, gen, lens, pages=None, extra_rows=0, layers=1):
    """A pool [pages][layers][K, V][kv heads][page][d], its sequences' pages
    scattered over it, the pages' counts of users, tables and lengths."""
    page, rows = case["page"], len(lens) + extra_rows
    held = [-(-n // page) for n in lens]
    pages = pages or sum(held) + max(4, sum(held) // 8) + extra_rows
    pool = _randn(gen, pages, layers, 2, case["hkv"], page, case["d"], dtype=DTYPE[case["dtype"]])
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    width = max(max(held), 1)
    tables = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(width, device="cuda")
    mine = torch.zeros((rows, width), dtype=torch.bool, device="cuda")
    mine[:len(lens)] = col < _ints(held)[:, None]
    tables[mine] = order[:sum(held)]
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:sum(held)].long()] = 1
    return dict(pool=pool, refs=refs, tables=tables, lens=_ints(lens + [0] * extra_rows))


_streams = {}


def _engine():
    """The engine on a stream that torch's own operations can be put on too."""
    from fable5_llm_amd import engine
    ctx = engine.default_context()
    if ctx not in _streams:
        _streams[ctx] = torch.cuda.Stream()
    ctx.set_stream(_streams[ctx])
    return ctx, _streams[ctx]


def prepare(case, seed):
    gen, kind, dt = _gen(seed), case["kind"], DTYPE[case["dtype"]]
    st = dict(case=case)
    if kind == "attend":
        st.update(_cache(case, gen, _lens(case)))
        st["q"] = _randn(gen, case["rows"], case["hq"], case["d"], dtype=dt)
        st["seqs"] = torch.randperm(case["rows"], device="cuda", generator=gen).to(torch.int32)
        st["out"] = torch.zeros_like(st["q"])
    elif kind == "append":
        lens, spans = _lens(case), _spans(case)
        st.update(_cache(case, gen, [max(a, b) for a, b in zip(lens, spans)]))
        st["k"], st["v"] = (_randn(gen, case["tokens"], case["hkv"], case["d"], dtype=dt)
                            for _ in range(2))
        # the last tokens of each sequence
        span = _ints(spans).long()
        st["seqs"] = torch.repeat_interleave(torch.arange(case["rows"], device="cuda"), span)
        first = (st["lens"].long() - span)[st["seqs"]]
        nth = torch.arange(case["tokens"], device="cuda") - (span.cumsum(0) - span)[st["seqs"]]
        st["pos"], st["seqs"] = (first + nth).to(torch.int32), st["seqs"].to(torch.int32)
    elif kind == "branch":
        st.update(_cache(case, gen, _lens(case), extra_rows=case["children"],
                         layers=case["layers"]))
        st["parents"] = _ints([i % case["rows"] for i in range(case["children"])])
        st["children"] = _ints([case["rows"] + i for i in range(case["children"])])
    elif kind == "compact":
        st.update(_cache(case, gen, _lens(case), pages=case["pages"], layers=case["layers"]))
        st["was"] = (st["refs"].clone(), st["tables"].clone())
    else:
        n, hk, hv, dk, dv = (case[k] for k in ("rows", "hk", "hv", "dk", "dv"))
        tokens = n if kind == "step" else case["tokens"]
        st["q"], st["k"] = (_randn(gen, tokens, hk, dk, dtype=dt) for _ in range(2))
        st["v"] = _randn(gen, tokens, hv, dv, dtype=dt)
        # decays from "forgets in a few tokens" to "keeps hundreds"
        st["g"] = -torch.exp(_randn(gen, tokens, hv) * 1.5 - 3.0)
        st["beta"] = torch.sigmoid(_randn(gen, tokens, hv))
        st["state"] = _randn(gen, n, hv, dk, dv) * 0.1
        st["slots"] = torch.randperm(n, device="cuda", generator=gen).to(torch.int32)
        st["out"] = torch.zeros_like(st["v"])
        if kind == "chunk":
            st["cu"] = _ints([0] + np.cumsum(_spans(case)).tolist())
    if own:      # the handles and workspaces that a program keeps
        from fable5_llm_amd import engine
        st["ctx"], st["stream"] = _engine()
        if "pool" in st:
            st["kv"] = engine.PagedKV(st["ctx"], st["pool"], st["refs"], st["tables"],
                                      st["lens"])
        if kind == "attend":
            st["ws"] = st["kv"].attend_workspace(case["rows"], case["hq"])
        if kind == "chunk":
            st["ws"] = st["ctx"].delta_chunk_workspace(case["tokens"], case["rows"], case["hv"])
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _OWN[kind](st)
    return _PLAIN[kind](st)


def _own_attend(st):
    st["kv"].attend_async(0, st["q"], st["seqs"], st["out"], st["ws"])
    return st["out"]


def _own_append(st):
    st["kv"].append_async(0, st["k"], st["v"], st["seqs"], st["pos"])
    return st["pool"]


def _own_branch(st):
    st["kv"].fork_async(st["parents"], st["children"])
    st["kv"].free_async(st["children"])
    return {k: st[k] for k in ("pool", "refs", "tables", "lens")}


def _own_compact(st):
    with torch.cuda.stream(st["stream"]):
        st["refs"].copy_(st["was"][0])
        st["tables"].copy_(st["was"][1])
    st["kv"].compact_async()
    return {k: st[k] for k in ("pool", "refs", "tables", "lens")}


def _own_step(st):
    st["ctx"].delta_step_async(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"],
                               st["out"], slots=st["slots"])
    return {"out": st["out"], "state": st["state"]}


def _own_chunk(st):
    st["ctx"].delta_chunk_async(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"],
                                st["out"], st["cu"], st["ws"], slots=st["slots"])
    return {"out": st["out"], "state": st["state"]}


_OWN = dict(attend=_own_attend, append=_own_append, branch=_own_branch, compact=_own_compact,
            step=_own_step, chunk=_own_chunk)


# ------------------------------------------------------------- plain forms
def _rows_of(pool, tables, which, n):
    """Layer 0's rows (which 0: keys, 1: values) of n tokens of each of the
    sequences that tables are of: [sequences, kv heads, n, d] in 32 bits."""
    page = pool.shape[4]
    at = tables[:, :-(-n // page)].long().clamp(min=0)
    x = pool[at, 0, which].float()                   # [sequences, pages, heads, page, d]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n]


def _plain_attend(st):
    case, seqs = st["case"], st["seqs"].long()
    hkv, hq, d, n = case["hkv"], case["hq"], case["d"], case["max_len"]
    lens, tables = st["lens"][seqs], st["tables"][seqs]
    q = st["q"].float().reshape(-1, hkv, hq // hkv, d) * (1.0 / math.sqrt(d))
    k = _rows_of(st["pool"], tables, 0, n).transpose(2, 3).contiguous()
    s = q @ k
    del k
    live = (torch.arange(n, device="cuda") < lens[:, None])[:, None, None]
    s = s.masked_fill(~live, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    o = (p @ _rows_of(st["pool"], tables, 1, n)) / torch.where(total > 0, total, 1.0)
    st["out"].copy_(o.reshape(-1, hq, d))
    return st["out"]


def _plain_append(st):
    page, pos = st["case"]["page"], st["pos"].long()
    at = st["tables"][st["seqs"].long(), pos // page].long()
    st["pool"][at, 0, 0, :, pos % page] = st["k"]
    st["pool"][at, 0, 1, :, pos % page] = st["v"]
    return st["pool"]


def _plain_branch(st):
    pool, refs, tables, lens, page = st["pool"], st["refs"], st["tables"], st["lens"], \
        st["case"]["page"]
    par, chi = st["parents"].long(), st["children"].long()
    n = lens[par].long()
    full, rest = n // page, n % page
    need = rest > 0
    free = torch.nonzero(refs == 0)[:, 0]
    new = free[(need.cumsum(0) - 1).clamp(min=0)]
    col = torch.arange(tables.shape[1], device="cuda")
    shared = col < full[:, None]
    last = (col == full[:, None]) & need[:, None]
    rows = torch.where(shared, tables[par],
                       torch.where(last, new[:, None].to(torch.int32), tables[chi]))
    old = tables[par[need], full[need]].long()
    tables[chi] = rows
    refs.index_add_(0, rows[shared].long(), torch.ones_like(rows[shared]))
    refs[new[need]] = 1
    kept = torch.arange(page, device="cuda") < rest[need][:, None]
    kept = kept[:, None, None, None, :, None]
    pool[new[need]] = torch.where(kept, pool[old], pool[new[need]])
    lens[chi] = lens[par]
    # and dropped again
    held = col < -(-lens[chi].long() // page)[:, None]
    mine = tables[chi][held].long()
    refs.index_add_(0, mine, -torch.ones_like(tables[chi][held]))
    lens[chi] = 0
    return {k: st[k] for k in ("pool", "refs", "tables", "lens")}


def _plain_compact(st):
    pool, refs, tables, page = st["pool"], st["refs"], st["tables"], st["case"]["page"]
    refs.copy_(st["was"][0])
    tables.copy_(st["was"][1])
    at = torch.arange(refs.shape[0], device="cuda")
    used = refs > 0
    count = used.sum()
    src = torch.nonzero(used & (at >= count))[:, 0]
    dst = torch.nonzero(~used & (at < count))[:, 0]
    pool[dst] = pool[src]
    to = at.to(torch.int32)
    to[src] = dst.to(torch.int32)
    held = torch.arange(tables.shape[1], device="cuda") < -(-st["lens"] // page)[:, None]
    tables.copy_(torch.where(held, to[tables.long().clamp(min=0)], tables))
    refs[dst] = refs[src]
    refs[src] = 0
    return {k: st[k] for k in ("pool", "refs", "tables", "lens")}


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)


def _plain_step(st):
    case, slots = st["case"], st["slots"].long()
    per = case["hv"] // case["hk"]
    q = _unit(st["q"].float()).repeat_interleave(per, 1) * (1.0 / math.sqrt(case["dk"]))
    k = _unit(st["k"].float()).repeat_interleave(per, 1)
    s = st["state"][slots] * torch.exp(st["g"])[..., None, None]
    u = st["beta"][..., None] * (st["v"].float() - (s * k[..., None]).sum(2))
    s = s + k[..., None] * u[..., None, :]
    st["state"][slots] = s
    st["out"].copy_((s * q[..., None]).sum(2))
    return {"out": st["out"], "state": st["state"]}


def _plain_chunk(st):
    case, slots, C = st["case"], st["slots"].long(), 64
    n, hk, hv, dk, dv = (case[k] for k in ("rows", "hk", "hv", "dk", "dv"))
    most = -(-max(_spans(case)) // C) * C
    cu = st["cu"].long()
    at = cu[:-1, None] + torch.arange(most, device="cuda")
    live = at < cu[1:, None]
    at = at.clamp(max=case["tokens"] - 1)

    def split(x):      # [tokens, heads, ...] -> [n, chunks, heads, C, ...], zeros past the end
        x = torch.where(live.view(n, most, *[1] * (x.dim() - 1)), x[at].float(), 0.0)
        return x.view(n, most // C, C, *x.shape[2:]).transpose(2, 3)

    q = split(_unit(st["q"].float()).repeat_interleave(hv // hk, 1)) * (1.0 / math.sqrt(dk))
    k = split(_unit(st["k"].float()).repeat_interleave(hv // hk, 1))
    v, g, beta = split(st["v"]), split(st["g"]), split(st["beta"])
    G = g.double().cumsum(-1)
    low = torch.ones(C, C, dtype=torch.bool, device="cuda").tril()
    decay = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], 0.0)).float() * low
    kT = k.transpose(-1, -2).contiguous()
    A = beta[..., None] * decay * (k @ kT) * low.tril(-1)
    T = torch.eye(C, device="cuda").expand(A.shape).contiguous()
    for i in range(1, C):      # (I + A) T = I, row by row
        T[..., i, :i] = -(A[..., i, None, :i] @ T[..., :i, :i])[..., 0, :]
    M = T * beta[..., None, :]
    P = decay * (q @ kT)
    rise, fall = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
    s = st["state"][slots]
    outs = []
    for c in range(most // C):
        u = M[:, c] @ (v[:, c] - rise[:, c] * (k[:, c] @ s))
        outs.append(rise[:, c] * (q[:, c] @ s) + P[:, c] @ u)
        s = rise[:, c, :, -1:] * s + kT[:, c] @ (fall[:, c] * u)
    st["state"][slots] = s
    o = torch.stack(outs, 1).transpose(2, 3).reshape(n, most, hv, dv)
    st["out"].copy_(o[live])
    return {"out": st["out"], "state": st["state"]}


_PLAIN = dict(attend=_plain_attend, append=_plain_append, branch=_plain_branch,
              compact=_plain_compact, step=_plain_step, chunk=_plain_chunk)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    kind = case["kind"]
    if kind == "attend":
        return _exact_attend(case, st)
    if kind == "append":
        flat = st["pool"].double()
        seqs, pos, tables = (st[k].cpu().numpy() for k in ("seqs", "pos", "tables"))
        pages = torch.from_numpy(tables[seqs, pos // case["page"]].astype(np.int64)).cuda()
        slot = torch.from_numpy((pos % case["page"]).astype(np.int64)).cuda()
        for which, x in ((0, st["k"]), (1, st["v"])):
            for h in range(case["hkv"]):
                flat[pages, 0, which, h, slot] = x[:, h].double()
        return flat
    if kind == "branch":
        return _exact_branch(case, st)
    if kind == "compact":
        return _exact_compact(case, st)
    return _exact_delta(case, st)


def _exact_attend(case, st):
    out = torch.zeros(case["rows"], case["hq"], case["d"], dtype=torch.float64, device="cuda")
    per = case["hq"] // case["hkv"]
    lens, seqs = st["lens"].tolist(), st["seqs"].tolist()
    for i, s in enumerate(seqs):
        n = lens[s]
        pages = st["tables"][s, :-(-n // case["page"])].long()
        for h in range(case["hkv"] if n else 0):
            k, v = (st["pool"][pages, 0, w, h].double().reshape(-1, case["d"])[:n]
                    for w in (0, 1))
            x = st["q"][i, h * per:(h + 1) * per].double()
            a = torch.softmax((k @ x.T).T / math.sqrt(case["d"]), -1)
            out[i, h * per:(h + 1) * per] = a @ v
    return out


def _host(st):
    return [st[k].cpu().numpy().copy() for k in ("refs", "tables", "lens")]


def _exact_branch(case, st):
    refs, tables, lens = _host(st)
    pool = st["pool"].double()
    page = case["page"]
    grown = []
    for p, c in zip(st["parents"].tolist(), st["children"].tolist()):
        full, rest = divmod(int(lens[p]), page)
        for j in range(full):
            tables[c, j] = tables[p, j]
            refs[tables[p, j]] += 1
        if rest:
            grown.append((p, c, full, rest))
    for p, c, full, rest in grown:
        new = int(np.flatnonzero(refs == 0)[0])
        refs[new], tables[c, full] = 1, new
        pool[new, ..., :rest, :] = pool[int(tables[p, full]), ..., :rest, :]
    for p, c in zip(st["parents"].tolist(), st["children"].tolist()):
        for j in range(-(-int(lens[p]) // page)):
            refs[tables[c, j]] -= 1
    return dict(pool=pool, refs=refs, tables=tables, lens=lens)


def _exact_compact(case, st):
    refs, tables, lens = _host(st)
    pool = st["pool"].double()
    used, to = int((refs > 0).sum()), {}
    holes = [p for p in range(used) if refs[p] == 0]
    for p in range(used, len(refs)):
        if refs[p]:
            to[p] = holes.pop(0)
    for src, dst in to.items():
        pool[dst] = pool[src]
        refs[dst], refs[src] = refs[src], 0
    for s in range(tables.shape[0]):
        for j in range(-(-int(lens[s]) // case["page"])):
            tables[s, j] = to.get(int(tables[s, j]), tables[s, j])
    return dict(pool=pool, refs=refs, tables=tables, lens=lens)


def _exact_delta(case, st):
    """Token by token: S <- e^g S; S <- S + k (beta (v - S^T k))^T; o = S^T q."""
    if case["kind"] == "step":
        spans = [1] * case["rows"]
    else:
        spans = _spans(case)
    start = np.concatenate([[0], np.cumsum(spans)[:-1]])
    order = np.argsort(spans)[::-1].copy()         # the longest first: a prefix is alive
    q, k, v, g, beta = (st[n].double() for n in ("q", "k", "v", "g", "beta"))
    q, k = (x / (x.square().sum(-1, keepdim=True) + EPS).sqrt() for x in (q, k))
    per = case["hv"] // case["hk"]
    state = st["state"].double()
    slot = st["slots"].long()[torch.from_numpy(order).cuda()]
    S, out = state[slot], torch.zeros_like(v)
    lens = np.array(spans)[order]
    for t in range(int(lens[0])):
        n = int((lens > t).sum())
        at = torch.from_numpy(start[order][:n] + t).cuda()
        kt, qt = (x[at].repeat_interleave(per, 1)[..., None, :] for x in (k, q))
        live = S[:n].mul_(g[at].exp()[..., None, None])
        u = beta[at][..., None, None] * (v[at][:, :, None] - kt @ live)
        live.add_(kt.transpose(-1, -2) * u)
        out[at] = (qt @ live)[:, :, 0] / math.sqrt(case["dk"])
    state[slot] = S
    return dict(out=out, state=state)
