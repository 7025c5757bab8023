"""What a chunk of a prompt goes through besides a step's sites, as cases that
can be timed and checked: where its tokens lie, their positions, their attention
over the paged cache, and what the head's logits say about them.

Kinds of case, and what each stands for:

  map      one `PagedKV.map_async`: from the requests' counts of new tokens, each
           token's sequence, position and slot of the cache, and the attention's
           pieces of work; once a step, for all layers
  append   one `PagedKV.append_rotary_async`: a layer's queries and keys
           normalised and rotated to their positions, keys and values written
           into their slots
  rotary   one `Context.rotary_async`: the same for queries and keys without a
           cache
  chunk    one `PagedKV.attend_chunk_async`: attention of the new tokens of each
           sequence over all that the sequence holds up to them
  logprobs one `Context.logprobs_async`: log probabilities of given tokens, the
           entropy of each row and its best alternatives

With `own` false the same results come from elementary torch operations in 32
bits (angles in 64).
"""
import math
import random

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
         "i32": torch.int32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "i32": 4}
EPS = 1e-6                           # of the heads' norms


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode batch's step, and a step of prompts of uneven lengths
        dict(name="map_decode", kind="map", rows=61, tokens=61, page=16, max_len=900),
        dict(name="map_prompts", kind="map", rows=300, tokens=16381, page=32, max_len=6000),
        # one token of the 9B shape's attention layers (16 query heads of 256, a
        # quarter of each rotated, 4 key-value heads) at the reference's context of
        # 511; a prompt through the same layer
        dict(name="append_one", kind="append", dtype="bf16", rows=1, tokens=1, hq=16, hkv=4,
             d=256, rot=64, halves=True, norm=True, scaled=False, page=16, max_len=511),
        dict(name="append_prompt", kind="append", dtype="bf16", rows=3, tokens=8191, hq=16,
             hkv=4, d=256, rot=64, halves=True, norm=True, scaled=False, page=64, max_len=9000),
        # full precision, pairs side by side, positions far out in a stretched context
        dict(name="rotary_far", kind="rotary", dtype="f32", tokens=777, hq=12, hkv=3, d=128,
             rot=128, halves=False, norm=False, scaled=True, max_pos=1000000),
        # the last part of a prompt at the reference's context
        dict(name="chunk_one", kind="chunk", dtype="bf16", rows=1, tokens=17, hq=16, hkv=4,
             d=256, page=16, max_len=511),
        # a serving step: prompts' chunks of uneven lengths, one of them padding
        dict(name="chunk_batch", kind="chunk", dtype="f16", rows=13, tokens=3001, hq=32, hkv=8,
             d=128, page=32, max_len=4099),
        # full precision, every query head with its own keys
        dict(name="chunk_f32", kind="chunk", dtype="f32", rows=5, tokens=1000, hq=8, hkv=8,
             d=64, page=16, max_len=2000),
        # a whole prompt at once
        dict(name="chunk_prompt", kind="chunk", dtype="bf16", rows=1, tokens=8192, hq=16, hkv=4,
             d=256, page=64, max_len=8192),
        # a question about a long document, where few tokens have to fill the chip
        dict(name="chunk_long", kind="chunk", dtype="bf16", rows=1, tokens=100, hq=32, hkv=8,
             d=128, page=64, max_len=131072),
        # the head's own 248,320 sums for one token; a prompt's tokens scored at once
        dict(name="logprobs_one", kind="logprobs", dtype="i32", rows=1, vocab=248320, k=20),
        dict(name="logprobs_prompt", kind="logprobs", dtype="bf16", rows=509, vocab=248320, k=5),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v))))


def draw(rng):
    kind = rng.choice(["map", "append", "append", "rotary", "chunk", "chunk", "chunk", "chunk",
                       "logprobs", "logprobs"])
    dtype, page = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([16, 32, 64])
    if kind == "map":
        rows = _log(rng, 1, 2000)
        return dict(kind=kind, rows=rows, tokens=_log(rng, rows, 16000), page=page,
                    max_len=_log(rng, 1, 20000))
    hkv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    hq = hkv * rng.choice([1, 2, 3, 4, 7, 8, 16])
    if kind in ("append", "rotary"):
        case = dict(kind=kind, dtype=dtype, hq=min(hq, 32 // hkv * hkv), hkv=hkv, d=d,
                    rot=16 * rng.randint(1, d // 16), halves=rng.random() < 0.6,
                    norm=rng.random() < 0.5, scaled=rng.random() < 0.4)
        if kind == "rotary":
            case.update(d=16 * rng.randint(1, 16), tokens=_log(rng, 1, 8000),
                        max_pos=_log(rng, 2, 2000000))
            case["rot"] = 16 * rng.randint(1, case["d"] // 16)
            return case
        rows = _log(rng, 1, 64)
        return dict(case, rows=rows, tokens=_log(rng, rows, 8000), page=page,
                    max_len=_log(rng, 1, 16000 // rows))
    if kind == "chunk":
        rows = _log(rng, 1, 40)
        case = dict(kind=kind, dtype=dtype, rows=rows, hq=hq, hkv=hkv, d=d, page=page,
                    tokens=_log(rng, rows, 16000),
                    max_len=_log(rng, 1, min(131072, (1 << 28) // (rows * hkv * d *
                                                                   SIZE[dtype]))))
        # scores of at most 2 GiB in the plain form, and queries of 256 MiB
        while rows * hq * max(_spans(case)) * max(_lens(case)) > 1 << 29 or \
                case["tokens"] * hq * d * SIZE[dtype] > 1 << 28:
            case["tokens"] = max(rows, case["tokens"] // 2)
            case["max_len"] = max(1, case["max_len"] * 3 // 4)
        return case
    return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32", "i32"]),
                rows=_log(rng, 1, 300), vocab=_log(rng, 2, 250000), k=rng.choice([0, 1, 5, 20, 32]))


def _spans(case):
    """New tokens of each sequence: `tokens` split at random places, none empty
    (a case's lengths are part of it, not of the seed)."""
    rows, tokens = case["rows"], case["tokens"]
    rng = random.Random("%d of %d" % (rows, tokens))
    cuts = sorted(rng.sample(range(1, tokens), rows - 1)) if rows > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [tokens])]


def _lens(case):
    """Tokens that each sequence holds, the new ones among them."""
    spans = _spans(case)
    rng = random.Random("%d of at most %d" % (case["rows"], case["max_len"]))
    lens = [max(n, _log(rng, 1, case["max_len"])) for n in spans]
    lens[0] = max(spans[0], case["max_len"])
    return lens


def _padded(case):
    """The row that is padding, where there are many."""
    return case["rows"] // 2 if case["kind"] in ("map", "chunk") and case["rows"] >= 8 else None


def _spare(case):
    """Places for tokens behind the last row's."""
    return 5 if _padded(case) is not None else 0


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * (12 + 8 * case["k"]),
                "flops": 5 * n}
    if kind == "map":
        t = case["tokens"]
        return {"bytes": 16 * case["rows"] + 4 * t // case["page"] + 16 * t, "flops": 0}
    e, d, t = SIZE[case["dtype"]], case["d"], case["tokens"]
    if kind in ("append", "rotary"):
        heads = case["hq"] + case["hkv"]
        flops = t * heads * (3 * case["rot"] + (4 * d if case["norm"] else 0))
        if kind == "append":
            heads += case["hkv"]
        return {"bytes": 2 * t * heads * d * e + 12 * t, "flops": flops}
    seen = held = rows = 0
    for i, (c, n) in enumerate(zip(_spans(case), _lens(case))):
        if i != _padded(case):
            seen += c * n - c * (c - 1) // 2
            held += n
        rows += c
    return {"bytes": (2 * held * case["hkv"] + 2 * rows * case["hq"]) * d * e,
            "flops": 4 * seen * case["hq"] * d}


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


def _cache(case, gen, heads, d, dtype):
    """A pool [pages][1 layer][K, V][kv heads][page][d], its sequences' pages
    scattered over it, the pages' counts of users, tables and lengths."""
    page, lens = case["page"], _lens(case)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + max(4, sum(held) // 8)
    pool = _randn(gen, pages, 1, 2, heads, page, d, dtype=dtype)
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    tables = torch.full((len(lens), max(held)), -1, dtype=torch.int32, device="cuda")
    mine = torch.arange(max(held), device="cuda") < _ints(held)[:, None]
    tables[mine] = order[:sum(held)]
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:sum(held)].long()] = 1
    return dict(pool=pool, refs=refs, tables=tables, lens=_ints(lens))


def _requests(case, gen):
    """The step's requests in any order: sequences (-1: padding) and counts."""
    order = torch.randperm(case["rows"], device="cuda", generator=gen)
    seqs, counts = order.to(torch.int32), _ints(_spans(case))[order]
    if _padded(case) is not None:
        seqs = torch.where(order == _padded(case), -1, seqs)
    return dict(seqs=seqs, counts=counts)


def _frequencies(case):
    """Radians a position of each pair, and what cosines and sines are multiplied
    by: base 10000; scaled, slow pairs are four times slower, fast ones as they
    are, a ramp between them."""
    rot = case["rot"]
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if not case["scaled"]:
        return f.cuda(), 1.0
    turns = 4096 * f / (2 * math.pi)          # of a pair over the trained context
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return (f * keep + f / 4 * (1 - keep)).cuda(), 0.1 * math.log(4.0) + 1.0


_streams = {}


def _engine():
    """The engine on a stream that torch's own operations can be put on too."""
    from fable5_llm_amd import engine
    ctx = engine.default_context()
    if ctx not in _streams:
        _streams[ctx] = torch.cuda.Stream()
    ctx.set_stream(_streams[ctx])
    return ctx


def prepare(case, seed):
    gen, kind = _gen(seed), case["kind"]
    st = dict(case=case)
    if kind == "logprobs":
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        if case["dtype"] == "i32":       # sums of products, 18 fraction bits
            st["logits"] = (_randn(gen, rows, vocab) * (3 << 18)).to(torch.int32)
        else:
            st["logits"] = (_randn(gen, rows, vocab) * 3).to(DTYPE[case["dtype"]])
        st["scale"] = 2.0 ** -18 if case["dtype"] == "i32" else 0.8
        st["ids"] = torch.randint(0, vocab, (rows,), device="cuda", generator=gen) \
            .to(torch.int32)
        f32 = dict(dtype=torch.float32, device="cuda")
        k = min(k, vocab)
        st["out"] = dict(logp=torch.zeros(rows, **f32), entropy=torch.zeros(rows, **f32),
                         top_logp=torch.zeros(rows, k, **f32),
                         top_ids=torch.zeros(rows, k, dtype=torch.int32, device="cuda"))
    elif kind == "map":
        st.update(_cache(case, gen, 1, 64, torch.bfloat16))
        st.update(_requests(case, gen))
    else:
        dt, t, hq, hkv, d = DTYPE[case["dtype"]], case["tokens"] + _spare(case), case["hq"], \
            case["hkv"], case["d"]
        st["q"] = _randn(gen, t, hq, d, dtype=dt)
        st["q_out"] = torch.zeros_like(st["q"])
        if kind != "rotary":
            st.update(_cache(case, gen, hkv, d, dt))
            st.update(_requests(case, gen))
        if kind != "chunk":
            st["k"] = _randn(gen, t, hkv, d, dtype=dt)
            st["freq"], st["amplitude"] = _frequencies(case)
            st["norms"] = [1.0 + 0.2 * _randn(gen, d) for _ in range(2)] if case["norm"] \
                else [None, None]
        if kind == "append":
            st["v"] = _randn(gen, t, hkv, d, dtype=dt)
            _, _, st["pos"], st["slots"] = _maps(st, t)
        if kind == "rotary":
            st["k_out"] = torch.zeros_like(st["k"])
            st["pos"] = torch.randint(0, case["max_pos"], (t,), device="cuda", generator=gen) \
                .to(torch.int32)
    if own:      # the handles, maps and workspaces that a program keeps
        st["ctx"] = _engine()
        if kind == "logprobs":
            st["ws"] = st["ctx"].logprobs_workspace(case["rows"], case["vocab"])
        if "pool" in st:
            from fable5_llm_amd import engine
            st["kv"] = engine.PagedKV(st["ctx"], st["pool"], st["refs"], st["tables"],
                                      st["lens"])
        if kind in ("map", "chunk"):
            st["maps"] = st["kv"].chunk_maps(case["rows"], case["tokens"] + _spare(case),
                                             case.get("hq", 1))
        if kind == "chunk":
            st["ws"] = st["kv"].attend_chunk_workspace(st["maps"])
            torch.cuda.synchronize()
            st["kv"].map_async(st["seqs"], st["counts"], st["maps"])
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _OWN[kind](st)
    return _PLAIN[kind](st)


def _own_map(st):
    m = st["maps"]
    st["kv"].map_async(st["seqs"], st["counts"], m)
    return dict(cu=m.cu, seqs=m.seqs, pos=m.pos, slots=m.slots)


def _layout(case):
    return "halves" if case["halves"] else "pairs"


def _own_append(st):
    st["kv"].append_rotary_async(0, st["q"], st["k"], st["v"], st["pos"], st["slots"],
                                 st["freq"], st["q_out"], layout=_layout(st["case"]),
                                 amplitude=st["amplitude"], q_norm=st["norms"][0],
                                 k_norm=st["norms"][1], eps=EPS)
    return dict(q=st["q_out"], pool=st["pool"])


def _own_rotary(st):
    st["ctx"].rotary_async(st["q"], st["k"], st["pos"], st["freq"], st["q_out"], st["k_out"],
                           layout=_layout(st["case"]), amplitude=st["amplitude"],
                           q_norm=st["norms"][0], k_norm=st["norms"][1], eps=EPS)
    return dict(q=st["q_out"], k=st["k_out"])


def _own_chunk(st):
    st["kv"].attend_chunk_async(0, st["q"], st["q_out"], st["maps"], st["ws"])
    return st["q_out"]


def _own_logprobs(st):
    o, some = st["out"], st["out"]["top_ids"].shape[1] > 0
    st["ctx"].logprobs_async(st["logits"], st["ids"], o["logp"], st["ws"], entropy=o["entropy"],
                             top_logp=o["top_logp"] if some else None,
                             top_ids=o["top_ids"] if some else None, scale=st["scale"])
    return o


_OWN = dict(map=_own_map, append=_own_append, rotary=_own_rotary, chunk=_own_chunk,
            logprobs=_own_logprobs)


# ------------------------------------------------------------- plain forms
def _maps(st, tokens):
    """cu, and each token's sequence, position and slot (-1: none)."""
    page, rows = st["case"]["page"], st["seqs"].shape[0]
    counts = st["counts"].long()
    cu = torch.cat([torch.zeros_like(counts[:1]), counts.cumsum(0)])
    t = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(cu[1:], t, right=True)
    live = row < rows
    row = row.clamp(max=rows - 1)
    seq = st["seqs"].long()[row]
    live &= seq >= 0
    seq = seq.clamp(min=0)
    pos = st["lens"].long()[seq] - counts[row] + t - cu[row]
    pos = torch.where(live, pos, 0)
    slot = st["tables"].long()[seq, pos // page] * page + pos % page
    none = torch.full_like(t, -1)
    return (cu.to(torch.int32), torch.where(live, seq, none).to(torch.int32),
            torch.where(live, pos, none).to(torch.int32), torch.where(live, slot, none))


def _plain_map(st):
    cu, seqs, pos, slots = _maps(st, st["case"]["tokens"] + _spare(st["case"]))
    return dict(cu=cu, seqs=seqs, pos=pos, slots=slots)


def _rotated(st, x, weight):
    """x [tokens, heads, d] in 32 bits, normalised and rotated."""
    case, x = st["case"], x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    angle = st["pos"].double()[:, None, None] * st["freq"]
    c, s = (f(angle).float() * st["amplitude"] for f in (torch.cos, torch.sin))
    rot = case["rot"]
    if case["halves"]:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(st):
    page, slot = st["case"]["page"], st["slots"]
    st["q_out"].copy_(_rotated(st, st["q"], st["norms"][0]))
    k = _rotated(st, st["k"], st["norms"][1]).to(st["pool"].dtype)
    st["pool"][slot // page, 0, 0, :, slot % page] = k
    st["pool"][slot // page, 0, 1, :, slot % page] = st["v"]
    return dict(q=st["q_out"], pool=st["pool"])


def _plain_rotary(st):
    st["q_out"].copy_(_rotated(st, st["q"], st["norms"][0]))
    st["k_out"].copy_(_rotated(st, st["k"], st["norms"][1]))
    return dict(q=st["q_out"], k=st["k_out"])


def _plain_chunk(st):
    case = st["case"]
    hkv, hq, d, page = case["hkv"], case["hq"], case["d"], case["page"]
    n, c = max(_lens(case)), max(_spans(case))
    counts, seqs = st["counts"].long(), st["seqs"].long()
    start = counts.cumsum(0) - counts
    at = start[:, None] + torch.arange(c, device="cuda")           # [rows, c]
    mine = torch.arange(c, device="cuda") < counts[:, None]
    q = st["q"][torch.where(mine, at, 0)].float() * (1.0 / math.sqrt(d))
    rows = q.shape[0]
    q = q.view(rows, c, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(rows, hkv, -1, d)
    tables = st["tables"][seqs.clamp(min=0), :-(-n // page)].long().clamp(min=0)

    def cached(which):
        x = st["pool"][tables, 0, which].float()
        return x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n]

    k = cached(0).transpose(2, 3).contiguous()
    s = (q @ k).view(rows, hkv, c, hq // hkv, n)
    del k
    pos = st["lens"].long()[seqs.clamp(min=0)] - counts
    last = torch.where(seqs >= 0, pos, -1 << 40)[:, None] + torch.arange(c, device="cuda")
    live = torch.arange(n, device="cuda") <= last[..., None]          # [rows, c, n]
    s.masked_fill_(~live[:, None, :, None], float("-inf"))
    s -= s.amax(-1, keepdim=True).clamp(min=-1e30)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    s /= torch.where(total > 0, total, 1.0)
    o = s.view(rows, hkv, -1, n) @ cached(1)
    o = o.view(rows, hkv, c, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(rows, c, hq, d)
    st["q_out"][at[mine]] = o[mine].to(st["q_out"].dtype)
    return st["q_out"]


def _plain_logprobs(st):
    x, k = st["logits"], st["out"]["top_ids"].shape[1]
    top = x.amax(-1, keepdim=True)
    y = (x.long() - top if x.dtype == torch.int32 else x.float() - top.float()).float()
    y *= st["scale"]
    log_sum = torch.log(torch.exp(y).sum(-1, keepdim=True))
    y -= log_sum
    ids = st["ids"].long()[:, None]
    out = dict(logp=y.gather(1, ids)[:, 0], entropy=-(torch.exp(y) * y).sum(-1))
    best = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k]
    return dict(out, top_logp=y.gather(1, best), top_ids=best.to(torch.int32))


_PLAIN = dict(map=_plain_map, append=_plain_append, rotary=_plain_rotary, chunk=_plain_chunk,
              logprobs=_plain_logprobs)


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
    return {"map": _exact_map, "append": _exact_rotary, "rotary": _exact_rotary,
            "chunk": _exact_chunk, "logprobs": _exact_logprobs}[case["kind"]](case, st)


def _exact_map(case, st):
    """Token by token, on the host."""
    seqs, counts, lens = (st[k].tolist() for k in ("seqs", "counts", "lens"))
    tables, page = st["tables"].cpu().numpy().astype(np.int64), case["page"]
    cu, out = [0], []
    for s, c in zip(seqs, counts):
        for j in range(c):
            p = lens[s] - c + j
            out.append((s, p, int(tables[s, p // page]) * page + p % page) if s >= 0
                       else (-1, -1, -1))
        cu.append(cu[-1] + c)
    out += [(-1, -1, -1)] * _spare(case)
    s, p, slot = (np.array(v) for v in zip(*out))
    return dict(cu=np.array(cu, np.int32), seqs=s.astype(np.int32), pos=p.astype(np.int32),
                slots=slot.astype(np.int64))


def _exact_rotary(case, st):
    def turn(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() \
                * weight.double()
        z = torch.exp(1j * st["pos"].double()[:, None] * st["freq"]) * st["amplitude"]
        y, rot = x.clone(), case["rot"]
        for i in range(rot // 2):
            a, b = (i, i + rot // 2) if case["halves"] else (2 * i, 2 * i + 1)
            w = torch.complex(x[:, :, a], x[:, :, b]) * z[:, i, None]
            y[:, :, a], y[:, :, b] = w.real, w.imag
        return y

    q, k = turn(st["q"], st["norms"][0]), turn(st["k"], st["norms"][1])
    if case["kind"] == "rotary":
        return dict(q=q, k=k)
    pool, page = st["pool"].double(), case["page"]
    for which, x in ((0, k), (1, st["v"].double())):
        for h in range(case["hkv"]):
            pool[st["slots"] // page, 0, which, h, st["slots"] % page] = x[:, h]
    return dict(q=q, pool=pool)


def _exact_chunk(case, st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    per, page, d = case["hq"] // case["hkv"], case["page"], case["d"]
    lens, t = st["lens"].tolist(), 0
    for s, c in zip(st["seqs"].tolist(), st["counts"].tolist()):
        if s >= 0:
            n = lens[s]
            pages = st["tables"][s, :-(-n // page)].long()
            late = torch.arange(n, device="cuda") > n - c + torch.arange(c, device="cuda")[:, None]
            for h in range(case["hkv"]):
                k, v = (st["pool"][pages, 0, w, h].double().reshape(-1, d)[:n] for w in (0, 1))
                for j in range(h * per, (h + 1) * per):
                    a = st["q"][t:t + c, j].double() @ k.T / math.sqrt(d)
                    a = torch.softmax(a.masked_fill_(late, float("-inf")), -1)
                    out[t:t + c, j] = a @ v
        t += c
    return out


def _exact_logprobs(case, st):
    rows, k = case["rows"], st["out"]["top_ids"].shape[1]
    out = dict(logp=[], entropy=[], top_logp=[], top_ids=[])
    for i in range(rows):
        raw = st["logits"][i].double()
        lp = torch.log_softmax(raw * st["scale"], -1)
        best = torch.argsort(-raw, stable=True)[:k]
        out["logp"].append(lp[int(st["ids"][i])])
        out["entropy"].append(-(lp.exp() * lp).sum())
        out["top_logp"].append(lp[best])
        out["top_ids"].append(best.to(torch.int32))
    return {name: torch.stack(v) for name, v in out.items()}
