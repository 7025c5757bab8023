"""The pages of a key-value cache on the device (PagedKV's extend, append,
fork, free, compact, copy) against the page model of page_model.py: counts,
tables, lengths and every token's content exactly, refusals that change
nothing, entries outside the cache, and replays of a captured sequence."""
import random

import numpy as np
import pytest
import torch

from fable5_llm_amd.engine import PagedKV
from page_model import Pages, Refused

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS, DIM, LAYERS = 2, 64, 2


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Both:
    """A cache on the device and its model, given the same calls."""

    def __init__(self, engine, pages, seqs, max_pages, page=16, dtype=torch.float32):
        self.eng, self.n = engine, 0
        self.kv = PagedKV.empty(engine, pages, LAYERS, HEADS, page, DIM, seqs, max_pages, dtype)
        self.m = Pages(pages, seqs, max_pages, page)

    def both(self, name, *lists):
        """One call on both; True where both took it."""
        args = [ints(x) for x in lists]
        torch.cuda.synchronize()
        getattr(self.kv, name + "_async")(*args)
        try:
            getattr(self.m, name)(*lists)
            ok = True
        except Refused:
            ok = False
        if ok:
            self.eng.sync()
        else:
            with pytest.raises(AssertionError, match="KV cache"):
                self.eng.sync()
        return ok

    def append(self, seqs, pos):
        """Tokens whose values name them, in every layer."""
        n = len(seqs)
        label = torch.arange(self.n, self.n + n, device=DEV)
        self.n += n
        base = (label[:, None, None] * 8).float()
        for layer in range(LAYERS):
            k = (base + layer).expand(n, HEADS, DIM).to(self.kv.pool.dtype).contiguous()
            v = (base + 4 + layer).expand(n, HEADS, DIM).to(self.kv.pool.dtype).contiguous()
            args = ints(seqs), ints(pos)
            torch.cuda.synchronize()
            self.kv.append_async(layer, k, v, *args)
            self.eng.sync()
        for i, (s, p) in enumerate(zip(seqs, pos)):
            if s >= 0:
                self.m.write(s, p, int(label[i]))

    def check(self):
        assert self.kv.refs.tolist() == self.m.refs
        assert self.kv.lens.tolist() == self.m.lens
        tables = self.kv.tables.tolist()
        pool = self.kv.pool.float().cpu().numpy()
        for s, n in enumerate(self.m.lens):
            held = self.m.held(n)
            assert tables[s][:held] == self.m.tables[s][:held], s
        for p, slots in enumerate(self.m.data):
            for t, x in enumerate(slots):
                if x is None:
                    continue
                for layer in range(LAYERS):
                    want = np.array([8 * x + layer, 8 * x + 4 + layer], np.float32)
                    got = pool[p, layer, :, :, t]
                    assert np.array_equal(got, np.broadcast_to(want[:, None, None], got.shape))


@pytest.mark.parametrize("seed,page", [(0, 16), (1, 32), (2, 64), (3, 16)])
def test_random_calls(engine, seed, page):
    rng = random.Random(seed)
    S = 14
    b = Both(engine, 50, S, 6, page)
    took = dict(extend=0, fork=0, free=0, compact=0, refused=0)
    for _ in range(60):
        op = rng.choice(["extend", "extend", "extend", "fork", "fork", "free", "compact"])
        if op == "extend":
            seqs = rng.sample(range(-1, S + (rng.random() < 0.1)), rng.randint(1, 5))
            old = list(b.m.lens)
            ok = b.both("extend", seqs, [rng.choice([0, 1, 3, page, 2 * page + 1]) for _ in seqs])
            if ok:
                new = [(s, t) for s in seqs if s >= 0 for t in range(old[s], b.m.lens[s])]
                rng.shuffle(new)
                if new:
                    b.append([s for s, _ in new] + [-1], [t for _, t in new] + [0])
        elif op == "fork":
            n = rng.randint(1, 4)
            empty = [s for s in range(S) if not b.m.lens[s]]
            kids = rng.sample(empty, min(n, len(empty))) if rng.random() < 0.8 \
                else [rng.randrange(S) for _ in range(n)]
            ok = b.both("fork", [rng.randrange(-1, S) for _ in kids], kids) if kids else True
        elif op == "free":
            ok = b.both("free", [rng.randrange(-1, S) for _ in range(rng.randint(1, 4))])
        else:
            ok = b.both("compact")
        took[op if ok else "refused"] += 1
        b.check()
    assert min(took.values()) > 0, took


def test_many_pages_and_a_long_list(engine):
    # more pages than one turn of the scans takes (16,384), more sequences than
    # a workgroup has threads, runs of pages longer than a thread writes
    S, pages = 2100, 40003
    kv = PagedKV.empty(engine, pages, 1, 1, 16, 64, S, 600, torch.float16)
    m = Pages(pages, S, 600, 16)
    rng = random.Random(9)
    order = rng.sample(range(S), S)
    counts = [rng.choice([1, 16, 17, 100, 400]) for _ in range(S)]
    counts[7] = 9600
    gone = rng.sample(range(S), 900)
    kids, parents = gone[:300], rng.choices([s for s in range(S) if s not in gone], k=300)
    args = [ints(v) for v in (order, counts, gone, parents, kids)]
    torch.cuda.synchronize()
    kv.extend_async(args[0], args[1])
    kv.free_async(args[2])
    kv.fork_async(args[3], args[4])
    engine.sync()
    m.extend(order, counts)
    m.free(gone)
    m.fork(parents, kids)
    assert kv.refs.tolist() == m.refs and kv.lens.tolist() == m.lens
    was = kv.pool.normal_().clone()
    tables = kv.tables.clone()
    torch.cuda.synchronize()
    kv.compact_async()
    engine.sync()
    m.compact()
    got = kv.tables.tolist()
    assert kv.refs.tolist() == m.refs
    assert all(got[s][:m.held(n)] == m.tables[s][:m.held(n)] for s, n in enumerate(m.lens))
    for s in (order[7], kids[0], order[50]):
        held = m.held(m.lens[s])
        assert torch.equal(kv.pool[kv.tables[s, :held].long()], was[tables[s, :held].long()])


@pytest.mark.parametrize("call,lists", [
    ("extend", ([0, 1], [1, 16 * 5])),             # one page too many
    ("extend", ([0, 0], [1, 1])), ("extend", ([5], [1])), ("extend", ([1], [-1])),
    ("extend", ([1], [16 * 7])), ("extend", ([1], [2 ** 31 - 1])),
    ("fork", ([0, 0], [3, 3])), ("fork", ([0], [1])), ("fork", ([3, 0], [4, 3])),
    ("fork", ([0], [0])), ("fork", ([5], [3])), ("fork", ([0], [5])),
])
def test_refusals_change_nothing(engine, call, lists):
    b = Both(engine, 9, 5, 6)
    assert b.both("extend", [0, 1, 2], [20, 33, 5])
    b.append([0, 1, 2], [19, 32, 4])
    assert b.both(call, *lists) is False
    b.check()
    assert b.both("extend", [4, 0], [17, 0])       # and the next call is its own
    b.check()


def test_fork_without_room_for_the_last_pages(engine):
    b = Both(engine, 7, 6, 6)
    assert b.both("extend", [0, 1], [40, 32])      # 3 + 2 pages, 2 free
    assert not b.both("fork", [0, 0, 0], [2, 3, 4])
    assert b.both("fork", [0, 1, 0], [2, 3, 4])    # sequence 1 needs none
    b.check()


def test_padding_and_empty_lists(engine):
    b = Both(engine, 9, 5, 6)
    assert b.both("extend", [-1, 2, -1], [7, 18, 900])
    assert b.both("fork", [-1, 2, 2], [0, -1, 1])
    assert b.both("fork", [3], [4])                # an empty parent
    assert b.both("free", [-1, 3, 2, 2])           # empty, and listed twice
    assert b.both("extend", [], []) and b.both("free", []) and b.both("fork", [], [])
    b.check()
    assert b.m.lens == [0, 18, 0, 0, 0]


def test_append_outside_the_cache_is_reported(engine):
    b = Both(engine, 9, 5, 6)
    assert b.both("extend", [0, 1], [20, 33])
    b.append([0], [19])
    k = torch.ones((1, HEADS, DIM), device=DEV)
    before = b.kv.pool.clone()
    for seq, pos in ((0, 20), (0, -1), (5, 0), (2, 0)):
        args = ints([seq]), ints([pos])
        torch.cuda.synchronize()
        b.kv.append_async(0, k, k, *args)
        with pytest.raises(AssertionError, match="outside the cache"):
            engine.sync()
    for page in (-1, 9, 2 ** 31 - 1):              # a table that names no page
        keep = int(b.kv.tables[0, 1])
        b.kv.tables[0, 1] = page
        args = ints([0]), ints([18])
        torch.cuda.synchronize()
        b.kv.append_async(0, k, k, *args)
        with pytest.raises(AssertionError, match="outside the cache"):
            engine.sync()
        b.kv.tables[0, 1] = keep
    assert torch.equal(b.kv.pool, before)
    args = ints([1])
    torch.cuda.synchronize()
    b.kv.append_async(1, k, k, args)               # without positions: the last token
    engine.sync()
    assert torch.equal(b.kv.pool[b.kv.tables[1, 2], 1, :, :, 0], torch.ones(2, HEADS, DIM,
                                                                           device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_append_strided_and_int16(engine, dtype):
    rng = np.random.default_rng(1)
    kv = PagedKV.empty(engine, 12, 1, 4, 16, 128, 3, 4, dtype)
    seqs, n = ints([2, 0, 1]), 3
    counts = ints([40, 17, 64])
    wide = torch.from_numpy(rng.normal(0, 1, (n, 3, 4, 128))).to(DEV).to(dtype)
    i16 = torch.from_numpy(rng.integers(-32768, 32768, (n, 6, 2 * 128)).astype(np.int16)).to(DEV)
    torch.cuda.synchronize()
    kv.extend_async(seqs, counts)
    # keys and values side by side in one row of a projection
    kv.append_async(0, wide[:, 0], wide[:, 2], seqs)
    # every other half row, as int16 with 9 fraction bits
    kv.append_async(0, i16[:, :4, 128:], i16[:, 2:, :128], ints([0, 1, 2]), ints([3, 4, 5]),
                    frac=9)
    engine.sync()
    for i, (s, c) in enumerate(((2, 40), (0, 17), (1, 64))):
        at = kv.pool[kv.tables[s, (c - 1) // 16], 0, :, :, (c - 1) % 16]
        assert torch.equal(at[0], wide[i, 0]) and torch.equal(at[1], wide[i, 2])
    for i in range(3):
        at = kv.pool[kv.tables[i, 0], 0, :, :, 3 + i]
        assert torch.equal(at[0], (i16[i, :4, 128:].double() / 512).to(dtype))
        assert torch.equal(at[1], (i16[i, 2:, :128].double() / 512).to(dtype))


def test_lists_of_the_largest_size(engine):
    # 2^20 entries, padding but for a few
    b = Both(engine, 60, 8, 6)
    n = 1 << 20
    def full(*at):
        x = [-1] * n
        for i, v in at:
            x[i] = v
        return x
    assert b.both("extend", full((5, 2), (n - 1, 0)), full((5, 20), (n - 1, 7)))
    b.append([2] * 20 + [0] * 7, list(range(20)) + list(range(7)))
    assert b.both("fork", full((0, 2), (n // 2, 0), (n - 1, 2)), full((0, 3), (n // 2, 4), (n - 1, 5)))
    b.check()
    assert b.both("free", full((0, 2), (n - 2, 2), (n - 1, 4)))
    b.check()


def test_a_list_that_asks_for_more_pages_than_an_integer_holds(engine):
    S, most = 1100, 1 << 21                        # 1100 times 2^21 pages: over 2^31
    zeros = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)
    kv = PagedKV(engine, torch.zeros(3, 1, 2, 1, 16, 64, device=DEV), zeros(3),
                 torch.empty(S, most, dtype=torch.int32, device=DEV), zeros(S))
    seqs, counts = ints(list(range(S))), ints([16 * most] * S)
    for n in (S, 1):
        torch.cuda.synchronize()
        kv.extend_async(seqs[:n], counts[:n])
        with pytest.raises(AssertionError, match="too few free pages"):
            engine.sync()
        assert not kv.refs.any() and not kv.lens.any()


def test_compact_reports_tables_that_disagree_with_the_counts(engine):
    b = Both(engine, 9, 5, 6)
    assert b.both("extend", [0, 1, 2], [40, 40, 20])
    assert b.both("free", [0])
    for wrong in (8, -3, 9):                       # a free page past the used ones; none at all
        keep = int(b.kv.tables[1, 0])
        b.kv.tables[1, 0] = wrong
        torch.cuda.synchronize()
        b.kv.compact_async()
        with pytest.raises(AssertionError, match="outside the cache"):
            engine.sync()
        assert int(b.kv.tables[1, 0]) == wrong
        b.kv.tables[1, 0] = keep
        if wrong == 8:                             # the first call moved the rest
            b.m.compact()
            b.kv.tables[1, 0] = b.m.tables[1][0]
    b.check()


def test_a_cache_ends_with_its_context(engine):
    from fable5_llm_amd.engine import Context
    ctx = Context(0)
    kv, other = (PagedKV.empty(ctx, 4, 1, 1, 16, 64, 2, 2, torch.float32) for _ in range(2))
    other.close()
    ctx.close()
    with pytest.raises(ValueError, match="null cache"):
        kv.free_async(ints([0]))
    kv.close()
    del kv, other


def test_copy_pages(engine):
    kv = PagedKV.empty(engine, 300, 3, 2, 16, 64, 1, 1, torch.bfloat16)
    kv.pool.normal_()
    want = kv.pool.clone()
    src, dst = [5, 299, -1, 7, 9, 11], [0, 1, 2, -1, 9, 298]
    for a, b in zip(src, dst):
        if a >= 0 and b >= 0:
            want[b] = want[a]
    args = ints(src), ints(dst)
    torch.cuda.synchronize()
    kv.copy_async(*args)
    engine.sync()
    assert torch.equal(kv.pool, want)
    for a, b in ((300, 0), (0, 300)):
        args = ints([a, 4]), ints([b, 3])
        torch.cuda.synchronize()
        kv.copy_async(*args)
        with pytest.raises(AssertionError, match="outside the cache"):
            engine.sync()
        want[3] = want[4]
        assert torch.equal(kv.pool, want)


def test_captured_calls_replay(engine):
    """A beam's step captured once: fork, one more token each, drop the
    parents; replayed from a saved state, with eager work between."""
    b = Both(engine, 40, 8, 6)
    assert b.both("extend", [0, 1], [40, 33])
    b.append([0] * 40 + [1] * 33, list(range(40)) + list(range(33)))
    state = [t.clone() for t in (b.kv.pool, b.kv.refs, b.kv.tables, b.kv.lens)]
    par, kid, one, old = ints([0, 0, 1]), ints([4, 5, 6]), ints([1, 1, 1]), ints([0, 1])
    k = torch.full((3, HEADS, DIM), 5.0, device=DEV)
    torch.cuda.synchronize()

    def step():
        b.kv.fork_async(par, kid)
        b.kv.extend_async(kid, one)
        b.kv.append_async(1, k, k, kid)
        b.kv.free_async(old)
        b.kv.compact_async()

    def restore():
        for t, s in zip((b.kv.pool, b.kv.refs, b.kv.tables, b.kv.lens), state):
            t.copy_(s)
        torch.cuda.synchronize()

    step()
    engine.sync()
    want = [t.clone() for t in (b.kv.pool, b.kv.refs, b.kv.tables, b.kv.lens)]
    restore()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(g, stream=side):
            engine.set_stream(side)
            step()
    finally:
        engine.set_stream(None)
    for _ in range(3):
        restore()
        g.replay()
        torch.cuda.synchronize()
        engine.sync()
        for t, w in zip((b.kv.pool, b.kv.refs, b.kv.tables, b.kv.lens), want):
            assert torch.equal(t, w)


def test_wrong_tensors_are_refused(engine):
    f32 = torch.float32
    kv = PagedKV.empty(engine, 4, 1, 2, 16, 64, 2, 2, f32)
    one = ints([0])
    k = torch.zeros((1, 2, 64), device=DEV)
    bad = [
        lambda: kv.append_async(0, k[:, :1], k[:, :1], one),
        lambda: kv.append_async(0, k, k.half(), one),
        lambda: kv.append_async(0, k.half(), k.half(), one),
        lambda: kv.append_async(1, k, k, one),
        lambda: kv.append_async(0, k, k, ints([0, 1])),
        lambda: kv.append_async(0, k, k, one.long()),
        lambda: kv.append_async(0, k, k, one, ints([0, 1])),
        lambda: kv.append_async(0, k.cpu(), k, one),
        lambda: kv.append_async(0, torch.zeros((1, 2, 128), device=DEV)[:, :, ::2], k, one),
        lambda: kv.append_async(0, torch.zeros(129, device=DEV)[1:].view(1, 2, 64), k, one),
        lambda: kv.extend_async(ints([0, 1]), one),
        lambda: kv.extend_async(one.cpu(), one),
        lambda: kv.fork_async(ints([[0]]), one),
        lambda: PagedKV(engine, kv.pool, kv.refs, kv.tables, ints([0])),
        lambda: PagedKV(engine, kv.pool, kv.refs[:3], kv.tables, kv.lens),
        lambda: PagedKV(engine, kv.pool.double(), kv.refs, kv.tables, kv.lens),
        lambda: PagedKV(engine, kv.pool[:, :, :1], kv.refs, kv.tables, kv.lens),
        lambda: PagedKV.empty(engine, 4, 1, 2, 8, 64, 2, 2, f32),
        lambda: PagedKV.empty(engine, 4, 1, 2, 16, 80, 2, 2, f32),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
    engine.sync()
