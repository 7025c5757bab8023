"""A refused reserve or fork stops its cache until the next sync has reported it:
the calls behind it, which count on it, change nothing, and the step can be made
again."""
import pytest
import torch

from fable5_llm_amd.engine import PagedKV
from test_gpu_kv import DEV, DIM, HEADS, LAYERS, Both, ints

pytestmark = pytest.mark.gpu


def state(kv):
    return [t.clone() for t in (kv.pool, kv.refs, kv.tables, kv.lens)]


def same(kv, want):
    return all(torch.equal(t, w) for t, w in zip((kv.pool, kv.refs, kv.tables, kv.lens), want))


def rows(n, value):
    return torch.full((n, HEADS, DIM), float(value), device=DEV)


@pytest.mark.parametrize("call,lists,why", [
    ("extend", ([0, 1], [13, 62]), "too few free pages"),   # 1 + 3 pages, 3 are free
    ("extend", ([0, 1], [1, 16 * 5]), "outside the cache"),  # 113 tokens of at most 96
    ("extend", ([0, 0], [1, 1]), "listed twice"),
    ("extend", ([0, 5], [1, 1]), "outside the cache"),
    ("extend", ([0, 1], [1, -1]), "outside the cache"),
    ("fork", ([0, 0], [3, 3]), "listed twice"),
    ("fork", ([0], [1]), "listed twice"),
    ("fork", ([0], [5]), "outside the cache"),
])
def test_the_calls_behind_a_refused_one_change_nothing(engine, call, lists, why):
    b = Both(engine, 9, 5, 6)
    assert b.both("extend", [0, 1, 2], [20, 33, 5])
    b.append([0, 1, 2], [19, 32, 4])
    want = state(b.kv)
    args, one, k = [ints(x) for x in lists], ints([1]), rows(2, 7)
    first, four, zero, page = ints([0, 1]), ints([4]), ints([0]), ints([8])
    torch.cuda.synchronize()
    getattr(b.kv, call + "_async")(*args)
    for layer in range(LAYERS):
        b.kv.append_async(layer, k, k, first)             # the step's new tokens
        b.kv.append_async(layer, k, k, first, ints([3, 4]))
    b.kv.extend_async(four, one)
    b.kv.append_async(0, k[:1], k[:1], four)
    b.kv.fork_async(zero, four)
    b.kv.free_async(first)
    b.kv.compact_async()
    b.kv.copy_async(zero, page)
    with pytest.raises(AssertionError, match=why):
        engine.sync()
    assert same(b.kv, want)
    engine.sync()                                         # reported once
    assert b.both("extend", [0, 4], [1, 3])               # and then all is as it was
    b.append([0, 4], [20, 2])
    b.check()
    assert b.both("free", [1]) and b.both("compact") and b.both("fork", [0], [3])
    b.check()


def test_a_fork_without_room_keeps_its_parents(engine):
    # a beam's step: fork, a token each, the parents dropped
    b = Both(engine, 6, 6, 6)
    assert b.both("extend", [0, 1], [40, 32])
    b.append([0] * 40 + [1] * 32, list(range(40)) + list(range(32)))
    want = state(b.kv)
    par, kid, one, old, k = ints([0, 0]), ints([2, 3]), ints([1, 1]), ints([0, 1]), rows(2, 7)
    torch.cuda.synchronize()
    for _ in range(2):
        b.kv.fork_async(par, kid)
        b.kv.extend_async(kid, one)
        b.kv.append_async(0, k, k, kid)
        b.kv.free_async(old)
        b.kv.compact_async()
        with pytest.raises(AssertionError, match="too few free pages"):
            engine.sync()
        assert same(b.kv, want)


def test_a_captured_step_that_runs_out_of_pages(engine):
    # replayed past the pool's end without a sync: stopped at the last token that
    # had room; after the sync and a free the same graph goes on
    b = Both(engine, 5, 3, 4)
    assert b.both("extend", [0, 1], [30, 17])             # 2 + 2 pages, one free
    b.append([0] * 30 + [1] * 17, list(range(30)) + list(range(17)))
    seqs, one = ints([0, 1]), ints([1, 1])
    k = rows(2, 0)
    count = torch.zeros(1, device=DEV)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(g, stream=side):
            engine.set_stream(side)
            count.add_(1.0)
            k.copy_(count.expand_as(k))
            b.kv.extend_async(seqs, one)
            for layer in range(LAYERS):
                b.kv.append_async(layer, k, k, seqs)
    finally:
        engine.set_stream(None)

    def tokens(s):
        kv, n = b.kv, int(b.kv.lens[s])
        return [float(kv.pool[kv.tables[s, t // 16], 1, 1, 0, t % 16, 0]) for t in range(n)]

    was = tokens(0), tokens(1)
    for _ in range(20):                 # 2 fill sequence 0's page, 14 more its third page
        g.replay()
    torch.cuda.synchronize()
    with pytest.raises(AssertionError, match="too few free pages"):
        engine.sync()
    assert b.kv.lens.tolist() == [45, 32, 0]              # 33: a page for each, one is free
    assert tokens(0) == was[0] + [float(i) for i in range(1, 16)]
    assert tokens(1) == was[1] + [float(i) for i in range(1, 16)]
    args = ints([0])
    torch.cuda.synchronize()
    b.kv.free_async(args)
    engine.sync()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        engine.sync()
    assert b.kv.lens.tolist() == [3, 35, 0]
    assert tokens(0) == [21.0, 22.0, 23.0]
    assert tokens(1) == was[1] + [float(i) for i in range(1, 16)] + [21.0, 22.0, 23.0]


def test_another_cache_of_the_context_goes_on(engine):
    a, b = Both(engine, 4, 3, 4), Both(engine, 4, 3, 4)
    assert a.both("extend", [0], [20]) and b.both("extend", [0], [20])
    two, many, one, zero, k = ints([0, 0]), ints([1, 1]), ints([1]), ints([0]), rows(1, 5)
    torch.cuda.synchronize()
    a.kv.extend_async(two, many)
    b.kv.extend_async(zero, one)
    b.kv.append_async(0, k, k, zero)
    with pytest.raises(AssertionError, match="listed twice"):
        engine.sync()
    assert a.kv.lens.tolist() == [20, 0, 0] and b.kv.lens.tolist() == [21, 0, 0]
    assert (b.kv.pool[b.kv.tables[0, 1], 0, :, :, 4] == 5).all()


def test_an_append_outside_the_cache_stops_nothing(engine):
    b = Both(engine, 9, 5, 6)
    assert b.both("extend", [0, 1], [20, 33])
    k, seqs, pos, zero, one = rows(2, 3), ints([0, 1]), ints([20, 32]), ints([0]), ints([1])
    torch.cuda.synchronize()
    b.kv.append_async(0, k, k, seqs, pos)
    b.kv.extend_async(zero, one)
    with pytest.raises(AssertionError, match="outside the cache"):
        engine.sync()
    assert b.kv.lens.tolist() == [21, 33, 0, 0, 0]
    assert (b.kv.pool[b.kv.tables[1, 2], 0, :, :, 0] == 3).all()
