"""Lists of many entries: right, and in a time that grows with the list and not
with its square (16 times the entries: 16 times the time, where it was 256; 64
stands between them)."""
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
