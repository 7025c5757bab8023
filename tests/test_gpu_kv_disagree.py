"""Compaction beside tables that name pages which no sequence holds: reported, the
entries left alone, every other sequence's tokens kept."""
import pytest
import torch

from test_gpu_kv import Both, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wrong", [0, 1, 2, 8, 9, -1])
def test_a_free_page_below_and_above_the_ones_in_use(engine, wrong):
    # sequence 0 held pages 0 to 2: free, and filled by the pages 5, 6 and 7 of the
    # five in use; 8 is free and stays so
    b = Both(engine, 9, 5, 6)
    assert b.both("extend", [0, 1, 2], [40, 33, 20])      # pages 0-2, 3-5, 6-7
    b.append([1] * 33 + [2] * 20, list(range(33)) + list(range(20)))
    assert b.both("free", [0])
    keep = int(b.kv.tables[1, 1])
    b.kv.tables[1, 1] = wrong
    torch.cuda.synchronize()
    b.kv.compact_async()
    with pytest.raises(AssertionError, match="outside the cache"):
        engine.sync()
    assert int(b.kv.tables[1, 1]) == wrong
    b.m.compact()
    b.kv.tables[1, 1] = b.m.tables[1][1]
    assert keep == 4
    b.check()
    assert b.both("compact")                              # and nothing is left to report
    b.check()


def test_every_entry_right_reports_nothing(engine):
    b = Both(engine, 40, 8, 6)
    assert b.both("extend", list(range(8)), [17, 33, 49, 1, 16, 64, 80, 5])
    for gone in ([1, 6], [0], [3, 4]):
        assert b.both("free", gone) and b.both("compact")
        b.check()
