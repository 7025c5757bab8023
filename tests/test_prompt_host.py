"""The checks of arguments of a step's maps and attention, the rotary positions and
the log probabilities on a machine without a GPU: the C ABI on the stand-in HIP
runtime (each refused call launches nothing), what is no device tensor, and the
frequencies of stretched contexts."""
import math
import types

import numpy as np
import pytest
import torch

import fake_hip
from fable5_llm_amd import mixers as M


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    return fake_hip.build(tmp_path_factory.mktemp("hip"))


@pytest.mark.parametrize("check", ["map", "attend", "rotary", "logprobs", "launches"])
def test_abi(runtime, check):
    assert fake_hip.run(runtime, "prompt_check.py", check) == "ok"


class Ctx:
    h, device = None, 0


@pytest.mark.parametrize("bad", [None, 3, np.zeros((2, 1, 64), np.float32), torch.zeros(2, 1, 64)])
def test_device_tensors_only(bad):
    with pytest.raises(ValueError, match="device tensor|needed"):
        M.rotary_args(Ctx, bad, None, None, bad, None, bad, bad, None, "halves", 1.0, None, None,
                      1e-6, 0, 0)
    with pytest.raises(ValueError, match="device tensor"):
        M.logprobs_args(Ctx, bad, None, None, bad, None, None, None, 1.0)


def test_maps_are_made_by_their_cache():
    kv = types.SimpleNamespace()
    for maps in (None, 3, types.SimpleNamespace(cache=kv)):
        with pytest.raises(ValueError, match="chunk_maps"):
            M.PagedKV._maps(kv, maps)
    m = M.ChunkMaps.__new__(M.ChunkMaps)
    m.cache = kv
    assert M.PagedKV._maps(kv, m) is m
    with pytest.raises(ValueError, match="another cache"):
        M.PagedKV._maps(types.SimpleNamespace(), m)


def test_frequencies():
    i = torch.arange(32, dtype=torch.float64)
    f, a = M.rotary_frequencies(64)
    assert a == 1 and torch.allclose(f, 10000.0 ** (-i / 32), rtol=1e-15)
    g, a = M.rotary_frequencies(64, stretch="positions", factor=8.0)
    assert a == 1 and torch.equal(g, f / 8)
    g, a = M.rotary_frequencies(64, base=500000.0, stretch="base", factor=4.0)
    own = 500000.0 ** (-i / 32)
    # the fastest as it was, the slowest slower by the factor, all by b^(-i / 31)
    assert a == 1 and torch.allclose(g, own * 4.0 ** (-i / 31), rtol=1e-14)
    g, a = M.rotary_frequencies(64, stretch="parts", factor=16.0, trained=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32])
    assert torch.allclose(g[turns <= 1], f[turns <= 1] / 16, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((g < f) & (g > f / 16))[between].all()
    assert math.isclose(a, 0.1 * math.log(16.0) + 1)
    for kw in (dict(rot=7), dict(rot=0), dict(rot=64, base=0.0), dict(rot=64, factor=0.5),
               dict(rot=64, stretch="some"), dict(rot=64, stretch="parts", factor=2.0),
               dict(rot=64, stretch="parts", factor=2.0, trained=4096, fast=1.0),
               dict(rot=2, stretch="base")):
        with pytest.raises(ValueError):
            M.rotary_frequencies(**kw)
