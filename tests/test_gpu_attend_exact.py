"""Attention over 16-bit caches: the output's own rounding is the only one that
counts.  Per output, with u half a step of the cache's type, A = sum p |v| / sum
p, X the largest sum |q k| scale of a row's scores and V the largest |v|:

    u |out|          the output's rounding (int16: half of one step instead)
  + u^2 A            a weight as the sum of two values of the type
  + 2^-39 n V        float16: what lies below the second value's last bit,
                     2^-25 of weights held 2^14 as large
  + 2^-24 A (X (D + 4) + n + 16)   scores, exponentials and sums in float32
"""
import math

import pytest
import torch

from test_gpu_attend import DEV, U, make, rows_of, run

pytestmark = pytest.mark.gpu


def check(kv, layer, q, seqs, got, scale=None, unit=1.0, out_unit=None):
    dim, u = kv.head_dim, U[kv.pool.dtype]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    lens, per = kv.lens.tolist(), q.shape[1] // kv.kv_heads
    q, got = q.double().cpu() * unit, got.double().cpu() * (out_unit or 1.0)
    low = 2.0 ** -39 if kv.pool.dtype == torch.float16 else 0.0
    for i, s in enumerate(seqs):
        n = lens[s]
        k, v = (x.repeat_interleave(per, 0) for x in rows_of(kv, layer, s, n))
        sc = (k @ q[i][:, :, None])[:, :, 0] * scale
        dots = (k.abs() @ q[i].abs()[:, :, None]) * scale
        X = dots[torch.isfinite(dots)].max().item()
        p = torch.softmax(sc, -1)[:, None]
        want, A = (p @ v)[:, 0], (p @ v.abs())[:, 0]
        tol = (0.5 * out_unit if out_unit else u * want.abs()) + u * u * A + low * n * v.abs().max() + \
            2.0 ** -24 * A * (X * (dim + 4) + n + 16)
        off = (got[i] - want).abs() / tol
        assert not torch.isnan(got[i]).any() and off.max() <= 1, (i, s, n, float(off.max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,heads,group,page", [(64, 2, 1, 16), (128, 2, 4, 32), (256, 1, 4, 16),
                                                  (256, 1, 17, 64)])
def test_weights_keep_more_bits_than_the_output(engine, dtype, dim, heads, group, page):
    gen = torch.Generator().manual_seed(dim + group)
    lens = [511, 1, 2, 33, 700, 96]
    kv = make(engine, gen, lens, heads, dim, page, dtype)
    q = torch.randn(len(lens), heads * group, dim, generator=gen).to(DEV).to(dtype)
    seqs = [3, 1, 0, 5, 4, 2]
    check(kv, 0, q, seqs, run(engine, kv, 0, q, seqs))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("empty", [(0,), (1,), (3,), (0, 1), (2, 3), (0, 2)])
def test_a_split_without_a_finite_score_weighs_nothing(engine, dtype, dim, empty):
    # four workgroups of 128 tokens a row: some with scores of -infinity alone,
    # the others' so far below zero that 2^score is 0
    gen = torch.Generator().manual_seed(dim)
    kv = make(engine, gen, [500, 400], 2, dim, 16, dtype)
    for s in (0, 1):
        for j, page in enumerate(kv.tables[s, :-(-[500, 400][s] // 16)].tolist()):
            kv.pool[page, 0, 0, :, :, 0] = -float("inf") if j // 8 in empty else -480.0
    q = torch.randn(2, 6, dim, generator=gen).to(DEV).to(dtype)
    q[:, :, 0] = 1.0
    out = run(engine, kv, 0, q, [0, 1], scale=1.0)
    check(kv, 0, q, [0, 1], out, scale=1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 256])
def test_int16_rows_over_keys_of_infinity(engine, dtype, dim):
    # q of every kind of bits (a byte of zeros above or below, either sign) against
    # keys that are infinite in one place: -infinity weighs nothing, and the rest
    # of the row is what it is without them; +infinity makes the row NaN
    steps = [256, 1, -1, 255, -255, -256, 127, 128, 129, -128, -32768, 32767, 32512, 3, 511, -512]
    gen = torch.Generator().manual_seed(dim)
    lens = [300] * len(steps)
    kv = make(engine, gen, lens, 1, dim, 16, dtype)
    q = torch.randint(-40, 41, (len(steps), 4, dim), generator=gen, dtype=torch.int16).to(DEV)
    for i, x in enumerate(steps):
        q[i, :, 5] = x
        for j in (0, 3, 18):
            kv.pool[kv.tables[i, j], 0, 0, :, 7, 5] = -float("inf") if x > 0 else float("inf")
    # 13 fraction bits: the largest q is 4, scores stay within a few
    out = run(engine, kv, 0, q, list(range(len(steps))), frac=13, out_frac=12)
    check(kv, 0, q, list(range(len(steps))), out, unit=2.0 ** -13, out_unit=2.0 ** -12)
    for i, x in enumerate(steps):
        kv.pool[kv.tables[i, 0], 0, 0, :, 7, 5] *= -1
    torch.cuda.synchronize()
    out = run(engine, kv, 0, q, list(range(len(steps))), frac=13, out_frac=12)
    assert (out == -32768).all()                   # NaN as int16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", [600.0, 1100.0, 1.2e4, 6e4])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_millions(engine, dtype, size, sign):
    # scores of 2^k for whole k, exact in float32 as 64 equal products; the
    # largest weighs 1, those 64 and more below it nothing, whatever their size
    kv = make(engine, torch.Generator().manual_seed(3), [300, 200], 1, 64, 16, dtype)
    near = 2.0 ** math.floor(math.log2(size))
    for s in (0, 1):
        for j, page in enumerate(kv.tables[s, :-(-[300, 200][s] // 16)].tolist()):
            kv.pool[page, 0, 0] = sign * near * (1.0 if sign < 0 else 0.5)
            if j == 5:
                kv.pool[page, 0, 0, :, 3] = sign * near * (0.5 if sign < 0 else 1.0)
    q = torch.full((2, 2, 64), near, device=DEV).to(dtype)
    out = run(engine, kv, 0, q, [0, 1], scale=1.0)
    for s in (0, 1):
        assert torch.equal(out[s], kv.pool[kv.tables[s, 5], 0, 1, :, 3].expand(2, -1))
