"""Attention over 16-bit caches: the output's own rounding is the only one that
counts.  Per output, with u half a step of the cache's type, A = sum p |v| / sum
p, X the largest sum |q k| scale of a row's scores and V the largest |v|:

    u |out|          the output's rounding
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


def check(kv, layer, q, seqs, got, scale=None):
    dim, u = kv.head_dim, U[kv.pool.dtype]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    lens, per = kv.lens.tolist(), q.shape[1] // kv.kv_heads
    q, got = q.double().cpu(), got.double().cpu()
    low = 2.0 ** -39 if kv.pool.dtype == torch.float16 else 0.0
    for i, s in enumerate(seqs):
        n = lens[s]
        k, v = (x.repeat_interleave(per, 0) for x in rows_of(kv, layer, s, n))
        sc = (k @ q[i][:, :, None])[:, :, 0] * scale
        X = (k.abs() @ q[i].abs()[:, :, None]).amax().item() * scale
        p = torch.softmax(sc, -1)[:, None]
        want, A = (p @ v)[:, 0], (p @ v.abs())[:, 0]
        tol = u * want.abs() + u * u * A + low * n * v.abs().max() + \
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
