"""Run by test_mixers_host.py in a process of its own, with the stand-in
runtime loaded before the library: mixers_check.py RUNTIME CHECK."""
import ctypes
import sys

import fake_hip

OK, E_HIP, E_ARG = 0, -5, -6
F32, BF16, F16, I16 = 0, 1, 2, 3

rt, lib = fake_hip.load(sys.argv[1])
P, I64 = ctypes.c_void_p, ctypes.c_int64
lib.w4a8_last_error.restype = ctypes.c_char_p
ctx = P()
assert lib.w4a8_ctx_create(0, ctypes.byref(ctx)) == OK
PTR, ODD = P(0x10000), P(0x10002)      # never followed: kernels do nothing here


def cache(dtype=BF16, pages=8, layers=2, heads=4, page=16, dim=128, seqs=3, max_pages=5,
          pool=PTR, refs=PTR, tables=PTR, lens=PTR):
    h = P()
    rc = lib.w4a8_kv_create(ctx, dtype, pages, layers, heads, page, dim, seqs, max_pages, pool,
                            refs, tables, lens, ctypes.byref(h))
    assert (rc == OK) == bool(h)
    return rc, h


def refused(call, *args, what=E_ARG):
    """The call with these arguments is refused and launches nothing."""
    before = rt.fake_launches()
    rc = call(*args)
    assert rc == what, (rc, args, lib.w4a8_last_error())
    assert rt.fake_launches() == before, args
    assert what == OK or lib.w4a8_last_error()


def check_cache():
    for page in (16, 64, 1024):
        rc, h = cache(page=page)
        assert rc == OK and lib.w4a8_kv_destroy(h) == OK
    for kw in (dict(dtype=I16), dict(dtype=-1), dict(pages=0), dict(layers=0), dict(heads=0),
               dict(page=8), dict(page=24), dict(page=2048), dict(dim=96), dict(dim=0),
               dict(seqs=0), dict(max_pages=0), dict(pool=None), dict(refs=None),
               dict(tables=None), dict(lens=None), dict(pool=ODD), dict(refs=ODD),
               dict(tables=ODD), dict(lens=ODD), dict(pages=(1 << 30) + 1),
               dict(max_pages=(1 << 20) + 1, page=1024)):
        refused(lambda kw=kw: cache(**kw)[0])
    assert lib.w4a8_kv_destroy(None) == OK
    rt.fake_set(1, 0, 0, 0)              # the clearing of its scratch fails
    assert cache()[0] == E_HIP
    rt.fake_set(0, 0, 0, 0)


def check_lists():
    _, h = cache()
    two = (lib.w4a8_kv_extend_async, lib.w4a8_kv_fork_async, lib.w4a8_kv_copy_async)
    for f in two:
        refused(f, None, PTR, PTR, 3)
        refused(f, h, None, PTR, 3)
        refused(f, h, PTR, None, 3)
        refused(f, h, PTR, PTR, -1)
        refused(f, h, PTR, PTR, (1 << 20) + 1)
        refused(f, h, None, None, 0, what=OK)
    refused(lib.w4a8_kv_free_async, None, PTR, 1)
    refused(lib.w4a8_kv_free_async, h, None, 1)
    refused(lib.w4a8_kv_free_async, h, None, 0, what=OK)
    refused(lib.w4a8_kv_compact_async, None)


def append(h, layer=0, dtype=BF16, frac=0, k=PTR, k0=512, k1=128, v=PTR, v0=512, v1=128,
           seqs=PTR, pos=None, n=3):
    return lib.w4a8_kv_append_async(h, layer, dtype, frac, k, I64(k0), I64(k1), v, I64(v0),
                                    I64(v1), seqs, pos, n)


def check_append():
    _, h = cache()
    assert append(h) == OK and append(h, dtype=I16, frac=8) == OK
    refused(lambda: append(h, n=0), what=OK)
    for kw in (dict(layer=-1), dict(layer=2), dict(dtype=F16), dict(dtype=F32), dict(dtype=4),
               dict(frac=-1), dict(frac=32), dict(k=None), dict(v=None), dict(k=ODD),
               dict(v=ODD), dict(k0=513), dict(k1=4), dict(v0=-8), dict(v1=1), dict(seqs=None),
               dict(n=-1)):
        refused(lambda kw=kw: append(h, **kw))
    refused(lambda: append(None))


def attend(h, layer=0, dtype=BF16, frac=0, out_frac=0, q=PTR, q0=1024, q1=128, out=PTR, o0=1024,
           o1=128, seqs=PTR, upto=None, rows=2, heads=8, ws=PTR, ws_bytes=1 << 24):
    return lib.w4a8_kv_attend_async(h, layer, dtype, frac, out_frac, q, I64(q0), I64(q1), out,
                                    I64(o0), I64(o1), seqs, upto, rows, heads,
                                    ctypes.c_double(0.1), ws, I64(ws_bytes))


def check_attend():
    _, h = cache(max_pages=500)
    b = I64()
    assert lib.w4a8_kv_attend_workspace(h, 2, 8, ctypes.byref(b)) == OK and b.value > 0
    assert attend(h, ws_bytes=b.value) == OK
    refused(lambda: attend(h, rows=0), what=OK)
    for kw in (dict(layer=2), dict(layer=-1), dict(dtype=F32), dict(frac=40), dict(out_frac=-2),
               dict(q=None), dict(out=None), dict(q=ODD), dict(out=ODD), dict(q0=1023),
               dict(q1=2), dict(o0=-1024), dict(o1=129), dict(seqs=None), dict(rows=-1),
               dict(heads=6), dict(heads=0), dict(ws=None), dict(ws=ODD),
               dict(ws_bytes=b.value - 1), dict(rows=(1 << 20) + 1), dict(rows=1 << 20, heads=16)):
        refused(lambda kw=kw: attend(h, **kw))
    refused(lambda: attend(None))
    refused(lib.w4a8_kv_attend_workspace, h, 2, 9, ctypes.byref(b))
    refused(lib.w4a8_kv_attend_workspace, h, 2, 8, None)


class Delta(ctypes.Structure):
    _fields_ = [(n, P) for n in ("q", "k", "v", "g", "beta", "state", "out", "slots", "cu",
                                 "ws")] + \
        [(n, I64) for n in ("ws_bytes", "q_token", "q_head", "k_token", "k_head", "v_token",
                            "v_head", "out_token", "out_head", "g_token", "beta_token", "tokens",
                            "rows", "hk", "hv", "dk", "dv", "nslots", "dtype", "frac",
                            "out_frac", "norm", "fresh")] + \
        [("scale", ctypes.c_double), ("eps", ctypes.c_double)]


def delta(**kw):
    d = Delta(q=PTR, k=PTR, v=PTR, g=PTR, beta=PTR, state=PTR, out=PTR, slots=PTR, cu=PTR, ws=PTR,
              ws_bytes=1 << 40, q_token=256, q_head=128, k_token=256, k_head=128, v_token=512,
              v_head=128, out_token=512, out_head=128, g_token=4, beta_token=4, tokens=3, rows=3,
              hk=2, hv=4, dk=128, dv=128, nslots=3, dtype=BF16, norm=1, scale=1.0, eps=1e-6)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def check_delta():
    step, chunk = lib.w4a8_delta_step_async, lib.w4a8_delta_chunk_async
    b = I64()

    def space(tokens=3, rows=3, hk=2, hv=4, dk=128, dtype=BF16, to=b):
        return lib.w4a8_delta_chunk_workspace(ctx, I64(tokens), I64(rows), I64(hk), I64(hv),
                                              I64(dk), dtype, None if to is None else ctypes.byref(to))
    sizes = []
    for dtype in (BF16, F16, F32):
        assert space(dtype=dtype) == OK
        sizes.append(b.value)
    assert 0 < sizes[0] < sizes[1] < sizes[2]
    for kw in (dict(tokens=-1), dict(rows=-1), dict(hk=0), dict(hv=1), dict(hv=1 << 16),
               dict(dk=32), dict(dtype=4), dict(to=None), dict(tokens=1 << 31)):
        refused(lambda kw=kw: space(**kw))
    for f in (step, chunk):
        assert f(ctx, ctypes.byref(delta())) == OK
        refused(f, ctx, None)
        refused(f, None, ctypes.byref(delta()))
        refused(f, ctx, ctypes.byref(delta(rows=0, tokens=0)), what=OK)
        for kw in (dict(dtype=4), dict(dtype=-1), dict(dk=96), dict(dv=24), dict(dv=8),
                   dict(dv=272), dict(hv=3), dict(hk=0), dict(hv=0), dict(rows=-1),
                   dict(tokens=-1), dict(tokens=(1 << 30) + 1), dict(rows=(1 << 20) + 1),
                   dict(rows=1 << 20, tokens=1 << 20, nslots=1 << 20), dict(nslots=-1), dict(frac=32),
                   dict(out_frac=-1), dict(slots=None, nslots=2), dict(q=None), dict(k=ODD.value),
                   dict(v=None), dict(out=ODD.value), dict(state=None), dict(state=ODD.value),
                   dict(g=None), dict(beta=ODD.value), dict(q_token=1), dict(k_head=4),
                   dict(v_token=-8), dict(out_head=7), dict(g_token=-1)):
            refused(f, ctx, ctypes.byref(delta(**kw)))
    refused(step, ctx, ctypes.byref(delta(tokens=4)))
    refused(chunk, ctx, ctypes.byref(delta(cu=None)))
    for n in ("v_token", "out_token"):
        refused(chunk, ctx, ctypes.byref(delta(**{n: (1 << 23) + 8})))
    refused(chunk, ctx, ctypes.byref(delta(ws=None)))
    refused(chunk, ctx, ctypes.byref(delta(ws=ODD.value)))
    for dtype, need in zip((BF16, F16, F32), sizes):
        assert chunk(ctx, ctypes.byref(delta(dtype=dtype, ws_bytes=need))) == OK
        refused(chunk, ctx, ctypes.byref(delta(dtype=dtype, ws_bytes=need - 1)))


def check_launches():
    """A launch that fails is the call's error, and the next call's is its own."""
    _, h = cache()
    for f in (lambda: append(h), lambda: attend(h), lambda: lib.w4a8_kv_compact_async(h),
              lambda: lib.w4a8_kv_extend_async(h, PTR, PTR, 2),
              lambda: lib.w4a8_kv_free_async(h, PTR, 2),
              lambda: lib.w4a8_delta_step_async(ctx, ctypes.byref(delta()))):
        rt.fake_set(1, 0, 0, 0)
        assert f() == E_HIP
        rt.fake_set(0, 0, 0, 0)
        assert f() == OK


globals()["check_" + sys.argv[2]]()
print("ok")
