"""Run by test_prompt_host.py in a process of its own, with the stand-in runtime
loaded before the library: prompt_check.py RUNTIME CHECK."""
import ctypes
import sys

import fake_hip

OK, E_HIP, E_ARG = 0, -5, -6
F32, BF16, F16, I16, I32 = 0, 1, 2, 3, 4

rt, lib = fake_hip.load(sys.argv[1])
P, I64, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double
lib.w4a8_last_error.restype = ctypes.c_char_p
ctx = P()
assert lib.w4a8_ctx_create(0, ctypes.byref(ctx)) == OK
PTR, ODD = P(0x10000), P(0x10002)      # never followed: kernels do nothing here
EIGHT = P(0x10008)


def cache(dtype=BF16, heads=4, page=16, dim=128, max_pages=5, layers=2):
    h = P()
    assert lib.w4a8_kv_create(ctx, dtype, 8, layers, heads, page, dim, 3, max_pages, PTR, PTR, PTR,
                              PTR, ctypes.byref(h)) == OK
    return h


def refused(call, what=E_ARG):
    """The call is refused and launches nothing."""
    before = rt.fake_launches()
    rc = call()
    assert rc == what, (rc, lib.w4a8_last_error())
    assert rt.fake_launches() == before
    assert what == OK or lib.w4a8_last_error()


def plan_bytes(h, rows=2, tokens=40, heads=8):
    b = I64()
    rc = lib.w4a8_kv_plan_bytes(h, rows, tokens, heads, ctypes.byref(b))
    return rc, b.value


def step(h, seqs=PTR, counts=PTR, rows=2, tokens=40, heads=8, cu=PTR, ts=PTR, pos=PTR, slots=PTR,
         plan=PTR, nbytes=1 << 30):
    return lib.w4a8_kv_map_async(h, seqs, counts, rows, tokens, heads, cu, ts, pos, slots, plan,
                                 I64(nbytes))


def check_map():
    h = cache()
    rc, need = plan_bytes(h)
    assert rc == OK and need > 0
    assert step(h, nbytes=need) == OK and step(h, rows=3000) == OK
    assert step(h, rows=0, tokens=0, seqs=None, counts=None, ts=None, pos=None, slots=None) == OK
    for kw in (dict(rows=-1), dict(tokens=-1), dict(rows=(1 << 20) + 1), dict(tokens=(1 << 20) + 1),
               dict(heads=0), dict(heads=6), dict(heads=1 << 17), dict(seqs=None),
               dict(counts=None), dict(cu=None), dict(ts=None), dict(pos=None), dict(slots=None),
               dict(slots=P(0x10004)), dict(seqs=ODD), dict(counts=ODD), dict(cu=ODD),
               dict(ts=ODD), dict(pos=ODD), dict(plan=None), dict(plan=EIGHT),
               dict(nbytes=need - 1)):
        refused(lambda kw=kw: step(h, **kw))
    refused(lambda: step(None))
    refused(lambda: plan_bytes(None)[0])
    refused(lambda: plan_bytes(h, heads=9)[0])
    refused(lambda: plan_bytes(h, rows=1 << 20, tokens=1 << 20, heads=512)[0])
    refused(lambda: lib.w4a8_kv_plan_bytes(h, 2, 40, 8, None))


def attend(h, layer=0, q=PTR, q0=1024, q1=128, dtype=BF16, frac=0, out=PTR, o0=1024, o1=128,
           plan=PTR, nbytes=1 << 30, rows=2, tokens=40, heads=8, scale=0.1, ws=PTR,
           ws_bytes=1 << 40):
    return lib.w4a8_kv_attend_chunk_async(h, layer, q, I64(q0), I64(q1), dtype, frac, out, I64(o0),
                                          I64(o1), plan, I64(nbytes), rows, tokens, heads,
                                          F64(scale), ws, I64(ws_bytes))


def check_attend():
    for dtype in (BF16, F16, F32):
        for dim in (64, 128, 256):
            h = cache(dtype=dtype, dim=dim, max_pages=500)
            b = I64()
            assert lib.w4a8_kv_attend_chunk_workspace(h, 2, 40, 8, ctypes.byref(b)) == OK
            assert b.value > 0
            assert attend(h, dtype=dtype, ws_bytes=b.value) == OK
            assert attend(h, dtype=I16, frac=12) == OK
    h = cache(max_pages=500)
    assert lib.w4a8_kv_attend_chunk_workspace(h, 2, 40, 8, ctypes.byref(b)) == OK
    need = plan_bytes(h)[1]
    refused(lambda: attend(h, tokens=0), OK)
    refused(lambda: attend(h, rows=0), OK)
    for kw in (dict(layer=2), dict(layer=-1), dict(dtype=F32), dict(dtype=F16), dict(frac=32),
               dict(frac=-1), dict(q=None), dict(out=None), dict(q=ODD), dict(out=ODD),
               dict(q0=1023), dict(q1=2), dict(o0=-1024), dict(o1=129), dict(plan=None),
               dict(plan=EIGHT), dict(nbytes=need - 1), dict(rows=-1), dict(heads=6),
               dict(tokens=-1), dict(ws=None), dict(ws=ODD), dict(ws_bytes=b.value - 1)):
        refused(lambda kw=kw: attend(h, **kw))
    refused(lambda: attend(None))
    refused(lambda: lib.w4a8_kv_attend_chunk_workspace(h, 2, 40, 8, None))
    refused(lambda: lib.w4a8_kv_attend_chunk_workspace(h, 2, 40, 9, ctypes.byref(b)))


class Rotary(ctypes.Structure):
    _fields_ = [(n, P) for n in ("q", "k", "v", "q_out", "k_out", "pos", "slots", "freq", "q_norm",
                                 "k_norm")] + \
        [(n, I64) for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head",
                            "q_out_token", "q_out_head", "k_out_token", "k_out_head", "tokens",
                            "q_heads", "k_heads", "dim", "rot", "pairs", "dtype", "frac",
                            "out_dtype", "out_frac")] + \
        [("amplitude", F64), ("eps", F64)]


def rotary(**kw):
    d = Rotary(q=PTR, k=PTR, v=PTR, q_out=PTR, k_out=PTR, pos=PTR, slots=PTR, freq=PTR, q_norm=PTR,
               k_norm=PTR, q_token=1024, q_head=128, k_token=512, k_head=128, v_token=512,
               v_head=128, q_out_token=1024, q_out_head=128, k_out_token=512, k_out_head=128,
               tokens=3, q_heads=8, k_heads=4, dim=128, rot=64, dtype=BF16, out_dtype=BF16,
               amplitude=1.0, eps=1e-6)
    for n, v in kw.items():
        setattr(d, n, v)
    return ctypes.byref(d)


def check_rotary():
    f, g, h = lib.w4a8_rotary_async, lib.w4a8_kv_append_rotary_async, cache()
    assert f(ctx, rotary()) == OK and g(h, 1, rotary()) == OK
    assert f(ctx, rotary(q_heads=0, q=None, q_out=None)) == OK
    assert f(ctx, rotary(k_heads=0, k=None, k_out=None)) == OK
    assert f(ctx, rotary(rot=0, freq=None, q_norm=None, k_norm=None)) == OK
    for out in (F32, BF16, F16, I16):
        assert f(ctx, rotary(dtype=I16, out_dtype=out)) == OK
    assert g(h, 0, rotary(dtype=I16, frac=8)) == OK
    refused(lambda: f(ctx, rotary(tokens=0)), OK)
    refused(lambda: f(None, rotary()))
    refused(lambda: f(ctx, None))
    refused(lambda: g(None, 0, rotary()))
    refused(lambda: g(h, 0, None))
    nan = float("nan")
    both = [dict(dtype=4), dict(dtype=-1), dict(frac=32), dict(frac=-1), dict(out_frac=99),
            dict(rot=24), dict(rot=144), dict(rot=-16), dict(freq=None), dict(freq=0x10004),
            dict(tokens=-1), dict(tokens=(1 << 20) + 1), dict(q_heads=-1), dict(q_heads=1 << 16),
            dict(q_norm=ODD.value), dict(k_norm=ODD.value), dict(amplitude=nan), dict(eps=nan),
            dict(eps=-1.0), dict(tokens=1 << 20, q_heads=200), dict(pos=None),
            dict(pos=ODD.value), dict(q=None), dict(q=ODD.value), dict(q_out=EIGHT.value),
            dict(q_token=3), dict(q_out_head=-8), dict(k=None), dict(k_token=4),
            dict(dtype=F16)]
    for kw in both + [dict(out_dtype=F32), dict(out_dtype=I16), dict(dim=0), dict(dim=24),
                      dict(dim=272), dict(k_out=None), dict(k_out_head=1), dict(k_heads=-1),
                      dict(q_heads=0, k_heads=0)]:
        refused(lambda kw=kw: f(ctx, rotary(**kw)))
    for kw in both + [dict(out_dtype=F16, dtype=F16), dict(dim=64), dict(k_heads=2),
                      dict(v=None), dict(v=ODD.value), dict(v_head=1), dict(slots=None),
                      dict(slots=0x10004)]:
        refused(lambda kw=kw: g(h, 0, rotary(**kw)))
    for layer in (-1, 2):
        refused(lambda: g(h, layer, rotary()))


class Logprobs(ctypes.Structure):
    _fields_ = [(n, P) for n in ("logits", "ids", "logp", "entropy", "top_logp", "top_ids",
                                 "ws")] + \
        [(n, I64) for n in ("ws_bytes", "row", "rows", "vocab", "k", "dtype")] + [("scale", F64)]


def logprobs(**kw):
    d = Logprobs(logits=PTR, ids=PTR, logp=PTR, entropy=PTR, top_logp=PTR, top_ids=PTR, ws=PTR,
                 ws_bytes=1 << 40, row=50000, rows=3, vocab=50000, k=8, dtype=F32, scale=1.0)
    for n, v in kw.items():
        setattr(d, n, v)
    return ctypes.byref(d)


def check_logprobs():
    f, b = lib.w4a8_logprobs_async, I64()

    def space(rows, vocab, to=b, c=ctx):
        return lib.w4a8_logprobs_workspace(c, I64(rows), I64(vocab),
                                           None if to is None else ctypes.byref(to))
    assert space(3, 50000) == OK and b.value > 0
    assert f(ctx, logprobs(ws_bytes=b.value)) == OK
    need = b.value
    for dtype in (F32, BF16, F16, I32):
        assert f(ctx, logprobs(dtype=dtype)) == OK
    assert f(ctx, logprobs(dtype=BF16, logits=ODD.value, row=50001)) == OK
    assert f(ctx, logprobs(ids=None, logp=None, entropy=None)) == OK
    assert f(ctx, logprobs(k=0, top_logp=None, top_ids=None)) == OK
    refused(lambda: f(ctx, logprobs(rows=0)), OK)
    assert space(0, 1) == OK and b.value == 0
    for args in ((-1, 5), ((1 << 20) + 1, 5), (3, 0), (3, (1 << 24) + 1)):
        refused(lambda args=args: space(*args))
    refused(lambda: space(3, 5, to=None))
    refused(lambda: space(3, 5, c=None))
    refused(lambda: f(None, logprobs()))
    refused(lambda: f(ctx, None))
    for kw in (dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(dtype=I16),
               dict(dtype=5), dict(dtype=-1), dict(k=-1), dict(k=33), dict(vocab=7, k=8),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(scale=1e-50), dict(logits=None),
               dict(logits=ODD.value), dict(row=-1), dict(ids=None), dict(logp=None),
               dict(top_logp=None), dict(top_ids=None), dict(entropy=ODD.value),
               dict(ids=ODD.value), dict(ws=None), dict(ws=EIGHT.value), dict(ws_bytes=need - 1)):
        refused(lambda kw=kw: f(ctx, logprobs(**kw)))


def check_launches():
    """A launch that fails is the call's error, and the next call's is its own."""
    h = cache(max_pages=500)
    for f in (lambda: step(h), lambda: attend(h),
              lambda: lib.w4a8_rotary_async(ctx, rotary()),
              lambda: lib.w4a8_kv_append_rotary_async(h, 0, rotary()),
              lambda: lib.w4a8_logprobs_async(ctx, logprobs())):
        rt.fake_set(1, 0, 0, 0)
        assert f() == E_HIP
        rt.fake_set(0, 0, 0, 0)
        assert f() == OK


globals()["check_" + sys.argv[2]]()
print("ok")
