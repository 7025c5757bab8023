"""The mixers between a step's sites, on device tensors: attention over a
paged key-value cache with the cache's pages (PagedKV), and the gated delta
rule (the delta_* methods of engine.Context).

Everything is enqueued on the context's stream and nothing waits.  Lists
(sequences, positions, pages, slots) are int32 device tensors, a negative
entry is padding; what they hold is checked on the device and reported, as an
AssertionError, by the next Context.sync().  Activations are float32,
bfloat16, float16 or the engine's own int16 with `frac` fraction bits; they
may be strided, with a contiguous last dimension, 16-byte aligned.  No output
or workspace overlaps an input or another output.

A call's tensors, lists and workspaces too, are used after it has returned:
they are made before the context's stream gets to the call, and kept, unwritten,
until the work is done (a tensor made in the call's own brackets is torch's
again at once).  A captured graph needs its PagedKVs open as long as it is
replayed.
"""
import ctypes
import math
import struct

from . import _native as N

_DTYPES = {}


def _dtypes():
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float32: N.DT_F32, torch.bfloat16: N.DT_BF16,
                        torch.float16: N.DT_F16, torch.int16: N.DT_I16,
                        torch.int32: None, None: torch.int32})
    return _DTYPES


def _on(t, ctx, name):
    try:
        if t.get_device() == ctx.device:
            return
    except AttributeError:
        pass
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{name}: must be a device tensor")
    raise ValueError(f"{name}: is on device {t.device.index}, the context on {ctx.device}")


def _act(t, ctx, name, shape, dtype=None):
    """(pointer, stride of dimension 0, of dimension 1) of an activation
    tensor of the given shape (and dtype, where one is given)."""
    _on(t, ctx, name)
    if t.shape != shape:
        raise ValueError(f"{name}: has shape {tuple(t.shape)}, the call takes {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: is {t.dtype}, the call takes {dtype}")
    s0, s1, s2 = t.stride()
    if s2 != 1 and shape[2] > 1:
        raise ValueError(f"{name}: its last dimension must be contiguous")
    # the stride of a dimension of one entry is never used
    return t.data_ptr(), s0 if shape[0] > 1 else 0, s1 if shape[1] > 1 else 0


def _list(t, ctx, name, n=None):
    """Pointer of an int32 list of n entries (any number where n is None)."""
    try:
        shape = t.shape
        if t.get_device() == ctx.device and len(shape) == 1 and (n is None or shape[0] == n) \
                and t.dtype is _DTYPES.get(None) and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _on(t, ctx, name)
    if t.dim() != 1 or _dtypes().get(t.dtype, 0) is not None or not t.is_contiguous():
        raise ValueError(f"{name}: must be a contiguous int32 vector")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name}: has {t.shape[0]} entries, the call takes {n}")
    return t.data_ptr()


def _gate(t, ctx, name, shape):
    import torch
    _on(t, ctx, name)
    if t.shape != shape or t.dtype != torch.float32:
        raise ValueError(f"{name}: must be float32 of shape {tuple(shape)}")
    if t.stride(1) != 1 and shape[1] > 1:
        raise ValueError(f"{name}: its last dimension must be contiguous")
    return t.data_ptr(), t.stride(0) if shape[0] > 1 else 0


def _workspace(ctx, nbytes):
    import torch
    return torch.empty(int(nbytes), dtype=torch.uint8, device=torch.device("cuda", ctx.device))


class PagedKV:
    """A key-value cache in pages, over the caller's device tensors:

      pool    [pages, layers, 2, kv_heads, page_tokens, head_dim], float32,
              bfloat16 or float16 (keys at 0, values at 1); page_tokens a power
              of two from 16 to 1024, head_dim 64, 128 or 256
      refs    int32 [pages]: how many sequences hold a page, 0: free
      tables  int32 [seqs, max_pages]: each sequence's pages
      lens    int32 [seqs]: its tokens

    Zeros in refs and lens are an empty cache; `PagedKV.empty` makes one.  All
    four are the cache's state and may be read, saved and restored by the
    caller between calls on the same stream.  Calls on one cache from several
    streams must be ordered by the caller."""

    def __init__(self, ctx, pool, refs, tables, lens):
        dt = _dtypes()
        for t, name, dims, types in (
                (pool, "pool", 6, (N.DT_F32, N.DT_BF16, N.DT_F16)), (refs, "refs", 1, (None,)),
                (tables, "tables", 2, (None,)), (lens, "lens", 1, (None,))):
            _on(t, ctx, name)
            if t.dim() != dims or not t.is_contiguous() or dt.get(t.dtype, -1) not in types:
                raise ValueError(f"{name}: a contiguous tensor of {dims} dimensions and a cache's "
                                 f"type is required, not {t.dtype} {tuple(t.shape)}")
        pages, layers, two, heads, page, dim = pool.shape
        if two != 2:
            raise ValueError("pool: the third dimension holds keys and values")
        if refs.shape[0] != pages or tables.shape[0] != lens.shape[0]:
            raise ValueError("refs has an entry per page, tables and lens one per sequence")
        h = ctypes.c_void_p()
        N.check(N.lib().w4a8_kv_create(
            ctx.h, dt[pool.dtype], pages, layers, heads, page, dim, tables.shape[0],
            tables.shape[1], pool.data_ptr(), refs.data_ptr(), tables.data_ptr(),
            lens.data_ptr(), ctypes.byref(h)), "kv_create")
        self.ctx, self.h = ctx, h
        ctx.caches.add(self)
        self.pool, self.refs, self.tables, self.lens = pool, refs, tables, lens
        self.kv_heads, self.page_tokens, self.head_dim = heads, page, dim
        self.scale = 1.0 / math.sqrt(dim)
        self.dtype, self._type, self._types = pool.dtype, dt[pool.dtype], dt

    @classmethod
    def empty(cls, ctx, pages, layers, kv_heads, page_tokens, head_dim, seqs, max_pages, dtype):
        """An empty cache with tensors of its own."""
        import torch
        dev = torch.device("cuda", ctx.device)
        ints = dict(dtype=torch.int32, device=dev)
        kv = cls(ctx, torch.zeros((pages, layers, 2, kv_heads, page_tokens, head_dim),
                                  dtype=dtype, device=dev),
                 torch.zeros(pages, **ints), torch.full((seqs, max_pages), -1, **ints),
                 torch.zeros(seqs, **ints))
        torch.cuda.synchronize(dev)   # the fills before the engine's stream uses them
        return kv

    def _act_type(self, t, name):
        dtype = t.dtype
        if dtype is self.dtype:
            return self._type
        if self._types.get(dtype) != N.DT_I16:
            raise ValueError(f"{name}: must be {self.dtype}, as the cache, or int16")
        return N.DT_I16

    def extend_async(self, seqs, counts):
        """Sequence seqs[i] grows by counts[i] tokens, pages added as needed:
        lowest free page first, in the order of the list, all or nothing.  A
        refused call (the next sync reports it) stops the cache until that
        sync: calls behind it change nothing."""
        p = _list(seqs, self.ctx, "seqs")
        N.check(N.lib().w4a8_kv_extend_async(
            self.h, p, _list(counts, self.ctx, "counts", seqs.shape[0]), seqs.shape[0]),
            "kv_extend")

    def append_async(self, layer, k, v, seqs, pos=None, frac=0):
        """Keys and values [n, kv_heads, head_dim] of n tokens of one layer, to
        sequence seqs[i] at position pos[i] (its last token without pos)."""
        n, dev = seqs.shape[0], self.ctx.device
        shape = (n, self.kv_heads, self.head_dim)
        dt = self._act_type(k, "k")
        if k.shape == shape and v.shape == shape and v.dtype is k.dtype \
                and k.get_device() == dev and v.get_device() == dev:
            (k0, k1, k2), (v0, v1, v2) = k.stride(), v.stride()
        else:
            k2 = None
        if k2 != 1 or v2 != 1 or n <= 1 or self.kv_heads == 1:   # refused, or unused strides
            kp, k0, k1 = _act(k, self.ctx, "k", shape)
            vp, v0, v1 = _act(v, self.ctx, "v", shape, k.dtype)
        else:
            kp, vp = k.data_ptr(), v.data_ptr()
        N.check(N.lib().w4a8_kv_append_async(
            self.h, layer, dt, frac, kp, k0, k1, vp, v0, v1, _list(seqs, self.ctx, "seqs"),
            None if pos is None else _list(pos, self.ctx, "pos", n), n), "kv_append")

    def attend_workspace(self, rows, q_heads):
        """Device memory for attend_async with this many rows and query heads;
        calls that can overlap, graphs' replays among them, need one each."""
        b = ctypes.c_int64()
        N.check(N.lib().w4a8_kv_attend_workspace(self.h, rows, q_heads, ctypes.byref(b)),
                "kv_attend_workspace")
        return _workspace(self.ctx, b.value)

    def attend_async(self, layer, q, seqs, out, ws, upto=None, scale=None, frac=0, out_frac=0):
        """out [rows, q_heads, head_dim] = attention of q over the tokens of
        sequence seqs[row] (the first upto[row] of them, where given).  scale:
        1 / sqrt(head_dim) unless given.  A row without tokens gets zeros."""
        n, hq = q.shape[0], q.shape[1]
        shape = (n, hq, self.head_dim)
        dt = self._act_type(q, "q")
        qp, q0, q1 = _act(q, self.ctx, "q", shape)
        op, o0, o1 = _act(out, self.ctx, "out", shape, q.dtype)
        _on(ws, self.ctx, "ws")
        if not ws.is_contiguous():
            raise ValueError("ws: must be contiguous")
        N.check(N.lib().w4a8_kv_attend_async(
            self.h, layer, dt, frac, out_frac, qp, q0, q1, op, o0, o1,
            _list(seqs, self.ctx, "seqs", n),
            None if upto is None else _list(upto, self.ctx, "upto", n), n, hq,
            self.scale if scale is None else scale, ws.data_ptr(), ws.nbytes), "kv_attend")

    def fork_async(self, parents, children):
        """Sequence children[i], empty, becomes a copy of parents[i]: full
        pages shared, the used tokens of the last page copied; all or nothing,
        and what it stops, as extend_async."""
        p = _list(parents, self.ctx, "parents")
        n = parents.shape[0]
        N.check(N.lib().w4a8_kv_fork_async(
            self.h, p, _list(children, self.ctx, "children", n), n), "kv_fork")

    def free_async(self, seqs):
        """The listed sequences become empty; pages no other holds are free."""
        N.check(N.lib().w4a8_kv_free_async(self.h, _list(seqs, self.ctx, "seqs"),
                                           seqs.shape[0]), "kv_free")

    def compact_async(self):
        """The pages in use become the pool's first; refs and tables follow."""
        N.check(N.lib().w4a8_kv_compact_async(self.h), "kv_compact")

    def copy_async(self, src, dst):
        """Page src[i] copied to page dst[i], whole."""
        n = src.shape[0]
        N.check(N.lib().w4a8_kv_copy_async(self.h, _list(src, self.ctx, "src"),
                                           _list(dst, self.ctx, "dst", n), n), "kv_copy")

    def close(self):
        """Frees the handle's scratch memory, not the caller's tensors; done
        by the context's close() too."""
        if self.h:
            N.lib().w4a8_kv_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            if self.h and self.ctx.h:
                self.close()
        except Exception:
            pass


# w4a8_delta: ten pointers, ws_bytes, ten strides, tokens, rows, hk, hv, dk, dv,
# nslots, dtype, frac, out_frac, norm, fresh, scale, eps
_DELTA = struct.Struct("=10Q23q2d")


def _delta_fault(ctx, q, k, v, g, beta, state, out):
    """What is wrong with the tensors of a delta-rule call, as a ValueError."""
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (g, "g"), (beta, "beta"), (state, "state"),
                    (out, "out")):
        _on(t, ctx, name)
    if q.dim() != 3 or v.dim() != 3 or state.dim() != 4:
        raise ValueError("q, k [tokens, hk, dk], v, out [tokens, hv, dv] and "
                         "state [slots, hv, dk, dv] are required")
    tokens, hk, dk = q.shape
    hv, dv = v.shape[1], v.shape[2]
    if _dtypes().get(q.dtype) is None:
        raise ValueError(f"q: float32, bfloat16, float16 or int16, not {q.dtype}")
    _act(q, ctx, "q", (tokens, hk, dk))
    _act(k, ctx, "k", (tokens, hk, dk), q.dtype)
    _act(v, ctx, "v", (tokens, hv, dv), q.dtype)
    _act(out, ctx, "out", (tokens, hv, dv), q.dtype)
    _gate(g, ctx, "g", (tokens, hv))
    _gate(beta, ctx, "beta", (tokens, hv))
    raise ValueError(f"state: must be contiguous float32 [slots, {hv}, {dk}, {dv}]")


def delta_args(ctx, q, k, v, g, beta, state, out, cu, ws, slots, scale, norm, eps, fresh, frac,
               out_frac):
    """The checked arguments of one delta-rule call, packed as w4a8_delta.
    The checks of the tensors are one condition (a step is a few microseconds
    on the device); what does not hold is told by _delta_fault."""
    dts, dev = _dtypes(), ctx.device
    try:
        qt = q.dtype
        dt = dts.get(qt)
        tokens, hk, dk = qs = q.shape
        _, hv, dv = vs = v.shape
        q0, q1, q2 = q.stride()
        k0, k1, k2 = k.stride()
        v0, v1, v2 = v.stride()
        o0, o1, o2 = out.stride()
        g0, g1 = g.stride()
        b0, b1 = beta.stride()
        slots_n, *heads = state.shape
        fine = (dt is not None and q.get_device() == dev and k.get_device() == dev
                and v.get_device() == dev and out.get_device() == dev and g.get_device() == dev
                and beta.get_device() == dev and state.get_device() == dev
                and k.dtype is qt and v.dtype is qt and out.dtype is qt
                and k.shape == qs and out.shape == vs and vs[0] == tokens
                and g.shape == beta.shape == (tokens, hv) and heads == [hv, dk, dv]
                and q2 == k2 == v2 == o2 == 1 and (g1 == b1 == 1 or hv == 1)
                and dts.get(g.dtype) == dts.get(beta.dtype) == dts.get(state.dtype) == N.DT_F32
                and state.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        fine = False
    if not fine:
        _delta_fault(ctx, q, k, v, g, beta, state, out)
    # the stride of a dimension of one entry is never used
    if tokens == 1:
        q0 = k0 = v0 = o0 = g0 = b0 = 0
    if hk == 1:
        q1 = k1 = 0
    if hv == 1:
        v1 = o1 = 0
    rows = tokens if cu is None else cu.shape[0] - 1
    if rows < 0:
        raise ValueError("cu: needs an entry per row and one more")
    wp, wb = 0, 0
    if ws is not None:
        _on(ws, ctx, "ws")
        if not ws.is_contiguous():
            raise ValueError("ws: must be contiguous")
        wp, wb = ws.data_ptr(), ws.nbytes
    return _DELTA.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
        state.data_ptr(), out.data_ptr(),
        0 if slots is None else _list(slots, ctx, "slots", rows),
        0 if cu is None else _list(cu, ctx, "cu"), wp, wb,
        q0, q1, k0, k1, v0, v1, o0, o1, g0, b0, tokens, rows, hk, hv, dk, dv, slots_n, dt,
        frac, out_frac, 1 if norm else 0, 1 if fresh else 0,
        1.0 / math.sqrt(dk) if scale is None else scale, eps)


def delta_workspace(ctx, tokens, rows, hv, hk, dk, dtype):
    b = ctypes.c_int64()
    dt = N.DT_F32 if dtype is None else _dtypes().get(dtype)
    if dt is None:
        raise ValueError(f"dtype: float32, bfloat16, float16 or int16, not {dtype}")
    N.check(N.lib().w4a8_delta_chunk_workspace(
        ctx.h, tokens, rows, hv if hk is None else hk, hv, dk, dt, ctypes.byref(b)),
        "delta_chunk_workspace")
    return _workspace(ctx, b.value)
