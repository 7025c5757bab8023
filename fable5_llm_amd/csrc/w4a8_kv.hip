// The pages of a key-value cache on the device: reserving, forking, freeing
// and compacting them, and writing new tokens' keys and values into them.
// Every decision (which page is free, what moves where) is taken from the
// device's own counts and tables, so that a step with them can be captured
// and replayed, and is the same from run to run: free pages are handed out
// lowest first, in the order of the list.
#include <algorithm>

#include "w4a8_mixers.h"

namespace w4a8 {

namespace {

constexpr int kOne = 1024;        // threads of the single-workgroup kernels
constexpr int kRefsPerThread = 16;
constexpr int kPiece = 16 << 10;  // bytes a workgroup copies at a time

__device__ __forceinline__ int32_t *marks(const KvCache &kv) { return kv.scratch + kKvHead; }
__device__ __forceinline__ int32_t *jobs(const KvCache &kv) { return marks(kv) + kv.seqs; }
__device__ __forceinline__ int32_t *list_a(const KvCache &kv) { return jobs(kv) + kv.seqs; }
__device__ __forceinline__ int32_t *list_b(const KvCache &kv) { return list_a(kv) + kv.pages; }

__device__ __forceinline__ int32_t held_pages(const KvCache &kv, int32_t len) {
  return (int32_t)(((int64_t)len + kv.page() - 1) >> kv.lg_page);
}

// what a reserve or a fork found wrong, by its first thread: reported, and the
// cache stopped; nothing more where the cache was stopped already
__device__ __forceinline__ void refuse(const KvCache &kv, int bad) {
  if (bad & kKvSkip) return;
  atomicOr(kv.err, bad);
  kv.scratch[kKvStop] = kv.err[1] + 1;
}

// exclusive scan of one value per thread of a kOne-thread workgroup, and the
// total; every thread of it calls
__device__ int scan_excl(int v, int *total) {
  __shared__ int sums[kOne / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();              // the last call's sums are read
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kOne / 64; ++w) {
    const int s = sums[w];
    before += w < wave ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

// the sum of one value per thread, or most where it is above that (what a list
// asks for can pass any integer); most and every value below 2^31
__device__ uint32_t sum_up_to(uint32_t v, uint32_t most) {
  __shared__ uint32_t sums[kOne / 64];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = min(v + __shfl_xor(v, d), most);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < kOne / 64; ++w) all = min(all + sums[w], most);
  return all;
}

// refs[p0 .. p0 + 16), pages past the end as 1 (in use) or 0
__device__ __forceinline__ void load_refs(const KvCache &kv, int p0, int past, int *r) {
  if (p0 + kRefsPerThread <= kv.pages) {
#pragma unroll
    for (int i = 0; i < kRefsPerThread / 4; ++i) {
      const int4 v = *(const int4 *)(kv.refs + p0 + 4 * i);
      r[4 * i] = v.x, r[4 * i + 1] = v.y, r[4 * i + 2] = v.z, r[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRefsPerThread; ++i) r[i] = p0 + i < kv.pages ? kv.refs[p0 + i] : past;
  }
}

// The counts of a thread's share of the first kOne * kRefsPerThread pages, so
// that the scans' first turn does not wait for them.
struct FirstRefs {
  int r[kRefsPerThread];
};
__device__ __forceinline__ FirstRefs first_refs(const KvCache &kv, int past) {
  FirstRefs f;
  load_refs(kv, (int)threadIdx.x * kRefsPerThread, past, f.r);
  return f;
}

// the need lowest free pages, in order, to list; how many there were (fewer
// than need: not enough).  One workgroup.
__device__ int find_free(const KvCache &kv, int need, int32_t *list, const FirstRefs &f) {
  int found = 0;
  for (int base = 0; base < kv.pages && found < need; base += kOne * kRefsPerThread) {
    int r[kRefsPerThread], mine = 0, all;
    const int p0 = base + (int)threadIdx.x * kRefsPerThread;
    if (base == 0) {
#pragma unroll
      for (int i = 0; i < kRefsPerThread; ++i) r[i] = f.r[i];
    } else {
      load_refs(kv, p0, 1, r);
    }
#pragma unroll
    for (int i = 0; i < kRefsPerThread; ++i) mine += r[i] == 0;
    int at = found + scan_excl(mine, &all);
#pragma unroll
    for (int i = 0; i < kRefsPerThread; ++i)
      if (r[i] == 0) {
        if (at < need) list[at] = p0 + i;
        ++at;
      }
    found += all;
  }
  __syncthreads();              // list is written (for this workgroup's reads)
  return found;
}

// ------------------------------------------------------------------ reserve
// One workgroup, bound by its dependent loads and barriers.  First pass: what
// is wrong with the list; second: the pages
// each sequence needs, their ranks by a scan in list order; nothing is written
// to the cache unless everything fits.
__global__ __launch_bounds__(kOne) void kv_extend_kernel(KvCache kv, const int32_t *seqs,
                                                         const int32_t *counts, int n) {
  __shared__ int bad;
  const FirstRefs refs = first_refs(kv, 1);
  const bool stopped = kv_stopped(kv);
  int32_t *mark = marks(kv), *list = list_a(kv);
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const uint32_t over = (uint32_t)kv.pages + 1;   // more than there are
  uint32_t need = 0;
  const int64_t most = (int64_t)kv.max_pages << kv.lg_page;
  for (int i = threadIdx.x; i < n; i += kOne) {
    const int s = seqs[i];
    if (s < 0) continue;
    if (s >= kv.seqs) {
      atomicOr(&bad, kErrKvRange);
      continue;
    }
    if (atomicAdd(mark + s, 1) != 0) atomicOr(&bad, kErrKvList);
    const int64_t len = kv.lens[s], c = counts[i];
    if (len < 0 || c < 0 || len + c > most || len + c > INT32_MAX)
      atomicOr(&bad, kErrKvRange);
    else
      need = min(need + held_pages(kv, (int32_t)(len + c)) - held_pages(kv, (int32_t)len), over);
  }
  if (stopped && threadIdx.x == 0) atomicOr(&bad, kKvSkip);
  const int all = (int)sum_up_to(need, over);     // synchronises: bad is whole
  const bool fine = bad == 0;
  __syncthreads();                                // and read by all
  if (fine && (all > kv.pages || (all > 0 && find_free(kv, all, list, refs) < all))) {
    if (threadIdx.x == 0) bad = kErrKvFull;
  }
  __syncthreads();
  if (!bad) {
    int from = 0;
    for (int base = 0; base < n; base += kOne) {
      const int i = base + threadIdx.x;
      const int s = i < n ? seqs[i] : -1;
      int h0 = 0, h1 = 0, len = 0, sum;
      if (s >= 0) {
        len = kv.lens[s];
        h0 = held_pages(kv, len);
        h1 = held_pages(kv, len + counts[i]);
      }
      const int at = from + scan_excl(h1 - h0, &sum);
      from += sum;
      // a thread writes its own sequence's few pages; a long run of them (a
      // prompt's) is written by its whole wavefront
      const int add = h1 - h0;
      if (s >= 0) {
        if (add <= 8)
          for (int j = 0; j < add; ++j) {
            const int p = list[at + j];
            kv.tables[(int64_t)s * kv.max_pages + h0 + j] = p;
            kv.refs[p] = 1;
          }
        kv.lens[s] = len + counts[i];
      }
      uint64_t lots = __ballot(s >= 0 && add > 8);
      while (lots) {
        const int src = __builtin_ctzll(lots);
        lots &= lots - 1;
        const int ws = __shfl(s, src), wh = __shfl(h0, src), wa = __shfl(add, src),
                  wat = __shfl(at, src);
        for (int j = threadIdx.x & 63; j < wa; j += 64) {
          const int p = list[wat + j];
          kv.tables[(int64_t)ws * kv.max_pages + wh + j] = p;
          kv.refs[p] = 1;
        }
      }
    }
  } else if (threadIdx.x == 0) {
    refuse(kv, bad);
  }
  for (int i = threadIdx.x; i < n; i += kOne) {
    const int s = seqs[i];
    if (s >= 0 && s < kv.seqs) atomicExch(mark + s, 0);
  }
}

// --------------------------------------------------------------------- fork
// First kernel, one workgroup (32 children and under 1,000 pages: 6.8 us, a chain
// of loads, marks and scans): the list's faults, a free page for each child
// of a parent whose last page is not full (jobs[child], -1 where none), the
// children's lengths.  scratch[0]: whether the second kernel runs.
__global__ __launch_bounds__(kOne) void kv_fork_kernel(KvCache kv, const int32_t *parents,
                                                       const int32_t *children, int n) {
  __shared__ int bad;
  const FirstRefs refs = first_refs(kv, 1);
  const bool stopped = kv_stopped(kv);
  int32_t *mark = marks(kv), *job = jobs(kv), *list = list_a(kv);
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  int need = 0;
  for (int i = threadIdx.x; i < n; i += kOne) {
    const int p = parents[i], c = children[i];
    if (p < 0 || c < 0) continue;
    if (p >= kv.seqs || c >= kv.seqs) {
      atomicOr(&bad, kErrKvRange);
      if (c < kv.seqs) atomicAdd(mark + c, 1);
      continue;
    }
    if (atomicAdd(mark + c, 1) != 0 || kv.lens[c] != 0) atomicOr(&bad, kErrKvList);
    const int64_t len = kv.lens[p];
    if (len < 0 || len > ((int64_t)kv.max_pages << kv.lg_page))
      atomicOr(&bad, kErrKvRange);
    else
      need += (len & (kv.page() - 1)) != 0;
  }
  int all;
  scan_excl(need, &all);
  for (int i = threadIdx.x; i < n; i += kOne) {   // a child that is a parent too
    const int p = parents[i], c = children[i];
    if (p >= 0 && c >= 0 && p < kv.seqs && atomicAdd(mark + p, 0) != 0)
      atomicOr(&bad, kErrKvList);
  }
  if (stopped && threadIdx.x == 0) atomicOr(&bad, kKvSkip);
  __syncthreads();
  const bool fine = bad == 0;
  if (fine && all > 0 && find_free(kv, all, list, refs) < all) {
    if (threadIdx.x == 0) bad = kErrKvFull;
  }
  __syncthreads();
  if (!bad) {
    int from = 0;
    for (int base = 0; base < n; base += kOne) {
      const int i = base + threadIdx.x;
      const int p = i < n ? parents[i] : -1, c = i < n ? children[i] : -1;
      const bool on = p >= 0 && c >= 0;
      const int len = on ? kv.lens[p] : 0;
      const int rest = (len & (kv.page() - 1)) != 0;
      int sum;
      const int at = from + scan_excl(rest, &sum);
      from += sum;
      if (on) {
        int page = -1;
        if (rest) {
          page = list[at];
          kv.refs[page] = 1;
        }
        job[c] = page;
        kv.lens[c] = len;
      }
    }
  } else if (threadIdx.x == 0) {
    refuse(kv, bad);
  }
  if (threadIdx.x == 0) kv.scratch[0] = bad == 0;
  for (int i = threadIdx.x; i < n; i += kOne) {
    const int p = parents[i], c = children[i];
    if (p >= 0 && c >= 0 && c < kv.seqs) atomicExch(mark + c, 0);
  }
}

// Second kernel, a row of workgroups per pair: the shared pages' entries and
// counts, and the used tokens of the last page, one run of memory per layer,
// keys or values, and head (32 children, 8 layers of 4 heads of 256: 4.6 us).
__global__ __launch_bounds__(256) void kv_fork_rows_kernel(KvCache kv, const int32_t *parents,
                                                           const int32_t *children) {
  if (kv.scratch[0] == 0) return;
  const int p = parents[blockIdx.x], c = children[blockIdx.x];
  if (p < 0 || c < 0) return;
  const int len = kv.lens[p], full = len >> kv.lg_page, rest = len & (kv.page() - 1);
  const int32_t *from = kv.tables + (int64_t)p * kv.max_pages;
  int32_t *to = kv.tables + (int64_t)c * kv.max_pages;
  for (int j = blockIdx.y * 256 + threadIdx.x; j < full; j += gridDim.y * 256) {
    const int page = from[j];
    to[j] = page;
    if ((uint32_t)page < (uint32_t)kv.pages)
      atomicAdd(kv.refs + page, 1);
    else
      atomicOr(kv.err, kErrKvRange);
  }
  if (!rest) return;
  const int dst = jobs(kv)[c], src = from[full];
  if (blockIdx.y == 0 && threadIdx.x == 0) to[full] = dst;
  if ((uint32_t)src >= (uint32_t)kv.pages) {
    if (threadIdx.x == 0) atomicOr(kv.err, kErrKvRange);
    return;
  }
  const int runs = kv.layers * 2 * kv.heads;
  const int64_t run = (int64_t)kv.page() * kv.dim * kv.esize;
  const int used = rest * kv.dim * kv.esize;   // a multiple of 128
  const uint8_t *a = kv.pool + src * kv.page_bytes;
  uint8_t *b = kv.pool + dst * kv.page_bytes;
  for (int r = blockIdx.y; r < runs; r += gridDim.y)
    for (int o = threadIdx.x * 16; o < used; o += 256 * 16)
      store16_nt(b + r * run + o, load16_nt(a + r * run + o));
}

// --------------------------------------------------------------------- free
// A workgroup per listed sequence, which takes its length: of the workgroups of
// one listed again, and of an empty one, there is nothing left to free.  2.8 us
// for 32 sequences of up to 1,500 tokens; 2^20 entries take 2^20 workgroups'
// time (each looking through those before it would be 2^39 comparisons).
__global__ __launch_bounds__(256) void kv_free_kernel(KvCache kv, const int32_t *seqs) {
  __shared__ int taken;
  const bool stopped = kv_stopped(kv);
  const int s = seqs[blockIdx.x];
  if (s < 0 || stopped) return;
  if (s >= kv.seqs) {
    if (threadIdx.x == 0) atomicOr(kv.err, kErrKvRange);
    return;
  }
  if (threadIdx.x == 0) taken = atomicExch(kv.lens + s, 0);
  __syncthreads();
  const int held = min(held_pages(kv, max(taken, 0)), kv.max_pages);
  const int32_t *row = kv.tables + (int64_t)s * kv.max_pages;
  for (int j = threadIdx.x; j < held; j += 256) {
    const int page = row[j];
    if ((uint32_t)page >= (uint32_t)kv.pages) {
      atomicOr(kv.err, kErrKvRange);
    } else if (atomicAdd(kv.refs + page, -1) <= 0) {
      atomicAdd(kv.refs + page, 1);
      atomicOr(kv.err, kErrKvRange);
    }
  }
}

// ------------------------------------------------------------------ compact
// First kernel, one workgroup: U pages are in use; the k-th page in use at U
// or above moves to the k-th free page below U (there are as many of either).
// list_a: the free pages that are filled.  list_b[page]: where a page at U or
// above goes; which page comes to a filled one; -1 for the others.  The counts
// move too.  scratch[0] = moves, scratch[1] = U.  8.3 us for 2,048 pages.
__global__ __launch_bounds__(kOne) void kv_compact_kernel(KvCache kv) {
  int32_t *holes = list_a(kv), *to = list_b(kv);
  FirstRefs refs = first_refs(kv, 0);
  if (kv_stopped(kv)) return;
  for (int p = threadIdx.x; p < kv.pages; p += kOne) to[p] = -1;
  int used = 0, U;
#pragma unroll
  for (int i = 0; i < kRefsPerThread; ++i) used += refs.r[i] != 0;
  const int turn = kOne * kRefsPerThread;
  for (int p0 = turn + (int)threadIdx.x * kRefsPerThread; p0 < kv.pages; p0 += turn) {
    int r[kRefsPerThread];
    load_refs(kv, p0, 0, r);
#pragma unroll
    for (int i = 0; i < kRefsPerThread; ++i) used += r[i] != 0;
  }
  scan_excl(used, &U);
  FirstRefs free = refs;          // past the last page: not free
#pragma unroll
  for (int i = 0; i < kRefsPerThread; ++i)
    if ((int)threadIdx.x * kRefsPerThread + i >= kv.pages) free.r[i] = 1;
  const int moves = find_free(kv, U, holes, free);   // free pages, lowest first, up to U of them
  // those below U are the holes: as many as pages in use at U or above
  int from = 0;
  for (int base = U / turn * turn; base < kv.pages; base += kOne * kRefsPerThread) {
    const int p0 = base + (int)threadIdx.x * kRefsPerThread;
    int r[kRefsPerThread], mine = 0, all;
    if (base == 0) {
#pragma unroll
      for (int i = 0; i < kRefsPerThread; ++i) r[i] = refs.r[i];
    } else {
      load_refs(kv, p0, 0, r);
    }
#pragma unroll
    for (int i = 0; i < kRefsPerThread; ++i) mine += r[i] != 0 && p0 + i >= U;
    int at = from + scan_excl(mine, &all);
    from += all;
#pragma unroll
    for (int i = 0; i < kRefsPerThread; ++i)
      if (r[i] != 0 && p0 + i >= U) {
        const int hole = at < min(moves, U) ? holes[at] : -1;
        if (hole >= 0) {
          to[p0 + i] = hole;
          to[hole] = p0 + i;
          kv.refs[hole] = r[i];
          kv.refs[p0 + i] = 0;
        }
        ++at;
      }
  }
  if (threadIdx.x == 0) {
    kv.scratch[0] = from;
    kv.scratch[1] = U;
  }
}

__device__ __forceinline__ void copy_piece(uint8_t *b, const uint8_t *a, int64_t o, int64_t end) {
  u32x4 v[kPiece / (256 * 16)];
#pragma unroll
  for (int u = 0; u < kPiece / (256 * 16); ++u) {
    const int64_t at = o + (u * 256 + (int)threadIdx.x) * 16;
    if (at < end) v[u] = load16_nt(a + at);
  }
#pragma unroll
  for (int u = 0; u < kPiece / (256 * 16); ++u) {
    const int64_t at = o + (u * 256 + (int)threadIdx.x) * 16;
    if (at < end) store16_nt(b + at, v[u]);
  }
}

// Second kernel: the tables follow, and the pages are copied, a piece per
// workgroup at a time.  Sources lie at U or above and destinations below, so
// no copy reads what another writes.  Bound by HBM: 238 MB read and written in
// 44 us, 5.4 TB/s.
__global__ __launch_bounds__(256) void kv_move_kernel(KvCache kv) {
  if (kv_stopped(kv)) return;
  const int moves = kv.scratch[0], U = kv.scratch[1];
  const int32_t *holes = list_a(kv), *to = list_b(kv);
  for (int s = blockIdx.x; s < kv.seqs; s += gridDim.x) {
    const int held = min(held_pages(kv, max(kv.lens[s], 0)), kv.max_pages);
    int32_t *row = kv.tables + (int64_t)s * kv.max_pages;
    for (int j = threadIdx.x; j < held; j += 256) {
      const int p = row[j];
      const bool page = (uint32_t)p < (uint32_t)kv.pages;
      const int q = page ? to[p] : -1;
      // no page, or one that no sequence held: at U or above it goes nowhere,
      // below U another one comes there
      if (!page || (p < U) != (q < 0)) atomicOr(kv.err, kErrKvRange);
      else if (q >= 0) row[j] = q;
    }
  }
  const int64_t pieces = (kv.page_bytes + kPiece - 1) / kPiece;
  for (int64_t w = blockIdx.x; w < moves * pieces; w += gridDim.x) {
    const int m = (int)(w / pieces);
    const int dst = holes[m], src = to[dst];
    copy_piece(kv.pool + dst * kv.page_bytes, kv.pool + src * kv.page_bytes,
               (w - m * pieces) * kPiece, kv.page_bytes);
  }
}

__global__ __launch_bounds__(256) void kv_copy_kernel(KvCache kv, const int32_t *src,
                                                      const int32_t *dst, int n) {
  if (kv_stopped(kv)) return;
  const int64_t pieces = (kv.page_bytes + kPiece - 1) / kPiece;
  for (int64_t w = blockIdx.x; w < n * pieces; w += gridDim.x) {
    const int m = (int)(w / pieces);
    const int a = src[m], b = dst[m];
    if (a < 0 || b < 0 || a == b) continue;
    if (a >= kv.pages || b >= kv.pages) {
      if (threadIdx.x == 0) atomicOr(kv.err, kErrKvRange);
      continue;
    }
    copy_piece(kv.pool + b * kv.page_bytes, kv.pool + a * kv.page_bytes,
               (w - m * pieces) * kPiece, kv.page_bytes);
  }
}

// ------------------------------------------------------------------- append
// A wavefront per token: its keys and values, 16 bytes of the cache a lane, are
// on their way while the token's place is looked up.  Bound by HBM where there
// are many: 16,381 tokens of 8 heads of 128 float16, 134 MB in 24 us; 61 tokens
// of 4 heads of 256: 3.4 us.
constexpr int kAppendWaves = 4;
template <typename T, bool I16>
__global__ __launch_bounds__(64 * kAppendWaves) void kv_append_kernel(KvCache kv, KvAppend a) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * kAppendWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= a.n) return;
  const int lg = __builtin_ctz(kv.dim / V);   // vectors of a head's row
  const int per = kv.heads << lg, all = 2 * per;
  auto load = [&](int x, T *v) {
    const int which = x >= per, y = x - which * per;
    const int h = y >> lg, d = (y - (h << lg)) * V;
    const int64_t at = i * (which ? a.v_token : a.k_token) + h * (which ? a.v_head : a.k_head) + d;
    const void *src = which ? a.v : a.k;
    if constexpr (I16) {
      int16_t w[V];
      __builtin_memcpy(w, (const int16_t *)src + at, sizeof(w));
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = (T)(w[j] * a.unit);
    } else {
      *(u32x4 *)v = load16_nt((const T *)src + at);
    }
  };
  alignas(16) T v[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (lane + 64 * u < all) load(lane + 64 * u, v[u]);
  const bool stopped = kv_stopped(kv);
  const int s = a.seqs[i];
  if (s < 0 || stopped) return;
  bool ok = s < kv.seqs;
  int page = -1, pos = 0;
  if (ok) {
    const int len = kv.lens[s];
    pos = a.pos ? a.pos[i] : len - 1;
    ok = pos >= 0 && pos < len && (pos >> kv.lg_page) < kv.max_pages;
    if (ok) page = kv.tables[(int64_t)s * kv.max_pages + (pos >> kv.lg_page)];
    ok = ok && (uint32_t)page < (uint32_t)kv.pages;
  }
  if (!ok) {
    if (lane == 0) atomicOr(kv.err, kErrKvRange);
    return;
  }
  uint8_t *base = kv.pool + page * kv.page_bytes +
                  ((int64_t)a.layer * 2 * kv.heads * kv.page() + (pos & (kv.page() - 1))) *
                      kv.dim * (int)sizeof(T);
  const int64_t row = (int64_t)kv.page() * kv.dim * (int)sizeof(T);   // from a head to the next
  for (int x0 = lane; x0 < all; x0 += 64 * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = x0 + 64 * u;
      if (x < all) {
        if (x0 != lane) load(x, v[u]);
        *(u32x4 *)(base + (x >> lg) * row + (x & ((1 << lg) - 1)) * 16) = *(const u32x4 *)v[u];
      }
    }
  }
}

}  // namespace

hipError_t launch_kv_extend(const KvCache &kv, const int32_t *seqs, const int32_t *counts,
                            int32_t n, hipStream_t s) {
  kv_extend_kernel<<<1, kOne, 0, s>>>(kv, seqs, counts, n);
  return hipGetLastError();
}

hipError_t launch_kv_fork(const KvCache &kv, const int32_t *parents, const int32_t *children,
                          int32_t n, hipStream_t s) {
  kv_fork_kernel<<<1, kOne, 0, s>>>(kv, parents, children, n);
  // a workgroup per run of a last page, up to 64; a launch has fewer than 2^32 threads
  const int runs = std::min(kv.layers * 2 * kv.heads, 64);
  const int rows = std::max(std::min(runs, (1 << 23) / n), 1);
  kv_fork_rows_kernel<<<dim3(n, rows), 256, 0, s>>>(kv, parents, children);
  return hipGetLastError();
}

hipError_t launch_kv_free(const KvCache &kv, const int32_t *seqs, int32_t n, hipStream_t s) {
  kv_free_kernel<<<n, 256, 0, s>>>(kv, seqs);
  return hipGetLastError();
}

hipError_t launch_kv_compact(const KvCache &kv, int num_cu, hipStream_t s) {
  kv_compact_kernel<<<1, kOne, 0, s>>>(kv);
  kv_move_kernel<<<num_cu * 8, 256, 0, s>>>(kv);
  return hipGetLastError();
}

hipError_t launch_kv_copy(const KvCache &kv, const int32_t *src, const int32_t *dst, int32_t n,
                          int num_cu, hipStream_t s) {
  const int64_t work = n * ((kv.page_bytes + kPiece - 1) / kPiece);
  const int grid = (int)(work < num_cu * 8 ? work : num_cu * 8);
  kv_copy_kernel<<<grid, 256, 0, s>>>(kv, src, dst, n);
  return hipGetLastError();
}

hipError_t launch_kv_append(const KvCache &kv, const KvAppend &a, hipStream_t s) {
  const int grid = (a.n + kAppendWaves - 1) / kAppendWaves, threads = 64 * kAppendWaves;
  const bool i16 = a.dtype == DT_I16;
  if (kv.dtype == DT_F32) {
    if (i16) kv_append_kernel<float, true><<<grid, threads, 0, s>>>(kv, a);
    else kv_append_kernel<float, false><<<grid, threads, 0, s>>>(kv, a);
  } else if (kv.dtype == DT_BF16) {
    if (i16) kv_append_kernel<__bf16, true><<<grid, threads, 0, s>>>(kv, a);
    else kv_append_kernel<__bf16, false><<<grid, threads, 0, s>>>(kv, a);
  } else {
    if (i16) kv_append_kernel<_Float16, true><<<grid, threads, 0, s>>>(kv, a);
    else kv_append_kernel<_Float16, false><<<grid, threads, 0, s>>>(kv, a);
  }
  return hipGetLastError();
}

}  // namespace w4a8
