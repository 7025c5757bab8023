// Attention of several new tokens of each sequence over a paged key-value
// cache, and where a step's tokens lie.
//
//   o_h = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q_h . k_t - m),
//
// over the tokens t up to the query's own, in one pass with a running maximum
// m and sum.
#include "w4a8_mfma_ops.h"

namespace w4a8 {

namespace {

// ---------------------------------------------------------------------- maps
// What a map writes is a word or two a token; it costs its launch and a chain of
// dependent loads: a row's words, its length, and its tokens' table entries.
constexpr int kOne = 1024;        // threads of a workgroup that takes in all rows

// exclusive scans of N values per thread of a kOne-thread workgroup, and their
// totals; every thread of it calls
template <int N>
__device__ void scan_excl(int (&v)[N], int (&total)[N]) {
  __shared__ int sums[kOne / 64][N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = v[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x[i], d);
      if (lane >= d) x[i] += y;
    }
  }
  __syncthreads();              // the last call's sums are read
  if (lane == 63) {
#pragma unroll
    for (int i = 0; i < N; ++i) sums[wave][i] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kOne / 64; ++w) {
      const int s = sums[w][i];
      before += w < wave ? s : 0;
      all += s;
    }
    v[i] = before + x[i] - v[i];
    total[i] = all;
  }
}

// the sums of two values per thread, at most 2^52 each
__device__ void sum_all(int64_t &v, int64_t &w) {
  __shared__ int64_t sums[kOne / 64][2];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    v += __shfl_xor(v, d);
    w += __shfl_xor(w, d);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6][0] = v;
    sums[threadIdx.x >> 6][1] = w;
  }
  __syncthreads();
  v = w = 0;
#pragma unroll
  for (int i = 0; i < kOne / 64; ++i) {
    v += sums[i][0];
    w += sums[i][1];
  }
}

struct MapRow {
  int seq, count, len;   // seq -1: padding
  int bad;
};
__device__ __forceinline__ MapRow map_row(const KvCache &kv, const KvMap &m, int row) {
  MapRow r{m.seqs[row], m.counts[row], 0, 0};
  if (r.count < 0) r.count = 0, r.bad = 1;
  if (r.seq >= kv.seqs) r.seq = -1, r.bad = 1;
  if (r.seq < 0) r.seq = -1;
  if (r.seq >= 0) {
    r.len = kv.lens[r.seq];
    if (r.len < r.count || r.len > ((int64_t)kv.max_pages << kv.lg_page)) {
      r.bad = 1;
      r.seq = -1;
      r.len = 0;
    }
  }
  return r;
}

// Keys of a part: L = the work (tiles of a row times its tokens, all rows) over
// the units that fill the chip, but no fewer than shape.least.
__device__ __forceinline__ int parts_of(int len, int64_t most) {
  return len > most ? (int)((len + most - 1) / most) : 1;
}
struct RowPlan {
  int tiles, parts;
  int add[4];                   // tokens, units, joins, parts of split rows
};
__device__ __forceinline__ RowPlan plan_of(const KvMap &m, const MapRow &r, int64_t most) {
  const int tiles = (r.count + m.shape.tokens - 1) / m.shape.tokens, n = parts_of(r.len, most);
  return {tiles, n, {r.count, tiles * n, n > 1 ? tiles : 0, n > 1 ? tiles * n : 0}};
}
__device__ __forceinline__ int64_t part_keys(const KvMap &m, int64_t work) {
  const int64_t most = (work + m.shape.split - 1) / m.shape.split;
  return most < m.shape.least ? m.shape.least : most;
}

// the last of n rows whose word (at stride) is at most v; word 0 is
template <int STRIDE>
__device__ __forceinline__ int row_of(const int32_t *words, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (words[STRIDE * mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

// token i, of row r that begins at token `first`; r.seq -1: of none
__device__ __forceinline__ void put_token(const KvCache &kv, const KvMap &m, int i,
                                          const MapRow &r, int first) {
  int pos = -1;
  int64_t slot = -1;
  if (r.seq >= 0) {
    pos = r.len - r.count + (i - first);
    const int page = kv.tables[(int64_t)r.seq * kv.max_pages + (pos >> kv.lg_page)];
    if ((uint32_t)page < (uint32_t)kv.pages)
      slot = ((int64_t)page << kv.lg_page) + (pos & (kv.page() - 1));
    else
      atomicOr(kv.err, kErrKvRange);
  }
  m.token_seqs[i] = r.seq;
  m.pos[i] = pos;
  m.slots[i] = slot;
}

// unit i, the at-th of row r's, whose tokens, joins and parts begin at `first`,
// `join` and `slot`: a row's tiles from its last tokens, which see the most keys,
// to its first, those of the same part of the keys side by side
__device__ __forceinline__ void put_unit(const KvMap &m, int i, int at, const MapRow &r, int n,
                                         int first, int join, int slot) {
  const int tokens = m.shape.tokens, tiles = (r.count + tokens - 1) / tokens;
  const int part = at / tiles, j = at - part * tiles, tile = tiles - 1 - j;
  const int tok = tile * tokens, ntok = min(tokens, r.count - tok);
  int pos0 = 0, k0 = 0, k1 = 0, mine = -1;
  bool none = false;                        // a part behind the tile's last key
  if (r.seq >= 0) {
    pos0 = r.len - r.count + tok;
    const int end = pos0 + ntok, per = ((end + n - 1) / n + 63) / 64 * 64;
    const int used = (int)(((int64_t)end + per - 1) / per);
    const int64_t from = (int64_t)part * per;
    none = from >= end;
    k0 = none ? 0 : (int)from;
    k1 = none ? 0 : (int)(from + per < end ? from + per : end);
    if (used > 1) mine = slot + j * n + part;
    if (n > 1 && part == 0)
      *(int4 *)(m.plan + kPlanHead + kUnitWords * m.shape.units +
                (int64_t)kJoinWords * (join + j)) = int4{first + tok, ntok, slot + j * n, used};
  }
  int4 *u = (int4 *)(m.plan + kPlanHead + (int64_t)kUnitWords * i);
  u[0] = int4{r.seq, first + tok, none ? 0 : ntok, pos0};
  u[1] = int4{k0, k1, mine, 0};
}

__device__ __forceinline__ void put_head(const KvMap &m, int units, int joins, bool fits) {
  *(int4 *)m.plan = int4{units, joins, fits, 0};
}

// Rows of a step whose units are put in order: 3,001 tokens of 13 rows 149 -> 131
// us, 2,000 of 20 rows 103 -> 83, a layer, for 1.5 us of the map (eight rows' sizes at a
// time; one after another 10).  Many rows' lie mixed as they come.
constexpr int kSorted = 128;

// Steps of up to kOne rows in one launch: every workgroup takes in all rows, a
// thread each, and then writes kOne tokens and units of its own.  61 rows of a token
// 8 us (7.9 under the profiler, of which an empty kernel is 4.4), 300 rows of 16,381
// tokens 9, 1,024 rows of a token 10.5; one workgroup for the rows and a second launch
// for the tokens took 11.6 and 14.6 for the first two.
__global__ __launch_bounds__(kOne) void kv_map_kernel(KvCache kv, KvMap m) {
  __shared__ int32_t at[6][kOne + 1];       // where a row's tokens, units, joins, parts begin,
                                            // its parts, its units' place in the plan
  __shared__ MapRow rows[kOne];
  const bool stopped = kv_stopped(kv);
  const int row = threadIdx.x;
  MapRow r{-1, 0, 0, 0};
  if (row < m.rows) r = map_row(kv, m, row);
  if (r.bad && blockIdx.x == 0) atomicOr(kv.err, kErrKvRange);
  int64_t sum = r.count;
  int64_t work = ((int64_t)r.count + m.shape.tokens - 1) / m.shape.tokens * r.len;
  sum_all(sum, work);
  const bool fits = sum <= m.tokens && !stopped;
  if (row == 0 && blockIdx.x == 0 && sum > m.tokens) atomicOr(kv.err, kErrKvRange);
  if (!fits) r = MapRow{-1, 0, 0, 0};
  RowPlan p = plan_of(m, r, part_keys(m, work));
  int all[4];
  scan_excl<4>(p.add, all);
  rows[row] = r;
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i][row] = p.add[i];
  at[4][row] = p.parts;
  at[5][row] = p.add[1];
  if (m.rows > 1 && m.rows <= kSorted && all[1] > m.shape.split) {
    // more units than the chip takes at once: the rows with the longest ones first,
    // in every workgroup the same way
    __shared__ int2 size[kSorted];          // keys of a unit, at most; units
    const int keys = r.len / p.parts, mine = p.tiles * p.parts;
    if (row < kSorted) size[row] = row < m.rows ? int2{keys, mine} : int2{0, 0};
    __syncthreads();
    if (row < m.rows) {
      int before = 0;
      for (int at8 = 0; at8 < m.rows; at8 += 8) {       // zeros behind the last
        int2 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = size[at8 + i];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          before += ((x[i].x > keys) | ((x[i].x == keys) & (at8 + i < row))) ? x[i].y : 0;
      }
      at[5][row] = before;
    }
  }
  if (blockIdx.x == 0) {
    if (row < m.rows) m.cu[row] = p.add[0];
    if (row == 0) {
      m.cu[m.rows] = all[0];
      put_head(m, all[1], all[2], fits);
    }
  }
  __syncthreads();
  const int i = blockIdx.x * kOne + threadIdx.x;
  if (i < m.tokens) {
    const int x = m.rows > 0 && i < all[0] ? row_of<1>(at[0], m.rows, i) : -1;
    put_token(kv, m, i, x < 0 ? MapRow{-1, 0, 0, 0} : rows[max(x, 0)], x < 0 ? 0 : at[0][x]);
  }
  if (i < all[1]) {
    const int x = row_of<1>(at[1], m.rows, i);
    const int nth = i - at[1][x];
    put_unit(m, at[5][x] + nth, nth, rows[x], at[4][x], at[0][x], at[2][x], at[3][x]);
  }
}

// More rows: first one workgroup, which leaves where rows' tokens, units, joins and
// parts begin behind the plan's joins, a round of loads for each kOne rows and another
// for their scans (2,000 rows of 16,000 tokens 19.6 us in all, 10.7 of them here; 1,025
// rows of a token 17.5);
__global__ __launch_bounds__(kOne) void kv_map_rows_kernel(KvCache kv, KvMap m) {
  int32_t *rows = m.plan + kPlanHead + kUnitWords * m.shape.units + kJoinWords * m.shape.joins;
  const bool stopped = kv_stopped(kv);
  int64_t sum = 0, work = 0;
  int bad = 0;
  for (int i = threadIdx.x; i < m.rows; i += kOne) {
    const MapRow r = map_row(kv, m, i);
    sum += r.count;
    bad |= r.bad;
    work += ((int64_t)r.count + m.shape.tokens - 1) / m.shape.tokens * r.len;
  }
  sum_all(sum, work);
  if (bad) atomicOr(kv.err, kErrKvRange);
  const bool fits = sum <= m.tokens && !stopped;
  if (threadIdx.x == 0 && sum > m.tokens) atomicOr(kv.err, kErrKvRange);
  const int64_t most = part_keys(m, work);
  int from[4] = {0, 0, 0, 0};
  for (int base = 0; base < m.rows; base += kOne) {
    const int i = base + threadIdx.x;
    MapRow r{-1, 0, 0, 0};
    if (i < m.rows && fits) r = map_row(kv, m, i);
    RowPlan p = plan_of(m, r, most);
    int all[4];
    scan_excl<4>(p.add, all);
    if (i < m.rows) {
      m.cu[i] = from[0] + p.add[0];
      *(int4 *)(rows + kRowWords * i) =
          int4{from[1] + p.add[1], from[2] + p.add[2], from[3] + p.add[3], p.parts};
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) from[x] += all[x];
  }
  if (threadIdx.x == 0) {
    m.cu[m.rows] = from[0];
    put_head(m, from[1], from[2], fits);
  }
}
// then a thread per token and unit.
__global__ __launch_bounds__(256) void kv_map_tokens_kernel(KvCache kv, KvMap m) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int32_t *rows =
      m.plan + kPlanHead + kUnitWords * m.shape.units + kJoinWords * m.shape.joins;
  const int4 head = *(const int4 *)m.plan;
  if (i < m.tokens) {
    const bool some = head.z && i < m.cu[m.rows];
    const int x = some ? row_of<1>(m.cu, m.rows, i) : 0;
    put_token(kv, m, i, some ? map_row(kv, m, x) : MapRow{-1, 0, 0, 0}, m.cu[x]);
  }
  if (head.z && i < head.x) {
    const int x = row_of<kRowWords>(rows, m.rows, i);
    const int4 at = *(const int4 *)(rows + kRowWords * x);
    put_unit(m, i, i - at.x, map_row(kv, m, x), at.w, m.cu[x], at.y, at.z);
  }
}

// ----------------------------------------------------------------- attention
constexpr int kWaves = 4, kThreads = 64 * kWaves;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// what exponents are taken against: the maximum, or 0 where no score is above
// -infinity, so that every weight there is 0 and not a NaN
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// Where a maximum (times scale) is this far from 0, its rounding (below that half of
// 2^-13) is no longer nothing to an exponent: in 2^(s scale - m scale) with m scale rounded
// it is a factor that all weights against m have, and those against the next maximum
// have another.  Two of them are 2^-13.5 of a weight at most, a sixth of what its own
// rounding to float16 may be.
constexpr float kFar = 2048.f;
// of scores, in powers of two; what is below 0 or 0 is part of q
__device__ __forceinline__ float scale_of(const Chunk &a) {
  return a.scale == 0.f ? 1.f : fabsf(a.scale);
}

struct Unit {
  int seq, tok, ntok, pos0, k0, k1, slot;
};
// A unit of the plan as it stands there, or one without tokens where it is not
// what a plan of this call can hold.
__device__ __forceinline__ Unit unit_of(const KvCache &kv, const Chunk &a, int64_t i) {
  const int4 *p = (const int4 *)(a.plan + kPlanHead + kUnitWords * i);
  const int4 x = p[0], y = p[1];
  const int units = __builtin_amdgcn_readfirstlane(a.plan[0]);
  Unit u{__builtin_amdgcn_readfirstlane(x.x), __builtin_amdgcn_readfirstlane(x.y),
         __builtin_amdgcn_readfirstlane(x.z), __builtin_amdgcn_readfirstlane(x.w),
         __builtin_amdgcn_readfirstlane(y.x), __builtin_amdgcn_readfirstlane(y.y),
         __builtin_amdgcn_readfirstlane(y.z)};
  if (i >= units) {
    u.ntok = 0;
    return u;
  }
  const int64_t most = (int64_t)kv.max_pages << kv.lg_page;
  if (u.seq >= kv.seqs || u.tok < 0 || u.ntok < 0 || u.ntok > a.shape.tokens ||
      (int64_t)u.tok + u.ntok > a.tokens || u.pos0 < 0 || u.k0 < 0 || u.k1 < 0 ||
      (u.k1 > 0 && u.k1 <= u.k0) || u.k1 > most || (int64_t)u.pos0 + u.ntok > most ||
      (u.seq < 0 && u.k1 > 0) || (u.k0 & 63) || u.slot >= a.shape.parts) {
    if (threadIdx.x == 0) atomicOr(kv.err, kErrKvRange);
    u.ntok = 0;
  }
  return u;
}

template <typename T>
__device__ __forceinline__ void store_four(T *p, const float *x) {
  typedef T x4 __attribute__((ext_vector_type(4)));
  *(x4 *)p = x4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
}
// four values of a head: rounded once
__device__ __forceinline__ void store_out(const Chunk &a, int cache_dtype, int64_t at,
                                          const float *x) {
  if (a.dtype == DT_I16) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    s16x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = (int16_t)fminf(fmaxf(rintf(x[i] * a.out_unit), -32768.f), 32767.f);
    *(s16x4 *)((int16_t *)a.out + at) = v;
  } else if (cache_dtype == DT_F32) {
    store_four((float *)a.out + at, x);
  } else if (cache_dtype == DT_BF16) {
    store_four((__bf16 *)a.out + at, x);
  } else {
    store_four((_Float16 *)a.out + at, x);
  }
}

template <typename T>
struct Of {
  typedef T x8 __attribute__((ext_vector_type(8)));
};

// Keys of a turn: 64, or 32 where a row of them is 512 bytes or more
template <int D, typename T>
constexpr int kTurn = D * sizeof(T) >= 512 ? 32 : 64;
// A turn's keys or values lie in LDS by rows, the order of a row's pieces of 16
// bytes changed by the row so that neither 16 rows' same piece (keys) nor four
// rows' runs of 64 bytes (values by columns) meet in a bank.
template <int ROW>
__device__ __forceinline__ constexpr int turn_of(int t) {
  return ROW == 128 ? ((t >> 1) & 1) << 2 | ((t >> 2) & 3) : (t & 3) << 2 | ((t >> 2) & 3);
}
template <int ROW>
__device__ __forceinline__ constexpr int lds_at(int t, int piece) {
  return t * ROW + ((piece ^ turn_of<ROW>(t)) << 4);
}

// A value that the compiler takes as new each time, so that what is made of it
// by an addition or two is made again and not kept in a register.
__device__ __forceinline__ int afresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// What the kernels of either width share: a unit's place, and a turn's keys and
// values on their way to LDS, by NW wavefronts.
template <int D, typename T, int NW>
struct Turns {
  static constexpr int KT = kTurn<D, T>, ROW = D * sizeof(T), BYTES = KT * ROW;
  static constexpr int BLOCKS = KT / 16;            // of 16 tokens, each in one page
  // A block's keys, or its values, are a job of 16 ROW bytes: a wavefront has
  // one or two (a block's keys and values), or shares one with another.
  static constexpr int JOBS = 2 * BLOCKS, SHARE = NW > JOBS ? NW / JOBS : 1;
  static constexpr int MINE = JOBS > NW ? JOBS / NW : 1;
  static constexpr int COPIES = 16 * ROW / 1024 / SHARE;
  static_assert(MINE <= 2 && (MINE == 1 || BLOCKS == NW) && COPIES >= 1, "copies");
  const KvCache &kv;
  const int32_t *table;
  int64_t plane, kbase;
  int k1, wave, page, lane_at;
  static constexpr uint32_t GOOD = (1u << BLOCKS) - 1;
  int bad;
  struct Pages { int p[BLOCKS]; };
  __device__ __forceinline__ Turns(const KvCache &kv, const Unit &u, int layer, int kvh, int wave)
      : kv(kv), table(kv.tables + (int64_t)u.seq * kv.max_pages),
        plane((int64_t)kv.page() * D), kbase(((int64_t)layer * 2 * kv.heads + kvh) * plane),
        k1(u.k1), wave(wave), page(kv.page()), bad(0) {
    const int at = (threadIdx.x & 63) * 16, row = at / ROW, piece = (at % ROW) >> 4;
    lane_at = row * ROW + ((piece ^ turn_of<ROW>(row)) << 4);
  }
  __device__ __forceinline__ Pages look_up(int t) const {
    Pages next;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      const int tt = t + 16 * j;
      next.p[j] = table[(tt < k1 ? tt : k1 - 1) >> kv.lg_page];
    }
    return next;
  }
  // the turn from t on, in these pages, to lds (keys, then values); a bit for each
  // block whose page is one of the pool's
  __device__ __forceinline__ uint32_t load(int t, const Pages &next, uint32_t lds) {
    uint32_t good = 0;
    int p[BLOCKS];
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      p[j] = __builtin_amdgcn_readfirstlane(next.p[j]);
      const bool ok = (uint32_t)p[j] < (uint32_t)kv.pages;
      good |= (ok ? 1u : 0u) << j;
      bad |= !ok;
      if (!ok) p[j] = 0;
    }
    const int job = MINE == 2 ? wave : wave / SHARE, j = job % BLOCKS, part = wave % SHARE;
    int mine = p[0];
#pragma unroll
    for (int x = 1; x < BLOCKS; ++x) mine = j == x ? p[x] : mine;
    const uint8_t *from = kv.pool + mine * kv.page_bytes +
                          (kbase + (int64_t)((t + 16 * j) & (page - 1)) * D) * (int)sizeof(T);
    const int at = afresh(lane_at);
#pragma unroll
    for (int x = 0; x < MINE; ++x) {
      const int which = MINE == 2 ? x : job / BLOCKS;
      const uint8_t *src = which ? from + kv.heads * plane * (int)sizeof(T) : from;
      const uint32_t to = lds + which * BYTES + j * 16 * ROW + part * COPIES * 1024;
      if constexpr (SHARE == 1) {
#pragma unroll
        for (int n = 0; n < COPIES; ++n)            // turn_of is a sum without carries
          copy16(src, (at ^ (turn_of<ROW>(n * 1024 / ROW) << 4)) + n * 1024, to + n * 1024);
      } else {
#pragma unroll
        for (int n = 0; n < COPIES; ++n) {
          const int i = part * COPIES + n;
          copy16(src, (at ^ (turn_of<ROW>(i * 1024 / ROW) << 4)) + i * 1024, to + n * 1024);
        }
      }
    }
    return good;
  }
};

// the copies of all but the last N are there, for every wavefront
template <int N>
__device__ __forceinline__ void turn_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Infinities and NaNs among a masked turn's values: 0 times one would reach the
// queries that do not see it, and what lies behind a sequence's end may be
// anything.  give(key): adds such values of a key that a query sees to its
// output; then they are taken out.  Every wavefront calls.  That comes before the
// turn's maximum, so an infinity may be all that a query's output holds while its
// maximum is -infinity, and its factor there is 1 and not 0.
template <typename T, typename Tn, int NW, typename Give>
__device__ __forceinline__ void take_out_odd(uint8_t *values, int *flag, Give give) {
  constexpr uint32_t E = sizeof(T) == 4 ? 0x7F800000u : __is_same(T, _Float16) ? 0x7C00u : 0x7F80u;
  auto odd_bits = [](uint32_t w) {
    if constexpr (sizeof(T) == 4) return (w & E) == E ? 0xFFFFFFFFu : 0u;
    return ((w & E) == E ? 0xFFFFu : 0u) | ((w >> 16 & E) == E ? 0xFFFF0000u : 0u);
  };
  bool odd = false;
  for (int at = threadIdx.x * 16; at < Tn::BYTES; at += NW * 1024) {
    const u32x4 w = *(const u32x4 *)(values + at);
    odd |= (odd_bits(w[0]) | odd_bits(w[1]) | odd_bits(w[2]) | odd_bits(w[3])) != 0;
  }
  if (odd) *flag = 1;
  __syncthreads();
  if (*flag == 0) return;
  for (int key = 0; key < Tn::KT; ++key) give(key);
  __syncthreads();
  for (int at = threadIdx.x * 16; at < Tn::BYTES; at += NW * 1024) {
    u32x4 w = *(const u32x4 *)(values + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= ~odd_bits(w[i]);
    *(u32x4 *)(values + at) = w;
  }
  if (threadIdx.x == 0) *flag = 0;
  __syncthreads();
}

// Outputs times a factor f >= 0, a power of two; where 32 bits hold none so small and
// f is 0, an infinity stays one and all else becomes 0: three factors of 2^-126 bring
// any number below the least.
template <int N, typename V>
__device__ __forceinline__ void fall_by(V (&o)[N], float f) {
  constexpr float LEAST = 1.17549435e-38f;          // 2^-126
  const bool none = f == 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] *= none ? LEAST : f;
  if (__any(none)) {
    const float again = none ? LEAST : 1.f;
#pragma unroll 1
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] *= again;
  }
}

struct Place {
  int kvh, h0, heads;        // key-value head, first query head, query heads
  int64_t unit;
  int part;                  // of a unit's parts: which tile of heads
};
__device__ __forceinline__ Place place_of(const KvCache &kv, const Chunk &a, int64_t i) {
  const int per = kv.heads * a.shape.tiles, group = a.hq / kv.heads;
  Place p;
  p.unit = i / per;
  p.part = (int)(i - p.unit * per);
  p.kvh = p.part / a.shape.tiles;
  const int first = (p.part - p.kvh * a.shape.tiles) * a.shape.heads;
  p.heads = min(a.shape.heads, group - first);
  p.h0 = p.kvh * group + first;
  return p;
}

__device__ __forceinline__ void zeros(const KvCache &kv, const Chunk &a, const Unit &u,
                                      const Place &p) {
  const float zero[4] = {0, 0, 0, 0};
  const int each = p.heads * kv.dim;
  for (int e = threadIdx.x * 4; e < u.ntok * each; e += blockDim.x * 4) {
    const int t = e / each, x = e - t * each;
    store_out(a, kv.dtype, (int64_t)(u.tok + t) * a.out_token + (p.h0 + x / kv.dim) * a.out_head +
                               x % kv.dim, zero);
  }
}

// Where four elements, 4 e .., of a row of a unit's part lie: 32 rows' side by
// side, as the lanes of a wavefront hold them; then (all rows') maximum, of scores
// before the scale so that large ones' differences are exact, and sum.
__device__ __forceinline__ float *part_at(const KvCache &kv, const Chunk &a, int slot,
                                          const Place &p, int row, int e) {
  const int per = kv.heads * a.shape.tiles;
  return a.part + (((int64_t)slot * per + p.part) * kChunkRows + (row & ~31)) * kv.dim +
         (e * 32 + (row & 31)) * 4;
}
__device__ __forceinline__ float *part_sums(const KvCache &kv, const Chunk &a, int slot,
                                            const Place &p, int row) {
  const int64_t per = kv.heads * a.shape.tiles;
  return a.part + a.shape.parts * per * kChunkRows * kv.dim +
         ((slot * per + p.part) * kChunkRows + row) * 2;
}

// Keys and values of 16 bits, on 32 x 32 x 16 matrix instructions: a wavefront has
// 32 of the unit's rows.  S^T = K q^T leaves 16 keys of one query in a lane, which
// are, rounded once to the cache's type, the B operand of o^T = V^T p^T as they
// are: no weight passes through LDS, and a query's maximum and sum are a lane's own
// and its partner's.  V is read by columns from where it lies by rows.  Keys and
// values of the next turn are copied to LDS while this one is worked on; a turn's 32
// or 64 keys serve 128 rows, so that LDS is read once for 128 operations a byte.
//
// No one unit is the bound: a wavefront's products, exponents and reads of LDS follow
// one another, and the two wavefronts of a SIMD cover each other in part.  8,192
// tokens of a prompt, 16 query heads of 256, take 533-571 us on several cards,
// 0.96-1.03 PFLOP/s, with the matrix units busy 45 % of the cycles at 1.9 of 2.4 GHz (a
// product of 8,192 x 8,192 x 8,192: 1.35-1.39 PFLOP/s, 70 % at 1.8), and no conflicts
// in LDS; 100 tokens over 131,072 keys, heads of 128, 291-300 us, 36 %.  At heads of
// 256 turns whose products begin before the last turn's weights are done gained
// nothing; at fewer that was not tried.  Short calls wait: 17 tokens over 511 keys,
// 10-11 us, of which 2 before the first turn, 1.1 a turn and 2.6 for the parts' stores.
//
// Weights are rounded once to the cache's type for the second product, beside the
// rounding of the output: errors against 64 bits of 1.25 to 1.42 times what the latter
// alone leaves (bfloat16 0.0022 for 0.0016, float16 0.00025 for 0.0002; two roundings
// of one size and no relation, so the square root of 2 at most).  As sums of two
// values, as for a single token, they leave none of it, for half as many products
// again: the prompt took 775 us where it takes 569, 100 tokens over 131,072 391 for 299,
// 17 over 511 15.1 for 14.6; and an infinite value would meet a second part of 0.
//
// At D = 256 (s - m) scale takes two operations, elsewhere one multiply-add and the
// branch for far maxima: that branch's registers do not fit beside 128 of out.
// At D = 64 registers are held to 128, four wavefronts a SIMD (8,192 tokens of a prompt,
// 64 heads of 64, 629 us; with the 140 that it takes otherwise 640).
template <int D, typename T>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void chunk_kernel(KvCache kv, Chunk a) {
  typedef Turns<D, T, kWaves> Tn;
  typedef typename Of<T>::x8 x8;
  constexpr int KT = Tn::KT, ROW = Tn::ROW, BYTES = Tn::BYTES;
  constexpr int KS = D / 16, NT = KT / 32, ND = D / 32;
  constexpr bool HALF = __is_same(T, _Float16);
  // weights are taken against a maximum that follows the largest score only when
  // that is SLACK above it, so that sums are rarely rescaled; a float16 weight's
  // exponent ends at 2^-24: weights there are 2^LIFT as large
  constexpr float LIFT = HALF ? 14.f : 0.f, SLACK = HALF ? 1.f : 8.f;
  __shared__ __align__(1024) uint8_t buf[2][2 * BYTES];
  __shared__ int odd;

  const Place P = place_of(kv, a, blockIdx.x);
  const Unit u = unit_of(kv, a, P.unit);
  if (u.ntok == 0) return;
  if (u.k1 == 0) return zeros(kv, a, u, P);
  const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Tn turns(kv, u, a.layer, P.kvh, wave);
  const typename Tn::Pages first = turns.look_up(u.k0), second = turns.look_up(u.k0 + KT);

  // this lane's query: row of the unit, its token and head
  const int row = wave * 32 + r, tok = row / P.heads, head = P.h0 + row - tok * P.heads;
  const bool on = tok < u.ntok;
  const bool work = wave * 32 < u.ntok * P.heads;
  const int last = u.pos0 + (on ? tok : 0);         // the last key it sees
  const int wave_last =                             // and any of this wavefront
      u.pos0 + min(u.ntok - 1, __builtin_amdgcn_readfirstlane((wave * 32 + 31) / P.heads));
  // a scale below 0 turns q, and 0 makes it 0 (a masked score is -infinity)
  const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;
  const float scale = scale_of(a);
  if (threadIdx.x == 0) odd = 0;
  x8 q[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int64_t e = (int64_t)(u.tok + tok) * a.q_token + head * a.q_head + 16 * s + 8 * g;
    const u32x4 w = on ? *(const u32x4 *)((const uint16_t *)a.q + e) : u32x4{0, 0, 0, 0};
    const uint32_t flip = sign < 0.f ? 0x80008000u : 0u, keep = sign == 0.f ? 0u : ~0u;
    q[s] = __builtin_bit_cast(x8, (w ^ flip) & keep);
  }
  // both slots, as soon as q and the pages are there
  const uint32_t lds = (uint32_t)(uintptr_t)buf;
  __builtin_amdgcn_sched_barrier(0);
  uint32_t good = turns.load(u.k0, first, lds);
  uint32_t after = turns.load(u.k0 + KT, second, lds + 2 * BYTES);

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -INFINITY, l = 0.f;                     // m: of scores before the scale
  // where this lane's keys (row r, piece g of each step) and the columns of
  // values that it reads for its group of 16 lie in LDS; a step, an element tile
  // and a second four keys turn bits of the place
  const int k_at = lds_at<ROW>(r, g);
  const int v_row = 4 * g + ((lane & 15) >> 2), v_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const int v_at = lds_at<ROW>(v_row, v_col >> 3) + (v_col & 4) * 2;

  auto body = [&](int t, const uint8_t *lds, uint32_t good, bool masked) {
    f32x16 sc[NT];
    const int kat = afresh(k_at);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[j][i] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const x8 k = *(const x8 *)(lds + (kat ^ (s << 5)) + 32 * j * ROW);
        sc[j] = mfma32(k, q[s], sc[j]);
        if (D == 256 && s % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
    // result i of tile j is key t + 32 j + 8 (i >> 2) + 4 g + (i & 3)
    if (masked) {
      const int end = min(last, u.k1 - 1) - t - 4 * g;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool off = (32 * j + 8 * (i >> 2) + (i & 3) > end) | !(good >> (2 * j + (i >> 3)) & 1);
          sc[j][i] = off ? -INFINITY : sc[j][i];
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[j][i]);
    if (__any((top - m) * scale > SLACK)) {         // from -infinity too
      top = fmaxf(top, __shfl_xor(top, 32));
      const float up = (top - m) * scale > SLACK ? top : m;
      const float fall = m == -INFINITY ? 1.f : exp2_of((m - up) * scale);
      m = up;
      l *= fall;
      fall_by(o, fall);
    }
    const float base = base_of(m);
    float sum = 0.f;
    if constexpr (D == 256) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = (sc[j][i] - base) * scale;
          sc[j][i] = exp2_of(LIFT > 0.f ? x + LIFT : x);
          sum += sc[j][i];
        }
    } else {
      float off = base * scale;
      const bool far = fabsf(off) >= kFar;
      if (__any(far)) {                             // of other queries, not a bit changes
#pragma unroll
        for (int j = 0; j < NT; ++j) sc[j] -= far ? base : 0.f;
        off = far ? 0.f : off;
      }
      off -= LIFT;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sc[j][i] = exp2_of(__builtin_fmaf(sc[j][i], scale, -off));
          sum += sc[j][i];
        }
    }
    l += sum;
    const int vat = afresh(v_at);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        x8 p;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (T)sc[j][8 * s + i];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          // row d of V transposed: eight keys of this lane's, four at a time
          u32x2 w[2];
#pragma unroll
          for (int x = 0; x < 2; ++x)
            w[x] = lds_columns(lds + BYTES + (vat ^ (d << 6) ^ (x << 5)) +
                               (32 * j + 16 * s + 8 * x) * ROW);
          o[d] = mfma32(__builtin_bit_cast(x8, w), p, o[d]);
          if (D == 256 && d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      }
  };
  // the infinities and NaNs among a key's values, to the queries that see it
  auto give = [&](int t, const uint8_t *values, uint32_t good, int key) {
    const bool sees = t + key <= last && t + key < u.k1 && (good >> (key >> 4) & 1);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int col = 32 * d + 8 * b + 4 * g;
        typedef T x4 __attribute__((ext_vector_type(4)));
        const x4 v = *(const x4 *)(values + lds_at<ROW>(key, col >> 3) + (col & 4) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = (float)v[i];
          o[d][4 * b + i] += sees && !(fabsf(y) < INFINITY) ? y : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  };

  typename Tn::Pages next = turns.look_up(u.k0 + 2 * KT);
  turn_barrier<Tn::MINE * Tn::COPIES>();
  const int full = min(u.pos0 + 1, u.k1);           // keys that every query sees
  for (int t = u.k0, b = 0; t < u.k1; t += KT, b ^= 1) {
    const uint8_t *now = buf[b];
    const bool masked = t + KT > full || good != Tn::GOOD;
    if (masked)
      take_out_odd<T, Tn, kWaves>((uint8_t *)now + BYTES, &odd,
                   [&](int key) { give(t, now + BYTES, good, key); });
    if (work && t <= wave_last) body(t, now, good, masked);
    turn_barrier<0>();
    good = after;
    if (t + 2 * KT < u.k1) {
      after = turns.load(t + 2 * KT, next, lds + b * 2 * BYTES);
      next = turns.look_up(t + 3 * KT);
    }
  }
  if (turns.bad && threadIdx.x == 0) atomicOr(kv.err, kErrKvRange);
  if (!on) return;
  l += __shfl_xor(l, 32);
  // result i of tile d is element 32 d + 8 (i >> 2) + 4 g + (i & 3)
  if (u.slot < 0) {
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    const int64_t at = (int64_t)(u.tok + tok) * a.out_token + head * a.out_head + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float x[4] = {o[d][4 * b] * inv, o[d][4 * b + 1] * inv, o[d][4 * b + 2] * inv,
                            o[d][4 * b + 3] * inv};
        store_out(a, kv.dtype, at + 32 * d + 8 * b, x);
      }
    return;
  }
  float *part = part_at(kv, a, u.slot, P, row, g);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *(f32x4 *)(part + (8 * d + 2 * b) * 128) =
          f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
  if (g == 0) {
    float *ml = part_sums(kv, a, u.slot, P, row);
    ml[0] = m;
    ml[1] = l;
  }
}

// Keys and values of 32 bits, on the float32 matrix instructions: 16 keys by 16
// queries, a wavefront's queries as C columns of tiles, so that q and out stay
// in 128 registers.  Weights stay in 32 bits.  At the float32 matrix rate, an eighth
// of the 16-bit one, this is bound by the matrix units once the chip is full: 4,096
// tokens of a prompt, 32 heads of 128, 1.17 ms, 117 of 153 TFLOP/s.  1,000 tokens of
// five rows over up to 2,000 keys, 8 heads of 64, take 27 us of 6 at that rate (few units
// of uneven length: the matrix units are busy 22 % of the cycles), and 6.5 for the
// join.
template <int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void chunk_f32_kernel(KvCache kv, Chunk a) {
  typedef Turns<D, float, NW> Tn;
  constexpr int C = kChunkRows / (16 * NW);
  constexpr int KT = Tn::KT, ROW = Tn::ROW, BYTES = Tn::BYTES;
  constexpr int KS = D / 16, NT = KT / 16, NC = D / 64;
  constexpr float SLACK = 8.f;
  __shared__ __align__(1024) uint8_t buf[2][2 * BYTES];
  __shared__ int odd;

  const Place P = place_of(kv, a, blockIdx.x);
  const Unit u = unit_of(kv, a, P.unit);
  if (u.ntok == 0) return;
  if (u.k1 == 0) return zeros(kv, a, u, P);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Tn turns(kv, u, a.layer, P.kvh, wave);
  const typename Tn::Pages first = turns.look_up(u.k0), second = turns.look_up(u.k0 + KT);

  int row[C], tok[C], head[C], last[C];
  bool on[C];
  const bool work = wave * 16 * C < u.ntok * P.heads;
  const int wave_last =
      u.pos0 + min(u.ntok - 1, __builtin_amdgcn_readfirstlane((wave * 16 * C + 16 * C - 1) / P.heads));
  f32x4 q[C][KS];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    row[c] = wave * 16 * C + 16 * c + r;
    tok[c] = row[c] / P.heads;
    head[c] = P.h0 + row[c] - tok[c] * P.heads;
    on[c] = tok[c] < u.ntok;
    last[c] = u.pos0 + (on[c] ? tok[c] : 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int64_t e = (int64_t)(u.tok + tok[c]) * a.q_token + head[c] * a.q_head + 16 * s + 4 * g;
      q[c][s] = f32x4{0, 0, 0, 0};
      if (on[c]) {
        q[c][s] = *(const f32x4 *)((const float *)a.q + e);
        if (a.scale < 0.f) q[c][s] = -q[c][s];
        if (a.scale == 0.f) q[c][s] = f32x4{0, 0, 0, 0};
      }
    }
  }
  const float scale = scale_of(a);
  if (threadIdx.x == 0) odd = 0;
  const uint32_t lds = (uint32_t)(uintptr_t)buf;
  __builtin_amdgcn_sched_barrier(0);
  uint32_t good = turns.load(u.k0, first, lds);
  uint32_t after = turns.load(u.k0 + KT, second, lds + 2 * BYTES);
  f32x4 o[C][NC * 4];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int d = 0; d < NC * 4; ++d) o[c][d] = f32x4{0, 0, 0, 0};
  float m[C], l[C];
#pragma unroll
  for (int c = 0; c < C; ++c) m[c] = -INFINITY, l[c] = 0.f;

  // a step of 16 elements and a key of the lane's four turn bits of the place
  const int k_at = lds_at<ROW>(r, g), v_at = lds_at<ROW>(4 * g, r);
  auto body = [&](int t, const uint8_t *lds, uint32_t good, bool masked) {
    f32x4 sc[C][NT];
    const int kat = afresh(k_at);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < C; ++c) sc[c][j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const f32x4 k = *(const f32x4 *)(lds + (kat ^ (s << 6)) + 16 * j * ROW);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < C; ++c) sc[c][j] = mfma16(k[i], q[c][s][i], sc[c][j]);
        if (s & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
    // result i of tile j is key t + 16 j + 4 g + i
    if (masked) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int end = min(last[c], u.k1 - 1) - t - 4 * g;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[c][j][i] = ((16 * j + i > end) | !(good >> j & 1)) ? -INFINITY : sc[c][j][i];
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[c][j][i]);
      if (__any((top - m[c]) * scale > SLACK)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float up = (top - m[c]) * scale > SLACK ? top : m[c];
        const float fall = m[c] == -INFINITY ? 1.f : exp2_of((m[c] - up) * scale);
        m[c] = up;
        l[c] *= fall;
        fall_by(o[c], fall);
      }
      const float base = base_of(m[c]);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[c][j][i] = exp2_of((sc[c][j][i] - base) * scale);
          l[c] += sc[c][j][i];
        }
    }
    const int vat = afresh(v_at);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < NC; ++d) {
          const f32x4 v = *(const f32x4 *)(lds + BYTES + (vat ^ (i << 6)) + 256 * d +
                                           (16 * j + i) * ROW);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < C; ++c)
              o[c][4 * d + e] = mfma16(v[e], sc[c][j][i], o[c][4 * d + e]);
          if (d & 1) __builtin_amdgcn_sched_barrier(0);
        }
  };
  auto give = [&](int t, const uint8_t *values, uint32_t good, int key) {
#pragma unroll
    for (int d = 0; d < NC; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 v = *(const f32x4 *)(values + lds_at<ROW>(key, 16 * d + 4 * g + i));
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const bool sees = t + key <= last[c] && t + key < u.k1 && (good >> (key >> 4) & 1);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[c][4 * d + e][i] += sees && !(fabsf(v[e]) < INFINITY) ? v[e] : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  };

  typename Tn::Pages next = turns.look_up(u.k0 + 2 * KT);
  turn_barrier<Tn::MINE * Tn::COPIES>();
  const int full = min(u.pos0 + 1, u.k1);           // keys that every query sees
  for (int t = u.k0, b = 0; t < u.k1; t += KT, b ^= 1) {
    const uint8_t *now = buf[b];
    const bool masked = t + KT > full || good != Tn::GOOD;
    if (masked)
      take_out_odd<float, Tn, NW>((uint8_t *)now + BYTES, &odd,
                   [&](int key) { give(t, now + BYTES, good, key); });
    if (work && t <= wave_last) body(t, now, good, masked);
    turn_barrier<0>();
    good = after;
    if (t + 2 * KT < u.k1) {
      after = turns.load(t + 2 * KT, next, lds + b * 2 * BYTES);
      next = turns.look_up(t + 3 * KT);
    }
  }
  if (turns.bad && threadIdx.x == 0) atomicOr(kv.err, kErrKvRange);
  // result i of o[4 d + e] is element (16 d + 4 g + i) * 4 + e
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float sum = l[c] + __shfl_xor(l[c], 16);
    sum += __shfl_xor(sum, 32);
    if (!on[c]) continue;
    const float inv = u.slot >= 0 ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    const int64_t at = (int64_t)(u.tok + tok[c]) * a.out_token + head[c] * a.out_head;
    float *part = u.slot >= 0 ? part_at(kv, a, u.slot, P, row[c], 0) : nullptr;
#pragma unroll
    for (int d = 0; d < NC; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = (16 * d + 4 * g + i) * 4;
        const float x[4] = {o[c][4 * d][i] * inv, o[c][4 * d + 1][i] * inv,
                            o[c][4 * d + 2][i] * inv, o[c][4 * d + 3][i] * inv};
        if (part) *(f32x4 *)(part + e * 32) = f32x4{x[0], x[1], x[2], x[3]};
        else store_out(a, kv.dtype, at + e, x);
      }
    if (part && g == 0) {
      float *ml = part_sums(kv, a, u.slot, P, row[c]);
      ml[0] = m[c];
      ml[1] = sum;
    }
  }
}

// The parts of a tile joined, with c = the scale in powers of two:
//   out = sum_s 2^(c (m_s - M)) o_s / sum_s 2^(c (m_s - M)) l_s.
// A thread takes four elements of a row; a workgroup ROWS rows and FOURS such fours
// of them (128 bytes of a part, 64 of out side by side), one tile's after another,
// so that few are launched where nothing was split.  Bound by its reads: 8.4 us behind
// 100 tokens over 131,072 keys; 4.4 where there is little, and as much where nothing is.
template <int D>
struct JoinShape {
  static constexpr int FOURS = D / 4 < 32 ? D / 4 : 32, ROWS = kThreads / FOURS;
  static constexpr int GROUPS = kChunkRows / ROWS * (D / 4 / FOURS);
};
template <int D>
__global__ __launch_bounds__(kThreads) void chunk_join_kernel(KvCache kv, Chunk a) {
  typedef JoinShape<D> J;
  constexpr int AT_ONCE = 4;
  const int per = kv.heads * a.shape.tiles;
  const float scale = scale_of(a);
  const int64_t all = min((int64_t)a.plan[1], a.shape.joins) * per * J::GROUPS;
  for (int64_t w = blockIdx.x; w < all; w += gridDim.x) {
    const int64_t unit = w / J::GROUPS;
    const int group = (int)(w - unit * J::GROUPS), rows = group % (kChunkRows / J::ROWS);
    const int row = rows * J::ROWS + threadIdx.x % J::ROWS;
    const int e = group / (kChunkRows / J::ROWS) * J::FOURS + threadIdx.x / J::ROWS;
    const Place P = place_of(kv, a, unit);
    const int4 j = *(const int4 *)(a.plan + kPlanHead + kUnitWords * a.shape.units +
                                   kJoinWords * P.unit);
    if (j.w <= 1 || j.x < 0 || j.y < 0 || j.y > a.shape.tokens ||
        (int64_t)j.x + j.y > a.tokens || j.z < 0 || (int64_t)j.z + j.w > a.shape.parts ||
        row >= j.y * P.heads)
      continue;
    float m = -INFINITY, l = 0.f;
    f32x4 o{0, 0, 0, 0};
    for (int s0 = 0; s0 < j.w; s0 += AT_ONCE) {
      f32x4 so[AT_ONCE];
      float sm[AT_ONCE], sl[AT_ONCE];
#pragma unroll
      for (int x = 0; x < AT_ONCE; ++x) {
        const int s = j.z + min(s0 + x, j.w - 1);
        const float *ml = part_sums(kv, a, s, P, row);
        so[x] = *(const f32x4 *)part_at(kv, a, s, P, row, e);
        sm[x] = ml[0];
        sl[x] = ml[1];
      }
#pragma unroll
      for (int x = 0; x < AT_ONCE; ++x) {
        if (s0 + x >= j.w) break;
        const float top = fmaxf(m, sm[x]), base = base_of(top);
        const float f = m == -INFINITY ? 1.f : exp2_of((m - base) * scale);
        const float y = exp2_of((sm[x] - base) * scale);
        m = top;
        l = l * f + sl[x] * y;
        f32x4 was[1] = {o}, part[1] = {so[x]};
        fall_by(was, f);
        fall_by(part, y);
        o = was[0] + part[0];
      }
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    const float x[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    const int tok = row / P.heads;
    store_out(a, kv.dtype, (int64_t)(j.x + tok) * a.out_token +
                               (P.h0 + row - tok * P.heads) * a.out_head + e * 4, x);
  }
}

template <int D>
void launch_dim(const KvCache &kv, const Chunk &a, uint32_t grid, hipStream_t s) {
  constexpr int F32 = D == 256 ? 8 : 4;
  if (kv.dtype == DT_F32) chunk_f32_kernel<D, F32><<<grid, 64 * F32, 0, s>>>(kv, a);
  else if (kv.dtype == DT_BF16) chunk_kernel<D, __bf16><<<grid, kThreads, 0, s>>>(kv, a);
  else chunk_kernel<D, _Float16><<<grid, kThreads, 0, s>>>(kv, a);
  const int64_t joins = kv.heads * a.shape.tiles * a.shape.joins * JoinShape<D>::GROUPS;
  if (joins)
    chunk_join_kernel<D><<<(uint32_t)(joins < a.most_joins ? joins : a.most_joins), kThreads, 0,
                           s>>>(kv, a);
}

}  // namespace

// A unit has up to kChunkRows rows: every query head of a key-value head that
// fits, and as many tokens.  A row's keys are split (kv_map_kernel) so that the
// units of `split` tiles' work fill the chip; with W = the sum over rows of
// tiles times tokens and L = W / split or more keys a part, parts beyond the
// first and tiles that are split are at most W / L each.
ChunkShape chunk_shape(const KvCache &kv, int64_t rows, int64_t tokens, int64_t hq, int num_cu) {
  ChunkShape c{};
  const int64_t group = hq / kv.heads;
  c.heads = (int32_t)(group < kChunkRows ? group : kChunkRows);
  c.tiles = (int32_t)((group + c.heads - 1) / c.heads);
  c.tokens = kChunkRows / c.heads;
  const int64_t per = (int64_t)kv.heads * c.tiles, most = rows < tokens ? rows : tokens;
  const int64_t tiles = tokens / c.tokens + most;
  // Two units a compute unit, as its LDS holds: 100 tokens over 131,072 keys 296 us
  // (one 362, four 303), 1,000 float32 tokens of five rows 33 (48, 33), 2,000 of twenty 83
  // (92, 106), 64 of two over up to 60,000 of 64 elements 44 (43, 58); the other way
  // 700 of three over up to 9,000 keys 54 (47, 62), 3,001 of thirteen 132 (127, 135)
  c.split = (2ll * num_cu + per - 1) / per;
  // two turns of the kernels.  17 tokens over 511 keys in parts of 64 keys and of 128:
  // 256 bfloat16 elements a key 14.3 and 15.8 us, float32 128 19.5 and 27.4, 256 28.3 and
  // 43.5; bfloat16 64 and 128 11 and 12 either way, float32 64 15.2 and 18.4.  1,000 tokens
  // of five rows over up to 2,000: float32 256 100 and 92, 128 53 and 53, 64 34 and
  // 34; bfloat16 256 36 and 34, 128 23 and 23, 64 18.9 and 17.7
  c.least = kv.dim * kv.esize >= 512 ? 64 : 128;
  const bool can = (((int64_t)kv.max_pages << kv.lg_page) > c.least) && tiles > 0;
  c.joins = can ? (tiles < c.split ? tiles : c.split) : 0;
  c.units = tiles + (can ? c.split : 0);
  c.parts = can ? c.joins + c.split : 0;
  return c;
}

int64_t chunk_workspace(const KvCache &kv, const ChunkShape &c) {
  return c.parts * kv.heads * c.tiles * kChunkRows * (kv.dim + 2) * 4;
}

hipError_t launch_kv_map(const KvCache &kv, const KvMap &m, hipStream_t s) {
  const int64_t n = m.tokens > m.shape.units ? m.tokens : m.shape.units;
  if (m.rows <= kOne) {
    const uint32_t grid = (uint32_t)((n + kOne - 1) / kOne);
    kv_map_kernel<<<grid ? grid : 1, kOne, 0, s>>>(kv, m);
  } else {
    kv_map_rows_kernel<<<1, kOne, 0, s>>>(kv, m);
    if (n > 0) kv_map_tokens_kernel<<<(uint32_t)((n + 255) / 256), 256, 0, s>>>(kv, m);
  }
  return hipGetLastError();
}

hipError_t launch_chunk(const KvCache &kv, const Chunk &a, hipStream_t s) {
  const uint32_t grid = (uint32_t)(kv.heads * a.shape.tiles * a.shape.units);
  if (grid == 0) return hipSuccess;
  if (kv.dim == 64) launch_dim<64>(kv, a, grid, s);
  else if (kv.dim == 128) launch_dim<128>(kv, a, grid, s);
  else launch_dim<256>(kv, a, grid, s);
  return hipGetLastError();
}

}  // namespace w4a8
