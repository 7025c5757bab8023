// What rows of logits say: log probabilities of given tokens, the rows' entropy
// and their best alternatives.  With y = scale x, m its maximum, Z = sum e^(y - m):
//
//   log p = y - m - log Z,  entropy = log Z - sum (y - m) e^(y - m) / Z
//
// in one pass over the logits with a running maximum (both terms of the entropy
// are positive).  The best k come from k of the row's blocks of kBlock logits:
// those whose maxima are the largest, the first of equals.  Each of the best
// logits lies in one, since the k blocks' maxima precede what lies elsewhere; so
// a second kernel reads k blocks again, and no more, whatever the values.
#include "w4a8_mixers.h"

namespace w4a8 {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kBlock = 1024;      // logits of a block
constexpr int kPer = kBlock / 64; // of a lane
constexpr int kList = 1024;       // candidates that are ranked in LDS
constexpr float kFar = 16777216.f; // 2^24: scaled logits of a last bit above 1 lie beyond

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Logits of type T: what their maximum is held as, differences to it, and an
// order on 32 bits (NaN: lowest; a zero has one place).
template <typename T>
struct Logit {
  typedef float Max;
  static constexpr Max none() { return -INFINITY; }
  static __device__ __forceinline__ Max of(T x) { return (float)x; }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return fmaxf(a, b); }
  // of three, a NaN none: without the steps that fmaxf takes for signalling ones
  static __device__ __forceinline__ Max larger(Max a, Max b, Max c) {
    float m;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
    return m;
  }
  // x - m; 0 below nothing at all
  static __device__ __forceinline__ float less(Max x, Max m) {
    return x - (m == -INFINITY ? 0.f : m);
  }
  static __device__ __forceinline__ uint32_t key(Max x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0u : b ^ ((int32_t)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
  }
  static __device__ __forceinline__ Max from_key(uint32_t k) {
    return k == 0 ? NAN : __uint_as_float(k ^ ((int32_t)k < 0 ? 0x80000000u : 0xFFFFFFFFu));
  }
};
template <>
struct Logit<int32_t> {
  typedef int32_t Max;
  static constexpr Max none() { return INT32_MIN; }
  static __device__ __forceinline__ Max of(int32_t x) { return x; }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return max(a, b); }
  static __device__ __forceinline__ Max larger(Max a, Max b, Max c) { return max(max(a, b), c); }
  static __device__ __forceinline__ float less(Max x, Max m) {
    return -(float)((uint32_t)m - (uint32_t)x);
  }
  static __device__ __forceinline__ uint32_t key(Max x) { return (uint32_t)x ^ 0x80000000u; }
  static __device__ __forceinline__ Max from_key(uint32_t k) { return (Max)(k ^ 0x80000000u); }
};

// the largest of 64 lanes' values, in lane 63: neighbours, fours, rows' halves and
// rows of 16, then rows one after another
__device__ __forceinline__ uint32_t largest_of_lanes(uint32_t x) {
#define W4A8_STEP(ctrl, rows) \
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xF, false))
  W4A8_STEP(0xB1, 0xF);    // quad_perm [1,0,3,2]
  W4A8_STEP(0x4E, 0xF);    // quad_perm [2,3,0,1]
  W4A8_STEP(0x141, 0xF);   // row_half_mirror
  W4A8_STEP(0x140, 0xF);   // row_mirror
  W4A8_STEP(0x142, 0xA);   // row_bcast15 -> rows 1, 3
  W4A8_STEP(0x143, 0xC);   // row_bcast31 -> rows 2, 3
#undef W4A8_STEP
  return x;
}

// A running maximum m with Z = sum 2^d and T = sum d 2^d, d = (x - m) scale (in
// powers of two)
template <typename T>
struct Sums {
  typename Logit<T>::Max m = Logit<T>::none();
  float Z = 0.f, S = 0.f;
  static __device__ __forceinline__ Sums from(const float *p) {
    Sums o;
    o.m = __builtin_bit_cast(typename Logit<T>::Max, p[0]);
    o.Z = p[1];
    o.S = p[2];
    return o;
  }
  __device__ __forceinline__ void put(float *p) const {
    p[0] = __builtin_bit_cast(float, m);
    p[1] = Z;
    p[2] = S;
  }
  // to a maximum that is no smaller
  __device__ __forceinline__ void raise(typename Logit<T>::Max to, float scale) {
    const float d = fmaxf(Logit<T>::less(m, to) * scale, -3e38f), f = exp2_of(d);
    S = f * (S + d * Z);
    if (f == 0.f) S = 0.f;          // 2^d without a bit left: d Z may be infinite
    Z *= f;
    m = to;
  }
  __device__ __forceinline__ void join_lanes(float scale) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      Sums o;
      o.m = __shfl_xor(m, d);
      o.Z = __shfl_xor(Z, d);
      o.S = __shfl_xor(S, d);
      join(o, scale);
    }
  }
  __device__ __forceinline__ void join(Sums o, float scale) {
    const auto to = Logit<T>::larger(m, o.m);
    raise(to, scale);
    o.raise(to, scale);
    Z += o.Z;
    S += o.S;
  }
};

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

// Element i of this lane's part of block b, in the order of memory: pieces of 16
// bytes, lane after lane.
template <typename T>
__device__ __forceinline__ int place(int i) {
  constexpr int V = 16 / sizeof(T);
  return (i / V * 64 + (int)(threadIdx.x & 63)) * V + i % V;
}
// A row starts at any element: its blocks are counted from the 16 bytes that its
// first lies in, `shift` elements into them, so that pieces are aligned; those
// that hold others' elements too are read one by one.
template <typename T>
__device__ __forceinline__ int shift_of(const T *row) {
  return (int)(((uintptr_t)row & 15) / sizeof(T));
}
template <typename T>
struct Piece {
  alignas(16) T x[kPer];
};
template <typename T>
__device__ __forceinline__ void load_block(Piece<T> &p, const T *row, int64_t vocab, int64_t first) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < kPer / V; ++j) {
    const int64_t at = first + place<T>(j * V);
    if (at >= 0 && at + V <= vocab) {
      *(u32x4 *)(p.x + j * V) = load16_nt(row + at);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at + i >= 0 && at + i < vocab) p.x[j * V + i] = row[at + i];
    }
  }
}

// First kernel: `splits` workgroups a row, a wavefront a block at a time.  Bound by
// HBM and the exponents beside it: 509 rows of 248,320 bfloat16 logits 48-49 us, 5.2 TB/s
// (reads alone reach 7.35).
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_sums_kernel(Logprobs a) {
  typedef Logit<T> L;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x - r * a.splits);
  const T *row = (const T *)a.logits + r * a.row;
  const int shift = shift_of(row);
  const int each = (a.blocks + a.splits - 1) / a.splits;
  const int b0 = split * each, b1 = min(b0 + each, a.blocks);
  Sums<T> sums;
  auto add = [&](const Piece<T> &p, int b, auto whole) {
    constexpr bool ALL = whole.value;
    const int64_t first = (int64_t)b * kBlock - shift;
    auto in = [&](int i) {
      const int64_t at = first + place<T>(i);
      return ALL || (at >= 0 && at < a.vocab);
    };
    auto top = L::none();
#pragma unroll
    for (int i = 0; i < kPer; i += 2)
      top = L::larger(in(i) ? L::of(p.x[i]) : L::none(), in(i + 1) ? L::of(p.x[i + 1]) : L::none(),
                      top);
    sums.raise(L::larger(sums.m, top), a.scale);
    float Z = 0.f, S = 0.f;
    bool done = false;
    if constexpr (ALL && !__is_same(T, int32_t)) {
      // one multiply-add a difference, against the scaled maximum as it is rounded;
      // what that is off by, half a power of two at most, is taken out of the sums
      const float ref = sums.m * a.scale;
      if (!__any(!(fabsf(ref) < kFar))) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const float d = __builtin_fmaf(L::of(p.x[i]), a.scale, -ref), e = exp2_of(d);
          Z += e;
          S += e * d;
        }
        done = !__any(S != S);              // a logit of -infinity: 0 times that
        const float off = __builtin_fmaf(sums.m, a.scale, -ref), f = exp2_of(-off);
        S = (S - off * Z) * f;
        Z *= f;
      }
    }
    if (!done) {
      Z = S = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float d = in(i) ? L::less(L::of(p.x[i]), sums.m) * a.scale : -INFINITY;
        const float e = exp2_of(d);
        Z += e;
        S += e * fmaxf(d, -3e38f);
      }
    }
    sums.Z += Z;
    sums.S += S;
    if (a.keys) {
      const uint32_t key = largest_of_lanes(L::key(top));
      if (lane == 63) a.keys[r * a.blocks + b] = key;
    }
  };
  Piece<T> p{}, next{};
  int b = b0 + wave;
  if (b < b1) load_block(p, row, a.vocab, (int64_t)b * kBlock - shift);
  for (; b < b1; b += kWaves) {
    if (b + kWaves < b1) load_block(next, row, a.vocab, (int64_t)(b + kWaves) * kBlock - shift);
    const int64_t first = (int64_t)b * kBlock - shift;
    if (first >= 0 && first + kBlock <= a.vocab) add(p, b, Flag<true>());
    else add(p, b, Flag<false>());
    p = next;
  }
  sums.join_lanes(a.scale);
  __shared__ float parts[kWaves][3];
  if (lane == 0) sums.put(parts[wave]);
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kWaves; ++w) sums.join(Sums<T>::from(parts[w]), a.scale);
  sums.put(a.parts + (r * a.splits + split) * 4);
}

// how many of the workgroup's threads say yes
__device__ __forceinline__ int count(int mine) {
  __shared__ int sums[kWaves];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) mine += __shfl_xor(mine, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = mine;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += sums[w];
  return all;
}
// the largest v of which `want` or more of what how_many(v) counts are at least v
template <typename F>
__device__ __forceinline__ uint32_t reached_by(int want, F how_many) {
  uint32_t v = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t to = v | 1u << bit;
    if (how_many(to) >= want) v = to;
  }
  return v;
}

// Second kernel, a workgroup per row: the splits' sums joined, the given token,
// and the best: the k blocks, what in them is at least the last of their maxima
// (k logits or more, mostly few more), and of those each one's rank.  What it
// waits for is two rounds of loads: sums, maxima and the token; the blocks.  With them
// those 509 rows' best five take 14 us, a row of int32 sums and its best 20 with both
// launches 18.5.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Logprobs a) {
  typedef Logit<T> L;
  constexpr int kLocal = 4096, kRanked = 1024;
  // a thread reads 16 bytes of a block, AT_ONCE of them before it looks at any
  constexpr int V = 16 / sizeof(T), SIDE = kThreads / (kBlock / V), AT_ONCE = 4;
  __shared__ float whole[3];
  __shared__ __align__(16) uint32_t keys[kLocal];
  __shared__ uint64_t list[kList];
  __shared__ int32_t blocks[32];
  __shared__ uint32_t smallest;
  __shared__ int listed;
  const int64_t r = blockIdx.x;
  const T *row = (const T *)a.logits + r * a.row;
  const int lane = threadIdx.x & 63, k = a.k, nb = min(k, a.blocks);
  const uint32_t *from = a.keys + r * a.blocks;
  const bool local = a.blocks <= kLocal;
  const int id = a.logp ? a.ids[r] : -1;
  if (k > 0 && local)
    for (int i = threadIdx.x; i < (a.blocks + 3) / 4 * 4; i += kThreads)
      keys[i] = i < a.blocks ? from[i] : 0u;
  T given{};
  if (threadIdx.x == 0 && id >= 0 && id < a.vocab) given = row[id];
  if (threadIdx.x < 64) {
    Sums<T> sums;
    for (int i = lane; i < a.splits; i += 64)
      sums.join(Sums<T>::from(a.parts + (r * a.splits + i) * 4), a.scale);
    sums.join_lanes(a.scale);
    if (lane == 0) {
      sums.put(whole);
      listed = 0;
    }
  }
  __syncthreads();
  const Sums<T> sums = Sums<T>::from(whole);
  const float logZ = log2f(sums.Z);
  auto logp = [&](typename L::Max x) {
    const float d = L::less(x, sums.m) * a.scale;
    // a row of -infinity alone: Z = 0
    return sums.Z == 0.f ? -INFINITY : (d - logZ) * 0.6931471805599453f;
  };
  if (threadIdx.x == 0) {
    if (id >= a.vocab) atomicOr(a.err, kErrToken);
    if (a.logp) a.logp[r] = id >= 0 && id < a.vocab ? logp(L::of(given)) : 0.f;
    if (a.entropy)
      a.entropy[r] = sums.Z == 0.f ? 0.f : (logZ - sums.S / sums.Z) * 0.6931471805599453f;
  }
  if (k == 0) return;

  // f(place, key, rank) of the first n of LDS's keys, in order of size and place;
  // `padded`, a multiple of 4, of them are there
  auto rank_keys = [&](int padded, int n, auto f) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t mine = keys[i];
      int rank = 0;
#pragma unroll 2
      for (int j = 0; j < padded; j += 4) {
        const u32x4 x = *(const u32x4 *)(keys + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) rank += (x[e] > mine) | ((x[e] == mine) & (j + e < i));
      }
      f(i, mine, rank);
    }
    __syncthreads();
  };
  // the k blocks, and the last one's maximum
  uint32_t least = 0;
  if (a.blocks <= k) {
    if ((int)threadIdx.x < a.blocks) blocks[threadIdx.x] = threadIdx.x;
    __syncthreads();
  } else if (a.blocks <= kRanked) {
    rank_keys((a.blocks + 3) / 4 * 4, a.blocks, [&](int i, uint32_t key, int rank) {
      if (rank < k) blocks[rank] = i;
      if (rank == k - 1) smallest = key;
    });
    least = smallest;
  } else {
    auto key_of = [&](int i) { return local ? keys[i] : from[i]; };
    least = reached_by(k, [&](uint32_t v) {
      int mine = 0;
      for (int i = threadIdx.x; i < a.blocks; i += kThreads) mine += key_of(i) >= v;
      return count(mine);
    });
    int above = 0;
    for (int i = threadIdx.x; i < a.blocks; i += kThreads) above += key_of(i) > least;
    int equals = k - count(above);         // so many of the first that equal it
    if (threadIdx.x < 64) {
      for (int base = 0, n = 0; base < a.blocks; base += 64) {
        const int i = base + lane;
        const uint32_t key = i < a.blocks ? key_of(i) : 0;
        const uint64_t same = __ballot(i < a.blocks && key == least);
        const int before = __popcll(same & ((1ull << lane) - 1));
        const bool take = i < a.blocks && (key > least || (key == least && before < equals));
        const uint64_t taken = __ballot(take);
        if (take) blocks[n + __popcll(taken & ((1ull << lane) - 1))] = i;
        n += __popcll(taken);
        equals -= min(equals, (int)__popcll(same));
      }
    }
    __syncthreads();
  }

  // The blocks' logits as 16 bytes a thread, of SIDE blocks at once, AT_ONCE times
  // before any is looked at: f(keys, first place).  Those of no row have key 0.
  const int shift = shift_of(row);
  const int side = SIDE == 1 ? 0 : (int)threadIdx.x / (kBlock / V);
  const int mine_at = ((int)threadIdx.x - side * (kBlock / V)) * V;
  auto each = [&](auto f) {
#pragma unroll 1
    for (int j0 = 0; j0 < nb; j0 += AT_ONCE * SIDE) {
      u32x4 x[AT_ONCE];
      int64_t at[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int b = j0 + j * SIDE + side;
        at[j] = b < nb ? (int64_t)blocks[b] * kBlock - shift + mine_at : a.vocab;
        // what lies beside a row's ends in its 16 bytes is read one by one below
        const bool whole = at[j] >= 0 && at[j] + V <= a.vocab;
        x[j] = whole ? *(const u32x4 *)(row + at[j]) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        struct Vec { T e[V]; };
        Vec v = __builtin_bit_cast(Vec, x[j]);
        const bool whole = at[j] >= 0 && at[j] + V <= a.vocab;
        uint32_t key[V];
#pragma unroll
        for (int e = 0; e < V; ++e) key[e] = whole ? L::key(L::of(v.e[e])) : 0u;
        if (!whole && at[j] < a.vocab) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (at[j] + e >= 0 && at[j] + e < a.vocab) key[e] = L::key(L::of(row[at[j] + e]));
        }
        f(key, at[j]);
      }
    }
  };
  if (a.blocks <= k && a.vocab > kList) {
    // no block was left out: the k-th of the threads' maxima
    uint32_t top = 0;
#pragma unroll 1
    for (int64_t i = threadIdx.x; i < a.vocab; i += kThreads) top = max(top, L::key(L::of(row[i])));
    keys[threadIdx.x] = top;
    __syncthreads();
    rank_keys(kThreads, kThreads, [&](int, uint32_t key, int rank) {
      if (rank == k - 1) smallest = key;
    });
    least = smallest;
  }
  auto put = [&](uint32_t key, int64_t at) {
    const int n = atomicAdd(&listed, 1);
    if (n < kList) list[n] = (uint64_t)key << 32 | (uint32_t)~(uint32_t)at;
  };
  each([&](const uint32_t *key, int64_t at) {
    uint32_t top = key[0];
#pragma unroll
    for (int e = 1; e < V; ++e) top = max(top, key[e]);
    if (top < least) return;
    for (int e = 0; e < V; ++e)
      if (at + e >= 0 && at + e < a.vocab && key[e] >= least) put(key[e], at + e);
  });
  __syncthreads();
  if (listed > kList) {
    // many at least as large: the k-th largest, and which of its equals count;
    // rarely needed, and kept short
    auto all = [&](auto f) {
      int mine = 0;
#pragma unroll 1
      for (int j = 0; j < nb * (kBlock / kThreads); ++j) {
        const int64_t at = (int64_t)blocks[j / (kBlock / kThreads)] * kBlock - shift +
                           j % (kBlock / kThreads) * kThreads + threadIdx.x;
        if (at >= 0 && at < a.vocab) mine += f(L::key(L::of(row[at])), at);
      }
      return count(mine);
    };
    const uint32_t kth = reached_by(k, [&](uint32_t v) {
      return all([&](uint32_t key, int64_t) { return key >= v; });
    });
    const int rest = k - all([&](uint32_t key, int64_t) { return key > kth; });
    // the place of the rest-th of them: not below the last whose earlier are fewer
    const uint32_t first = ~reached_by(rest, [&](uint32_t v) {
      return all([&](uint32_t key, int64_t at) { return key == kth && ~(uint32_t)at >= v; });
    });
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    all([&](uint32_t key, int64_t at) {
      if (key > kth || (key == kth && (uint32_t)at <= first)) put(key, at);
      return 0;
    });
  }
  const int n = min(listed, kList);
  // only a row of NaNs has fewer: any indices
  for (int i = n + threadIdx.x; i < k; i += kThreads) {
    a.top_ids[r * k + i] = i;
    a.top_logp[r * k + i] = NAN;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += list[j] > mine;
    if (rank < k) {
      a.top_ids[r * k + rank] = (int32_t)~(uint32_t)mine;
      a.top_logp[r * k + rank] = logp(L::from_key((uint32_t)(mine >> 32)));
    }
  }
}

template <typename T>
void launch_typed(const Logprobs &a, hipStream_t s) {
  logprobs_sums_kernel<T><<<(uint32_t)(a.rows * a.splits), kThreads, 0, s>>>(a);
  logprobs_kernel<T><<<(uint32_t)a.rows, kThreads, 0, s>>>(a);
}

}  // namespace

// Blocks of a row, counted from the 16 bytes that it starts in, and workgroups
// that share them: sixteen a CU (509 rows of 248,320 64.5 us, with eight 65.2), but at
// least a block for each wavefront.
int logprobs_blocks(int64_t vocab) { return (int)((vocab + 7 + kBlock - 1) / kBlock); }
int logprobs_splits(int64_t rows, int64_t vocab, int num_cu) {
  const int64_t blocks = logprobs_blocks(vocab), most = (blocks + kWaves - 1) / kWaves;
  const int64_t want = (16ll * num_cu + rows - 1) / rows;
  return (int)(want < most ? want : most);
}
int64_t logprobs_workspace(int64_t rows, int64_t vocab, int num_cu) {
  return rows * (logprobs_splits(rows, vocab, num_cu) * 16ll + logprobs_blocks(vocab) * 4ll);
}

hipError_t launch_logprobs(const Logprobs &a, hipStream_t s) {
  if (a.dtype == DT_F32) launch_typed<float>(a, s);
  else if (a.dtype == DT_BF16) launch_typed<__bf16>(a, s);
  else if (a.dtype == DT_F16) launch_typed<_Float16>(a, s);
  else launch_typed<int32_t>(a, s);
  return hipGetLastError();
}

}  // namespace w4a8
