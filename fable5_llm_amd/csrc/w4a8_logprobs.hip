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

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Logits of type T: what their maximum is held as, differences to it, and an
// order on 32 bits (NaN: lowest; a zero has one place).
template <typename T>
struct Logit {
  typedef float Max;
  static constexpr Max none() { return -INFINITY; }
  static __device__ __forceinline__ Max of(T x) { return (float)x; }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return fmaxf(a, b); }
  // x - m; 0 below nothing at all
  static __device__ __forceinline__ float less(Max x, Max m) {
    return x - (m == -INFINITY ? 0.f : m);
  }
  static __device__ __forceinline__ uint32_t key(Max x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0u : b ^ ((int32_t)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
  }
};
template <>
struct Logit<int32_t> {
  typedef int32_t Max;
  static constexpr Max none() { return INT32_MIN; }
  static __device__ __forceinline__ Max of(int32_t x) { return x; }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return max(a, b); }
  static __device__ __forceinline__ float less(Max x, Max m) {
    return -(float)((uint32_t)m - (uint32_t)x);
  }
  static __device__ __forceinline__ uint32_t key(Max x) { return (uint32_t)x ^ 0x80000000u; }
};

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

// First kernel: `splits` workgroups a row, a wavefront a block at a time.
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
    for (int i = 0; i < kPer; ++i)
      if (in(i)) top = L::larger(top, L::of(p.x[i]));
    sums.raise(L::larger(sums.m, top), a.scale);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float d = in(i) ? L::less(L::of(p.x[i]), sums.m) * a.scale : -INFINITY;
      const float e = exp2_of(d);
      sums.Z += e;
      sums.S += e * fmaxf(d, -3e38f);   // a logit of -infinity: 0, not 0 times that
    }
    if (a.keys) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) top = L::larger(top, __shfl_xor(top, d));
      if (lane == 0) a.keys[r * a.blocks + b] = L::key(top);
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
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t to = v | 1u << bit;
    if (how_many(to) >= want) v = to;
  }
  return v;
}

// Second kernel, a workgroup per row: the splits' sums joined, the given token,
// and the best: the k blocks, what in them is at least the last of their maxima
// (k logits or more, mostly few more), and of those each one's rank.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Logprobs a) {
  typedef Logit<T> L;
  __shared__ float whole[3];
  __shared__ uint32_t keys[4096];
  __shared__ uint64_t list[kList];
  __shared__ int32_t blocks[32];
  __shared__ int listed;
  const int64_t r = blockIdx.x;
  const T *row = (const T *)a.logits + r * a.row;
  const int lane = threadIdx.x & 63;
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
  auto logp = [&](T x) {
    const float d = L::less(L::of(x), sums.m) * a.scale;
    // a row of -infinity alone: Z = 0
    return sums.Z == 0.f ? -INFINITY : (d - logZ) * 0.6931471805599453f;
  };
  if (threadIdx.x == 0) {
    const int id = a.ids ? a.ids[r] : -1;
    if (a.logp) {
      if (id >= a.vocab) atomicOr(a.err, kErrToken);
      a.logp[r] = id >= 0 && id < a.vocab ? logp(row[id]) : 0.f;
    }
    if (a.entropy)
      a.entropy[r] = sums.Z == 0.f ? 0.f : (logZ - sums.S / sums.Z) * 0.6931471805599453f;
  }
  if (a.k == 0) return;

  // the k blocks, in the order of the row
  const uint32_t *from = a.keys + r * a.blocks;
  const bool local = a.blocks <= 4096;
  if (local)
    for (int i = threadIdx.x; i < a.blocks; i += kThreads) keys[i] = from[i];
  __syncthreads();
  auto key_of = [&](int i) { return local ? keys[i] : from[i]; };
  const int k = a.k, nb = min(k, a.blocks);
  uint32_t least = 0;
  if (a.blocks > k)
    least = reached_by(k, [&](uint32_t v) {
      int mine = 0;
      for (int i = threadIdx.x; i < a.blocks; i += kThreads) mine += key_of(i) >= v;
      return count(mine);
    });
  int above = 0;
  for (int i = threadIdx.x; i < a.blocks; i += kThreads) above += key_of(i) > least;
  int equals = nb - count(above);          // so many of the first that equal it
  if (a.blocks <= k) {
    if ((int)threadIdx.x < a.blocks) blocks[threadIdx.x] = threadIdx.x;
    __syncthreads();
  } else if (threadIdx.x < 64) {
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

  // what in them is at least v, by its key and place: every thread its own
  const int shift = shift_of(row);
  auto each = [&](auto f) {
    for (int j = 0; j < nb; ++j) {
      const int64_t first = (int64_t)blocks[j] * kBlock - shift;
#pragma unroll
      for (int i = 0; i < kBlock / kThreads; ++i) {
        const int64_t at = first + i * kThreads + threadIdx.x;
        if (at >= 0 && at < a.vocab) f(L::key(L::of(row[at])), (uint32_t)at);
      }
    }
  };
  auto list_up = [&](uint32_t v, uint32_t last) {     // those of v itself up to place last
    each([&](uint32_t key, uint32_t at) {
      if (key > v || (key == v && at <= last)) {
        const int n = atomicAdd(&listed, 1);
        if (n < kList) list[n] = (uint64_t)key << 32 | (uint32_t)~at;
      }
    });
    __syncthreads();
  };
  if (a.blocks <= k && a.vocab > kList) {
    // no block was left out: the k-th of the threads' maxima
    uint32_t top = 0;
    each([&](uint32_t key, uint32_t) { top = max(top, key); });
    least = reached_by(k, [&](uint32_t v) { return count(top >= v); });
  }
  list_up(least, 0xFFFFFFFFu);
  if (listed > kList) {
    // many at least as large: the k-th largest, and which of its equals count
    const uint32_t kth = reached_by(k, [&](uint32_t v) {
      int mine = 0;
      each([&](uint32_t key, uint32_t) { mine += key >= v; });
      return count(mine);
    });
    int more = 0;
    each([&](uint32_t key, uint32_t) { more += key > kth; });
    const int rest = k - count(more);
    // the place of the rest-th of them: not below the last whose earlier are fewer
    const uint32_t first = ~reached_by(rest, [&](uint32_t v) {
      int mine = 0;
      each([&](uint32_t key, uint32_t at) { mine += key == kth && ~at >= v; });
      return count(mine);
    });
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    list_up(kth, first);
  }
  const int n = min(listed, kList);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > mine;
    if (rank < k) {
      const uint32_t at = ~(uint32_t)mine;
      a.top_ids[r * k + rank] = (int32_t)at;
      a.top_logp[r * k + rank] = logp(row[at]);
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
// that share them: eight a CU, but at least a block for each wavefront.
int logprobs_blocks(int64_t vocab) { return (int)((vocab + 7 + kBlock - 1) / kBlock); }
int logprobs_splits(int64_t rows, int64_t vocab, int num_cu) {
  const int64_t blocks = logprobs_blocks(vocab), most = (blocks + kWaves - 1) / kWaves;
  const int64_t want = (8ll * num_cu + rows - 1) / rows;
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
