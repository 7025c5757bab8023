// The gated delta rule.  Per value head, with a state S [dk][dv]:
//
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q
//
// (q and k divided by their norms first where asked).  Both dot products of a
// token are taken of the old state in one pass over it: S^T q after the update
// is e^g S^T q + (k . q) u.
#include <algorithm>

#include "w4a8_mixers.h"

namespace w4a8 {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ float to_float(T x, float unit) {
  if constexpr (sizeof(T) == 2 && __is_same(T, int16_t)) return (float)x * unit;
  else return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_float(float x, float out_unit) {
  if constexpr (__is_same(T, int16_t))
    return (int16_t)fminf(fmaxf(rintf(x * out_unit), -32768.f), 32767.f);
  else
    return (T)x;
}

// The slot of a row's state, -1 for none: a padded row, or a slot that an
// earlier row names too or that lies outside the states, which is reported.
// The whole workgroup asks, of a call with one token a row.
__device__ __forceinline__ int slot_of(const Delta &p, int row, bool tell) {
  const int slot = p.slots ? p.slots[row] : row;
  int taken = 0;
  if (p.slots && slot >= 0)
    for (int j = threadIdx.x; j < row; j += blockDim.x) taken |= p.slots[j] == slot;
  taken = __syncthreads_or(taken) || slot >= p.nslots;
  if (taken && tell && threadIdx.x == 0) atomicOr(p.err, kErrDelta);
  return taken ? -1 : slot;
}

// The same for the rows kCheck part .., one a thread of a workgroup of kCheck,
// which compares them with all earlier ones, a tile (of kTile, in LDS) of them at
// a time.
constexpr int kCheck = 256, kTile = 8 * kCheck;
__device__ __forceinline__ int claim_slot(const Delta &p, int part, int32_t *tile) {
  const int first = part * kCheck, j = first + (int)threadIdx.x;
  const int slot = j >= p.rows ? -1 : p.slots ? p.slots[j] : j;
  bool taken = slot >= p.nslots;
  for (int base = 0; p.slots && base < first + kCheck; base += kTile) {
    int32_t x[kTile / kCheck];
#pragma unroll
    for (int i = 0; i < kTile / kCheck; ++i) {
      const int at = base + i * kCheck + (int)threadIdx.x;
      x[i] = at < p.rows ? p.slots[at] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTile / kCheck; ++i) tile[i * kCheck + threadIdx.x] = x[i];
    __syncthreads();
    const int whole = min(first - base, kTile);      // of them, all earlier than this part's
#pragma unroll 16
    for (int k = 0; k < whole; k += 4) {
      const int4 t = *(const int4 *)(tile + k);
      taken |= (t.x == slot) | (t.y == slot) | (t.z == slot) | (t.w == slot);
    }
    if (whole < kTile)
#pragma unroll 16
      for (int k = 0; k < kCheck; k += 4) {
        const int4 t = *(const int4 *)(tile + whole + k);
        const int mine = (int)threadIdx.x - k;      // rows of it before this thread's
        taken |= ((t.x == slot) & (mine > 0)) | ((t.y == slot) & (mine > 1)) |
                 ((t.z == slot) & (mine > 2)) | ((t.w == slot) & (mine > 3));
      }
  }
  taken = taken && slot >= 0;
  if (__syncthreads_or(taken) && threadIdx.x == 0) atomicOr(p.err, kErrDelta);
  return taken ? -1 : slot;
}

// Of many rows, each workgroup of delta_step_kernel looking through the earlier
// ones costs more than a kernel that does it once, and leaves a row's slot where
// the row's workgroups will write their outputs, in the first 4 bytes of each
// one's columns: 2^20 rows of 4 heads 567 -> 33 ms (8.5 of them the states'),
// 65,536 of 1 head 0.76 -> 0.61, 16,384 of 4 0.31 -> 0.25; but 16,384 of 1 0.08
// -> 0.16, so it is done where rows have workgroups enough.
constexpr int kManyRows = 16384, kManyUnits = 65536;
template <typename T>
__global__ __launch_bounds__(kCheck) void delta_claim_kernel(Delta p) {
  __shared__ __align__(16) int32_t tile[kTile];
  const int slot = claim_slot(p, blockIdx.x, tile);
  const int64_t row = (int64_t)blockIdx.x * kCheck + threadIdx.x;
  if (row >= p.rows) return;
  for (int h = 0; h < p.hv; ++h)
    for (int col = 0; col < p.dv; col += 64)
      *(int32_t *)((T *)p.out + row * p.out_token + h * p.out_head + col) = slot;
}

// One token of each row: a wavefront holds 16 columns of a head's state in
// registers, lane (rg, cq) = (lane >> 2, lane & 3) its rows NR rg .. and
// columns 4 cq .., so that a state is read and written once, in 64-byte runs.
// Bound by that: 125 rows of 32 heads of 128 x 128, 527 MB in 106 us, 4.97 TB/s,
// what a large copy reaches; one row, 4.2 MB, 4.9 us of which 2 are a launch's.
template <int DK, typename T>
__global__ __launch_bounds__(256) void delta_step_kernel(Delta p) {
  constexpr int NR = DK / 16;
  const int row = blockIdx.x, h = blockIdx.y;
  int slot;
  if (p.claimed) {
    slot = *(const int32_t *)((const T *)p.out + row * p.out_token + h * p.out_head +
                              blockIdx.z * 64);
    __syncthreads();             // read by all before it is written over
  } else {
    slot = slot_of(p, row, h == 0 && blockIdx.z == 0);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rg = lane >> 2, col = (blockIdx.z * 4 + wave) * 16 + (lane & 3) * 4;
  if (col >= p.dv) return;
  T *out = (T *)p.out + row * p.out_token + h * p.out_head + col;
  if (slot < 0) {
    if (rg == 0)
      for (int c = 0; c < 4; ++c) out[c] = (T)0;
    return;
  }
  float *S = p.state + (((int64_t)slot * p.hv + h) * p.dk + rg * NR) * p.dv + col;
  f32x4 s[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) s[i] = *(const f32x4 *)(S + (int64_t)i * p.dv);
  const int hk = h / (p.hv / p.hk);
  const T *q = (const T *)p.q + row * p.q_token + hk * p.q_head + rg * NR;
  const T *k = (const T *)p.k + row * p.k_token + hk * p.k_head + rg * NR;
  const T *v = (const T *)p.v + row * p.v_token + h * p.v_head + col;
  float qv[NR], kv[NR];
  float qq = 0.f, kk = 0.f, kq = 0.f;
  f32x4 pk{0, 0, 0, 0}, pq{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    qv[i] = to_float(q[i], p.unit);
    kv[i] = to_float(k[i], p.unit);
    qq += qv[i] * qv[i];
    kk += kv[i] * kv[i];
    kq += kv[i] * qv[i];
    pk += s[i] * kv[i];
    pq += s[i] * qv[i];
  }
#pragma unroll
  for (int d = 4; d < 64; d <<= 1) {
    qq += __shfl_xor(qq, d);
    kk += __shfl_xor(kk, d);
    kq += __shfl_xor(kq, d);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      pk[c] += __shfl_xor(pk[c], d);
      pq[c] += __shfl_xor(pq[c], d);
    }
  }
  const float rq = (p.norm ? 1.f / sqrtf(qq + p.eps) : 1.f) * p.scale;
  const float rk = p.norm ? 1.f / sqrtf(kk + p.eps) : 1.f;
  const float e = expf(p.g[row * p.g_token + h]), beta = p.beta[row * p.beta_token + h];
  f32x4 u;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    u[c] = beta * (to_float(v[c], p.unit) - e * rk * pk[c]);
    const float o = rq * (e * pq[c] + rk * kq * u[c]);
    if (rg == 0) out[c] = from_float<T>(o, p.out_unit);
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) *(f32x4 *)(S + (int64_t)i * p.dv) = s[i] * e + u * (kv[i] * rk);
}

// ------------------------------------------------------------ whole prompts
// A prompt goes in chunks of C = 64 tokens.  With G the running sum of g in a
// chunk, S0 the state before it, and rows of q, k, v as matrices, the tokens'
// u are the solution of a triangular system (strictly lower A):
//
//   A_tj = beta_t e^(G_t - G_j) k_t . k_j  (j < t),   M = (I + A)^-1 diag(beta)
//   U = M (V - diag(e^G) K S0)
//   O = scale (diag(e^G) Q S0 + P U),  P_tj = e^(G_t - G_j) q_t . k_j  (j <= t)
//   S = e^(G_C) S0 + K^T diag(e^(G_C - G)) U
//
// M and P of every chunk do not depend on the state: delta_prep_kernel makes
// them, all chunks at once; delta_scan_kernel then walks a row's chunks, a
// workgroup per head and 16 columns of the state, which stays in registers.
// Decays are differences of sums of g in 64 bits (an e^g of 0 among them
// would otherwise cost the others their bits), and each is at most 1 where g
// is at most 0.
//
// The products run on the bfloat16 matrix instructions with float32 sums: a
// float32 operand is the sum of three bfloat16 values, exactly (float16 and
// int16 of two, bfloat16 of one), and of the products of two operands' terms
// those below 2^-24 are left out.  So a state keeps its 24 bits through a
// prompt; a norm of q or k is a factor of its row, applied to the sums.
// (Exactly: from 2^-103 up to where bfloat16 ends, 2^128 - 2^119.)  From a token
// with an infinity or a NaN in k, v, g or beta on, its head's outputs, for v its
// column's alone, and the state are NaN; the tokens before it are what they are
// without it.
constexpr int C = 64;
constexpr int kTriBytes = 6 * 3 * 64 * 16;       // M or P: operands of tri_of, three terms
constexpr int kVecFloats = 256;                  // a, b, c of 64 tokens, e^(G_C) 64 times
constexpr int kHeadBytes = 2 * kTriBytes + kVecFloats * 4;   // of a chunk and value head
// K and Q of a chunk and key head, as operands
constexpr int64_t rows_bytes(int64_t dk, int terms) { return 2 * C * dk * 2 * terms; }
constexpr float kNoDecay = -200.f;               // e^g is 0 in float32 from here on down

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// terms of what goes into outputs alone
template <typename T>
constexpr int out_terms() {
  return __is_same(T, __bf16) || __is_same(T, _Float16) ? 2 : 3;
}
template <typename T>
struct Terms {
  static constexpr int n = sizeof(T) == 4 ? 3 : __is_same(T, __bf16) ? 1 : 2;
};

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma4(f32x4 a, f32x4 b, f32x4 c) {   // 16 x 16 x 16, float32
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}
template <int N>
struct Int {
  static constexpr int value = N;
};
// sum of the products of terms a[i] b[j] with i + j <= L
template <int NA, int NB, int L>
__device__ __forceinline__ f32x4 mfma_terms(const bf16x8 *a, const bf16x8 *b, f32x4 c) {
#pragma unroll
  for (int i = NA - 1; i >= 0; --i)
#pragma unroll
    for (int j = NB - 1; j >= 0; --j)
      if (i + j <= L) c = mfma(a[i], b[j], c);
  return c;
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// x[0 .. M) as a sum of N vectors of bfloat16, a pair of values per conversion
// (whose result is kept as one word: taken apart, the compiler converts each
// value again, 17 instructions a pair instead of 11)
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  uint32_t w = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
  asm("" : "+v"(w));
  return w;
}
template <int N, int M, typename V>
__device__ __forceinline__ void split(const float *x, V *t) {
  uint32_t w[N][M / 2];
#pragma unroll
  for (int j = 0; j < M / 2; ++j) {
    float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i][j] = pair_of(a, b);
      a -= __builtin_bit_cast(float, w[i][j] << 16);
      b -= __builtin_bit_cast(float, w[i][j] & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) __builtin_memcpy(&t[i], w[i], sizeof(V));
}

// Barrier of the workgroup for LDS alone: loads from memory stay in flight,
// and what waits for them is not moved up across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  __builtin_amdgcn_sched_barrier(0);
}

// The order of a chunk's tokens in an operand of k-steps s = 0, 1: slot j of
// lane group g is token 32 s + 16 (j >> 2) + 4 g + (j & 3), so that a lane's
// four results of row tiles 2 s and 2 s + 1 are its own eight slots.  The state's
// rows d are in the same order.
// M and P as operands: row tile w (of 16 tokens) and k-step s <= w / 2
__device__ __forceinline__ constexpr int tri_of(int w, int s) {
  return w < 2 ? w : w == 2 ? 2 + s : 4 + s;
}

// first chunk of a row in the workspace: rows do not share chunks
__device__ __forceinline__ int first_chunk(const Delta &p, int row) {
  return p.cu[row] / C + row;
}

// Chunks that the workspace has room for, and where behind them the
// findings on the rows lie: each row's slot (-1: none), then for every kCheck rows whether
// the bounds of one of them are out of order.
__device__ __forceinline__ int64_t chunks_of(const Delta &p) { return p.tokens / C + p.rows; }
__device__ __forceinline__ int32_t *row_slots(const Delta &p, int64_t chunk_bytes) {
  return (int32_t *)((uint8_t *)p.ws + chunks_of(p) * chunk_bytes);
}
__device__ __forceinline__ int32_t *row_faults(const Delta &p, int64_t chunk_bytes) {
  return row_slots(p, chunk_bytes) + p.rows;
}

// The findings on rows kCheck part .., by a workgroup of kCheck threads: what it
// finds wrong is reported here.
__device__ void check_rows(const Delta &p, int part, int32_t *slots, int32_t *faults,
                           int32_t *tile) {
  const int j = part * kCheck + (int)threadIdx.x;
  const bool on = j < p.rows;
  const int t0 = on ? p.cu[j] : 0, t1 = on ? p.cu[j + 1] : 0;
  const int slot = claim_slot(p, part, tile);
  if (on) slots[j] = slot;
  const int bad = __syncthreads_or(t0 < 0 || t1 < t0 || t1 > p.tokens);
  if (threadIdx.x == 0) {
    faults[part] = bad;
    if (bad) atomicOr(p.err, kErrDelta);
  }
}

// Which row chunk `slot` of the workspace belongs to, -1: none (a row's chunks
// are fewer than its room, or its bounds are out of order).  The last row whose
// first chunk is not behind it, looked for among blockDim.x rows at a time; the
// whole workgroup asks.
__device__ __forceinline__ int row_of(const Delta &p, int slot) {
  int lo = 0, n = p.rows;
  while (n > 1) {
    const int step = (n + (int)blockDim.x - 1) / (int)blockDim.x, at = (int)threadIdx.x * step;
    const int before = __syncthreads_count(at < n && first_chunk(p, lo + at) <= slot);
    if (before == 0) return -1;
    lo = __builtin_amdgcn_readfirstlane(lo + (before - 1) * step);
    n = __builtin_amdgcn_readfirstlane(min(step, n - (before - 1) * step));
  }
  const int t0 = p.cu[lo], t1 = p.cu[lo + 1], at = slot - (t0 / C + lo);
  if (t0 < 0 || t1 < t0 || t1 > p.tokens || at < 0 || at >= (t1 - t0 + C - 1) / C) return -1;
  return lo;
}

// A chunk in the workspace: M, P and factors per value head, rows per key head;
// the chunks of a head lie side by side.
template <int DK, typename T>
struct Space {
  static constexpr int64_t kRows = rows_bytes(DK, Terms<T>::n);
  uint8_t *ws;
  int64_t chunks, chunk, heads;
  __device__ Space(const Delta &p, int64_t c)
      : ws((uint8_t *)p.ws), chunks(chunks_of(p)), chunk(c), heads(p.hv) {}
  // of a chunk, all heads
  static __device__ int64_t bytes(const Delta &p) {
    return (int64_t)p.hv * kHeadBytes + p.hk * kRows;
  }
  __device__ uint8_t *head(int h) const { return ws + (h * chunks + chunk) * kHeadBytes; }
  // 0: K, 1: Q
  __device__ bf16x8 *rows(int hk, int which) const {
    return (bf16x8 *)(ws + heads * chunks * kHeadBytes + (hk * chunks + chunk) * kRows +
                      which * (kRows / 2));
  }
};

// A workgroup per chunk, key head and share of its value heads, and behind the
// chunks' one per kCheck rows for the findings on them.  It lays K and
// Q out as the operands that delta_scan_kernel reads, in whole lines (read where
// they lie, rows of a prompt 4 KB apart all fall to one channel of the L2: the
// scan of 8192 tokens, 16 key heads of 128, took 34 us more).  Tiles of M and P
// are made transposed (rows j, columns t), which leaves a lane with four
// neighbouring slots of their operand: nothing is rearranged.
//
// Bound by memory: 8192 bfloat16 tokens, 16 key and 32 value heads of 128, 67 MB
// read and 195 MB written in 64-69 us (3.9 TB/s).  M and P, which no cache holds
// until they are read, are written past them: prep and scan 268 -> 244 us; K and
// Q too, 257.
template <int DK, typename T>
__global__ __launch_bounds__(256, 2) void delta_prep_kernel(Delta p) {
  constexpr int NK = Terms<T>::n, NS = DK / 32, LD = 68, HEADS = 4;
  __shared__ bf16x8 Ks[4][NS][NK][64];             // K by row tiles, as operand
  __shared__ double Gs[HEADS][C];                  // log2(e) times the running sum of g
  __shared__ __align__(16) float betas[HEADS][C], rks[C], rqs[C];
  __shared__ int firsts[HEADS];
  __shared__ __align__(16) float At[C * LD];       // A transposed
  __shared__ __align__(16) float Tt[4][16 * 20];   // its diagonal blocks' inverses, transposed
  const int slot = blockIdx.x, hk = blockIdx.y;
  if (slot >= chunks_of(p)) {
    const int64_t bytes = Space<DK, T>::bytes(p);
    static_assert(sizeof(At) >= kTile * sizeof(int32_t), "no tile of slots");
    if (hk == 0 && blockIdx.z == 0)
      check_rows(p, slot - (int)chunks_of(p), row_slots(p, bytes), row_faults(p, bytes),
                 (int32_t *)At);
    return;
  }
  const int row = row_of(p, slot);
  if (row < 0) return;
  const int chunk = slot - first_chunk(p, row);
  const int t0 = p.cu[row] + chunk * C, len = min(C, p.cu[row + 1] - t0);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Space<DK, T> space(p, slot);
  const int per = p.hv / p.hk, share = (per + (int)gridDim.z - 1) / (int)gridDim.z;
  const int head0 = blockIdx.z * share, head1 = min(per, head0 + share);
  const bool rows_too = blockIdx.z == 0;           // the first share writes K and Q

  // rows 16 w + r of x, elements 32 s + 8 g .., as terms (zeros past the
  // chunk's end), written as operand; the sum of their squares
  bf16x8 kw[NS][NK], qw[NS][NK];
  auto load = [&](const void *x, int64_t token, int64_t head, bf16x8 (*f)[NK], int which) {
    const int t = 16 * w + r;
    const bool on = t < len;
    const T *src = (const T *)x + (t0 + min(t, len - 1)) * token + hk * head + 8 * g;
    float sum = 0.f;
    bf16x8 *out = space.rows(hk, which) + lane;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      T v[8];
      *(u32x4 *)v = *(const u32x4 *)(src + 32 * s);
      if constexpr (sizeof(T) == 4) *(u32x4 *)(v + 4) = *(const u32x4 *)(src + 32 * s + 4);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = on ? to_float(v[j], p.unit) : 0.f;
        sum += y[j] * y[j];
      }
      split<NK, 8>(y, f[s]);
#pragma unroll
      for (int i = 0; i < NK; ++i)
        if (rows_too) out[((w * NS + s) * NK + i) * 64] = f[s][i];
    }
    sum += __shfl_xor(sum, 16);
    return sum + __shfl_xor(sum, 32);
  };
  const float kk2 = load(p.k, p.k_token, p.k_head, kw, 0);
  const float qq2 = load(p.q, p.q_token, p.q_head, qw, 1);
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < NK; ++i) Ks[w][s][i][lane] = kw[s][i];
  if (g == 0) {
    const bool on = 16 * w + r < len;
    rks[16 * w + r] = !on ? 0.f : !finite(kk2) ? NAN : p.norm ? 1.f / sqrtf(kk2 + p.eps) : 1.f;
    rqs[16 * w + r] = !on ? 0.f : (p.norm ? 1.f / sqrtf(qq2 + p.eps) : 1.f) * p.scale;
  }
  __syncthreads();
  // k_j . k_t and k_j . q_t, j = 16 c + 4 g + i, t = 16 w + r, up to the diagonal
  f32x4 kk[4], kq[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    kk[c] = kq[c] = f32x4{0, 0, 0, 0};
    if (c <= w)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        bf16x8 kc[NK];
#pragma unroll
        for (int i = 0; i < NK; ++i) kc[i] = Ks[c][s][i][lane];
        kk[c] = mfma_terms<NK, NK, 2>(kc, kw[s], kk[c]);
        kq[c] = mfma_terms<NK, NK, 2>(kc, qw[s], kq[c]);
      }
  }
  // row tile w of M (which 0) or P out of its transposed tiles X[c], c <= w
  auto store = [&](uint8_t *ws, auto which, const f32x4 *X) {
    constexpr int N = which.value ? out_terms<T>() : 3;
    bf16x8 *out = (bf16x8 *)(ws + which.value * kTriBytes) + lane;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (s <= w >> 1) {
        bf16x8 t[3];
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = X[2 * s + (j >> 2)][j & 3];
        split<N, 8>(x, t);
#pragma unroll
        for (int i = 0; i < N; ++i)
          __builtin_nontemporal_store(t[i], &out[(tri_of(w, s) * 3 + i) * 64]);
      }
  };

  for (int first = head0; first < head1; first += HEADS) {
    const int count = min(HEADS, head1 - first);
    if (w < count) {   // a wavefront per head: its tokens' factors
      const int h = hk * per + first + w;
      const bool on = lane < len;
      const int64_t t = t0 + min(lane, len - 1);
      float gt = on ? p.g[t * p.g_token + h] : 0.f;
      gt = gt < kNoDecay ? kNoDecay : gt;          // a NaN stays one
      const float bt = on ? p.beta[t * p.beta_token + h] : 0.f;
      double G = gt * 1.4426950408889634;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(G, d);
        if (lane >= d) G += y;
      }
      // from the first token on whose k, g or beta is no number, M is 0 and a NaN
      const uint64_t odd = __ballot(!finite((float)G) || !finite(bt) || !finite(rks[lane]));
      const int first = odd ? __builtin_ctzll(odd) : C;
      if (lane == 0) firsts[w] = first;
      Gs[w][lane] = G;
      betas[w][lane] = lane < first ? bt : 0.f;
      const double GC = __shfl(G, 63);
      float *vec = (float *)(space.head(h) + 2 * kTriBytes);
      vec[lane] = !on ? 0.f : lane < first ? exp2_of((float)G) * rks[lane] : NAN;
      vec[64 + lane] = on ? exp2_of((float)G) * rqs[lane] : 0.f;
      vec[128 + lane] = on ? exp2_of((float)(GC - G)) * rks[lane] : 0.f;
      vec[192 + lane] = exp2_of((float)GC);
    }
    for (int b = 0; b < count; ++b) {
      uint8_t *ws = space.head(hk * per + first + b);
      __syncthreads();               // Gs, betas; the last head's At, Tt are read
      {
        const int t = 16 * w + r;
        const double Gt = Gs[b][t];
        const float rqt = rqs[t], bt = betas[b][t] * rks[t];
        const int before = min(t, t < firsts[b] ? C : 0);   // of the tokens that A_t has
        f32x4 P[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          P[c] = f32x4{0, 0, 0, 0};
          if (c <= w) {
            const f32x4 rkj = *(const f32x4 *)(rks + 16 * c + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = 16 * c + 4 * g + i;
              const float dec = exp2_of((float)(Gt - Gs[b][j])) * rkj[i];
              At[j * LD + t] = j < before ? bt * dec * kk[c][i] : 0.f;
              P[c][i] = j <= t ? rqt * dec * kq[c][i] : 0.f;
            }
          }
        }
        store(ws, Int<1>(), P);
      }
      __syncthreads();
      {   // the inverse of diagonal block w: lane r column r, by substitution
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i == r ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < 15; ++j) {
          const float *a = At + (16 * w + j) * LD + 16 * w;
#pragma unroll
          for (int i = j + 1; i < 16; ++i) x[i] -= a[i] * x[j];
        }
        if (g == 0)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *(f32x4 *)(Tt[w] + r * 20 + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
      }
      __syncthreads();
      {   // block row w of the inverse T, transposed: with T (I + A) = I,
          // T_wc^T = -T_cc^T sum_(c < k <= w) A_kc^T T_wk^T
        f32x4 X[4];
#pragma unroll
        for (int c = 3; c >= 0; --c) {
          X[c] = f32x4{0, 0, 0, 0};
          if (c == w) {
#pragma unroll
            for (int i = 0; i < 4; ++i) X[c][i] = Tt[c][(4 * g + i) * 20 + r];
          } else if (c < w) {
            f32x4 acc{0, 0, 0, 0};
#pragma unroll
            for (int k = c + 1; k < 4; ++k)
              if (k <= w)
                acc = mfma4(*(const f32x4 *)(At + (16 * c + r) * LD + 16 * k + 4 * g), X[k], acc);
            X[c] = mfma4(-*(const f32x4 *)(Tt[c] + r * 20 + 4 * g), acc, X[c]);
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) X[c] *= *(const f32x4 *)(betas[b] + 16 * c + 4 * g);
        store(ws, Int<0>(), X);
      }
    }
    __syncthreads();                 // betas are read
  }
}

// A workgroup per row, value head and 16 columns of the state, eight
// wavefronts on 16 tokens each: the chain of a chunk, S0 -> V - a K S0 -> U ->
// S, on four of them and the outputs, b Q S0 + P U, on the other four, so that
// the chain's trips through LDS are filled with the outputs' products.  Where
// there is one row, a chunk's chain is what bounds the kernel, and beside it the
// bytes that a CU's vector cache passes on (each column tile reads K, Q, M and P
// for itself).  So operands are loaded as soon as an earlier chunk has used
// their registers, the factors once per workgroup, and K transposed for the
// update comes out of LDS by transposed reads instead of from memory again.
// 8192 bfloat16 tokens of 32 heads of 128 x 128: 192-203 us, 1.5 us a chunk; of
// 8 heads, a quarter of the chip, 1.1 us a chunk.
//
// Wavefront w of the chain has rows 32 w .. of the state too: lane (r, g) rows
// 32 w + 8 g + 4 e + i of column r, in register S[e][i], which is its slots of
// the state as an operand; its results of U are slots of that operand likewise.
//
// Outputs are rounded to 16 bits (bfloat16, float16): two terms of their
// operands, an error of 2^-17, are enough for them (8192 bfloat16 tokens with
// three: 255 us, not 245).
//
// Key heads of 64 of 16-bit values are held to the registers of two workgroups a
// CU: 8 prompts of 1000 float16 tokens, 32 heads of 64 x 128, 235 us; 245 without.
template <int DK, typename T>
__global__ __launch_bounds__(512, DK == 64 && sizeof(T) == 2 ? 4 : 1) void
delta_scan_kernel(Delta p) {
  constexpr int NK = Terms<T>::n, NS = DK / 32;
  constexpr int OT = out_terms<T>();
  __shared__ bf16x8 Sb[3][NS][64];                // the state, k-step s by wavefront s
  __shared__ __align__(16) bf16x4 Rb[3][2][64][2], Ub[OT][2][64][2], Wb[3][2][64][2];
  __shared__ __align__(16) T Ts[8][16 * 16];      // a wavefront's tokens' values or outputs
  __shared__ __align__(16) uint8_t Kl[NK][C * DK * 2];   // K by rows, see k_at
  __shared__ __align__(16) float Fs[2][kVecFloats];   // a chunk's factors and the next one's
  __shared__ int seen;                            // whether a chunk of the row was odd
  __shared__ __align__(16) int odds[4];           // this one's tokens, by wavefront,
  __shared__ int firsts[4][16];                   // and each column's first odd one
  const int tiles = p.dv / 16, units = p.rows * p.hv, each = (units + 7) / 8;
  // a head's columns, and heads that share keys, on one XCD (workgroups go
  // round the eight of them)
  const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
  const int unit = xcd * each + at / tiles;
  if (at / tiles >= each || unit >= units) return;
  const int row = unit / p.hv, h = unit - row * p.hv, hk = h / (p.hv / p.hk);
  const int32_t *faults = row_faults(p, Space<DK, T>::bytes(p));
  const int slot = row_slots(p, Space<DK, T>::bytes(p))[row];
  int bad = 0;
  for (int i = threadIdx.x; i < (p.rows + kCheck - 1) / kCheck; i += 512) bad |= faults[i];
  if (__syncthreads_or(bad)) return;              // reported by delta_prep_kernel
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int col = (at % tiles) * 16 + r;
  const int begin = p.cu[row], end = p.cu[row + 1];
  if (slot < 0) {
    T *out = (T *)p.out + h * p.out_head + col;
    for (int t = begin + (int)(threadIdx.x >> 4); t < end; t += 32) out[t * p.out_token] = (T)0;
    return;
  }
  const int n = (end - begin + C - 1) / C;
  if (n == 0) {                                   // no tokens: the state stays, or is cleared
    float *state = p.state + ((int64_t)slot * p.hv + h) * DK * p.dv + col;
    if (p.fresh)
      for (int d = threadIdx.x >> 4; d < DK; d += 32) state[(int64_t)d * p.dv] = 0.f;
    return;
  }
  // of the chunk whose operands are loaded next
  const Space<DK, T> space(p, first_chunk(p, row));
  const uint8_t *ws = space.head(h);
  // row tile w of M (which 0) or P, terms i of k-step s
  auto tri = [&](int which, int s, int i) -> const bf16x8 & {
    return ((const bf16x8 *)(ws + which * kTriBytes) + (tri_of(w, s) * 3 + i) * 64)[lane];
  };
  // a, b or c of tokens 16 w + 4 g ..
  auto factor = [&](int ch, int which) {
    return *(const f32x4 *)(Fs[ch & 1] + 64 * which + 16 * w + 4 * g);
  };
  // Values and outputs move in pieces of 16 bytes, PIECES a row of 16 columns
  // (single values would be four loads and four stores for one), and change
  // between pieces and results' places in LDS, within a wavefront.  piece_at:
  // where this lane's lies, in bytes from a chunk's first token; past the
  // chunk's end of len tokens the last one's is read, whose factors and
  // columns of M and P are zeros.
  constexpr int PIECES = sizeof(T);
  const int prow = (lane / PIECES) & 15, piece = lane % PIECES;
  T *tile = &Ts[wave][0];
  auto piece_at = [&](int len, int64_t token) {
    return (uint32_t)(min(16 * w + prow, len - 1) * (int)token + col - r) * (uint32_t)sizeof(T) +
           (uint32_t)piece * 16;
  };
  // A token is odd in a column whose V - a K S0 is no finite number (k, v, g, beta
  // or the state were not).  0 times it would spoil the tokens before it in the
  // chunk's products.  So a row in which one was seen is walked again, from its
  // state, which is written last, and then the column's tokens from the first odd
  // one on are taken out of the products, and made NaN through Q S0 and the state's
  // factor.  (Decided in the chain of every chunk, six ragged prompts took 38.4 us,
  // not 37.3.  And no branch stands between a product and the first use of its
  // result: the compiler does not always wait for it across one.)
  auto any_odd = [&](int4 o) {
    return __builtin_amdgcn_readfirstlane(o.x | o.y | o.z | o.w) != 0;
  };
  auto first_odd = [&]() {
    int first = C;
    for (int i = 0; i < 4; ++i)
      if (odds[i]) first = min(first, firsts[i][r]);
    return first;
  };
  auto exchange = [&]() {                         // a wavefront's writes before its reads
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  };

  auto chain = [&](auto upper, auto again) {
    constexpr bool AGAIN = again.value;
    constexpr bool HI = upper.value;              // w >= 2: two k-steps of M
    constexpr bool STATE = NS == 4 || !HI;        // rows of the state
    float *state = p.state + (((int64_t)slot * p.hv + h) * DK + 32 * w + 8 * g) * p.dv + col;
    f32x4 S[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (STATE && !p.fresh) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) S[e][i] = state[(int64_t)(4 * e + i) * p.dv];
    }
    auto put_state = [&]() {
      bf16x8 t[3];
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = S[j >> 2][j & 3];
      split<3, 8>(x, t);
#pragma unroll
      for (int i = 0; i < 3; ++i) Sb[i][w][lane] = t[i];
    };
    auto put_rows = [&](bf16x4 (*b)[2][64][2], f32x4 x, auto terms) {
      bf16x4 t[3];
      const float y[4] = {x[0], x[1], x[2], x[3]};
      split<terms.value, 4>(y, t);
#pragma unroll
      for (int i = 0; i < terms.value; ++i) b[i][w >> 1][lane][w & 1] = t[i];
    };
    const uint8_t *kb = (const uint8_t *)space.rows(hk, 0);
    // K goes to LDS by rows, in the order of the pieces of 16 bytes changed so
    // that neither these writes (a lane's token is 16 w + r) nor the transposed
    // reads (16 lanes: 4 tokens of a group, 4 pieces each) meet in a bank
    constexpr int TURN = DK == 128 ? 0 : 1;
    auto turn_of = [&](int t) { return ((t >> TURN) & (DK == 128 ? 3 : 1)) << 2 | ((t >> 2) & 3); };
    auto k_at = [&](int t, int at) { return t * DK * 2 + ((at ^ turn_of(t)) * 16); };
    const int kt_at = k_at(4 * g + (r >> 2), 4 * w + (r & 3));
    const uint8_t *vb = (const uint8_t *)((const T *)p.v + begin * p.v_token + h * p.v_head);
    const int64_t v_step = p.v_token * C * (int)sizeof(T);
    uint32_t v_at = piece_at(C, p.v_token);
    struct In {
      bf16x8 k[NS][NK], m[2][3];
      u32x4 v;
    };
    const uint8_t *const kb0 = kb, *const vb0 = vb, *const ws0 = ws;
    auto next = [&](int ch) {                     // its operands are loaded from here on
      ch = min(ch, n - 1);
      kb = kb0 + ch * space.kRows;
      vb = vb0 + ch * v_step;
      ws = ws0 + (int64_t)ch * kHeadBytes;
      if (end - begin - ch * C < C) v_at = piece_at(end - begin - ch * C, p.v_token);
    };
    auto load_rows = [&](In &x) {
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int s = 0; s < NS; ++s)
          x.k[s][i] = ((const bf16x8 *)kb + ((w * NS + s) * NK + i) * 64)[lane];
      x.v = *(const u32x4 *)(vb + v_at);
    };
    auto load_solve = [&](In &x) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        x.m[0][i] = tri(0, 0, i);
        if constexpr (HI) x.m[1][i] = tri(0, 1, i);
      }
    };
    // K transposed as operand: rows d = 32 w + 8 (m >> 2) + 4 e + (m & 3) of
    // tile e, four tokens of a lane's slots at a time
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_x4;
    auto transposed = [&](int s, int e, int i) {
      s16x4 t[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        t[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_x4 *)(Kl[i] + kt_at + (32 * s + 16 * j) * DK * 2 + 8 * e));
      bf16x8 x;
      __builtin_memcpy(&x, t, sizeof(x));
      return x;
    };
    // U and W once more without the odd tokens; the first one of the column
    auto without_odd = [&](int ch, In &x) {
      auto take_out = [&](bf16x4 (*b)[2][64][2], auto terms, int first) {
        for (int i = 0; i < terms.value; ++i)
          for (int e = 0; e < 4; ++e)
            if (16 * w + 4 * g + e >= first) b[i][w >> 1][lane][w & 1][e] = (__bf16)0.f;
      };
      const int first = first_odd();
      take_out(Rb, Int<3>(), first);
      lds_barrier();
      const uint8_t *const after = ws;
      ws = ws0 + (int64_t)ch * kHeadBytes;
      load_solve(x);
      bf16x8 b[2][3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        b[0][i] = *(const bf16x8 *)Rb[i][0][lane];
        if constexpr (HI) b[1][i] = *(const bf16x8 *)Rb[i][1][lane];
      }
      f32x4 u = mfma_terms<3, 3, 2>(x.m[0], b[0], f32x4{0, 0, 0, 0});
      if constexpr (HI) u = mfma_terms<3, 3, 2>(x.m[1], b[1], u);
      put_rows(Wb, u * factor(ch, 2), Int<3>());
      put_rows(Ub, u, Int<OT>());
      take_out(Wb, Int<3>(), first);
      take_out(Ub, Int<OT>(), first);
      lds_barrier();
      ws = after;
      load_solve(x);
      return first;
    };
    // Loads go out behind a segment's reads of LDS, in the time those take.
    auto step = [&](int ch, In &x) {
      const int len = min(C, end - begin - ch * C);
      {
        bf16x8 sb[NS][3];
        T v[4];
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int i = 0; i < 3; ++i) sb[s][i] = Sb[i][s][lane];
        *(u32x4 *)(tile + prow * 16 + piece * (16 / (int)sizeof(T))) = x.v;
        exchange();
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = tile[(4 * g + i) * 16 + r];
        const f32x4 a = factor(ch, 0);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 ks{0, 0, 0, 0}, z;
#pragma unroll
        for (int s = 0; s < NS; ++s) ks = mfma_terms<NK, 3, 2>(x.k[s], sb[s], ks);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          z[i] = (16 * w + 4 * g + i < len ? to_float(v[i], p.unit) : 0.f) - a[i] * ks[i];
        put_rows(Rb, z, Int<3>());
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int i = 0; i < NK; ++i) *(bf16x8 *)(Kl[i] + k_at(16 * w + r, 4 * s + g)) = x.k[s][i];
      }
      lds_barrier();
      next(ch + 1);
      bf16x8 kt[2][2][NK];
      {
        bf16x8 b[2][3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          b[0][i] = *(const bf16x8 *)Rb[i][0][lane];
          if constexpr (HI) b[1][i] = *(const bf16x8 *)Rb[i][1][lane];
        }
        const f32x4 c = factor(ch, 2);
        if constexpr (STATE)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < NK; ++i) kt[s][e][i] = transposed(s, e, i);
        __builtin_amdgcn_sched_barrier(0);
        load_rows(x);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 u = mfma_terms<3, 3, 2>(x.m[0], b[0], f32x4{0, 0, 0, 0});
        if constexpr (HI) u = mfma_terms<3, 3, 2>(x.m[1], b[1], u);
        put_rows(Wb, u * c, Int<3>());
        put_rows(Ub, u, Int<OT>());
      }
      lds_barrier();
      int4 o4{0, 0, 0, 0};
      if constexpr (AGAIN) o4 = *(const int4 *)odds;
      if constexpr (STATE) {
        bf16x8 b[2][3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          b[0][i] = *(const bf16x8 *)Wb[i][0][lane];
          b[1][i] = *(const bf16x8 *)Wb[i][1][lane];
        }
        float fall = Fs[ch & 1][192];
        __builtin_amdgcn_sched_barrier(0);
        load_solve(x);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (AGAIN)
          if (any_odd(o4)) {
            if (without_odd(ch, x) < C) fall = NAN;
#pragma unroll
            for (int i = 0; i < 3; ++i) {
              b[0][i] = *(const bf16x8 *)Wb[i][0][lane];
              b[1][i] = *(const bf16x8 *)Wb[i][1][lane];
            }
          }
        S[0] *= fall;
        S[1] *= fall;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          S[0] = mfma_terms<NK, 3, 2>(kt[s][0], b[s], S[0]);
          S[1] = mfma_terms<NK, 3, 2>(kt[s][1], b[s], S[1]);
        }
        put_state();
      } else {
        load_solve(x);
        if constexpr (AGAIN)
          if (any_odd(o4)) without_odd(ch, x);
      }
      lds_barrier();
    };
    // the first chunks' operands, in the order of the loop, so that its waits
    // are for what it uses
    In in;
    if constexpr (STATE) put_state();
    next(0);
    __builtin_amdgcn_sched_barrier(0);
    load_rows(in);
    __builtin_amdgcn_sched_barrier(0);
    load_solve(in);
    lds_barrier();
    for (int ch = 0; ch < n; ++ch) step(ch, in);
    if constexpr (!AGAIN) lds_barrier();            // the last outputs were looked at
    if constexpr (STATE)
      if (AGAIN || !seen)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) state[(int64_t)(4 * e + i) * p.dv] = S[e][i];
  };

  auto output = [&](auto upper, auto again) {
    constexpr bool AGAIN = again.value, LATE = NS * NK <= 4;
    constexpr bool HI = upper.value;
    const uint8_t *qb = (const uint8_t *)space.rows(hk, 1);
    uint8_t *ob = (uint8_t *)((T *)p.out + begin * p.out_token + h * p.out_head);
    const int64_t o_step = p.out_token * C * (int)sizeof(T);
    const uint32_t o_at = piece_at(C, p.out_token);
    bf16x8 q[NS][NK], m[2][OT];
    f32x4 o{0, 0, 0, 0}, factors;
    const uint8_t *const qb0 = qb, *const ws0 = ws;
    // a chunk's rows of Q and their factors; its rows of P
    auto load_rows = [&](int ch, bf16x8 (*q)[NK]) {
      qb = qb0 + ch * space.kRows;
      ws = ws0 + (int64_t)ch * kHeadBytes;
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int s = 0; s < NS; ++s)
          q[s][i] = ((const bf16x8 *)qb + ((w * NS + s) * NK + i) * 64)[lane];
    };
    // a chunk's factors go to LDS for every wavefront, by the first of these
    auto load_factors = [&](int ch) {
      if (w == 0) factors = ((const f32x4 *)(ws0 + (int64_t)ch * kHeadBytes + 2 * kTriBytes))[lane];
    };
    auto put_factors = [&](int ch) {
      if (w == 0) *(f32x4 *)(Fs[ch & 1] + 4 * lane) = factors;
    };
    auto load_weights = [&](int ch) {
      ws = ws0 + (int64_t)ch * kHeadBytes;
#pragma unroll
      for (int i = 0; i < OT; ++i) {
        m[0][i] = tri(1, 0, i);
        if constexpr (HI) m[1][i] = tri(1, 1, i);
      }
    };
    auto write = [&](int ch) {
      const int len = min(C, end - begin - ch * C);
#pragma unroll
      for (int i = 0; i < 4; ++i) tile[(4 * g + i) * 16 + r] = from_float<T>(o[i], p.out_unit);
      exchange();
      const u32x4 x = *(const u32x4 *)(tile + prow * 16 + piece * (16 / (int)sizeof(T)));
      if (lane < 16 * PIECES && 16 * w + prow < len) store16_nt(ob + o_at, x);
      ob += o_step;
      if constexpr (!AGAIN)                         // an odd token's outputs are
        if (__any(!finite(o[0]) || !finite(o[1]) || !finite(o[2]) || !finite(o[3])) && lane == 0)
          seen = 1;
    };
    // whether V - a K S0 of this wavefront's tokens, by its first terms, is odd
    auto look_for_odd = [&]() {
      bool odd[4], any = false;
      uint32_t z[2];
      __builtin_memcpy(z, &Rb[0][w >> 1][lane][w & 1], sizeof(z));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        odd[e] = (z[e >> 1] >> (16 * (e & 1)) & 0x7F80) == 0x7F80;
        any |= odd[e];
      }
      any = __any(any);
      if (any) {
        int first = C;
#pragma unroll
        for (int e = 3; e >= 0; --e) first = odd[e] ? 16 * w + 4 * g + e : first;
        first = min(first, __shfl_xor(first, 16));
        first = min(first, __shfl_xor(first, 32));
        if (g == 0) firsts[w][r] = first;
      }
      if (lane == 0) odds[w] = any;
    };
    load_factors(0);
    load_rows(0, q);
    load_weights(0);
    put_factors(0);
    lds_barrier();
    for (int ch = 0; ch < n; ++ch) {
      // beside the chain's first segment the last chunk's outputs are written,
      // beside its second Q S0 is made, beside its third P U: no segment has
      // more than its share of the loads and stores.  Q of one term leaves the
      // registers for the next chunk's beside it: Q S0 is read beside the second
      // segment and made beside the third (8192 bfloat16 tokens 258 -> 245 us).
      if (ch) write(ch - 1);
      load_factors(min(ch + 1, n - 1));
      lds_barrier();
      bf16x8 sb[NS][OT], qn[NS][NK];
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < OT; ++i) sb[s][i] = Sb[i][s][lane];
      const f32x4 b = factor(ch, 1);
      if constexpr (AGAIN) look_for_odd();
      auto q_state = [&]() {
        o = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; ++s) o = mfma_terms<NK, OT, OT - 1>(q[s], sb[s], o);
        o *= b;
      };
      if constexpr (LATE) {
        load_rows(min(ch + 1, n - 1), qn);
        lds_barrier();
        q_state();
        __builtin_memcpy(q, qn, sizeof(q));
      } else {
        q_state();
        load_rows(min(ch + 1, n - 1), q);
        lds_barrier();
      }
      bf16x8 ub[2][OT];
      auto get_u = [&]() {
#pragma unroll
        for (int i = 0; i < OT; ++i) {
          ub[0][i] = *(const bf16x8 *)Ub[i][0][lane];
          if constexpr (HI) ub[1][i] = *(const bf16x8 *)Ub[i][1][lane];
        }
      };
      int4 o4{0, 0, 0, 0};
      if constexpr (AGAIN) o4 = *(const int4 *)odds;
      get_u();
      if constexpr (AGAIN)
        if (any_odd(o4)) {
          const int first = first_odd();
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = 16 * w + 4 * g + i < first ? o[i] : NAN;
          lds_barrier();                            // the chain's, in without_odd
          lds_barrier();
          get_u();
        }
      o = mfma_terms<OT, OT, OT - 1>(m[0], ub[0], o);
      if constexpr (HI) o = mfma_terms<OT, OT, OT - 1>(m[1], ub[1], o);
      load_weights(min(ch + 1, n - 1));
      put_factors(ch + 1);
      lds_barrier();
    }
    write(n - 1);
    if constexpr (!AGAIN) lds_barrier();
  };
  // the same number of barriers on every way
  auto walk = [&](auto again) {
    ws = space.head(h);
    if (wave < 4) {
      if (w < 2) chain(Int<0>(), again);
      else chain(Int<1>(), again);
    } else {
      if (w < 2) output(Int<0>(), again);
      else output(Int<1>(), again);
    }
  };
  if (threadIdx.x == 0) seen = 0;                 // chain and outputs meet before it is used
  walk(Int<0>());
  if (seen) walk(Int<1>());
}

template <int DK, typename T>
void launch_typed(const Delta &d, int num_cu, hipStream_t s) {
  if (!d.cu) {
    if (d.claimed) delta_claim_kernel<T><<<(d.rows + kCheck - 1) / kCheck, kCheck, 0, s>>>(d);
    delta_step_kernel<DK, T><<<dim3(d.rows, d.hv, (d.dv + 63) / 64), 256, 0, s>>>(d);
    return;
  }
  // A key head's value heads one after another where the chunks fill the chip
  // twice, otherwise each in a workgroup of its own (which lays out K and Q
  // again, but for the writing), up to that: 9 chunks of 16 key and 32 value
  // heads 30.9 -> 27.9 us with the scan, 48 of 1 and 8 97.5 -> 72.5; beyond it,
  // 31 chunks of 16 and 32, 70 -> 75.
  const int64_t units = (d.tokens / C + (int64_t)d.rows) * d.hk;
  const int shares =
      (int)std::max<int64_t>(std::min<int64_t>(d.hv / d.hk, 2 * num_cu / units), 1);
  const int parts = (d.rows + kCheck - 1) / kCheck;
  delta_prep_kernel<DK, T><<<dim3(d.tokens / C + d.rows + parts, d.hk, shares), 256, 0, s>>>(d);
  const int64_t each = ((int64_t)d.rows * d.hv + 7) / 8;
  delta_scan_kernel<DK, T><<<(uint32_t)(8 * each * (d.dv / 16)), 512, 0, s>>>(d);
}

template <int DK>
void launch_dim(const Delta &d, int num_cu, hipStream_t s) {
  if (d.dtype == DT_F32) launch_typed<DK, float>(d, num_cu, s);
  else if (d.dtype == DT_BF16) launch_typed<DK, __bf16>(d, num_cu, s);
  else if (d.dtype == DT_F16) launch_typed<DK, _Float16>(d, num_cu, s);
  else launch_typed<DK, int16_t>(d, num_cu, s);
}

}  // namespace

int64_t delta_workspace(int64_t tokens, int64_t rows, int64_t hk, int64_t hv, int64_t dk,
                        int dtype) {
  const int terms = dtype == DT_F32 ? Terms<float>::n
                    : dtype == DT_BF16 ? Terms<__bf16>::n : Terms<_Float16>::n;
  const int64_t findings = 4 * (rows + (rows + kCheck - 1) / kCheck);
  return (tokens / C + rows) * (hv * kHeadBytes + hk * rows_bytes(dk, terms)) +
         (findings + 15) / 16 * 16;
}

hipError_t launch_delta(Delta d, int num_cu, hipStream_t s) {
  d.claimed = !d.cu && d.slots && d.rows >= kManyRows &&
              (int64_t)d.rows * d.hv * ((d.dv + 63) / 64) >= kManyUnits;
  if (d.dk == 64) launch_dim<64>(d, num_cu, s);
  else launch_dim<128>(d, num_cu, s);
  return hipGetLastError();
}

}  // namespace w4a8
