// Attention of one new token per row over a paged key-value cache.
//
//   o_h = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q_h . k_t - m),
//
// in one pass over the cache with a running maximum m and sum; a row's tokens
// are split over workgroups when there are few rows, each split leaving its
// maximum, sum and unnormalised output for a second kernel to join.
//
// The query heads that share a key-value head (up to 16 at a time) are the
// columns of the matrix instructions, so that keys and values are read once.
// A wavefront takes 32 tokens at a time (16 of a float32 cache) and keeps them
// in registers from the load to the product, without LDS:
//   scores^T = K Q^T: lane (r, g) = (lane & 15, lane >> 4) holds 16 bytes of
//     token r at every 64-byte step of the head, the instruction's A operand;
//     the result's lane holds tokens 4 g + i of head r.
//   out^T = V^T P^T: those are the 8 (or 4) k-slots of lane group g in the
//     B operand, so P goes from one product to the next as it lies.  The A
//     operand wants one element of d of those tokens: a lane loads 16 bytes of
//     each of its group's tokens (16 lanes: a row's whole 256 bytes) and picks
//     the pairs apart with byte permutes.  The order of d over lanes and
//     instructions is free, and is undone where out is written.
#include "w4a8_mixers.h"

namespace w4a8 {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// what exponents are taken against: the maximum, or 0 where no score is above
// -infinity, so that every weight there is 0 and not a NaN
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Barrier of the workgroup for LDS alone: loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  __builtin_amdgcn_sched_barrier(0);
}

// Per cache type: a lane's 16 bytes as matrix operand.
template <typename T>
struct Half {
  typedef T x8 __attribute__((ext_vector_type(8)));
};

struct Range {
  int seq, n, t0, t1, used;   // the row's tokens, this split's, splits in use
};

// the row's length and this split's tokens of it: whole chunks, the same
// count for every split but the last
__device__ __forceinline__ Range range_of(const KvCache &kv, const Attend &a, int row, int split) {
  Range r{a.seqs[row], 0, 0, 0, 0};
  if (r.seq >= 0 && r.seq < kv.seqs) {
    int n = kv.lens[r.seq];
    const int64_t most = (int64_t)kv.max_pages << kv.lg_page;
    if (n > most) n = (int)most;
    if (a.upto) n = min(n, a.upto[row]);
    r.n = max(n, 0);
  }
  const int each = max((r.n + a.splits - 1) / a.splits, 1);
  const int per = (each + kAttendChunk - 1) / kAttendChunk * kAttendChunk;
  r.used = (int)(((int64_t)r.n + per - 1) / per);
  const int64_t t0 = (int64_t)split * per;
  r.t0 = __builtin_amdgcn_readfirstlane((int)(t0 < r.n ? t0 : r.n));
  r.t1 = __builtin_amdgcn_readfirstlane((int)(t0 + per < r.n ? t0 + per : r.n));
  return r;
}

template <typename T>
__device__ __forceinline__ void store_row(T *p, const float *x, int n) {
#pragma unroll
  for (int i = 0; i < n; ++i) p[i] = (T)x[i];
}

// out[d .. d + n) of a head: rounded once
__device__ __forceinline__ void store_out(const Attend &a, int cache_dtype, int64_t at,
                                          const float *x, int n) {
  if (a.dtype == DT_I16) {
    int16_t *p = (int16_t *)a.out + at;
    for (int i = 0; i < n; ++i)
      p[i] = (int16_t)fminf(fmaxf(rintf(x[i] * a.out_unit), -32768.f), 32767.f);
  } else if (cache_dtype == DT_F32) {
    store_row((float *)a.out + at, x, n);
  } else if (cache_dtype == DT_BF16) {
    store_row((__bf16 *)a.out + at, x, n);
  } else {
    store_row((_Float16 *)a.out + at, x, n);
  }
}

// I16: q is int16 (its value of a step is part of a.scale), exact as the sum
// of two 8-bit values of the cache's type, both of q's sign and neither zero
// unless q is: times an infinite key they are that infinity, not a NaN.  Over a
// 16-bit cache P goes into the second product as the sum of two values of that
// type, off by half a step squared (bfloat16 2^-16, float16 2^-22) of a weight,
// so that the output's own rounding is the only one that counts.
// Workgroups: key-value heads fastest, then a row's splits, then rows.  Two a CU
// at least, but for heads of 256 of float32 (whose registers are far over that)
// and of int16 rows, which two a CU make no faster.  A head of 256 of 16-bit
// values is held to that by keeping q in LDS: 244 registers (with q in
// registers, six values spilled: two rows of 131,072 tokens 177 us, so 167.5;
// one row of 511 tokens 9.9, so 10.3).
//
// Bound by the reading of keys and values where the cache is long: 2 rows of
// 131,072 tokens, 4 heads of 256, 1.07 GB in 164 us, 6.5 TB/s (int16 rows the
// same).  Short ones are latency, four loads one after another and one turn of
// the tiles: 8.5 us for one row of 511 tokens.
template <int D, typename T, bool I16>
__global__ __launch_bounds__(64 * kWaves, D == 256 && (I16 || sizeof(T) == 4) ? 1 : 2) void
attend_kernel(KvCache kv, Attend a) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int kTok = F32 ? 16 : 32;              // tokens of a turn
  constexpr int NT = kTok / 16;                    // 16-token tiles of them
  constexpr int KS = F32 ? D / 16 : D / 32;        // 64-byte steps of a key
  constexpr int VEC = F32 ? 4 : (D == 64 ? 4 : 8); // elements of a value load
  constexpr int NC = D / (16 * VEC);               // loads of a value row
  constexpr int ROWS = F32 ? 4 : 8;                // value rows of a lane group
  constexpr int QT = I16 && !F32 ? 2 : 1;          // values that q is the sum of
  constexpr int PT = F32 ? 1 : 2;                  // and that P is
  constexpr int LD = D + 4;                        // floats of a head's row in LDS
  // a float16 weight's exponent ends at 2^-24: weights there are 2^14 as large,
  // and so are their sum and the output until it is divided by it
  constexpr float LIFT = __is_same(T, _Float16) ? 14.f : 0.f;
  __shared__ float obuf[2][16 * LD];
  __shared__ float mbuf[kWaves][16], lbuf[kWaves][16];
  // q in LDS where registers are short
  constexpr bool QL = D == 256 && !F32;
  constexpr int QS = QL ? KS / kWaves : KS;        // steps of q a wavefront holds
  __shared__ __align__(16) T qbuf[QL ? QT * KS : 1][64][8];

  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.hq / kv.heads, tiles = (group + 15) / 16;
  const int heads_all = kv.heads * tiles, unit = blockIdx.x / heads_all;
  const int tile = blockIdx.x - unit * heads_all, kvh = tile / tiles;
  const int h0 = (tile - kvh * tiles) * 16;
  const int row = unit / a.splits, split = unit - row * a.splits;
  const int heads = min(16, group - h0);           // of this tile
  const Range R = range_of(kv, a, row, split);
  if (R.seq >= kv.seqs && split == 0 && threadIdx.x == 0) atomicOr(kv.err, kErrKvRange);
  const int hq = kvh * group + h0 + r;             // this lane's query head
  if (R.used == 0 && split == 0) {                 // nothing to attend to: zeros
    const float zero[4] = {0, 0, 0, 0};
    for (int e = threadIdx.x * 4; e < heads * D; e += 64 * kWaves * 4)
      store_out(a, kv.dtype,
                row * a.out_row + (kvh * group + h0 + e / D) * a.out_head + e % D, zero, 4);
  }
  if (split >= R.used) return;

  // q as B operand: head r, elements 8 g .. (4 g ..) of each step; a wavefront
  // makes every fourth step where they go to LDS
  typedef typename Half<T>::x8 x8;
  x8 qh[QT][F32 ? 1 : QS];
  f32x4 qf[F32 ? KS : 1];
  {
    const int64_t at = row * a.q_row + hq * a.q_head;
    const bool on = r < heads;
#pragma unroll
    for (int n = 0; n < QS; ++n) {
      const int s = QL ? n * kWaves + wave : n;
      if constexpr (F32) {
        const int64_t e = at + s * 16 + g * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          qf[n][i] = !on ? 0.f : I16 ? (float)((const int16_t *)a.q)[e + i]
                                     : ((const float *)a.q)[e + i];
      } else {
        const int64_t e = at + s * 32 + g * 8;
        const u32x4 w = on ? *(const u32x4 *)((const T *)a.q + e) : u32x4{0, 0, 0, 0};
        if constexpr (I16) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int x = (int16_t)(w[i >> 1] >> (16 * (i & 1)));
            const int lo = x < 0 ? -(-x & 255) : x & 255, hi = x - lo;
            const bool both = hi != 0 && lo != 0;
            qh[0][n][i] = (T)(both ? (float)hi : 0.5f * (float)x);
            qh[1][n][i] = (T)(both ? (float)lo : 0.5f * (float)x);
          }
        } else {
          qh[0][n] = __builtin_bit_cast(x8, w);
        }
      }
    }
  }

  const int page = kv.page(), lg = kv.lg_page;
  const int32_t *table = kv.tables + (int64_t)R.seq * kv.max_pages;
  const int64_t plane = (int64_t)page * D;          // elements of a head's page
  const int64_t kbase = (((int64_t)a.layer * 2) * kv.heads + kvh) * plane;

  f32x4 acc[NC * VEC];
#pragma unroll
  for (int i = 0; i < NC * VEC; ++i) acc[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.f;
  int bad = 0;

  // the pages of a turn's 16-token tiles, looked up a turn ahead; a tile past
  // the end, or whose page is none of the pool's, reads page 0 and is masked
  int next[NT];
  auto look_up = [&](int t) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int tt = t + 16 * j;
      next[j] = table[(tt < R.t1 ? tt : R.t0) >> lg];
    }
  };
  // a lane's bytes from a tile's first row: the tile's address is the same in
  // every lane
  const uint32_t k_at = (r * D + g * (F32 ? 4 : 8)) * (int)sizeof(T);
  const uint32_t v_at = (4 * g * D + r * VEC) * (int)sizeof(T);
  const uint8_t *vp[NT];
  int lim[NT];                                      // tokens below it count
  u32x4 kr[NT][KS], vr[ROWS][NC];
  auto load_keys = [&](int t) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int tt = t + 16 * j;
      int p = __builtin_amdgcn_readfirstlane(tt < R.t1 ? next[j] : 0);
      lim[j] = R.t1;
      if ((uint32_t)p >= (uint32_t)kv.pages) {
        bad = 1;
        p = 0;
        lim[j] = 0;
      }
      const uint8_t *kp = kv.pool + p * kv.page_bytes +
                          (kbase + (int64_t)(tt & (page - 1)) * D) * (int)sizeof(T);
      vp[j] = kp + kv.heads * plane * (int)sizeof(T);
#pragma unroll
      for (int s = 0; s < KS; ++s) kr[j][s] = load16_nt(kp + k_at + 64 * s);
    }
    look_up(t + kWaves * kTok);
  };
  auto load_values = [&]() {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint8_t *src =
            vp[i >> 2] + v_at + ((i & 3) * D + c * 16 * VEC) * (int)sizeof(T);
        if constexpr (VEC * sizeof(T) == 16) {
          vr[i][c] = load16_nt(src);
        } else {
          const u32x2 y = __builtin_nontemporal_load((const u32x2 *)src);
          vr[i][c] = u32x4{y.x, y.y, 0, 0};
        }
      }
  };
  f32x4 sc[NT];
  // scores of tokens t + 16 j + 4 g + i for head r
  auto scores = [&]() {
    int at = lane;
    if constexpr (QL) asm volatile("" : "+v"(at));  // read again every turn, not kept
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      sc[j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (F32) {
          const f32x4 k4 = __builtin_bit_cast(f32x4, kr[j][s]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[i], qf[s][i], sc[j], 0, 0, 0);
        } else {
          const x8 k8 = __builtin_bit_cast(x8, kr[j][s]);
#pragma unroll
          for (int q = 0; q < QT; ++q) {
            if constexpr (QL) sc[j] = mfma(k8, *(const x8 *)qbuf[q * KS + s][at], sc[j]);
            else sc[j] = mfma(k8, qh[q][s], sc[j]);
          }
        }
      }
    }
  };
  // the weights of tokens t .., and their values added up.  The next turn's
  // keys may be in flight already: lims are this turn's.
  auto weigh = [&](int t, const int *lim) {
    float top = m;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool live = t + 16 * j + 4 * g + i < lim[j];
        sc[j][i] = live ? sc[j][i] * a.scale : -INFINITY;
        top = fmaxf(top, sc[j][i]);
      }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float base = base_of(top), fall = exp2_of(m - base);
    m = top;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[j][i] = exp2_of(sc[j][i] - base + LIFT);   // a base of millions has no bits for LIFT
        sum += sc[j][i];
      }
    l = l * fall + sum;
    if (__any(fall != 1.f)) {
#pragma unroll
      for (int i = 0; i < NC * VEC; ++i) acc[i] *= fall;
    }
    // what lies in a masked value row may be anything: not a factor of 0
    if (t + kTok > R.t1 || lim[0] == 0 || lim[NT - 1] == 0) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (t + 16 * (i >> 2) + 4 * g + (i & 3) >= lim[i >> 2])
#pragma unroll
          for (int c = 0; c < NC; ++c) vr[i][c] = u32x4{0, 0, 0, 0};
    }
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const f32x4 v4 = __builtin_bit_cast(f32x4, vr[i][c]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[c * VEC + e] =
                __builtin_amdgcn_mfma_f32_16x16x4f32(v4[e], sc[0][i], acc[c * VEC + e], 0, 0, 0);
        }
    } else {
      x8 p[PT];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = sc[i >> 2][i & 3];
        p[0][i] = (T)w;
        p[1][i] = (T)(w - (float)p[0][i]);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = __builtin_amdgcn_perm(vr[2 * i + 1][c][e >> 1], vr[2 * i][c][e >> 1],
                                         e & 1 ? 0x07060302u : 0x05040100u);
          const x8 v = __builtin_bit_cast(x8, w);
#pragma unroll
          for (int q = 0; q < PT; ++q) acc[c * VEC + e] = mfma(v, p[q], acc[c * VEC + e]);
        }
    }
  };
  // A turn's registers are loaded with the next turn's keys once its scores are
  // made, and with its values once those are added up, so that a tile of each
  // wavefront is in flight throughout.
  constexpr int kStep = kWaves * kTok;
  int t = R.t0 + wave * kTok;
  if (t < R.t1) {
    look_up(t);
    load_keys(t);
    __builtin_amdgcn_sched_barrier(0);
    load_values();
  }
  if constexpr (QL) {
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int n = 0; n < QS; ++n) *(x8 *)qbuf[q * KS + n * kWaves + wave][lane] = qh[q][n];
    lds_barrier();
  }
  if (t < R.t1) {
    for (; t + kStep < R.t1; t += kStep) {
      int now[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) now[j] = lim[j];
      scores();
      load_keys(t + kStep);
      __builtin_amdgcn_sched_barrier(0);
      weigh(t, now);
      load_values();
      __builtin_amdgcn_sched_barrier(0);
    }
    scores();
    weigh(t, lim);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (bad && lane == 0) atomicOr(kv.err, kErrKvRange);

  // the wavefronts' parts on one maximum, then added: 2, 3 to 0, 1, then 1 to 0
  if (g == 0) {
    mbuf[wave][r] = m;
    lbuf[wave][r] = l;
  }
  __syncthreads();
  float top = mbuf[0][r], L = 0.f;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, mbuf[w][r]);
  const float M = base_of(top);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) L += lbuf[w][r] * exp2_of(mbuf[w][r] - M);
  const float mine = exp2_of(m - M);
#pragma unroll
  for (int i = 0; i < NC * VEC; ++i) acc[i] *= mine;
  // element e of load c and result i is d = (16 c + 4 g + i) VEC + e
  auto put = [&](float *o) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
          *(f32x4 *)(o + r * LD + (16 * c + 4 * g + i) * VEC + e) =
              f32x4{acc[c * VEC + e][i], acc[c * VEC + e + 1][i], acc[c * VEC + e + 2][i],
                    acc[c * VEC + e + 3][i]};
  };
  auto add = [&](const float *o) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          const f32x4 x = *(const f32x4 *)(o + r * LD + (16 * c + 4 * g + i) * VEC + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[c * VEC + e + k][i] += x[k];
        }
  };
  if (wave >= 2) put(obuf[wave - 2]);
  __syncthreads();
  if (wave < 2) add(obuf[wave]);
  __syncthreads();
  if (wave == 1) put(obuf[0]);
  __syncthreads();
  if (wave != 0) return;
  add(obuf[0]);
  if (r >= heads) return;
  if (R.used == 1) {
    const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = acc[c * VEC + e][i] * inv;
        store_out(a, kv.dtype, row * a.out_row + hq * a.out_head + (16 * c + 4 * g + i) * VEC, x,
                  VEC);
      }
    return;
  }
  const int64_t slot = ((int64_t)row * a.hq + hq) * a.splits + split;
  float *part = a.part + slot * D;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VEC; e += 4)
        *(f32x4 *)(part + (16 * c + 4 * g + i) * VEC + e) =
            f32x4{acc[c * VEC + e][i], acc[c * VEC + e + 1][i], acc[c * VEC + e + 2][i],
                  acc[c * VEC + e + 3][i]};
  if (g == 0) {
    float *ml = a.part + (int64_t)a.rows * a.hq * a.splits * D + slot * 2;
    ml[0] = top;                // -infinity where nothing weighs: no bound on the others'
    ml[1] = L;
  }
}

// The splits of a row and head joined: out = sum_s 2^(m_s - M) o_s / sum_s
// 2^(m_s - M) l_s.  A workgroup per row and head, D / 4 threads per split; what
// it waits for is a chain of small loads, so the first two splits of a thread
// are on their way before it knows how many there are.  One row of 16 heads of
// 256 and 4 splits 1.9-2.7 us, two rows of 64 splits 5.5.
constexpr int kJoin = 256;
template <int D>
__global__ __launch_bounds__(kJoin) void attend_join_kernel(KvCache kv, Attend a) {
  constexpr int LANES = D / 4, GROUPS = kJoin / LANES, EARLY = 2;
  __shared__ f32x4 obuf[GROUPS][LANES];
  __shared__ float mbuf[GROUPS], lbuf[GROUPS];
  const int row = blockIdx.x, h = blockIdx.y;
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int64_t slot = ((int64_t)row * a.hq + h) * a.splits;
  const float *part = a.part + slot * D + lane * 4;
  const float *ml = a.part + (int64_t)a.rows * a.hq * a.splits * D + slot * 2;
  f32x4 ahead[EARLY];
  float am[EARLY], al[EARLY];
#pragma unroll
  for (int e = 0; e < EARLY; ++e) {
    const int s = min(grp + e * GROUPS, a.splits - 1);
    ahead[e] = *(const f32x4 *)(part + (int64_t)s * D);
    am[e] = ml[2 * s];
    al[e] = ml[2 * s + 1];
  }
  const int used = range_of(kv, a, row, 0).used;
  if (used <= 1) return;
  // this group's splits on one maximum
  float m = -INFINITY, l = 0.f;
  f32x4 o{0, 0, 0, 0};
  auto add = [&](float sm, float sl, f32x4 so) {
    const float top = fmaxf(m, sm), base = base_of(top);
    const float x = exp2_of(m - base), y = exp2_of(sm - base);
    m = top;
    l = l * x + sl * y;
    o = o * x + so * y;
  };
#pragma unroll
  for (int e = 0; e < EARLY; ++e)
    if (grp + e * GROUPS < used) add(am[e], al[e], ahead[e]);
#pragma unroll 4
  for (int s = grp + EARLY * GROUPS; s < used; s += GROUPS)
    add(ml[2 * s], ml[2 * s + 1], *(const f32x4 *)(part + (int64_t)s * D));
  obuf[grp][lane] = o;
  if (lane == 0) {
    mbuf[grp] = m;
    lbuf[grp] = l;
  }
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int k = 1; k < GROUPS; ++k) add(mbuf[k], lbuf[k], obuf[k][lane]);
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  const float x[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  store_out(a, kv.dtype, row * a.out_row + h * a.out_head + lane * 4, x, 4);
}

template <int D, typename T>
void launch_typed(const KvCache &kv, const Attend &a, uint32_t grid, hipStream_t s) {
  if (a.dtype == DT_I16) attend_kernel<D, T, true><<<grid, 64 * kWaves, 0, s>>>(kv, a);
  else attend_kernel<D, T, false><<<grid, 64 * kWaves, 0, s>>>(kv, a);
}

template <int D>
void launch_dim(const KvCache &kv, const Attend &a, uint32_t grid, hipStream_t s) {
  if (kv.dtype == DT_F32) launch_typed<D, float>(kv, a, grid, s);
  else if (kv.dtype == DT_BF16) launch_typed<D, __bf16>(kv, a, grid, s);
  else launch_typed<D, _Float16>(kv, a, grid, s);
  if (a.splits > 1) attend_join_kernel<D><<<dim3(a.rows, a.hq), kJoin, 0, s>>>(kv, a);
}

}  // namespace

// Splits of a row: workgroups for the chip twice over at least, and no more than
// 512 tokens of the most that a table holds in one (the host knows no row's
// length; a longer split is what a ragged batch waits for), but no more than 16
// for that (each is a part to join), and none of less than a chunk.  Measured: 48
// ragged rows to 4099, 8 key-value heads of 128, in 9 splits 37.5 us, in 3 51; 8
// rows of 3450 in 8 25.8, in 16 29.5; 24 rows of 9216 in 16 151, in 3 168.
int attend_splits(const KvCache &kv, int64_t rows, int64_t hq, int num_cu) {
  const int64_t group = hq / kv.heads, base = rows * kv.heads * ((group + 15) / 16);
  const int64_t most = (((int64_t)kv.max_pages << kv.lg_page) + kAttendChunk - 1) / kAttendChunk;
  const int64_t fill = (2ll * num_cu + base - 1) / base;
  const int64_t even = most > 64 ? 16 : (most + 3) / 4;
  const int64_t want = fill > even ? fill : even;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

int64_t attend_workspace(const KvCache &kv, int64_t rows, int64_t hq, int num_cu) {
  const int64_t splits = attend_splits(kv, rows, hq, num_cu);
  return splits > 1 ? rows * hq * splits * (kv.dim + 2) * 4 : 0;
}

hipError_t launch_attend(const KvCache &kv, const Attend &a, hipStream_t s) {
  const int group = a.hq / kv.heads, tiles = (group + 15) / 16;
  const uint32_t grid = (uint32_t)(kv.heads * tiles) * a.rows * a.splits;
  if (kv.dim == 64) launch_dim<64>(kv, a, grid, s);
  else if (kv.dim == 128) launch_dim<128>(kv, a, grid, s);
  else launch_dim<256>(kv, a, grid, s);
  return hipGetLastError();
}

}  // namespace w4a8
