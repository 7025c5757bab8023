// Heads normalised and rotated to their tokens' positions, and the same with
// keys and values written into a paged cache.
//
//   y = x / sqrt(mean x^2 + eps) w        (where weights are given)
//   (a, b) -> amplitude (a cos t - b sin t, b cos t + a sin t),  t = pos freq_i
//
// for the pairs i of the first `rot` elements: (i, i + rot / 2), or (2 i, 2 i + 1).
#include "w4a8_mixers.h"

namespace w4a8 {

namespace {

constexpr int kThreads = 256;

template <typename T>
struct Unit {
  static __device__ __forceinline__ float in(T x, float) { return (float)x; }
  static __device__ __forceinline__ T out(float x, float) { return (T)x; }
};
template <>
struct Unit<int16_t> {
  static __device__ __forceinline__ float in(int16_t x, float unit) { return x * unit; }
  static __device__ __forceinline__ int16_t out(float x, float per) {
    return (int16_t)fminf(fmaxf(rintf(x * per), -32768.f), 32767.f);
  }
};

// eight elements as they lie in memory, and as numbers
template <typename T>
struct Raw {
  u32x4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw<T> load8(const void *p, int64_t at) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    r.w[i] = load16_nt((const u32x4 *)((const T *)p + at) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void numbers(float *x, const Raw<T> &r, float unit) {
  struct Eight { T v[8]; };
  const Eight e = __builtin_bit_cast(Eight, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Unit<T>::in(e.v[i], unit);
}
template <typename T>
__device__ __forceinline__ void store8(void *p, int64_t at, const float *x, float per) {
  alignas(16) T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Unit<T>::out(x[i], per);
#pragma unroll
  for (int i = 0; i < (int)sizeof(v) / 16; ++i)
    ((u32x4 *)((T *)p + at))[i] = ((const u32x4 *)v)[i];
}

// cos and sin of a turn's `t` (in turns): its nearest quarter is taken off in 64
// bits, so that far positions keep 32 bits of their angle, and what is left, at
// most pi / 4, goes through the first terms of either series (what is left out is
// below 2^-29 of the result)
__device__ __forceinline__ void turned(double t, float &c, float &s) {
  const double quarter = rint(4.0 * t);
  const float x = (float)(t - 0.25 * quarter) * 6.2831853071795865f, y = x * x;
  const float sn =
      x + x * y *
              (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880 - y / 39916800))));
  const float cs =
      1.f +
      y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320 - y / 3628800))));
  const int q = (int)(quarter - 4.0 * floor(0.25 * quarter));
  const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
  c = q == 1 || q == 2 ? -a : a;
  s = q >= 2 ? -b : b;
}

// Lanes: a head has a power of two of them, 16 elements each: eight pairs, or 16
// elements that are not rotated, which come from and go to one lane, so that out
// may be in.  U heads of a token at a time share its angles.  Many tokens are bound
// by HBM (8,191 tokens of 16 + 4 + 4 heads of 256 into the cache 50 us, 4.1 TB/s read
// and written), few by one chain of loads and angles (777 tokens 7.1 us under the
// profiler, one token 4.4, as an empty kernel).
template <typename IN, typename OUT, int U>
__global__ __launch_bounds__(kThreads) void rotary_kernel(KvCache kv, Rotary a) {
  const int lanes = a.lanes, lane = threadIdx.x & (lanes - 1);
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
  const int all = a.hq + a.hk * (a.slots ? 2 : 1), groups = (all + U - 1) / U;
  const int64_t token = item / groups;
  if (token >= a.tokens) return;
  const int h0 = (int)(item - token * groups) * U, heads = min(U, all - h0);
  const bool here = lane * 16 < a.dim, rotated = lane * 16 < a.rot;
  const bool split = rotated && !a.pairs;
  const int at0 = split ? 8 * lane : 16 * lane, at1 = split ? a.rot / 2 + 8 * lane : at0 + 8;
  Raw<IN> raw[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u;
    if (u < heads && here) {
      const bool q = h < a.hq, k = h < a.hq + a.hk;
      const void *src = q ? a.q : k ? a.k : a.v;
      const int64_t at =
          q ? token * a.q_token + h * a.q_head
            : k ? token * a.k_token + (h - a.hq) * a.k_head
                : token * a.v_token + (h - a.hq - a.hk) * a.v_head;
      raw[u][0] = load8<IN>(src, at + at0);
      raw[u][1] = load8<IN>(src, at + at1);
    } else {
      raw[u][0] = raw[u][1] = Raw<IN>{};
    }
  }
  const int pos = a.pos[token];
  int64_t slot = 0;
  if (a.slots) {
    const bool stopped = kv_stopped(kv);
    slot = a.slots[token];
    if (pos >= 0 && slot >= (int64_t)kv.pages << kv.lg_page) {
      if (lane == 0) atomicOr(kv.err, kErrKvRange);
      slot = -1;
    }
    if (stopped) slot = -1;
  }
  if (pos < 0 || slot < 0) return;            // every lane of the head
  float c[8], s[8];
  if (rotated && h0 < a.hq + a.hk) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      turned((double)pos * (a.freq[8 * lane + i] * 0.15915494309189535), c[i], s[i]);
      c[i] *= a.amplitude;
      s[i] *= a.amplitude;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u;
    if (u >= heads) break;
    const bool q = h < a.hq, k = h < a.hq + a.hk;
    float x[16];
    numbers(x, raw[u][0], a.unit);
    numbers(x + 8, raw[u][1], a.unit);
    const float *w = q ? a.q_norm : k ? a.k_norm : nullptr;
    if (w) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += x[i] * x[i];
      for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor(sum, d);
      const float inv = 1.f / sqrtf(sum * a.per_dim + a.eps);
      if (here) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= inv * w[at0 + i];
          x[8 + i] *= inv * w[at1 + i];
        }
      }
    }
    if (!here) continue;
    if (k && rotated) {
      auto turn = [&](int i, int ia, int ib) {
        const float p = x[ia], r = x[ib];
        x[ia] = p * c[i] - r * s[i];
        x[ib] = r * c[i] + p * s[i];
      };
      if (a.pairs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(i, 2 * i, 2 * i + 1);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(i, i, 8 + i);
      }
    }
    if (q || !a.slots) {
      void *dst = q ? a.q_out : a.k_out;
      const int64_t at = q ? token * a.q_out_token + h * a.q_out_head
                           : token * a.k_out_token + (h - a.hq) * a.k_out_head;
      store8<OUT>(dst, at + at0, x, a.out_per);
      store8<OUT>(dst, at + at1, x + 8, a.out_per);
    } else {
      const int which = k ? 0 : 1, kh = h - a.hq - (k ? 0 : a.hk);
      uint8_t *base = kv.pool + (slot >> kv.lg_page) * kv.page_bytes;
      const int64_t at =
          ((((int64_t)a.layer * 2 + which) * kv.heads + kh) * kv.page() + (slot & (kv.page() - 1))) *
          kv.dim;
      store8<OUT>(base, at + at0, x, 1.f);
      store8<OUT>(base, at + at1, x + 8, 1.f);
    }
  }
}

template <typename IN, typename OUT>
void launch_typed(const KvCache &kv, const Rotary &a, int num_cu, hipStream_t s) {
  const int all = a.hq + a.hk * (a.slots ? 2 : 1), each = kThreads / a.lanes;
  // Angles cost as much as heads do: by sixes 8,191 tokens into the cache take 51 us,
  // by ones 68.  Below eight workgroups a compute unit of lane groups of one head,
  // those end sooner: 777 tokens of 15 float32 heads 10.8 us, by sixes 12.2.
  const int64_t items = (int64_t)a.tokens * all, few = (int64_t)num_cu * 8 * each;
  auto blocks = [&](int u) {
    return (uint32_t)(((int64_t)a.tokens * ((all + u - 1) / u) + each - 1) / each);
  };
  if (items > few) rotary_kernel<IN, OUT, 6><<<blocks(6), kThreads, 0, s>>>(kv, a);
  else rotary_kernel<IN, OUT, 1><<<blocks(1), kThreads, 0, s>>>(kv, a);
}

}  // namespace

hipError_t launch_rotary(const KvCache &kv, const Rotary &a, int num_cu, hipStream_t s) {
  if (a.in_dtype == DT_F32) launch_typed<float, float>(kv, a, num_cu, s);
  else if (a.in_dtype == DT_BF16) launch_typed<__bf16, __bf16>(kv, a, num_cu, s);
  else if (a.in_dtype == DT_F16) launch_typed<_Float16, _Float16>(kv, a, num_cu, s);
  else if (a.out_dtype == DT_F32) launch_typed<int16_t, float>(kv, a, num_cu, s);
  else if (a.out_dtype == DT_BF16) launch_typed<int16_t, __bf16>(kv, a, num_cu, s);
  else if (a.out_dtype == DT_F16) launch_typed<int16_t, _Float16>(kv, a, num_cu, s);
  else launch_typed<int16_t, int16_t>(kv, a, num_cu, s);
  return hipGetLastError();
}

}  // namespace w4a8
