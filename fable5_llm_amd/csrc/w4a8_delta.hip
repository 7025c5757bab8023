// The gated delta rule.  Per value head, with a state S [dk][dv]:
//
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q
//
// (q and k divided by their norms first where asked).  Both dot products of a
// token are taken of the old state in one pass over it: S^T q after the update
// is e^g S^T q + (k . q) u.
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

// The tokens of a row and the slot of its state (-1: none, its tokens' out is
// zeros).  A slot that an earlier row names too, or outside the states, and
// bounds that do not lie in order within the tokens, are reported.
struct Row {
  int t0, t1, slot;
};
__device__ __forceinline__ Row row_of(const Delta &p, int row, int *flag) {
  Row r;
  int bad = 0, taken = 0;
  r.t0 = p.cu ? p.cu[row] : row;
  r.t1 = p.cu ? p.cu[row + 1] : row + 1;
  if (r.t0 < 0 || r.t1 < r.t0 || r.t1 > p.tokens) {
    bad = 1;
    r.t0 = r.t1 = 0;
  }
  r.slot = p.slots ? p.slots[row] : row;
  if (p.slots && r.slot >= 0)
    for (int j = threadIdx.x; j < row; j += blockDim.x) taken |= p.slots[j] == r.slot;
  taken = __syncthreads_or(taken) || r.slot >= p.nslots;
  if (taken) r.slot = -1;
  *flag = bad | taken;
  return r;
}

// A wavefront holds 16 columns of a head's state in registers: lane (rg, cq) =
// (lane >> 2, lane & 3) rows NR rg .. and columns 4 cq .., and takes the
// row's tokens one after another.
template <int DK, typename T>
__global__ __launch_bounds__(256) void delta_serial_kernel(Delta p) {
  constexpr int NR = DK / 16;
  const int row = blockIdx.x, h = blockIdx.y;
  int flag;
  const Row R = row_of(p, row, &flag);
  if (flag && threadIdx.x == 0 && h == 0 && blockIdx.z == 0) atomicOr(p.err, kErrDelta);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rg = lane >> 2, col = (blockIdx.z * 4 + wave) * 16 + (lane & 3) * 4;
  if (col >= p.dv) return;
  T *out = (T *)p.out + h * p.out_head + col;
  if (R.slot < 0) {
    if (rg == 0)
      for (int t = R.t0; t < R.t1; ++t)
        for (int c = 0; c < 4; ++c) out[t * p.out_token + c] = (T)0;
    return;
  }
  if (R.t0 == R.t1) {
    if (!p.fresh) return;
  }
  float *S = p.state + (((int64_t)R.slot * p.hv + h) * p.dk + rg * NR) * p.dv + col;
  f32x4 s[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i)
    s[i] = p.fresh ? f32x4{0, 0, 0, 0} : *(const f32x4 *)(S + (int64_t)i * p.dv);
  const int hk = h / (p.hv / p.hk);
  const T *q = (const T *)p.q + hk * p.q_head + rg * NR;
  const T *k = (const T *)p.k + hk * p.k_head + rg * NR;
  const T *v = (const T *)p.v + h * p.v_head + col;
  for (int t = R.t0; t < R.t1; ++t) {
    float qv[NR], kv[NR];
    float qq = 0.f, kk = 0.f, kq = 0.f;
    f32x4 pk{0, 0, 0, 0}, pq{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      qv[i] = to_float(q[t * p.q_token + i], p.unit);
      kv[i] = to_float(k[t * p.k_token + i], p.unit);
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
    const float e = expf(p.g[t * p.g_token + h]), beta = p.beta[t * p.beta_token + h];
    f32x4 u, o;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = beta * (to_float(v[t * p.v_token + c], p.unit) - e * rk * pk[c]);
      o[c] = rq * (e * pq[c] + rk * kq * u[c]);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) s[i] = s[i] * e + u * (kv[i] * rk);
    if (rg == 0)
#pragma unroll
      for (int c = 0; c < 4; ++c) out[t * p.out_token + c] = from_float<T>(o[c], p.out_unit);
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) *(f32x4 *)(S + (int64_t)i * p.dv) = s[i];
}

template <int DK>
void launch_serial(const Delta &d, hipStream_t s) {
  const dim3 grid(d.rows, d.hv, (d.dv + 63) / 64);
  if (d.dtype == DT_F32) delta_serial_kernel<DK, float><<<grid, 256, 0, s>>>(d);
  else if (d.dtype == DT_BF16) delta_serial_kernel<DK, __bf16><<<grid, 256, 0, s>>>(d);
  else if (d.dtype == DT_F16) delta_serial_kernel<DK, _Float16><<<grid, 256, 0, s>>>(d);
  else delta_serial_kernel<DK, int16_t><<<grid, 256, 0, s>>>(d);
}

}  // namespace

int64_t delta_workspace(int64_t, int64_t, int64_t) { return 0; }

hipError_t launch_delta(const Delta &d, hipStream_t s) {
  if (d.dk == 64) launch_serial<64>(d, s);
  else launch_serial<128>(d, s);
  return hipGetLastError();
}

}  // namespace w4a8
