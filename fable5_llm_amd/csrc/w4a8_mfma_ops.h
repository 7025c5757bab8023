// The matrix instructions on 32 x 32 and 16 x 16 tiles and what feeds them,
// for the attention of several tokens (w4a8_chunk.hip).
#pragma once
#include "w4a8_mixers.h"

namespace w4a8 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 32 x 32 x 16: lane (r, g) = (lane & 31, lane >> 5) holds elements 8 g .. of
// row (column) r of either operand; result i of it is row 8 (i >> 2) + 4 g +
// (i & 3) of column r
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// 16 x 16 x 4: lane (r, g) = (lane & 15, lane >> 4) holds element g of row
// (column) r; result i of it is row 4 g + i of column r
__device__ __forceinline__ f32x4 mfma16(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// 16 lanes' 8 bytes, taken as 4 rows (lane >> 2) of 4 pieces (lane & 3) of 4
// elements, come back as columns: lane m gets element m & 3 of piece m >> 2 of
// each row
__device__ __forceinline__ u32x2 lds_columns(const void *p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_x4 *)p));
}

// 16 bytes a lane from memory (a uniform address and a lane's offset) into LDS
// at a uniform address and 16 bytes a lane from there (M0: one wait state between its
// write and the copy, which nothing else puts there).  The compiler does not
// count them: a wait for them comes before the barrier that their readers wait at.
__device__ __forceinline__ void copy16(const void *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}

}  // namespace w4a8
