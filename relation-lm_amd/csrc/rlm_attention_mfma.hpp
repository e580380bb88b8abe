// Matrix-core operands of the attention kernels: products, packing, and the LDS layout of tiles.
// (The products and the sums of bf16 parts also serve rlm_linear_4bit.hip.)
#pragma once

#include <type_traits>

#include "rlm_attention.hpp"

namespace rlm {
namespace attention {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef const __attribute__((address_space(3))) s16x8* lds_s16x8;
typedef const __attribute__((address_space(3))) float* lds_f32;

// 16-byte pieces of an LDS row of at most 32 DC features: a power of two, LEAST at least.
template <typename T, int DC, int LEAST = 8>
constexpr int pitch() {
  constexpr int pieces = DC * 32 * static_cast<int>(sizeof(T)) / 16;
  return pieces <= LEAST ? LEAST : pieces <= 8 ? 8 : pieces <= 16 ? 16 : pieces <= 32 ? 32 : 64;
}

// c + a b over 32 (16-bit types) or 16 (fp32: four steps of four) features or keys.
__device__ __forceinline__ f32x4 product(s16x8 a, s16x8 b, f32x4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 product(s16x8 a, s16x8 b, f32x4 c, f16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// fp32: lane group g of a step has feature 4 g + i of the lane's four.
__device__ __forceinline__ f32x4 product(float4 a, float4 b, f32x4 c, float) {
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
}
// Two weights in the 16-bit type.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bf16) { return pack_bf16x2(lo, hi); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi, f16) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
}

// x as a sum of N bf16 numbers each.
template <int N>
__device__ __forceinline__ void split(float (&x)[8], s16x8 (&part)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      if (n + 1 < N) {
        x[2 * i] -= bf16_lo(w[i]);
        x[2 * i + 1] -= bf16_hi(w[i]);
      }
    }
    part[n] = __builtin_bit_cast(s16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// 16-byte pieces of an LDS row: rows of 8 pieces alternate between the halves of the 16 piece
// columns that the banks form, so their swizzle goes by pairs of rows (of 4: by four rows).
template <int PITCH>
__device__ __forceinline__ int swizzle(int row) {
  return PITCH == 4 ? (row >> 2) & 3 : PITCH == 8 ? (row >> 1) & 7 : row & 15;
}

// Lane l reads four values of key l / 16 * 4 + l % 16 / 4 at `at` and gets four keys of value
// feature l % 16; eight keys, of the two 16-key groups `apart` bytes from each other.
__device__ __forceinline__ s16x8 read_values(uint32_t at, uint32_t apart) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)static_cast<uintptr_t>(at));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)static_cast<uintptr_t>(at + apart));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace attention
}  // namespace rlm
