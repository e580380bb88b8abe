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

// ---- Caches of 8 bits: e4m3 codes, exact in bf16, met by operands that are sums of bf16 parts.

struct code8 {
  uint8_t bits;
};
__device__ __forceinline__ float code_to_f32(code8 c) {
  return __builtin_amdgcn_cvt_f32_fp8(c.bits, 0);
}

// A row's scale, NaN where it is not finite: an infinite one would give a score of -inf or +inf by the sign of
// the codes' product, and so drop its row or not.
__device__ __forceinline__ float scale_or_nan(float s) {
  return __builtin_fabsf(s) < INFINITY ? s : __builtin_nanf("");
}

// Parts of a query, and of the weights that meet the values.
template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : __is_same(T, f16) ? 2 : 1;
template <typename T>
constexpr int kWeightParts = sizeof(T) == 4 ? 3 : 2;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2* lds_i32x2;
typedef const __attribute__((address_space(3))) f32x4* lds_f32x4;

// 16-byte pieces of an LDS row of at most 16 PIECES codes, and where a row's pieces stand: 32 rows
// of one piece column, as a transposing read takes them, spread over all banks.
constexpr int code_pitch(int pieces) {
  return pieces <= 2 ? 2 : pieces <= 4 ? 4 : pieces <= 8 ? 8 : 16;
}
template <int PITCH>
__device__ __forceinline__ int code_swizzle(int row) {
  return PITCH == 2 ? (row >> 3) & 1 : swizzle<PITCH>(row);
}

// Eight codes as bf16.
__device__ __forceinline__ s16x8 decode8(uint32_t lo, uint32_t hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true)};
  return __builtin_bit_cast(s16x8, x);
}

// Eight elements of a query as bf16 parts.
template <typename T>
__device__ __forceinline__ void load_parts(const T* src, bool there, s16x8 (&part)[kParts<T>]) {
  if constexpr (__is_same(T, bf16)) {
    uint4 x = *reinterpret_cast<const uint4*>(src);
    if (!there) x = make_uint4(0, 0, 0, 0);
    part[0] = __builtin_bit_cast(s16x8, x);
  } else {
    float x[8];
    const float4 lo = load4(src), hi = load4(src + 4);
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
    x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = there ? x[e] : 0.0f;
    split<kParts<T>>(x, part);
  }
}

// The first of the eight features of a row of codes that lane group `quad` has for product j (an order
// that gives a lane 16 neighbouring codes where it can).
template <int DC>
__device__ __forceinline__ int code_feature(int j, int quad) {
  return j < DC / 2 * 2 ? 64 * (j / 2) + 16 * quad + 8 * (j & 1) : 32 * j + 8 * quad;
}
// The key of 32 whose codes lane (r, quad) reads for a transposing read: the keys of a lane group's
// weights, 4 quad .. + 3 and 16 + 4 quad .. + 3.
__device__ __forceinline__ int code_row(int r, int quad) {
  return 4 * quad + ((r >> 1) & 3) + 16 * (r >> 3);
}

}  // namespace attention
}  // namespace rlm
