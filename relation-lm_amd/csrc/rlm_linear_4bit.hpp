// What the kernels of the products with 4-bit weights share: the call's parameters, codes and
// scales as they are read.
#pragma once

#include "rlm_attention_mfma.hpp"
#include "rlm_common.hpp"
#include "rlm_fastdiv.hpp"

namespace rlm {
namespace linear4 {

using attention::product;
using attention::s16x8;

constexpr int kDeep = 128;  // inputs of a tile of codes

enum Activation { kNone = -1, kSilu = 0, kGelu = 1 };

struct LinearParams {
  const void* x;
  int64_t x_s;                  // row stride
  const uint4* codes[2];        // [NT][KT][64]
  const void* scales[2];        // [G][N]
  const void* zeros[2];         // or null
  const void* bias;             // or null
  int bias_dtype;
  void* out;
  int M, N, K, KT, NT;
  int group;
  FastDiv by_group_tiles;       // group / 128 where that is above 1
  int activation;
  bool wide_x, wide_s;          // whole accesses of inputs; of four scales
};

template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
template <typename T>
using matrix_t = typename std::conditional<sizeof(T) == 4, bf16, T>::type;
// What the matrix unit sees of code c: kBase<T> + c.
template <typename T>
constexpr float kBase = sizeof(T) == 4 ? -8.0f : 16.0f;

// Eight codes as an operand.  Codes 2 i and 2 i + 1 are at bits 4 i and 16 + 4 i.
template <typename T>
__device__ __forceinline__ s16x8 decode(uint32_t w) {
  uint32_t o[4];
  // (The base in a vector register: an and-or takes one constant.)
  uint32_t one;
  if constexpr (__is_same(T, f16)) {
    constexpr uint32_t kMask = 0x03c003c0u;  // fp16 of 16: mantissa bits 9..6
    asm("v_mov_b32 %0, 0x4c004c00" : "=v"(one));
    o[0] = ((w << 6) & kMask) | one;
    o[1] = ((w << 2) & kMask) | one;
    o[2] = ((w >> 2) & kMask) | one;
    o[3] = ((w >> 6) & kMask) | one;
  } else {
    constexpr uint32_t kMask = 0x00780078u;  // bf16 of 16: mantissa bits 6..3
    asm("v_mov_b32 %0, 0x41804180" : "=v"(one));
    o[0] = ((w << 3) & kMask) | one;
    o[1] = ((w >> 1) & kMask) | one;
    o[2] = ((w >> 5) & kMask) | one;
    o[3] = ((w >> 9) & kMask) | one;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = __float_as_uint(bf16_lo(o[i]) - 24.0f);
        const uint32_t hi = __float_as_uint(bf16_hi(o[i]) - 24.0f);
        o[i] = (lo >> 16) | hi;  // whole numbers: the low halves are zeros
      }
    }
  }
  return __builtin_bit_cast(s16x8, make_uint4(o[0], o[1], o[2], o[3]));
}

// Eight codes as c - 8 in bf16, in the order 0 4 1 5 2 6 3 7.  e4m3 below 2^-5 is n 2^-9 for its low four bits
// n: a code's byte 0x80 + (8 - c) or c - 8 is the difference in sign and magnitude, which one conversion a
// pair makes bf16.  17 instructions; through fp32, as above, 28.
__device__ __forceinline__ s16x8 decode_less_8(uint32_t w) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  bf16x2 o[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t c = (h == 0 ? w : w >> 4) & 0x0f0f0f0fu;
    const uint32_t low = 0x88888888u - c;  // of c <= 8, which its bytes' signs say
    const uint32_t is_low = __builtin_amdgcn_perm(low << 8, low, 0x090b080au);
    const uint32_t code = (low & is_low) | (c & 0x07070707u & ~is_low);
    o[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code, 512.0f, false);
    o[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code, 512.0f, true);
  }
  return __builtin_bit_cast(s16x8, o);
}

// Ones as an operand.
template <typename T>
__device__ __forceinline__ s16x8 ones() {
  constexpr uint32_t kOnes = __is_same(T, f16) ? 0x3c003c00u : 0x3f803f80u;
  return __builtin_bit_cast(s16x8, make_uint4(kOnes, kOnes, kOnes, kOnes));
}

// Raw values of four neighbouring scales or zero points (WIDE: one access), and one of them.
template <typename S, bool WIDE>
struct Four {
  typedef typename std::conditional<sizeof(S) == 4, uint32_t, uint16_t>::type one_t;
  struct Each {
    one_t e[4];
  };
  typename std::conditional<sizeof(S) == 4, uint4, uint2>::type v;
  // lane_off: this lane's byte offsets in a row, row_off: the row's.
  __device__ __forceinline__ void load(rsrc_t r, const uint32_t (&lane_off)[WIDE ? 1 : 4],
                                       uint32_t row_off) {
    if constexpr (WIDE && sizeof(S) == 4) {
      v = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, lane_off[0], row_off, 0));
    } else if constexpr (WIDE) {
      v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, lane_off[0], row_off, 0));
    } else {
      Each x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(S) == 4)
          x.e[i] = __builtin_amdgcn_raw_buffer_load_b32(r, lane_off[i], row_off, 0);
        else
          x.e[i] = __builtin_amdgcn_raw_buffer_load_b16(r, lane_off[i], row_off, 0);
      }
      v = __builtin_bit_cast(decltype(v), x);
    }
  }
  __device__ __forceinline__ float at(int i) const {
    return to_f32(__builtin_bit_cast(S, __builtin_bit_cast(Each, v).e[i]));
  }
};

__device__ __forceinline__ uint32_t word_of(const uint4& w, int i) {
  return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
}

__device__ __forceinline__ float activated(int activation, float x) {
  return activation == kSilu ? x / (1.0f + expf(-x)) : gelu_erf(x);
}

// Outputs n .. n + 3 of a token from the sums of its one or two (G) products.
template <typename T, int G>
__device__ __forceinline__ void finish(const LinearParams& p, int token, int n,
                                       const f32x4 (&v)[G]) {
  if (token >= p.M || n >= p.N) return;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = v[0][e];
    if constexpr (G == 2) y[e] = activated(p.activation, y[e]) * v[G - 1][e];
    if (p.bias != nullptr) y[e] += load_any_f(p.bias, p.bias_dtype, min(n + e, p.N - 1));
  }
  T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(token) * p.N + n;
  if (p.N % 4 == 0) {
    put4<T>(dst, y[0], y[1], y[2], y[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) dst[e] = from_f32<T>(y[e]);
  }
}

// Many tokens: tiles of tokens in LDS shared by the weight rows of a workgroup
// (rlm_linear_4bit_tile.hpp), which has 256 rows and 128 tokens, 128 and 64 in two parts of the inputs,
// or 64 and 64 in four parts (16-bit inputs).
enum TileShape { kWide, kMiddle, kSmall };
hipError_t tile_launch_bf16(const LinearParams& p, TileShape shape, int products, int scale_dtype,
                            hipStream_t stream);
hipError_t tile_launch_f16(const LinearParams& p, TileShape shape, int products, int scale_dtype,
                           hipStream_t stream);
hipError_t tile_launch_f32(const LinearParams& p, TileShape shape, int products, int scale_dtype,
                           hipStream_t stream);

}  // namespace linear4
}  // namespace rlm
