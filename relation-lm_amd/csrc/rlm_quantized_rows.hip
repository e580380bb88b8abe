// Rows of an 8-bit cache read back in a float type: out[b, i, h] = cache[b, row, h] * scale[b, row, h],
// row = rows[b, i] or i.  The product is rounded to fp32 and then to the type: a code of 4 bits times a scale
// of 24 may pass fp32, and where that first rounding lands on a 16-bit tie (1 of 2^16) it may be the other neighbour.
//
// Bound: memory, 1 + 4 / D bytes read and the type's written for each feature: 4 x 16384 rows of 4 heads
// of 128 features in bf16 (102 MB, which the MALL holds) take 16.4 us, 6.2 TB/s; 8 x 640 named rows of 3
// of 64 take 4.1, a launch and two round trips.
#include "rlm_common.hpp"
#include "rlm_fastdiv.hpp"

namespace rlm {
namespace {

constexpr int kThreads = 256;
constexpr int kRounds = 4;  // accesses of a thread

struct RowsParams {
  const uint8_t* cache;
  const float* scale;
  int64_t c_sb, c_st, c_sh, s_sb, s_st, s_sh;
  const void* rows;       // [B,N], or null
  int rows_dtype;
  int64_t r_sb, r_sn;
  void* out;              // [B,N,Hk,D]
  int64_t T, N;
  int Hk, D;
  uint32_t pieces;        // of a batch row: N * Hk * D / V
  FastDiv by_groups, by_pieces, by_heads;
};

// Eight codes as fp32.
__device__ __forceinline__ void decode8(uint2 codes, float (&x)[8]) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int c = static_cast<int>(w == 0 ? codes.x : codes.y);
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
    const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
    x[4 * w] = lo[0], x[4 * w + 1] = lo[1], x[4 * w + 2] = hi[0], x[4 * w + 3] = hi[1];
  }
}

// V: features of one access, eight or (unaligned shapes) one.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void rows_kernel(RowsParams p) {
  uint32_t group;
  const int64_t b = p.by_groups.div(blockIdx.x, group);
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const uint32_t i = (group * kRounds + k) * kThreads + threadIdx.x;
    if (i >= p.pieces) return;
    uint32_t piece, h;
    const uint32_t n = p.by_heads.div(p.by_pieces.div(i, piece), h);
    const int64_t row = p.rows == nullptr
                            ? static_cast<int64_t>(n)
                            : load_any_i(p.rows, p.rows_dtype, b * p.r_sb + n * p.r_sn);
    const bool there = row >= 0 && row < p.T;
    float x[V], s = 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = 0.0f;
    if (there) {
      const uint8_t* src = p.cache + b * p.c_sb + row * p.c_st + h * p.c_sh + V * piece;
      s = p.scale[b * p.s_sb + row * p.s_st + h * p.s_sh];
      if constexpr (V == 8)
        decode8(*reinterpret_cast<const uint2*>(src), x);
      else
        x[0] = __builtin_amdgcn_cvt_f32_fp8(*src, 0);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] *= s;
    }
    T* dst = static_cast<T*>(p.out) + (b * p.pieces + i) * V;
    if constexpr (V == 8) {
      put4<T>(dst, x[0], x[1], x[2], x[3]);
      put4<T>(dst + 4, x[4], x[5], x[6], x[7]);
    } else {
      *dst = from_f32<T>(x[0]);
    }
  }
}

template <typename T>
hipError_t launch(RowsParams& p, int64_t B, bool wide, hipStream_t stream) {
  const int64_t per_group = kThreads * kRounds;
  const int64_t groups = (p.pieces + per_group - 1) / per_group;
  RLM_TRY(check_launch("quantized_rows", B * groups, kThreads));
  p.by_groups = FastDiv(static_cast<uint32_t>(groups));
  const dim3 grid(static_cast<unsigned>(B * groups));
  if (wide)
    hipLaunchKernelGGL((rows_kernel<T, 8>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((rows_kernel<T, 1>), grid, dim3(kThreads), 0, stream, p);
  return launch_status("quantized_rows");
}

}  // namespace
}  // namespace rlm

using namespace rlm;

extern "C" hipError_t rlm_quantized_rows(const rlm_tensor* cache, const rlm_tensor* scale,
                                         const rlm_tensor* rows, const rlm_tensor* out,
                                         hipStream_t stream) {
  clear_error();
  RLM_TRY(check_strided(cache, "cache", 4));
  RLM_TRY(check_dtype_is(cache, "cache", RLM_F8E4M3));
  const int64_t B = cache->shape[0], T = cache->shape[1], Hk = cache->shape[2],
                D = cache->shape[3];
  RLM_TRY(check_scales(scale, "scale", B, T, Hk));
  RLM_TRY(check_dense(out, "out", 4));
  RLM_TRY(check_dtype_float(out, "out"));
  RowsParams p{};
  p.N = T;
  if (rows != nullptr) {
    RLM_REQUIRE(is_index_dtype(rows->dtype), "rows: expected an int32/int64 tensor");
    RLM_TRY(check_strided(rows, "rows", 2));
    RLM_TRY(check_dim(rows, "rows", 0, B));
    p.N = rows->shape[1];
    p.rows = rows->data;
    p.rows_dtype = rows->dtype;
    p.r_sb = rows->stride[0], p.r_sn = rows->stride[1];
  }
  const int64_t want[4] = {B, p.N, Hk, D};
  for (int i = 0; i < 4; ++i) RLM_TRY(check_dim(out, "out", i, want[i]));
  if (B == 0 || p.N == 0 || Hk == 0 || D == 0) return hipSuccess;
  p.cache = static_cast<const uint8_t*>(cache->data);
  p.c_sb = cache->stride[0], p.c_st = cache->stride[1], p.c_sh = cache->stride[2];
  p.scale = static_cast<const float*>(scale->data);
  p.s_sb = scale->stride[0], p.s_st = scale->stride[1], p.s_sh = scale->stride[2];
  p.out = out->data;
  p.T = T;
  p.Hk = static_cast<int>(Hk);
  p.D = static_cast<int>(D);
  bool wide = D % 8 == 0 && (reinterpret_cast<uintptr_t>(out->data) & 15u) == 0 &&
              (reinterpret_cast<uintptr_t>(cache->data) & 7u) == 0;
  for (int i = 0; i < 3; ++i)
    wide = wide && (cache->shape[i] <= 1 || cache->stride[i] % 8 == 0);
  const int64_t pieces = p.N * Hk * D / (wide ? 8 : 1);
  RLM_REQUIRE(pieces < (int64_t(1) << 31) - kThreads * kRounds && Hk < (int64_t(1) << 31) &&
                  B < (int64_t(1) << 31) && D < (int64_t(1) << 31),
              "quantized_rows: too many features of a batch row for one call");
  p.pieces = static_cast<uint32_t>(pieces);
  p.by_pieces = FastDiv(static_cast<uint32_t>(D / (wide ? 8 : 1)));
  p.by_heads = FastDiv(static_cast<uint32_t>(Hk));
  switch (out->dtype) {
    case RLM_F32: return launch<float>(p, B, wide, stream);
    case RLM_BF16: return launch<bf16>(p, B, wide, stream);
    default: return launch<f16>(p, B, wide, stream);
  }
}
