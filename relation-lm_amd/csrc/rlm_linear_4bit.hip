// Products with weights of 4 bits: out[m][n] = sum_k x[m][k] (c[n][k] - z[g][n]) s[g][n], g = k / group,
// and the gated form act(x Wg^T) * (x Wu^T).
//
// A code c goes into the matrix unit as 16 + c, which is exact in bf16 and fp16 and takes one
// and-or for two codes: the code's bits are the mantissa bits below 2^4's exponent.  The group's
// sum is taken back to c - z with the sum of its inputs, which a product with ones gives in the
// same layout:
//   sum_k x_k (c_k - z) = sum_k x_k (16 + c_k) - (16 + z) sum_k x_k,
// so a group costs two multiply-adds per output, whatever its zero points.  fp32 inputs enter as
// three bf16 parts and codes as c - 8, whose sums cancel less.
//
// Weights are laid out in operand order: a lane's 16 bytes are its codes of four matrix
// instructions (16 rows of weights, 32 inputs each), a wave's load is 1 KiB in a row.  A
// workgroup has R tiles of 16 weight rows; its waves share out the inputs and add up in LDS, in
// the waves' order.
#include "rlm_common.hpp"
#include "rlm_attention_mfma.hpp"

namespace rlm {
namespace {

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
  void* out;                    // [M][N]
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
  if constexpr (__is_same(T, f16)) {
    constexpr uint32_t kMask = 0x03c003c0u, kOne = 0x4c004c00u;  // fp16 of 16: mantissa bits 9..6
    o[0] = ((w << 6) & kMask) | kOne;
    o[1] = ((w << 2) & kMask) | kOne;
    o[2] = ((w >> 2) & kMask) | kOne;
    o[3] = ((w >> 6) & kMask) | kOne;
  } else {
    constexpr uint32_t kMask = 0x00780078u, kOne = 0x41804180u;  // bf16 of 16: mantissa bits 6..3
    o[0] = ((w << 3) & kMask) | kOne;
    o[1] = ((w >> 1) & kMask) | kOne;
    o[2] = ((w >> 5) & kMask) | kOne;
    o[3] = ((w >> 9) & kMask) | kOne;
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

// Ones as an operand.
template <typename T>
__device__ __forceinline__ s16x8 ones() {
  constexpr uint32_t kOnes = __is_same(T, f16) ? 0x3c003c00u : 0x3f803f80u;
  return __builtin_bit_cast(s16x8, make_uint4(kOnes, kOnes, kOnes, kOnes));
}

// Inputs k .. k + 7 of a row as an operand (fp32: as three), 0 past the row's end.
template <typename T>
__device__ __forceinline__ void load_x(const LinearParams& p, const T* row, int k,
                                       s16x8 (&part)[kParts<T>]) {
  if constexpr (sizeof(T) == 2) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (p.wide_x) {
      x = *reinterpret_cast<const uint4*>(row + (k < p.K ? k : 0));
      if (k >= p.K) x = make_uint4(0, 0, 0, 0);
    } else {
      uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        e[i] = k + i < p.K ? reinterpret_cast<const uint16_t*>(row)[k + i] : uint16_t{0};
      struct Raw {
        uint16_t e[8];
      } raw;
#pragma unroll
      for (int i = 0; i < 8; ++i) raw.e[i] = e[i];
      x = __builtin_bit_cast(uint4, raw);
    }
    part[0] = __builtin_bit_cast(s16x8, x);
  } else {
    float x[8];
    if (p.wide_x) {
      const float4 lo = load4(row + (k < p.K ? k : 0)), hi = load4(row + (k < p.K ? k + 4 : 4));
      x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
      x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = k < p.K ? x[i] : 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = k + i < p.K ? row[k + i] : 0.0f;
    }
    attention::split<3>(x, part);
  }
}

// Four neighbouring values of a row of scales or zero points.
template <typename S>
__device__ __forceinline__ f32x4 load_s(const LinearParams& p, const S* row, int n) {
  if (p.wide_s) {
    const float4 v = load4(row + (n < p.N ? n : 0));
    return f32x4{v.x, v.y, v.z, v.w};
  }
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32(row[min(n + i, p.N - 1)]);
  return v;
}

__device__ __forceinline__ float activated(int activation, float x) {
  return activation == kSilu ? x / (1.0f + expf(-x)) : gelu_erf(x);
}

// MT token tiles of 16, R tiles of 16 weight rows, G matrices; CH matrix instructions to a group
// (four also where a group is several tiles of codes).
template <typename T, typename S, int MT, int R, int G, int CH>
__global__ __launch_bounds__(512) void linear_4bit_kernel(LinearParams p) {
  constexpr int NP = kParts<T>;
  extern __shared__ __align__(16) char lds[];  // [wave][G][MT][64] f32x4
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int W = blockDim.x / kWave;
  const int r = lane & 15, quad = lane >> 4;
  const int nt0 = blockIdx.x * R;
  const int m0 = blockIdx.y * 16 * MT;

  const T* rows[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)  // tokens past the last read its row; their outputs are not kept
    rows[t] = static_cast<const T*>(p.x) + static_cast<int64_t>(min(m0 + 16 * t + r, p.M - 1)) * p.x_s;

  f32x4 total[G][R][MT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) total[g][i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (int kt = wave; kt < p.KT; kt += W) {
    uint4 words[G][R];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < R; ++i)
        words[g][i] =
            p.codes[g][(static_cast<int64_t>(min(nt0 + i, p.NT - 1)) * p.KT + kt) * kWave + lane];
#pragma unroll
    for (int c = 0; c < 4 / CH; ++c) {
      f32x4 acc[G][R][MT], sum[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < R; ++i) acc[g][i][t] = sum[t];
      }
#pragma unroll
      for (int s = c * CH; s < (c + 1) * CH; ++s) {
        s16x8 x[MT][NP];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          load_x<T>(p, rows[t], kDeep * kt + 32 * s + 8 * quad, x[t]);
#pragma unroll
          for (int n = 0; n < NP; ++n) sum[t] = product(ones<T>(), x[t][n], sum[t], matrix_t<T>{});
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const uint32_t w = s == 0 ? words[g][i].x : s == 1 ? words[g][i].y
                               : s == 2 ? words[g][i].z : words[g][i].w;
            const s16x8 a = decode<T>(w);
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int n = 0; n < NP; ++n)
                acc[g][i][t] = product(a, x[t][n], acc[g][i][t], matrix_t<T>{});
          }
      }
      // The group's scale and zero point, from its first input on; tiles past the last group
      // (their inputs are zeros) take the last one's.
      const int first = kDeep * kt + 32 * c * CH;
      const int at = min(CH < 4 ? first / (32 * CH)
                                : static_cast<int>(p.by_group_tiles.div(static_cast<uint32_t>(kt))),
                         (p.K - 1) / p.group);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int n = 16 * min(nt0 + i, p.NT - 1) + 4 * quad;
          const int64_t line = static_cast<int64_t>(at) * p.N;
          const f32x4 scale = load_s<S>(p, static_cast<const S*>(p.scales[g]) + line, n);
          f32x4 off = f32x4{8.0f, 8.0f, 8.0f, 8.0f};
          if (p.zeros[g] != nullptr) off = load_s<S>(p, static_cast<const S*>(p.zeros[g]) + line, n);
          off += kBase<T>;
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              total[g][i][t][e] =
                  fmaf(scale[e], fmaf(-off[e], sum[t][e], acc[g][i][t][e]), total[g][i][t][e]);
        }
    }
  }

  f32x4* sums = reinterpret_cast<f32x4*>(lds);
  T* out = static_cast<T*>(p.out);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int t = 0; t < MT; ++t) sums[((wave * G + g) * MT + t) * kWave + lane] = total[g][i][t];
    __syncthreads();
    for (int t = wave; t < MT; t += W) {
      f32x4 v[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        v[g] = sums[(g * MT + t) * kWave + lane];
        for (int w = 1; w < W; ++w) v[g] += sums[((w * G + g) * MT + t) * kWave + lane];
      }
      const int token = m0 + 16 * t + r, n = 16 * (nt0 + i) + 4 * quad;
      if (token >= p.M || n >= p.N) continue;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = v[0][e];
        if constexpr (G == 2) y[e] = activated(p.activation, y[e]) * v[G - 1][e];
        if (p.bias != nullptr) y[e] += load_any_f(p.bias, p.bias_dtype, min(n + e, p.N - 1));
      }
      T* dst = out + static_cast<int64_t>(token) * p.N + n;
      if (p.N % 4 == 0) {
        put4<T>(dst, y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.N) dst[e] = from_f32<T>(y[e]);
      }
    }
  }
}

template <typename T, typename S, int MT, int R, int G, int CH>
hipError_t launch(const LinearParams& p, hipStream_t stream) {
  const char* name = G == 2 ? "gated_linear_4bit" : "linear_4bit";
  int waves = 1;
  while (waves < 8 && waves < p.KT) waves *= 2;
  const dim3 grid((p.NT + R - 1) / R, (p.M + 16 * MT - 1) / (16 * MT));
  RLM_REQUIRE(grid.y < 65536u, "%s: too many tokens for one call", name);
  RLM_TRY(check_launch(name, static_cast<int64_t>(grid.x) * grid.y, kWave * waves));
  const size_t lds = static_cast<size_t>(waves) * G * MT * kWave * 16;
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(&linear_4bit_kernel<T, S, MT, R, G, CH>),
        hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    RLM_REQUIRE(e == hipSuccess, "%s: %zu bytes of LDS refused: %s", name, lds,
                hipGetErrorString(e));
  }
  hipLaunchKernelGGL((linear_4bit_kernel<T, S, MT, R, G, CH>), grid, dim3(kWave * waves), lds,
                     stream, p);
  return launch_status(name);
}

template <typename T, typename S, int G, int CH>
hipError_t launch_tokens(const LinearParams& p, hipStream_t stream) {
  if (p.M <= 16) return launch<T, S, 1, 1, G, CH>(p, stream);
  if (p.M <= 32) return launch<T, S, 2, 1, G, CH>(p, stream);
  return launch<T, S, 4, 1, G, CH>(p, stream);
}

template <typename T, typename S, int G>
hipError_t launch_group(const LinearParams& p, hipStream_t stream) {
  if (p.group == 32) return launch_tokens<T, S, G, 1>(p, stream);
  if (p.group == 64) return launch_tokens<T, S, G, 2>(p, stream);
  return launch_tokens<T, S, G, 4>(p, stream);
}

template <int G>
hipError_t launch_types(const LinearParams& p, int dtype, int scale_dtype, hipStream_t stream) {
  if (dtype == RLM_F32) return launch_group<float, float, G>(p, stream);
  if (dtype == RLM_BF16)
    return scale_dtype == RLM_F32 ? launch_group<bf16, float, G>(p, stream)
                                  : launch_group<bf16, bf16, G>(p, stream);
  return scale_dtype == RLM_F32 ? launch_group<f16, float, G>(p, stream)
                                : launch_group<f16, f16, G>(p, stream);
}

struct Weight {
  const rlm_tensor *codes, *scales, *zeros;
  const char *codes_name, *scales_name, *zeros_name;
};

hipError_t linear(const rlm_tensor* input, const Weight (&weights)[2], int count,
                  int64_t group_size, const rlm_tensor* bias, int activation,
                  const rlm_tensor* out, hipStream_t stream) {
  RLM_TRY(check_rows(input, "input"));
  RLM_TRY(check_dtype_float(input, "input"));
  const int64_t M = input->shape[0], K = input->shape[1];
  RLM_REQUIRE(K >= 1 && K <= (int64_t(1) << 24), "input: width must be in [1, 2^24], got %lld",
              (long long)K);
  RLM_REQUIRE(M < (int64_t(1) << 22), "input: at most 2^22 - 1 rows, got %lld", (long long)M);
  RLM_REQUIRE(group_size == 32 || group_size == 64 ||
                  (group_size >= 128 && group_size % 128 == 0 && group_size <= (int64_t(1) << 24)),
              "group_size must be 32, 64 or a multiple of 128, got %lld", (long long)group_size);
  const int64_t groups = (K + group_size - 1) / group_size, KT = (K + kDeep - 1) / kDeep;
  LinearParams p{};
  RLM_REQUIRE(weights[0].scales != nullptr && weights[0].scales->ndim == 2,
              "%s: expected a [groups, N] tensor", weights[0].scales_name);
  const int64_t N = weights[0].scales->shape[1];
  RLM_REQUIRE(N >= 1 && N <= (int64_t(1) << 24), "%s: outputs must be in [1, 2^24], got %lld",
              weights[0].scales_name, (long long)N);
  const int64_t NT = (N + 15) / 16;
  const int64_t per_scale = 4 * dtype_size(weights[0].scales->dtype);
  p.wide_s = N % 4 == 0;
  for (int g = 0; g < count; ++g) {
    const Weight& w = weights[g];
    RLM_TRY(check_dense(w.codes, w.codes_name, 4));
    RLM_TRY(check_dtype_is(w.codes, w.codes_name, RLM_I32));
    const int64_t want[4] = {NT, KT, kWave, 4};
    for (int i = 0; i < 4; ++i) RLM_TRY(check_dim(w.codes, w.codes_name, i, want[i]));
    RLM_REQUIRE((reinterpret_cast<uintptr_t>(w.codes->data) & 15u) == 0,
                "%s must be 16-byte aligned", w.codes_name);
    p.codes[g] = static_cast<const uint4*>(w.codes->data);
    RLM_REQUIRE((w.zeros == nullptr) == (weights[0].zeros == nullptr),
                "%s and %s: both or neither", weights[0].zeros_name, w.zeros_name);
    const rlm_tensor* const vectors[2] = {w.scales, w.zeros};
    for (int i = 0; i < (w.zeros == nullptr ? 1 : 2); ++i) {
      const rlm_tensor* t = vectors[i];
      const char* name = i == 0 ? w.scales_name : w.zeros_name;
      RLM_TRY(check_dense(t, name, 2));
      RLM_TRY(check_dim(t, name, 0, groups));
      RLM_TRY(check_dim(t, name, 1, N));
      RLM_REQUIRE(t->dtype == RLM_F32 || t->dtype == input->dtype,
                  "%s: expected float32 or the input's %s, got %s", name, dtype_name(input->dtype),
                  dtype_name(t->dtype));
      RLM_TRY(check_same_dtype(t, name, weights[0].scales, weights[0].scales_name));
      p.wide_s = p.wide_s && reinterpret_cast<uintptr_t>(t->data) % per_scale == 0;
    }
    p.scales[g] = w.scales->data;
    p.zeros[g] = w.zeros == nullptr ? nullptr : w.zeros->data;
  }
  if (bias != nullptr) {
    RLM_TRY(check_dense(bias, "bias", 1));
    RLM_TRY(check_dtype_float(bias, "bias"));
    RLM_TRY(check_dim(bias, "bias", 0, N));
    p.bias = bias->data;
    p.bias_dtype = bias->dtype;
  }
  RLM_TRY(check_dense(out, "out", 2));
  RLM_TRY(check_same_dtype(out, "out", input, "input"));
  RLM_TRY(check_dim(out, "out", 0, M));
  RLM_TRY(check_dim(out, "out", 1, N));
  RLM_REQUIRE((reinterpret_cast<uintptr_t>(out->data) & 15u) == 0, "out must be 16-byte aligned");
  if (M == 0) return hipSuccess;
  const int64_t per_vec = 16 / dtype_size(input->dtype);
  p.x = input->data;
  p.x_s = input->stride[0];
  p.wide_x = K % 8 == 0 && (reinterpret_cast<uintptr_t>(input->data) & 15u) == 0 &&
             (M <= 1 || input->stride[0] % per_vec == 0);
  p.out = out->data;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.KT = static_cast<int>(KT);
  p.NT = static_cast<int>(NT);
  p.group = static_cast<int>(group_size);
  p.by_group_tiles = FastDiv(static_cast<uint32_t>(std::max<int64_t>(group_size / kDeep, 1)));
  p.activation = activation;
  return count == 2 ? launch_types<2>(p, input->dtype, weights[0].scales->dtype, stream)
                    : launch_types<1>(p, input->dtype, weights[0].scales->dtype, stream);
}

}  // namespace
}  // namespace rlm

using namespace rlm;

extern "C" hipError_t rlm_linear_4bit(const rlm_tensor* input, const rlm_tensor* codes,
                                      const rlm_tensor* scales, const rlm_tensor* zeros,
                                      int64_t group_size, const rlm_tensor* bias,
                                      const rlm_tensor* out, hipStream_t stream) {
  clear_error();
  const Weight weights[2] = {{codes, scales, zeros, "codes", "scales", "zeros"}, {}};
  return linear(input, weights, 1, group_size, bias, kNone, out, stream);
}

extern "C" hipError_t rlm_gated_linear_4bit(const rlm_tensor* input, const rlm_tensor* gate_codes,
                                            const rlm_tensor* gate_scales,
                                            const rlm_tensor* gate_zeros,
                                            const rlm_tensor* up_codes,
                                            const rlm_tensor* up_scales, const rlm_tensor* up_zeros,
                                            int64_t group_size, int32_t activation,
                                            const rlm_tensor* out, hipStream_t stream) {
  clear_error();
  RLM_REQUIRE(activation == kSilu || activation == kGelu,
              "activation must be 0 (x / (1 + exp(-x))) or 1 (GELU), got %d", activation);
  const Weight weights[2] = {
      {gate_codes, gate_scales, gate_zeros, "gate_codes", "gate_scales", "gate_zeros"},
      {up_codes, up_scales, up_zeros, "up_codes", "up_scales", "up_zeros"}};
  return linear(input, weights, 2, group_size, nullptr, activation, out, stream);
}
