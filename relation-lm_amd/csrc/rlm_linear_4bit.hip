// Products with weights of 4 bits: out[m][n] = sum_k x[m][k] (c[n][k] - z[g][n]) s[g][n], g = k / group,
// and the gated form act(x Wg^T) * (x Wu^T).
//
// A code c goes into the matrix unit as 16 + c, which is exact in bf16 and fp16 and takes one
// and-or for two codes: the code's bits are the mantissa bits below 2^4's exponent.  The group's
// sum is taken back to c - z with the sum of its inputs, which a product with ones gives in the
// same layout:
//   sum_k x_k (c_k - z) = sum_k x_k (16 + c_k) - (16 + z) sum_k x_k,
// so a group costs two multiply-adds per output, whatever its zero points.  fp32 inputs enter as
// three bf16 parts, and codes as c - 8: sums of 16 + c are 10 to 50 times as large as what is left of
// them, which outputs of 16 bits do not show and outputs of 32 do (with inputs of one sign, 1104 wide,
// 3e-6 of the outputs' size in place of 6e-8).
//
// Weights are laid out in operand order: a lane's 16 bytes are its codes of four matrix
// instructions (16 rows of weights, 32 inputs each), a wave's load is 1 KiB in a row.  A
// workgroup has R tiles of 16 weight rows; its waves share out the inputs and add up in LDS, in
// the waves' order.
//
// Bound: memory, once the launch is paid.  One token of 4096 -> 11008 gated (48 MB of codes, scales and zero
// points) takes 13.1 us, 8 of 8192 -> 8192 (36 MB) 12.0, where an empty call takes about 5; one of 2304 -> 576
// 5.5.  Scales are kept as they were loaded until they are used: converted where they are loaded, each
// load waited for the one before (14.3 in place of 12.0).
#include "rlm_linear_4bit.hpp"

namespace rlm {
namespace {

using namespace linear4;

// Bytes of inputs that a workgroup keeps in LDS: as the faster way, and instead of reading them an
// element at a time.
constexpr int kMaxStaged = 36 * 1024, kMostStaged = 144 * 1024;
constexpr int kMaxWaves = 8;
constexpr int kManyTiles = 512;        // 16-row tiles of a weight from which a workgroup has two

// Eight inputs as they are in memory.
template <typename T>
struct Eight {
  uint4 part[sizeof(T) / 2];
  // Inputs k .. k + 7 of a row in whole accesses (past the row's end: its first ones).
  __device__ __forceinline__ void load(const T* row, int k, int K) {
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h)
      part[h] = reinterpret_cast<const uint4*>(row + (k < K ? k : 0))[h];
  }
  // The same an input at a time, 0 past the row's end.
  __device__ __forceinline__ void load_each(const T* row, int k, int K) {
    struct Raw {
      T e[8];
    } raw;
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.e[i] = k + i < K ? row[k + i] : T{};
    *this = __builtin_bit_cast(Eight, raw);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h) part[h] = make_uint4(0, 0, 0, 0);
  }
  // As an operand (fp32: as three).
  __device__ __forceinline__ void operands(s16x8 (&to)[kParts<T>]) const {
    if constexpr (sizeof(T) == 2) {
      to[0] = __builtin_bit_cast(s16x8, part[0]);
    } else {
      struct Raw {
        float e[8];
      };
      const Raw raw = __builtin_bit_cast(Raw, *this);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = raw.e[i];
      attention::split<3>(v, to);
    }
  }
};

// Bytes between the staged rows of two tokens: one 16-byte piece more than their inputs, so that
// a piece column of 16 tokens spreads over the banks.
template <typename T>
constexpr int64_t staged_pitch(int KT) {
  return static_cast<int64_t>(KT) * kDeep * sizeof(T) + 16;
}

// MT token tiles of 16, R tiles of 16 weight rows, G matrices; CH matrix instructions to a group
// (four also where a group is several tiles of codes); U tiles of codes loaded at a time, the next U
// while these are worked on.  STAGED: the tokens' inputs are put into LDS first (one token tile),
// else they come with the codes.  WIDE: whole accesses (of inputs: where they are not staged).
template <typename T, typename S, int MT, int R, int G, int CH, int U, bool WIDE, bool STAGED>
__global__ __launch_bounds__(kMaxWaves* kWave) void linear_4bit_kernel(LinearParams p,
                                                                         FastDiv by_rows) {
  constexpr int NP = kParts<T>, C = 4 / CH;
  extern __shared__ __align__(16) char lds[];  // inputs; later [wave][G][R][MT][64] f32x4
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int W = blockDim.x / kWave;
  const int r = lane & 15, quad = lane >> 4;
  // (Token blocks in a grid's y would end at 65535.)
  uint32_t row_block;
  const int m0 = static_cast<int>(by_rows.div(blockIdx.x, row_block)) * 16 * MT;

  struct Batch {
    uint4 words[U][G][R];
    Four<S, WIDE> scale[U][C][G][R], zero[U][C][G][R];
    Eight<T> x[STAGED ? 1 : U][4][MT];
  };
  const T* rows[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)  // tokens past the last read its row; their outputs are not kept
    rows[t] = static_cast<const T*>(p.x) + static_cast<int64_t>(min(m0 + 16 * t + r, p.M - 1)) * p.x_s;
  const bool zeros = p.zeros[0] != nullptr;
  // Codes and scales by uniform offsets.  Rows past the last read others', and nobody keeps their
  // outputs.
  const int nt0 = static_cast<int>(row_block) * R;
  const int first = min(nt0, p.NT - R);  // R <= NT; the last workgroup may begin in the one before
  rsrc_t codes[G], scales[G], zero_points[G];
  const int groups = (p.K + p.group - 1) / p.group;
  const uint32_t line = static_cast<uint32_t>(p.N) * sizeof(S);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    codes[g] = make_rsrc(p.codes[g] + static_cast<int64_t>(first) * p.KT * kWave,
                         static_cast<uint32_t>(R) * p.KT * 1024u);
    scales[g] = make_rsrc(p.scales[g], groups * line);
    zero_points[g] = make_rsrc(p.zeros[g], groups * line);
  }
  uint32_t lane_off[R][WIDE ? 1 : 4];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < (WIDE ? 1 : 4); ++e)
      lane_off[i][e] = min(16 * (first + i) + 4 * quad + e, p.N - (WIDE ? 4 : 1)) * sizeof(S);
  auto load = [&](int k0, Batch& t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kt = min(k0 + u * W, p.KT - 1);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < R; ++i)
          t.words[u][g][i] = __builtin_bit_cast(
              uint4, __builtin_amdgcn_raw_buffer_load_b128(
                         codes[g], 16u * lane, (static_cast<uint32_t>(i) * p.KT + kt) * 1024u, 0));
    }
    auto vectors = [&](const rsrc_t* of, Four<S, WIDE> (&to)[U][C][G][R]) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          // Past the last input, the last group's.
          const int kt = min(k0 + u * W, p.KT - 1);
          const int at = min(CH < 4 ? C * kt + c
                                    : static_cast<int>(p.by_group_tiles.div(static_cast<uint32_t>(kt))),
                             groups - 1);
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < R; ++i) to[u][c][g][i].load(of[g], lane_off[i], at * line);
        }
    };
    vectors(scales, t.scale);
    if (zeros) vectors(zero_points, t.zero);
    if constexpr (!STAGED) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int k = kDeep * min(k0 + u * W, p.KT - 1) + 32 * s + 8 * quad;
            if constexpr (WIDE)
              t.x[u][s][i].load(rows[i], k, p.K);
            else
              t.x[u][s][i].load_each(rows[i], k, p.K);
          }
    }
  };

  const int pitch = static_cast<int>(staged_pitch<T>(p.KT));
  Batch cur, next;
  load(wave, cur);
  if constexpr (STAGED) {
    const int tokens = min(16, p.M - m0);
    const int per = p.KT * (kDeep / 8);  // pieces of eight inputs
    for (int token = 0; token < tokens; ++token) {
      const T* row = static_cast<const T*>(p.x) + static_cast<int64_t>(m0 + token) * p.x_s;
      for (int i = threadIdx.x; i < per; i += blockDim.x) {
        const int k = 8 * i;
        Eight<T> x;
        x.clear();
        if (p.wide_x) {
          if (k < p.K) x.load(row, k, p.K);
        } else {
          x.load_each(row, k, p.K);
        }
        *reinterpret_cast<Eight<T>*>(lds + token * pitch + k * sizeof(T)) = x;
      }
    }
    __syncthreads();
  }
  const char* staged = lds + min(r, p.M - 1 - m0) * pitch;

  f32x4 total[G][R][MT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) total[g][i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (int k0 = wave; k0 < p.KT; k0 += W * U) {
    if (k0 + W * U < p.KT) load(k0 + W * U, next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kt = k0 + u * W;
      if (u > 0 && kt >= p.KT) break;
#pragma unroll
      for (int c = 0; c < C; ++c) {
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
          const int k = kDeep * kt + 32 * s + 8 * quad;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            Eight<T> e;
            if constexpr (STAGED) {
              e = *reinterpret_cast<const Eight<T>*>(staged + k * sizeof(T));
            } else {
              e = cur.x[u][s][t];
              if (kDeep * (kt + 1) > p.K && k >= p.K) e.clear();
            }
            e.operands(x[t]);
#pragma unroll
            for (int n = 0; n < NP; ++n)
              sum[t] = product(ones<T>(), x[t][n], sum[t], matrix_t<T>{});
          }
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < R; ++i) {
              const s16x8 a = decode<T>(word_of(cur.words[u][g][i], s));
#pragma unroll
              for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < NP; ++n)
                  acc[g][i][t] = product(a, x[t][n], acc[g][i][t], matrix_t<T>{});
            }
        }
        auto add = [&](auto off) {
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int t = 0; t < MT; ++t)
                  total[g][i][t][e] = fmaf(cur.scale[u][c][g][i].at(e),
                                           fmaf(-off(g, i, e), sum[t][e], acc[g][i][t][e]),
                                           total[g][i][t][e]);
        };
        if (zeros)
          add([&](int g, int i, int e) { return kBase<T> + cur.zero[u][c][g][i].at(e); });
        else
          add([&](int, int, int) { return kBase<T> + 8.0f; });
      }
    }
    cur = next;
  }

  if constexpr (STAGED) __syncthreads();  // the inputs have been read
  f32x4* sums = reinterpret_cast<f32x4*>(lds);
  constexpr int kSums = G * R * MT;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t)
        sums[(wave * kSums + (g * R + i) * MT + t) * kWave + lane] = total[g][i][t];
  __syncthreads();
  for (int j = wave; j < R * MT; j += W) {
    if (first + j / MT < nt0) continue;
    f32x4 v[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      v[g] = sums[(g * R * MT + j) * kWave + lane];
      for (int w = 1; w < W; ++w) v[g] += sums[(w * kSums + g * R * MT + j) * kWave + lane];
    }
    finish<T, G>(p, m0 + 16 * (j % MT) + r, 16 * (first + j / MT) + 4 * quad, v);
  }
}

template <typename T, typename S, int MT, int R, int G, int CH, int U, bool WIDE, bool STAGED>
hipError_t launch(const LinearParams& p, hipStream_t stream) {
  const char* name = G == 2 ? "gated_linear_4bit" : "linear_4bit";
  int waves = 1;
  while (waves < kMaxWaves && waves < p.KT) waves *= 2;
  const int64_t row_blocks = (p.NT + R - 1) / R, token_blocks = (p.M + 16 * MT - 1) / (16 * MT);
  RLM_TRY(check_launch(name, row_blocks * token_blocks, kWave * waves));
  size_t bytes = static_cast<size_t>(waves) * G * R * MT * kWave * 16;
  if (STAGED) bytes = std::max<size_t>(bytes, std::min(p.M, 16) * staged_pitch<T>(p.KT));
  if (bytes > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(&linear_4bit_kernel<T, S, MT, R, G, CH, U, WIDE, STAGED>),
        hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    RLM_REQUIRE(e == hipSuccess, "%s: %zu bytes of LDS refused: %s", name, bytes,
                hipGetErrorString(e));
  }
  hipLaunchKernelGGL((linear_4bit_kernel<T, S, MT, R, G, CH, U, WIDE, STAGED>),
                     dim3(static_cast<unsigned>(row_blocks * token_blocks)), dim3(kWave * waves),
                     bytes, stream, p, FastDiv(static_cast<uint32_t>(row_blocks)));
  return launch_status(name);
}

// Measured (us, bf16 or fp16, groups of 128; 8 waves):
//   staged, 1 token: tiles in flight 2 x 1 / 2 x 2 / 2 x 4    4096 to 11008 gated 13.3 / 15.3 / 22.9
//                    8192 to 8192, rows tiles 2 / 1           10.1 / 11.6    to 28672 28.4 / 31.4
//   8 tokens of 8192 to 8192: inputs with the codes 12.9 (one row tile 17.2), staged (131 KB of LDS) 15.8
// Sixteen waves to a workgroup: 1 token gated 16.3, 8192 to 28672 32.9.
template <typename T, typename S, int G, int CH>
hipError_t launch_tokens(const LinearParams& p, hipStream_t stream) {
  if (p.M <= 16 && p.M * staged_pitch<T>(p.KT) <= (p.wide_x ? kMaxStaged : kMostStaged)) {
    if (!p.wide_s) return launch<T, S, 1, 1, G, CH, 1, false, true>(p, stream);
    if constexpr (G == 1)
      if (p.NT >= kManyTiles) return launch<T, S, 1, 2, G, CH, 1, true, true>(p, stream);
    return launch<T, S, 1, 1, G, CH, G == 2 || CH == 1 ? 1 : 2, true, true>(p, stream);
  }
  if (!p.wide_s || !p.wide_x) return launch<T, S, 2, 1, G, CH, 1, false, false>(p, stream);
  if (p.M <= 16) {
    if constexpr (G == 1)
      if (p.NT >= kManyTiles) return launch<T, S, 1, 2, G, CH, 1, true, false>(p, stream);
    return launch<T, S, 1, 1, G, CH, 1, true, false>(p, stream);
  }
  return launch<T, S, 2, 1, G, CH, 1, true, false>(p, stream);
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

// Whether many tokens share tiles, and how.
bool tile_shape(const LinearParams& p, int dtype, int products, TileShape* shape) {
  // 32-bit offsets: a workgroup's tokens, the codes and the scales below 1 GiB each.  (Larger weights take the
  // kernel for few tokens, which reads them once for every 32.)
  if (p.M <= 32 || p.x_s >= (int64_t(1) << 21) ||
      static_cast<int64_t>(p.NT) * p.KT >= (int64_t(1) << 20) ||
      static_cast<int64_t>((p.K + p.group - 1) / p.group) * p.N >= (int64_t(1) << 28))
    return false;
  const int64_t rows = static_cast<int64_t>(p.NT) * products;
  if (!p.wide_x || !p.wide_s) {  // (one shape)
    *shape = kMiddle;
    return true;
  }
  // Modelled times (us).  Few tokens: the weights once for every 32.  Tiles: rounds of workgroups, steps of 128
  // inputs (two or four parts of them at once), a step's time by the group's size.  Measured (tokens, outputs,
  // width, group; few tokens / wide / middle / small):
  //   plain  64,4096,4096,128: 20 / 65 / 31 / 23     333,2304,768,32: 20 / 30 / 16 / 15    ,128: 14 / 22 / 12 / 11
  //          333,4096,4096,32: 110 / 126 / 62 / 77   ,64: 85 / 88 / 45 / 53                ,128: 82 / 68 / 35 / 45
  //          1024,4096,4096,32: 324 / 127 / 83 / 153 ,64: 247 / 90 / 60 / 106              ,128: 241 / 69 / 45 / 89
  //          4096,4096,4096,32: 1288 / 258 / 316 / 610  ,64: 978 / 183 / 220 / 416         ,128:  - / 139 / 165 / 348
  //   gated  64,4096,4096,128: 24 / 70 / 33 / 24     333,2304,768,32: 33 / 32 / 18 / 30    ,128: 19 / 24 / 14 / 21
  //          333,4096,4096,32: 153 / 128 / 88 / 119  ,64: 116 / 92 / 63 / 84               ,128: 105 / 73 / 48 / 71
  //          1024,4096,4096,32: 445 / 139 / 175 / 312   ,64:  - / 98 / 120 / 220           ,128: 310 / 76 / 92 / 181
  //   fp32   64,4096,4096,64: 45 / 211 / 89          333,2304,768,32: 43 / 57 / 28
  //          333,4096,4096,32: 242 / 258 / 117       ,128: 226 / 207 / 80
  //          1024,4096,4096,32: 712 / 265 / 232      ,64: 676 / 226 / 184                  ,128: 666 / 211 / 158
  //          4096,4096,4096,32: 2840 / 540 / 954     ,64: 2720 / 466 / 754                 ,128: 2670 / 424 / 638
  //          gated 333,2304,768,128: 48 / 48 / 24    1024,4096,4096,128: 775 / 210 / 313
  // (fp32 tiles with codes as 16 + c.  As c - 8 both shapes take 2 to 10% longer -- wide, 4096 tokens: 552, 493,
  // 437; middle, 1024: 237, 192, 168 -- which leaves the choice as it is.)
  const bool is32 = dtype == RLM_F32;
  const int ch = p.group == 32 ? 0 : p.group == 64 ? 1 : 2;
  constexpr double kWideStep[] = {3.65, 2.43, 1.83}, kSmallStep[] = {4.0, 2.43, 2.05},
                   kMiddleStep[] = {3.35, 2.25, 1.6}, kMiddleTwo[] = {4.85, 3.35, 2.4};
  auto rounds = [&](int tiles, int tokens, int resident) {
    const int64_t groups = (rows + tiles - 1) / tiles * ((p.M + tokens - 1) / tokens);
    return static_cast<double>((groups + resident - 1) / resident);
  };
  const double rate = is32            ? (products == 2 ? 1.1e6 : 0.8e6)
                      : products == 2 ? (ch == 0 ? 2.5e6 : 3.3e6)
                                      : (ch == 0 ? 1.75e6 : 2.35e6);
  const double few = 5.0 + (p.M + 31) / 32 * (static_cast<double>(rows) * p.KT * 2048.0) / rate;
  constexpr double kWide32[] = {8.0, 6.9, 6.4}, kMiddle32[] = {7.0, 5.5, 4.7};
  const double wide = 9.0 + rounds(16, 128, 256) * p.KT * (is32 ? kWide32 : kWideStep)[ch];
  const double one = rounds(8, 64, 256) * (is32 ? kMiddle32 : kMiddleStep)[ch];
  const double two = is32 ? one : rounds(8, 64, 512) * kMiddleTwo[ch];
  const double middle = 7.0 + (p.KT + 1) / 2 * std::min(one, two);
  const double small =
      is32 ? middle : rounds(4, 64, 256) * (6.8 + (p.KT + 3) / 4 * kSmallStep[ch]);
  *shape = wide <= middle && wide <= small ? kWide : middle <= small ? kMiddle : kSmall;
  return few > std::min(wide, std::min(middle, small));
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
  RLM_REQUIRE(groups * N < (int64_t(1) << 29), "%s: fewer than 2^29 elements, got %lld",
              weights[0].scales_name, (long long)(groups * N));
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
  TileShape shape;
  if (tile_shape(p, input->dtype, count, &shape))
    return (input->dtype == RLM_BF16  ? tile_launch_bf16
            : input->dtype == RLM_F16 ? tile_launch_f16
                                      : tile_launch_f32)(p, shape, count, weights[0].scales->dtype,
                                                         stream);
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
