// Products with 4-bit weights for many tokens: x tiles in LDS shared by the weight rows of a workgroup.
//
// A workgroup of eight waves has 128 tokens and 256 weight rows (gated: 128 rows of each weight), a
// wave 64 by 64 of them.  Inputs come by DMA into LDS, 128 of each token at a time, the next 128 on
// their way while these are worked on; codes come from memory straight into registers in operand
// order and are decoded by the two waves that need them.  Per group, total += s acc with
// acc = sum (16 + c) x; what the 16 and the zero point add,
//   sum_g (16 + z_g) s_g X_g,   X_g = the group's sum of inputs,
// is itself a product over groups: each wave sums 16 of the workgroup's tokens with ones as the other
// operand, and every 32 groups (16 + z) s and X meet as sums of three bf16 parts (six products, to
// 2^-24 of their size).
#include "rlm_linear_4bit.hpp"

namespace rlm {
namespace {

using namespace linear4;

constexpr int kThreads = 512;
constexpr int kTokens = 128;                     // of a workgroup
constexpr int kStage = kTokens * kDeep * 2;      // bytes of inputs in LDS
constexpr int kChunks = 32;                      // groups whose sums are kept
constexpr int kSumPitch = kChunks + 4;           // floats of a token's sums
constexpr int kLds = 2 * kStage + kTokens * kSumPitch * 4;

__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

typedef const __attribute__((address_space(3))) s16x8* lds_frag;
typedef const __attribute__((address_space(3))) f32x4* lds_f32x4;
typedef __attribute__((address_space(3))) float* lds_float;

// Four neighbouring scales at a byte offset, as they are and as fp32.
template <typename S>
using four_t = typename std::conditional<sizeof(S) == 4, uint4, uint2>::type;
template <typename S>
__device__ __forceinline__ four_t<S> load_four(rsrc_t r, uint32_t lane_off, uint32_t off) {
  if constexpr (sizeof(S) == 4)
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, lane_off, off, 0));
  else
    return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, lane_off, off, 0));
}
template <typename S>
__device__ __forceinline__ float one_of(const four_t<S>& v, int e) {
  struct Four {
    S e[4];
  };
  return to_f32(__builtin_bit_cast(Four, v).e[e]);
}

// G products; CH matrix instructions to a group (four also where a group is several tiles).
template <typename T, typename S, int G, int CH>
__global__ __launch_bounds__(kThreads, 2) void linear_4bit_tile_kernel(LinearParams p, FastDiv by_rows) {
  constexpr int R = 4 / G;                       // 16-row tiles of a wave, of each weight
  constexpr int C = 4 / CH;                      // groups of a tile of codes
  extern __shared__ __align__(1024) char lds[];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, quad = lane >> 4;
  // Neighbouring workgroups of an XCD share tokens and, a row of workgroups later, weights.
  uint32_t row_block;
  const uint32_t token_block =
      by_rows.div(static_cast<uint32_t>(xcd_tile(blockIdx.x, gridDim.x)), row_block);
  const int m0 = static_cast<int>(token_block) * kTokens;
  const int rq = wave & 3, half = wave >> 2;     // rows' quarter, tokens' half
  const int nt0 = static_cast<int>(row_block) * 4 * R + rq * R;

  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  // This lane's pieces of a stage: rows of 16 pieces, swizzled so that a piece column spreads
  // over all banks.
  constexpr int kDma = kStage / 16 / kThreads;
  const T* base = static_cast<const T*>(p.x) + static_cast<int64_t>(m0) * p.x_s;
  const int rows = min(kTokens, p.M - m0);
  const rsrc_t x_rows = make_rsrc(base, 0x7ffffff0u);
  uint32_t x_off[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int row = (wave * kDma + i) * 4 + (lane >> 4);
    x_off[i] = static_cast<uint32_t>(min(row, rows - 1) * static_cast<int>(p.x_s) * 2 +
                                     16 * ((lane & 15) ^ (row & 15)));
  }
  auto issue = [&](int kt) {
    const uint32_t to =
        __builtin_amdgcn_readfirstlane(lds0 + (kt & 1) * kStage + wave * kDma * 1024);
    if (kDeep * (kt + 1) <= p.K) {
#pragma unroll
      for (int i = 0; i < kDma; ++i)
        lds_dma16(x_rows, to + 1024u * i, x_off[i], 2u * kDeep * kt);
    } else {  // pieces past the inputs come as zeros
#pragma unroll
      for (int i = 0; i < kDma; ++i) {
        const int row = (wave * kDma + i) * 4 + (lane >> 4);
        const bool there = kDeep * kt + 8 * ((lane & 15) ^ (row & 15)) < p.K;
        lds_dma16(x_rows, to + 1024u * i, there ? x_off[i] + 2u * kDeep * kt : kNoOffset);
      }
    }
  };
  // Tiles of codes and scales by uniform offsets; rows past the last read others', and nobody keeps
  // their outputs.
  auto tile_of = [&](int i) { return min(nt0 + i, p.NT - 1); };
  rsrc_t codes[G], scales[G];
  const uint32_t code_bytes = static_cast<uint32_t>(p.NT) * p.KT * 1024u;
  const int groups = (p.K + p.group - 1) / p.group;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    codes[g] = make_rsrc(p.codes[g], code_bytes);
    scales[g] = make_rsrc(p.scales[g], static_cast<uint32_t>(groups) * p.N * sizeof(S));
  }
  auto load_words = [&](int kt, uint4 (&w)[G][R]) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < R; ++i)
        w[g][i] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(
                       codes[g], 16u * lane, (static_cast<uint32_t>(tile_of(i)) * p.KT + kt) * 1024u, 0));
  };

  float total[G][R][4][4];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[g][i][t][e] = 0.0f;

  uint4 words[G][R];
  load_words(0, words);
  issue(0);

  // Sums kept, 32 chunks of each token.
  const uint32_t sums0 = lds0 + 2 * kStage;
  const uint32_t my_sum = sums0 + (64 * half + 16 * rq + r) * kSumPitch * 4;
  auto group_of = [&](int chunk) {  // a chunk's group; past the last input, the last one
    const int at = CH < 4 ? chunk : static_cast<int>(p.by_group_tiles.div(static_cast<uint32_t>(chunk)));
    return min(at, groups - 1);
  };
  const uint32_t x_row = (64 * half + r) * 256 + ((quad ^ r) << 4);

  for (int kt = 0; kt < p.KT; ++kt) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    barrier();  // these inputs are in LDS for every wave, the other stage has been read
    if (kt + 1 < p.KT) issue(kt + 1);
    uint4 next[G][R];
    load_words(min(kt + 1, p.KT - 1), next);
    const uint32_t x_at = lds0 + (kt & 1) * kStage + x_row;
    auto inputs = [&](int s, s16x8 (&x)[4]) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        x[t] = *(lds_frag)static_cast<uintptr_t>((x_at ^ (64u * s)) + 4096u * t);
    };
    s16x8 x[4];
    inputs(0, x);
    // (A loop where it has several rounds: unrolled, it spills.)
#pragma unroll 1
    for (int c = 0; c < C; ++c) {
      const int chunk = C * kt + c;
      const uint32_t line = static_cast<uint32_t>(group_of(chunk)) * p.N;
      four_t<S> scale[G][R];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < R; ++i)
          scale[g][i] = load_four<S>(scales[g], min(4 * quad, p.N - 4 - 16 * tile_of(i)) * sizeof(S),
                                     (line + 16 * tile_of(i)) * sizeof(S));
      f32x4 acc[G][R][4], sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[g][i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < CH; ++s) {
        s16x8 x_next[4];
        inputs((c * CH + s + 1) & 3, x_next);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const s16x8 a = decode<T>(word_of(words[g][i], s));
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[g][i][t] = product(a, x[t], acc[g][i][t], T{});
          }
        __builtin_amdgcn_sched_barrier(0);  // operands of one step and the next live at once
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (rq == t) sum = product(ones<T>(), x[t], sum, T{});
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = x_next[t];
      }
      if (quad == 0)
        *(lds_float)static_cast<uintptr_t>(my_sum + 4 * (chunk % kChunks)) = sum[0];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              total[g][i][t][e] =
                  fmaf(one_of<S>(scale[g][i], e), acc[g][i][t][e], total[g][i][t][e]);
      if constexpr (CH < 4) {  // the next chunk's words to the front
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const uint4 w = words[g][i];
            words[g][i] = CH == 1 ? make_uint4(w.y, w.z, w.w, w.x) : make_uint4(w.z, w.w, w.x, w.y);
          }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < R; ++i) words[g][i] = next[g][i];

    const int end = C * (kt + 1);
    if (end % kChunks != 0 && kt + 1 != p.KT) continue;
    // total -= ((16 + z) s) X over the kept chunks.
    const int first = (end - 1) / kChunks * kChunks;
    barrier();
    s16x8 xs[4][3];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t at = sums0 + (64 * half + 16 * t + r) * kSumPitch * 4 + 32 * quad;
      const f32x4 lo = *(lds_f32x4)static_cast<uintptr_t>(at);
      const f32x4 hi = *(lds_f32x4)static_cast<uintptr_t>(at + 16);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = e < 4 ? lo[e] : hi[e - 4];
        v[e] = first + 8 * quad + e < end ? v[e] : 0.0f;
      }
      attention::split<3>(v, xs[t]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int n = min(16 * (nt0 + i) + r, p.N - 1);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int chunk = first + 8 * quad + e;
          const int64_t at = static_cast<int64_t>(group_of(min(chunk, end - 1))) * p.N + n;
          float z = 8.0f;
          if (p.zeros[g] != nullptr) z = to_f32(static_cast<const S*>(p.zeros[g])[at]);
          v[e] = chunk < end ? (kBase<T> + z) * to_f32(static_cast<const S*>(p.scales[g])[at]) : 0.0f;
        }
        s16x8 cs[3];
        attention::split<3>(v, cs);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
          a = product(cs[2], xs[t][0], a, bf16{});
          a = product(cs[0], xs[t][2], a, bf16{});
          a = product(cs[1], xs[t][1], a, bf16{});
          a = product(cs[1], xs[t][0], a, bf16{});
          a = product(cs[0], xs[t][1], a, bf16{});
          a = product(cs[0], xs[t][0], a, bf16{});
#pragma unroll
          for (int e = 0; e < 4; ++e) total[g][i][t][e] -= a[e];
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }

#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 v[G];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[g][e] = total[g][i][t][e];
      finish<T, G>(p, m0 + 64 * half + 16 * t + r, 16 * (nt0 + i) + 4 * quad, v);
    }
}

template <typename T, typename S, int G, int CH>
hipError_t launch(const LinearParams& p, hipStream_t stream) {
  const char* name = G == 2 ? "gated_linear_4bit" : "linear_4bit";
  const int64_t row_blocks = (p.NT + 16 / G - 1) / (16 / G);
  const int64_t token_blocks = (p.M + kTokens - 1) / kTokens;
  RLM_TRY(check_launch(name, row_blocks * token_blocks, kThreads));
  const hipError_t e = hipFuncSetAttribute(
      reinterpret_cast<const void*>(&linear_4bit_tile_kernel<T, S, G, CH>),
      hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  RLM_REQUIRE(e == hipSuccess, "%s: %d bytes of LDS refused: %s", name, kLds, hipGetErrorString(e));
  hipLaunchKernelGGL((linear_4bit_tile_kernel<T, S, G, CH>),
                     dim3(static_cast<unsigned>(row_blocks * token_blocks)), dim3(kThreads), kLds,
                     stream, p, FastDiv(static_cast<uint32_t>(row_blocks)));
  return launch_status(name);
}

template <typename T, typename S, int G>
hipError_t launch_group(const LinearParams& p, hipStream_t stream) {
  if (p.group == 32) return launch<T, S, G, 1>(p, stream);
  if (p.group == 64) return launch<T, S, G, 2>(p, stream);
  return launch<T, S, G, 4>(p, stream);
}

template <int G>
hipError_t launch_types(const LinearParams& p, int dtype, int scale_dtype, hipStream_t stream) {
  if (dtype == RLM_BF16)
    return scale_dtype == RLM_F32 ? launch_group<bf16, float, G>(p, stream)
                                  : launch_group<bf16, bf16, G>(p, stream);
  return scale_dtype == RLM_F32 ? launch_group<f16, float, G>(p, stream)
                                : launch_group<f16, f16, G>(p, stream);
}

}  // namespace

namespace linear4 {

bool tile_fits(const LinearParams& p, int dtype) {
  // 16-bit inputs in whole pieces, four scales at a time; a workgroup's tokens, the codes and the
  // scales below 2 GiB each.
  return dtype != RLM_F32 && p.wide_x && p.wide_s && p.x_s < (int64_t(1) << 22) &&
         static_cast<int64_t>(p.NT) * p.KT < (int64_t(1) << 20) &&
         static_cast<int64_t>((p.K + p.group - 1) / p.group) * p.N < (int64_t(1) << 28);
}

hipError_t tile_launch(const LinearParams& p, int products, int dtype, int scale_dtype,
                       hipStream_t stream) {
  return products == 2 ? launch_types<2>(p, dtype, scale_dtype, stream)
                       : launch_types<1>(p, dtype, scale_dtype, stream);
}

}  // namespace linear4
}  // namespace rlm
