// Products with 4-bit weights for many tokens: x tiles in LDS shared by the weight rows of a workgroup.
// (Instances: rlm_linear_4bit_bf16.hip, rlm_linear_4bit_f16.hip, rlm_linear_4bit_f32.hip.)
//
// A wave has 64 weight rows (gated: 32 of each weight) and 64 tokens, a workgroup WR by WT waves of them
// for each of WK parts of the inputs.  Inputs come by DMA into LDS, 128 of each token at a time, the
// next 128 on their way while these are worked on, and so do the step's scales; codes come from memory
// straight into registers in operand order.  Per group, total += s acc with acc = sum (16 + c) x; what the 16 and the zero point
// add,
//   sum_g (16 + z_g) s_g X_g,   X_g = the group's sum of inputs,
// is itself a product over groups: the waves that share tokens each sum some of them, with ones as the
// other operand, and every 32 (or 16) groups (16 + z) s and X meet as sums of three bf16 parts (six
// products, to 2^-24 of their size).  The parts of the inputs are added in LDS at the end, in order.
//
// Bound: instructions, and what a barrier a step leaves idle.  A wave's step of 64 rows, 64 tokens and 128
// inputs has 71 products (64 of weights, 4 of input sums, 3 of what is taken back) and about 220 other vector
// instructions (128 decode, 64 scale); each keeps its unit busy 45% of the time and waits take 30%.
// 4096 tokens of 4096 -> 4096 take 140 us in groups of 128 (980 TFLOP/s; the vendor's bf16 product of 8192
// reaches 1560), 183 of 64 and 257 of 32, whose sums are scaled two and four times as often.  With the scales
// loaded in the step that uses them 161 / 276 / 267.  Rows that are no whole accesses: 184 with 4095 outputs, 320 with 4095 inputs too.
//
// fp32 inputs are staged as they are and split into three bf16 parts as they are read (24 bits; three
// products a part of codes), and codes meet them as c - 8, so that only z - 8 is taken back: 438 us in groups of
// 128, 314 TFLOP/s, where the vendor's fp32 product does 150.  (Codes as 16 + c: 419, and errors 42 times as
// large with 304 inputs of one sign; decoding takes 36 instructions more to 32 inputs.)
#pragma once

#include "rlm_linear_4bit.hpp"

namespace rlm {
namespace linear4 {

__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

typedef const __attribute__((address_space(3))) s16x8* lds_frag;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) u32x4* lds_piece;
typedef const __attribute__((address_space(3))) f32x4* lds_f32x4;
typedef __attribute__((address_space(3))) float* lds_float;

// Groups whose sums are kept, and the floats between two tokens' sums.
template <int WK>
constexpr int kChunks = WK == 1 ? 32 : 16;
template <int WK>
constexpr int kSumPitch = kChunks<WK> + 4;
// Bytes of a step's scales of one weight: C groups of ROWS rows, in whole loads of a wave.
template <typename S, int C, int ROWS>
constexpr int kScaleBytes = (C * ROWS * static_cast<int>(sizeof(S)) + 255) / 256 * 256;
template <typename T, typename S, int G, int CH, int WR, int WT, int WK>
constexpr int kTileLds = WK * (64 * WT * (2 * static_cast<int>(sizeof(T)) * kDeep + 4 * kSumPitch<WK>) +
                               2 * G * kScaleBytes<S, 4 / CH, WR * 64 / G>);

// Sixteen bytes of inputs at any address: those below K.
template <typename T>
__device__ __forceinline__ u32x4 piece_of_inputs(const T* row, int k, int K) {
  constexpr int kEach = 16 / static_cast<int>(sizeof(T));
  u32x4 v = {0, 0, 0, 0};
  if (k + kEach <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    struct Raw {
      T e[kEach];
    } raw;
#pragma unroll
    for (int i = 0; i < kEach; ++i) raw.e[i] = k + i < K ? row[k + i] : T{};
    v = __builtin_bit_cast(u32x4, raw);
  }
  return v;
}

// G products; CH matrix instructions to a group (four also where a group is several tiles).  ALIGNED:
// inputs by DMA; EVEN: scales by DMA.
template <typename T, typename S, int G, int CH, int WR, int WT, int WK, bool ALIGNED, bool EVEN>
__global__ __launch_bounds__(WR* WT* WK* kWave, WK == 4 || (sizeof(T) == 4 && WK == 2) ? 1 : 2) void linear_4bit_tile_kernel(LinearParams p,
                                                                                FastDiv by_rows) {
  constexpr int R = 4 / G;                       // 16-row tiles of a wave, of each weight
  constexpr int C = 4 / CH;                      // groups of a tile of codes
  constexpr int kTokens = 64 * WT;               // of a workgroup
  constexpr bool k32 = sizeof(T) == 4;
  typedef matrix_t<T> M;                          // what the matrix unit multiplies
  constexpr int kBytes = static_cast<int>(sizeof(T)) * kDeep;  // of a token's inputs
  constexpr int kPieces = kBytes / 16;
  constexpr int kStage = kTokens * kBytes;
  constexpr int NC = kChunks<WK>, kPitch = kSumPitch<WK>;
  constexpr int kRows = WR * 16 * R;              // of each weight
  constexpr int kScales = kScaleBytes<S, C, kRows>;
  typedef const __attribute__((address_space(3)))
      typename std::conditional<sizeof(S) == 4, u32x4, u32x2>::type* lds_scales;
  extern __shared__ __align__(1024) char lds[];  // [WK][2] stages, [WK] sums, [WK][2][G] scales
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, quad = lane >> 4;
  // Neighbouring workgroups of an XCD share tokens and, a row of workgroups later, weights.
  uint32_t row_block;
  const uint32_t token_block =
      by_rows.div(static_cast<uint32_t>(xcd_tile(blockIdx.x, gridDim.x)), row_block);
  const int m0 = static_cast<int>(token_block) * kTokens;
  const int rq = wave % WR, half = wave / WR % WT, kq = wave / (WR * WT);
  const int nt0 = static_cast<int>(row_block) * WR * R + rq * R;
  const int mate = wave % (WR * WT);             // of the waves that share a part of the inputs
  // This part's tiles of codes.
  const int per = (p.KT + WK - 1) / WK;
  const int kt0 = kq * per, tiles = min(per, p.KT - kt0);  // (none or fewer for the last parts)

  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const uint32_t stages = lds0 + kq * 2 * kStage;
  // Rows of pieces of 16 bytes, swizzled so that a piece column spreads over all banks.  A wave brings four
  // rows at a time (fp32: two): those of load j for j = mate, mate + WR WT, ...
  constexpr int kTogether = kWave / kPieces;
  constexpr int kBring = kTokens / kTogether / (WR * WT);
  const T* base = static_cast<const T*>(p.x) + static_cast<int64_t>(m0) * p.x_s;
  const int rows = min(kTokens, p.M - m0);
  const uint32_t row_bytes = static_cast<uint32_t>(p.x_s) * sizeof(T);
  // (Rows past the last are out of range and come as zeros.)
  const rsrc_t x_rows = make_rsrc(base, static_cast<uint32_t>(rows - 1) * row_bytes + sizeof(T) * p.K);
  const int groups = (p.K + p.group - 1) / p.group;
  auto group_of = [&](int chunk) {  // a chunk's group; past the last input, the last one
    const int at = CH < 4 ? chunk : static_cast<int>(p.by_group_tiles.div(static_cast<uint32_t>(chunk)));
    return min(at, groups - 1);
  };
  // Tiles of codes and scales by uniform offsets; rows past the last read others', and nobody keeps
  // their outputs.
  auto tile_of = [&](int i) { return min(nt0 + i, p.NT - 1); };
  rsrc_t codes[G], scales[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    codes[g] = make_rsrc(p.codes[g], static_cast<uint32_t>(p.NT) * p.KT * 1024u);
    scales[g] = make_rsrc(p.scales[g], static_cast<uint32_t>(groups) * p.N * sizeof(S));
  }
  // A step's scales: four bytes to a lane, groups after each other (rows past the last read others').
  const uint32_t scales0 = lds0 + WK * (2 * kStage + kTokens * kPitch * 4) + kq * 2 * G * kScales;
  auto issue_scales = [&](int i) {
    constexpr int kEach = 4 / static_cast<int>(sizeof(S)), kUnits = kRows / kEach;  // of a group
    constexpr int kLoads = kScales / 256;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int n = 0; n < (kLoads + WR * WT - 1) / (WR * WT); ++n) {
        const int j = mate + n * WR * WT;
        if (kLoads % (WR * WT) != 0 && j >= kLoads) break;
        const int unit = j * kWave + lane, c = unit / kUnits;
        const uint32_t at =
            static_cast<uint32_t>(group_of(C * (kt0 + i) + (CH < 4 ? min(c, C - 1) : 0))) * p.N +
            row_block * kRows + unit % kUnits * kEach;
        lds_dma4(scales[g],
                 __builtin_amdgcn_readfirstlane(scales0 + ((i & 1) * G + g) * kScales + j * 256),
                 at * static_cast<uint32_t>(sizeof(S)));
      }
  };
  // The same through registers, an element to a lane: loaded with the step's inputs, written behind the
  // products of the step before.
  constexpr int kMates = WR * WT * kWave, kOwn = EVEN ? 1 : (C * kRows + kMates - 1) / kMates;
  typedef typename std::conditional<sizeof(S) == 4, uint32_t, uint16_t>::type one_t;
  one_t own[G][kOwn];
  auto load_scales = [&](int i) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int n = 0; n < kOwn; ++n) {
        const int unit = mate * kWave + n * kMates + lane, c = min(unit / kRows, C - 1);
        const uint32_t at = (static_cast<uint32_t>(group_of(C * (kt0 + i) + c)) * p.N +
                             row_block * kRows + unit % kRows) * static_cast<uint32_t>(sizeof(S));
        if constexpr (sizeof(S) == 4)
          own[g][n] = __builtin_amdgcn_raw_buffer_load_b32(scales[g], at, 0, 0);
        else
          own[g][n] = __builtin_amdgcn_raw_buffer_load_b16(scales[g], at, 0, 0);
      }
  };
  auto write_scales = [&](int i) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int n = 0; n < kOwn; ++n) {
        const int unit = mate * kWave + n * kMates + lane;
        if (C * kRows % kMates == 0 || unit < C * kRows)
          *(__attribute__((address_space(3))) one_t*)static_cast<uintptr_t>(
              scales0 + ((i & 1) * G + g) * kScales + unit * static_cast<uint32_t>(sizeof(S))) = own[g][n];
      }
  };
  auto issue = [&](int i) {
    const int kt = kt0 + i;
    const uint32_t to = __builtin_amdgcn_readfirstlane(stages + (i & 1) * kStage);
    if constexpr (EVEN)
      issue_scales(i);
    else
      load_scales(i);
#pragma unroll
    for (int n = 0; n < kBring; ++n) {
      const int j = mate + n * WR * WT;
      const int at = kTogether * j + lane / kPieces;  // row
      const int k = kDeep * kt + 16 / static_cast<int>(sizeof(T)) * (lane % kPieces ^ (at & 15));
      if constexpr (ALIGNED) {
        const uint32_t off = static_cast<uint32_t>(at) * row_bytes + sizeof(T) * k;
        lds_dma16(x_rows, to + 1024u * j, kDeep * (kt + 1) <= p.K || k < p.K ? off : kNoOffset);
      } else {
        *(lds_piece)static_cast<uintptr_t>(to + 1024u * j + 16 * lane) =
            piece_of_inputs(base + static_cast<int64_t>(min(at, rows - 1)) * p.x_s, k, p.K);
      }
    }
  };
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
  load_words(min(kt0, p.KT - 1), words);
  if (tiles > 0) {
    issue(0);
    if (!EVEN) write_scales(0);
  }

  // Sums kept, NC chunks of each token of this part.
  const uint32_t sums0 = lds0 + WK * 2 * kStage + (kq * kTokens + 64 * half) * kPitch * 4;
  const uint32_t x_row = (64 * half + r) * kBytes + (((k32 ? 2 * quad : quad) ^ r) << 4);

  for (int n = 0; n < per; ++n) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    barrier();  // these inputs are in LDS for every wave, the other stage has been read
    if (n + 1 < tiles) issue(n + 1);
    if (n < tiles) {
      const int kt = kt0 + n;
      uint4 next[G][R];
      load_words(min(kt + 1, p.KT - 1), next);
      const uint32_t x_at = stages + (n & 1) * kStage + x_row;
      auto inputs = [&](int s, s16x8 (&x)[4]) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          x[t] = *(lds_frag)static_cast<uintptr_t>((x_at ^ (64u * s)) + 4096u * t);
      };
      // Eight fp32 inputs of token tile t.
      auto eight = [&](int s, int t, float (&v)[8]) {
        const uint32_t at = (x_at ^ (128u * s)) + 8192u * t;
        const f32x4 lo = *(lds_f32x4)static_cast<uintptr_t>(at);
        const f32x4 hi = *(lds_f32x4)static_cast<uintptr_t>(at ^ 16u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < 4 ? lo[e] : hi[e - 4];
      };
      s16x8 x[4];
      if constexpr (!k32) inputs(0, x);
      // (A loop where it has several rounds: unrolled, it spills.)
#pragma unroll 1
      for (int c = 0; c < C; ++c) {
        Four<S, true> scale[G][R];
        f32x4 acc[G][R][4], sum[4 / WR];
#pragma unroll
        for (int t = 0; t < 4 / WR; ++t) sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < R; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[g][i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (k32) {
          float alone[4 / WR] = {};
#pragma unroll
          for (int s = 0; s < CH; ++s) {
            const int at = (c * CH + s) & 3;
            s16x8 a[G][R];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int i = 0; i < R; ++i) a[g][i] = decode_less_8(word_of(words[g][i], s));
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              float v[8];
              eight(at, t, v);
              float paired[8] = {v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};  // as the codes
              s16x8 parts[3];
              attention::split<3>(paired, parts);
#pragma unroll
              for (int n = 2; n >= 0; --n)
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                  for (int i = 0; i < R; ++i) acc[g][i][t] = product(a[g][i], parts[n], acc[g][i][t], M{});
            }
            // The token tiles that this wave sums.
#pragma unroll
            for (int t = 0; t < 4 / WR; ++t) {
              float v[8];
              eight(at, t * WR + (WR == 1 ? 0 : rq), v);
              alone[t] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            }
          }
#pragma unroll
          for (int t = 0; t < 4 / WR; ++t) sum[t][0] = attention::rows_sum(alone[t]);
        } else {
#pragma unroll
          for (int s = 0; s < CH; ++s) {
            s16x8 x_next[4];
            inputs((c * CH + s + 1) & 3, x_next);
            // The token tiles that this wave sums.
            s16x8 mine[4 / WR];
#pragma unroll
            for (int t = 0; t < 4 / WR; ++t)
              mine[t] = WR == 1 ? x[t]
                                : *(lds_frag)static_cast<uintptr_t>((x_at ^ (64u * ((c * CH + s) & 3))) +
                                                                    4096u * (t * WR + rq));
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int i = 0; i < R; ++i) {
                const s16x8 a = decode<M>(word_of(words[g][i], s));
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[g][i][t] = product(a, x[t], acc[g][i][t], T{});
              }
#pragma unroll
            for (int t = 0; t < 4 / WR; ++t) sum[t] = product(ones<T>(), mine[t], sum[t], T{});
#pragma unroll
            for (int t = 0; t < 4; ++t) x[t] = x_next[t];
          }
        }
        if (quad == 0) {
#pragma unroll
          for (int t = 0; t < 4 / WR; ++t)
            *(lds_float)static_cast<uintptr_t>(sums0 + ((16 * (t * WR + rq) + r) * kPitch +
                                                        (C * n + c) % NC) * 4) = sum[t][0];
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < R; ++i)
            scale[g][i].v = __builtin_bit_cast(
                decltype(scale[g][i].v),
                *(lds_scales)static_cast<uintptr_t>(
                    scales0 + ((n & 1) * G + g) * kScales +
                    (c * kRows + 16 * (rq * R + i) + 4 * quad) * static_cast<uint32_t>(sizeof(S))));
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < R; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                total[g][i][t][e] = fmaf(scale[g][i].at(e), acc[g][i][t][e], total[g][i][t][e]);
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
      if (!EVEN && n + 1 < tiles) write_scales(n + 1);
    }

    // total -= ((16 + z) s) X over the kept chunks.
    const int done = C * (n + 1);
    if (done % NC != 0 && n + 1 != per) continue;
    barrier();
    const int kept = (done - 1) / NC * NC;                     // the first one, of this part's,
    const int end = min(done, C * tiles);                      // and behind the last
    if (kept >= end) continue;
    s16x8 xs[4][3];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t at = sums0 + (16 * t + r) * kPitch * 4 + 32 * min(quad, NC / 8 - 1);
      const f32x4 lo = *(lds_f32x4)static_cast<uintptr_t>(at);
      const f32x4 hi = *(lds_f32x4)static_cast<uintptr_t>(at + 16);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = e < 4 ? lo[e] : hi[e - 4];
        v[e] = kept + 8 * quad + e < end ? v[e] : 0.0f;
      }
      attention::split<3>(v, xs[t]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int row = min(16 * (nt0 + i) + r, p.N - 1);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int chunk = min(kept + 8 * quad + e, end - 1);
          const int64_t at = static_cast<int64_t>(group_of(C * kt0 + chunk)) * p.N + row;
          float z = 8.0f;
          if (p.zeros[g] != nullptr) z = to_f32(static_cast<const S*>(p.zeros[g])[at]);
          v[e] = kept + 8 * quad + e < end
                     ? (kBase<T> + z) * to_f32(static_cast<const S*>(p.scales[g])[at]) : 0.0f;
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

  const int token0 = m0 + 64 * half + r, out0 = 16 * nt0 + 4 * quad;
  if constexpr (WK == 1) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 v[G];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[g][e] = total[g][i][t][e];
        finish<T, G>(p, token0 + 16 * t, out0 + 16 * i, v);
      }
  } else {
    // Part kq finishes the token tiles kq, kq + WK, ...
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    barrier();
    f32x4* parts = reinterpret_cast<f32x4*>(lds);  // [wave][G][R][4][64]
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          parts[(((wave * G + g) * R + i) * 4 + t) * kWave + lane] =
              f32x4{total[g][i][t][0], total[g][i][t][1], total[g][i][t][2], total[g][i][t][3]};
    barrier();
    for (int t = kq; t < 4; t += WK)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        f32x4 v[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          v[g] = parts[(((mate * G + g) * R + i) * 4 + t) * kWave + lane];
#pragma unroll
          for (int w = 1; w < WK; ++w)
            v[g] += parts[((((w * WR * WT + mate) * G + g) * R + i) * 4 + t) * kWave + lane];
        }
        finish<T, G>(p, token0 + 16 * t, out0 + 16 * i, v);
      }
  }
}

template <typename T, typename S, int G, int CH, int WR, int WT, int WK, bool ALIGNED, bool EVEN>
hipError_t launch_tile(const LinearParams& p, hipStream_t stream) {
  const char* name = G == 2 ? "gated_linear_4bit" : "linear_4bit";
  constexpr int kThreads = WR * WT * WK * kWave, kLds = kTileLds<T, S, G, CH, WR, WT, WK>;
  static_assert(WK == 1 || kThreads * 256 <= WK * 2 * 64 * WT * kDeep * static_cast<int>(sizeof(T)), "parts in the stages");
  const int64_t row_blocks = (p.NT + WR * 4 / G - 1) / (WR * 4 / G);
  const int64_t token_blocks = (p.M + 64 * WT - 1) / (64 * WT);
  RLM_TRY(check_launch(name, row_blocks * token_blocks, kThreads));
  const auto kernel = &linear_4bit_tile_kernel<T, S, G, CH, WR, WT, WK, ALIGNED, EVEN>;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  RLM_REQUIRE(e == hipSuccess, "%s: %d bytes of LDS refused: %s", name, kLds, hipGetErrorString(e));
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(row_blocks * token_blocks)), dim3(kThreads),
                     kLds, stream, p, FastDiv(static_cast<uint32_t>(row_blocks)));
  return launch_status(name);
}

template <typename T, typename S, int G, int CH>
hipError_t launch_shape(const LinearParams& p, TileShape shape, hipStream_t stream) {
  if (!p.wide_x) return launch_tile<T, S, G, CH, 2, 1, 2, false, false>(p, stream);
  if (!p.wide_s) return launch_tile<T, S, G, CH, 2, 1, 2, true, false>(p, stream);
  if (shape == kWide) return launch_tile<T, S, G, CH, 4, 2, 1, true, true>(p, stream);
  if constexpr (sizeof(T) == 2)  // (four parts of fp32 inputs do not fit)
    if (shape == kSmall) return launch_tile<T, S, G, CH, 1, 1, 4, true, true>(p, stream);
  return launch_tile<T, S, G, CH, 2, 1, 2, true, true>(p, stream);
}
template <typename T, typename S, int G>
hipError_t launch_group_tile(const LinearParams& p, TileShape shape, hipStream_t stream) {
  if (p.group == 32) return launch_shape<T, S, G, 1>(p, shape, stream);
  if (p.group == 64) return launch_shape<T, S, G, 2>(p, shape, stream);
  return launch_shape<T, S, G, 4>(p, shape, stream);
}
template <typename T>
hipError_t launch_tile_type(const LinearParams& p, TileShape shape, int products, int scale_dtype,
                            hipStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (scale_dtype != RLM_F32)
      return products == 2 ? launch_group_tile<T, T, 2>(p, shape, stream)
                           : launch_group_tile<T, T, 1>(p, shape, stream);
  return products == 2 ? launch_group_tile<T, float, 2>(p, shape, stream)
                       : launch_group_tile<T, float, 1>(p, shape, stream);
}

}  // namespace linear4
}  // namespace rlm
