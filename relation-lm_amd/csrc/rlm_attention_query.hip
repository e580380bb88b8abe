// Attention over a window and picked blocks, one query to a workgroup: single tokens, ring caches, and
// prompts that the shared tiles (rlm_attention_tile.hip) do not take or that are faster here.
//
// A workgroup has up to 16 query heads of one query and key head (the rows or columns of a
// matrix product) and shares the query's keys among its waves, 32 at a time; where there are fewer
// such items than half the CUs (fp32: see below), workgroups share the value features of each.  The keys are one
// list: the window's positions, then every picked block's; a lane finds one of a tile's keys
// -- its cache row and whether it counts -- and hands it to the lanes that load it, so blocks
// shorter than a tile share one.  A key that does not count (past the position, in the window
// already, a block named twice) is replaced by one of the tile that does, with weight 0: what
// its own row holds is never read.
//
// The products are those of the shared tiles, S^T = K Q^T and O^T += V^T P^T: keys straight
// from memory into operands, 16-bit values through a piece of LDS of the wave's own for the
// transposing reads.  fp32 uses v_mfma_f32_16x16x4_f32, whose operands need no transposing: the
// features of the first product are summed in an order that gives a lane four neighbours.
//
// 16-bit types: the weights are rounded to the type for the second product, which takes no other
// operands (half a step, relative to each weight; the outputs of the measured cases are 0.0020 to 0.0021
// off in bf16, where weights of 32 bits would leave the output's own rounding, 0.0016); scores, maxima,
// sums and outputs stay fp32.
//
// Bound: the latency of three dependent reads (positions and picks; keys and values; the merge
// of the waves), and the memory's rate for large batches: every row is read once per key head.
// 8 queries of 9 heads on 3 of 64 features, a window of 64 and four blocks of 32: 5.2 us.  20
// queries of 32 heads on 4 of 128 over caches of 131072 rows, a window of 512 and 16 blocks of 64:
// 19.8 us, 3.2 TB/s of the rows it needs.  With one head to a key head only one of a product's 16
// rows is used: 666 fp32 queries of 8 heads of 32, 32.3 us, two thirds of the issue slots taken.
#include "rlm_attention.hpp"
#include "rlm_attention_mfma.hpp"

namespace rlm {
namespace {

using namespace attention;

constexpr int kKeys = 32;  // keys of a wave's tile

template <typename T>
constexpr bool kIs32 = sizeof(T) == 4;

__device__ const uint4 zeros[64] = {};  // a row of values

// DC: head dim in 32s; PARTS workgroups have a share of the value features each.
template <typename T, int DC, int MAXW, int PARTS>
__global__ __launch_bounds__(MAXW* kWave) void attend_query_kernel(Params p) {
  constexpr int DT = 2 * DC / PARTS;                       // value features in 16s
  constexpr int kPitch = pitch<T, DC / PARTS, 4>();                   // 16-byte pieces of an LDS row
  constexpr int kRow = 16 * kPitch;
  extern __shared__ __align__(1024) char lds[];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, quad = lane >> 4;
  const int W = blockDim.x / kWave;
  uint32_t chunk, hk, step;
  // The parts of an item a grid apart: on one XCD where 8 divides the items.
  uint32_t part = 0;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) part += blockIdx.x >= i * p.items;
  const uint32_t item = blockIdx.x - part * p.items;
  const int first = 16 * DT * part;  // value feature
  const int64_t b = p.by_queries.div(p.by_kv.div(p.by_chunks.div(item, chunk), hk), step);
  const int in_group = static_cast<int>(chunk) * p.heads_per_chunk + r;
  const bool row_ok = r < p.heads_per_chunk && in_group < p.G;
  const int head = static_cast<int>(hk) * p.G + (row_ok ? in_group : 0);
  const int D = p.D;

  const int64_t t = position_of(p, b, step);
  const int32_t* picks = p.blocks + b * p.blk_sb + step * p.blk_st + hk * p.blk_sh;
  int32_t pick = lane < p.TOP ? picks[lane] : -1;

  typedef typename std::conditional<kIs32<T>, float4, s16x8>::type frag_t;
  constexpr int kFrags = kIs32<T> ? 2 * DC : DC;   // 16-byte pieces of a lane's row
  constexpr int kFeatures = kIs32<T> ? 4 : 8;  // in each
  const int d0 = kFeatures * quad;             // and between them 4 kFeatures
  frag_t qf[kFrags];
  {
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + step * p.q_st + head * p.q_sh;
#pragma unroll
    for (int j = 0; j < kFrags; ++j) {
      const int d = d0 + 4 * kFeatures * j;
      uint4 x = *reinterpret_cast<const uint4*>(src + (d < D ? d : 0));
      if (!(d < D && row_ok)) x = make_uint4(0, 0, 0, 0);
      qf[j] = __builtin_bit_cast(frag_t, x);
    }
  }

  // Positions seen: [low, high), of which [start, high) are the window's.
  const int64_t high = p.ring ? t + 1 : (t + 1 < p.T ? t + 1 : p.T);
  const int64_t low = p.ring && t + 1 > p.T ? t + 1 - p.T : 0;
  int64_t start = t - p.local_window + 1;
  start = start > low ? start : low;
  const uint32_t near = high > start ? static_cast<uint32_t>(high - start) : 0;
  // Blocks named before, or wholly unseen, name nothing.
  for (int i = 0; i + 1 < p.TOP; ++i) {
    const int32_t other = __builtin_amdgcn_readlane(pick, i);
    if (lane > i && pick == other) pick = -1;
  }
  {
    const int64_t at = pick * p.BS;
    if (at >= start || at >= high || at + p.BS <= low) pick = -1;
  }
  const uint64_t named = __builtin_amdgcn_ballot_w64(pick >= 0);
  // Of the named ones the list holds every position (up to the last one named).
  const uint32_t last_pick = named == 0 ? 0 : 64 - __builtin_clzll(named);
  const uint32_t BS = static_cast<uint32_t>(p.BS);
  const uint32_t keys = near + last_pick * BS;
  const uint32_t tiles = (keys + kKeys - 1) / kKeys;

  const T* kbase = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vbase = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const uint32_t mine = lds0 + wave * kKeys * kRow;

  f32x4 acc[DT];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int j = 0; j < DT; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (uint32_t tile = wave; tile < tiles; tile += W) {
    // Lane i (and i + 32): key i of the tile.
    const uint32_t key = tile * kKeys + (lane & (kKeys - 1));
    uint32_t off;
    const uint32_t at_pick = key >= near ? p.by_block.div(key - near, off) : 0;
    const int32_t block = __shfl(pick, static_cast<int>(at_pick < 63 ? at_pick : 63), kWave);
    const int64_t position = key < near ? start + key : block * p.BS + off;
    const bool counts = key < near || (key < keys && block >= 0 && position >= low &&
                                       position < start && position < high);
    const uint32_t mask = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(counts));
    if (mask == 0) continue;
    int32_t row = static_cast<int32_t>(p.ring ? position & (p.T - 1) : position);
    const int32_t some = __builtin_amdgcn_readlane(row, __builtin_ctz(mask));
    row = counts ? row : some;

    f32x4 s[2];
    frag_t kf[2][kFrags];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const T* src = kbase + static_cast<int64_t>(__shfl(row, 16 * kt + r, kWave)) * p.k_st;
#pragma unroll
      for (int j = 0; j < kFrags; ++j) {
        const int d = d0 + 4 * kFeatures * j;
        kf[kt][j] = *reinterpret_cast<const frag_t*>(src + (d < D ? d : 0));
      }
    }
    if constexpr (!kIs32<T>) {
      // The values' rows into the wave's LDS, pieces where the swizzle puts them (pieces past
      // the head dim hold anything: they are features that nobody reads).  Keys that do not
      // count have values of 0: their weight 0 times an infinity of the row that stands for them
      // would be NaN.
#pragma unroll
      for (int i = 0; i < kKeys * kPitch / kWave; ++i) {
        const int to = i * (kWave / kPitch) + lane / kPitch;
        const int piece = (lane % kPitch) ^ swizzle<kPitch>(to);
        const T* src = vbase + static_cast<int64_t>(__shfl(row, to, kWave)) * p.v_st +
                       (first + 8 * piece < D ? first + 8 * piece : 0);
        src = (mask >> to) & 1 ? src : reinterpret_cast<const T*>(zeros);
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(src),
            (__attribute__((address_space(3))) void*)static_cast<uintptr_t>(mine + i * kWave * 16), 16, 0, 0);
      }
    }
    float vs[kIs32<T> ? DT : 1][2][4];
    if constexpr (kIs32<T>) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T* src =
              vbase + static_cast<int64_t>(__shfl(row, 16 * kt + 4 * quad + i, kWave)) * p.v_st;
          src = (mask >> (16 * kt + 4 * quad + i)) & 1 ? src : reinterpret_cast<const T*>(zeros);
#pragma unroll
          for (int j = 0; j < DT; ++j) {
            const int d = first + 16 * j + r;
            vs[j][kt][i] = src[d < D ? d : 0];
          }
        }
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < kFrags; ++j) {
        if (d0 + 4 * kFeatures * j >= D) kf[kt][j] = frag_t{};  // past the head dim
        s[kt] = product(kf[kt][j], qf[j], s[kt], T{});
      }
    }
    float x[2][4], top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[kt][i] = (mask >> (16 * kt + 4 * quad + i)) & 1 ? s[kt][i] * p.scale_log2 : -INFINITY;
        top = fmaxf(top, x[kt][i]);
      }
    top = fmaxf(m, rows_max(top));
    const float base = top == -INFINITY ? 0.0f : top;
    const float fade = __builtin_amdgcn_exp2f(m - base);
    m = top;
    l *= fade;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[kt][i] = __builtin_amdgcn_exp2f(x[kt][i] - base);
        l += x[kt][i];
      }
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[j] *= fade;
    if constexpr (kIs32<T>) {
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vs[j][kt][i], x[kt][i], acc[j], 0, 0, 0);
    } else {
      const uint4 weights =
          make_uint4(pack2(x[0][0], x[0][1], T{}), pack2(x[0][2], x[0][3], T{}),
                     pack2(x[1][0], x[1][1], T{}), pack2(x[1][2], x[1][3], T{}));
      const int vrow = 4 * quad + (r >> 2);
      const uint32_t value0 = mine + vrow * kRow +
                              ((((r & 3) >> 1) ^ swizzle<kPitch>(vrow)) << 4) + (r & 1) * 8;
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      wave_sync();
#pragma unroll
      for (int j = 0; j < DT; ++j)
        acc[j] = product(read_values(value0 ^ (32u * j), 16 * kRow),
                         __builtin_bit_cast(s16x8, weights), acc[j], T{});
      wave_sync();  // the values have been read
    }
  }
  l = rows_sum(l);

  const int64_t row = (b * p.Tq + step) * p.Hq + head;
  T* out = static_cast<T*>(p.out) + row * D;
  auto write = [&](int j, f32x4 v, float inv) {
    const int d = first + 16 * j + 4 * quad;
    if (row_ok && d < D) put4<T>(out + d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  };
  auto write_lse = [&](float base, float total) {
    if (row_ok && quad == 0 && part == 0)
      p.lse[row] = total == 0.0f ? -INFINITY : (base + __builtin_amdgcn_logf(total)) * kLn2;
  };
  if (W == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < DT; ++j) write(j, acc[j], inv);
    write_lse(m, l);
    return;
  }
  // The waves' sums, in the waves' order; each wave finishes its share of the features.
  __syncthreads();
  f32x4* sums = reinterpret_cast<f32x4*>(lds);                         // [W][DT][64]
  float2* stats = reinterpret_cast<float2*>(sums + W * DT * kWave);    // [W][16]: base, sum
#pragma unroll
  for (int j = 0; j < DT; ++j) sums[(wave * DT + j) * kWave + lane] = acc[j];
  if (quad == 0) stats[wave * 16 + r] = make_float2(m, l);
  __syncthreads();
  if (wave >= DT) return;
  float top = -INFINITY;
  for (int w = 0; w < W; ++w) top = fmaxf(top, stats[w * 16 + r].x);
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  for (int w = 0; w < W; ++w) {
    const float2 of = stats[w * 16 + r];
    total += of.y * __builtin_amdgcn_exp2f(of.x - base);
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  for (int j = wave; j < DT; j += W) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int w = 0; w < W; ++w)
      v += sums[(w * DT + j) * kWave + lane] * __builtin_amdgcn_exp2f(stats[w * 16 + r].x - base);
    write(j, v, inv);
  }
  if (wave == 0) write_lse(top, total);
}

template <typename T, int DC, int MAXW, int PARTS>
hipError_t launch(const Params& p, hipStream_t stream) {
  constexpr int DT = 2 * DC / PARTS;
  constexpr int kPitch = pitch<T, DC / PARTS, 4>();
  // Waves of a query: enough to fill the chip, and one tile each at least.
  const int64_t tiles = (p.local_window + p.TOP * p.BS + kKeys - 1) / kKeys;
  int waves = 1;
  while (waves < MAXW && waves < tiles && static_cast<int64_t>(p.items) * waves < 4096) waves *= 2;
  RLM_TRY(check_launch("routed_attention", int64_t{PARTS} * p.items, kWave * waves));
  const size_t values = sizeof(T) == 4 ? 0 : static_cast<size_t>(waves) * kKeys * 16 * kPitch;
  const size_t merge = waves == 1 ? 0 : static_cast<size_t>(waves) * (DT * kWave * 16 + 16 * 8);
  const size_t lds = std::max(values, merge);
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(&attend_query_kernel<T, DC, MAXW, PARTS>),
        hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    RLM_REQUIRE(e == hipSuccess, "routed_attention: %zu bytes of LDS refused: %s", lds,
                hipGetErrorString(e));
  }
  hipLaunchKernelGGL((attend_query_kernel<T, DC, MAXW, PARTS>), dim3(PARTS * p.items),
                     dim3(kWave * waves), lds, stream, p);
  return launch_status("routed_attention");
}

// Parts of the value features.  Each part computes the weights anew and reads the keys again (from
// the L2 that they share), but its values, its sums and their merge are the shorter for it.
// As many as leave every workgroup a CU of its own.  Measured, one part / two / four (us; single
// tokens, a window of 512 and 16 blocks of 64):
//   bf16, 128 features    8 items: 20.9 / 17.3 / 15.6    64: 24.1 / 19.5 / 17.7
//                         128: 26.1 / 21.9               192: 31.1 / 42.8
//   bf16, 64 features     8 items: 11.6 / 10.6           128: 13.3 / 13.3
//   fp32, 64 features     8 items: 25.8 / 21.5           128: 28.9 / 24.6    256: 35 / 50
// fp32 beyond 64 features fills the registers with a tile's keys and values.  96 and 128 features
// take three and four parts while two workgroups to a CU hold them (one part / all):
//   128 features    8 items: 54 / 31    128: 95 / 56    132: 98 / 97    512: 294 / 359
//                   256 items that are 64 neighbouring queries: 27 / 49
//    96 features    8 items: 44 / 27    128: 75 / 49    256 items of neighbours: 27 / 34
// 256 features always take two, one part spilling (8 items: 221 / 67; 4096: 6274 / 3278).
// Waves: sixteen, but eight where sixteen would spill (bf16, 128 features, one part, 16 / 8 waves:
// 256 items 40 / 34, 1024 162 / 153; two parts, 128 items 21.9 / 20.2; four parts fit, and 64 items
// of 5120 keys take 47 / 54).  At 256 features one part of eight waves still spills 3 registers; single
// tokens over 512 keys: 256 items 25.3, 512 50, 1024 107, 4096 378.
constexpr int kUnits = 256;  // compute units
template <typename T, int DC>
hipError_t launch_parts(const Params& p, hipStream_t stream) {
  if constexpr (kIs32<T> && DC == 8) {
    return launch<T, DC, 8, 2>(p, stream);
  } else if constexpr (kIs32<T> && DC >= 3) {
    return DC * p.items <= 2 * kUnits ? launch<T, DC, 8, DC>(p, stream)
                                      : launch<T, DC, 8, 1>(p, stream);
  } else {
    constexpr int kWaves = DC == 8 || (kIs32<T> && DC == 2) ? 8 : 16;
    constexpr int kFewer = DC == 4 ? 8 : kWaves;
    const uint32_t room = kUnits / p.items;
    if constexpr (DC >= 4)
      if (room >= 4) return launch<T, DC, kWaves, 4>(p, stream);
    if constexpr (DC == 3)
      if (room >= 3) return launch<T, DC, kWaves, 3>(p, stream);
    if constexpr (DC % 2 == 0)
      if (room >= 2) return launch<T, DC, kFewer, 2>(p, stream);
    return launch<T, DC, kFewer, 1>(p, stream);
  }
}
template <typename T>
hipError_t launch_type(const Params& p, hipStream_t stream) {
  const int dc = (p.D + 31) / 32;
  if (dc <= 1) return launch_parts<T, 1>(p, stream);
  if (dc <= 2) return launch_parts<T, 2>(p, stream);
  if (dc <= 3) return launch_parts<T, 3>(p, stream);
  if (dc <= 4) return launch_parts<T, 4>(p, stream);
  return launch_parts<T, 8>(p, stream);
}

}  // namespace

namespace attention {

hipError_t query_launch(const Params& p, int dtype, hipStream_t stream) {
  if (dtype == RLM_F32) return launch_type<float>(p, stream);
  if (dtype == RLM_BF16) return launch_type<bf16>(p, stream);
  return launch_type<f16>(p, stream);
}

}  // namespace attention
}  // namespace rlm
