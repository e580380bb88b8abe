// Attention over a window and picked blocks of caches in 8 bits, one query to a workgroup.
//
// The work is laid out as for 16-bit caches (rlm_attention_query.hip): a workgroup has up to 16 query
// heads of one query and key head, its waves share the query's list of keys 32 at a time, keys that
// do not count are replaced by one that does with weight 0, and few items share out their value features.
//
// e4m3 codes are exact in bf16, so all products are bf16 ones whose other operand is a sum of
// bf16 parts.  A bf16 query is one, an fp16 query two (both exact), an fp32 query three (24 bits).  A row's
// scale is a factor of its score, or of its weight after the sum of the weights:
//   s_p = scale ks_p (q . c_p),   out = sum_p (w_p vs_p) c'_p / sum_p w_p.
// These products of weight and scale are two parts (within 2^-18 of themselves; as one, 2^-9, bf16 outputs
// would be 0.0023 off where their own rounding is 0.0017), or three for fp32.
//
// Keys come from memory straight into operands, 16 codes to a lane and load: lane group g has
// features 64 i + 16 g .. + 15, an order of the sum that the query's operand shares.  Values come by
// DMA into LDS as they are; ds_read_b64_tr_b8 gives a lane eight keys of one feature.
//
// Bound: few items wait, a launch, position and picks, keys and values, the merge: 8 queries of 9 heads on 3
// of 64 features over 192 keys take 5.7 us, 16 of 32 on 4 of 128 over 1536 keys (26 MB) 14.0, in three
// tiles a wave.  Many items read: 1024 of 8 queries' heads on 8 of 128 over 1536 keys (402 MB) 94 us, 4.3 TB/s.
// Tiles of 64 keys: 14.1 in place of 13.8, 29 in place of 26 with 512 items, 96 in place of 94.
#include "rlm_attention.hpp"
#include "rlm_attention_mfma.hpp"

namespace rlm {
namespace {

using namespace attention;

constexpr int kKeys = 32;  // keys of a wave's tile

// DC: head dim in 32s; SHARES workgroups have a share of the value features each.
template <typename T, int DC, int MAXW, int SHARES>
__global__ __launch_bounds__(MAXW* kWave) void attend_codes_kernel(Params p) {
  constexpr int NP = kParts<T>, NW = kWeightParts<T>;
  constexpr int DT = 2 * DC / SHARES;           // value features in 16s
  constexpr int kPitch = code_pitch(DT);
  constexpr int kRow = 16 * kPitch;
  constexpr int kValues = kKeys * kRow;         // bytes of a wave's values, and then
  constexpr int kPiece = kValues + 2 * kKeys * 4;  // of the key and value scales
  extern __shared__ __align__(1024) char lds[];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, quad = lane >> 4;
  const int W = blockDim.x / kWave;
  uint32_t chunk, hk, step;
  uint32_t share = 0;
#pragma unroll
  for (int i = 1; i < SHARES; ++i) share += blockIdx.x >= i * p.items;
  const uint32_t item = blockIdx.x - share * p.items;
  const int first = 16 * DT * share;  // value feature
  const int64_t b = p.by_queries.div(p.by_kv.div(p.by_chunks.div(item, chunk), hk), step);
  const int in_group = static_cast<int>(chunk) * p.heads_per_chunk + r;
  const bool row_ok = r < p.heads_per_chunk && in_group < p.G;
  const int head = static_cast<int>(hk) * p.G + (row_ok ? in_group : 0);
  const int D = p.D;

  const int64_t t = position_of(p, b, step);
  const int32_t* picks = p.blocks + b * p.blk_sb + step * p.blk_st + hk * p.blk_sh;
  int32_t pick = lane < p.TOP ? picks[lane] : -1;

  auto feature = [&](int j) { return code_feature<DC>(j, quad); };
  s16x8 qf[DC][NP];
  {
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + step * p.q_st + head * p.q_sh;
#pragma unroll
    for (int j = 0; j < DC; ++j) {
      const int d = feature(j);
      load_parts<T>(src + (d < D ? d : 0), d < D && row_ok, qf[j]);
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
  const uint32_t last_pick = named == 0 ? 0 : 64 - __builtin_clzll(named);
  const uint32_t BS = static_cast<uint32_t>(p.BS);
  const uint32_t keys = near + last_pick * BS;
  const uint32_t tiles = (keys + kKeys - 1) / kKeys;

  const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + b * p.v_sb + hk * p.v_sh;
  // The lower half of the wave loads a tile's key scales, the upper half its value scales.
  const float* sbase = lane < kKeys ? p.ks + b * p.ks_sb + hk * p.ks_sh
                                    : p.vs + b * p.vs_sb + hk * p.vs_sh;
  const int64_t s_st = lane < kKeys ? p.ks_st : p.vs_st;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const uint32_t mine = lds0 + wave * kPiece;

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

    const float scale = sbase[row * s_st];
    // The key codes; past the head dim a lane has the row's first codes, which meet zeros.
    uint4 kw[2][DC / 2 + 1];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint8_t* src = kbase + static_cast<int64_t>(__shfl(row, 16 * kt + r, kWave)) * p.k_st;
#pragma unroll
      for (int i = 0; i < DC / 2; ++i) {
        const int d = 64 * i + 16 * quad;
        kw[kt][i] = *reinterpret_cast<const uint4*>(src + (d < D ? d : 0));
      }
      if constexpr (DC % 2 != 0) {
        const int d = 32 * (DC - 1) + 8 * quad;
        const uint2 x = *reinterpret_cast<const uint2*>(src + (d < D ? d : 0));
        kw[kt][DC / 2] = make_uint4(x.x, x.y, 0, 0);
      }
    }
    // The values' rows into the wave's LDS, pieces where the swizzle puts them (pieces past the
    // head dim hold anything: they are features that nobody reads).
#pragma unroll
    for (int i = 0; i < kKeys * kPitch / kWave; ++i) {
      const int to = i * (kWave / kPitch) + lane / kPitch;
      const int d = first + 16 * ((lane % kPitch) ^ code_swizzle<kPitch>(to));
      const uint8_t* src =
          vbase + static_cast<int64_t>(__shfl(row, to, kWave)) * p.v_st + (d < D ? d : 0);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(src),
          (__attribute__((address_space(3))) void*)static_cast<uintptr_t>(mine + i * kWave * 16), 16,
          0, 0);
    }
    *(__attribute__((address_space(3))) float*)static_cast<uintptr_t>(mine + kValues + 4 * lane) =
        scale_or_nan(scale);
    wave_sync();

    float x[8], top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < DC; ++j) {
        const uint4 w = kw[kt][j / 2];
        const s16x8 kf = j & 1 ? decode8(w.z, w.w) : decode8(w.x, w.y);
#pragma unroll
        for (int n = 0; n < NP; ++n) s = product(kf, qf[j][n], s, bf16{});
      }
      const f32x4 ks = *(lds_f32x4)static_cast<uintptr_t>(mine + kValues + 64 * kt + 16 * quad);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[4 * kt + i] = (mask >> (16 * kt + 4 * quad + i)) & 1
                            ? s[i] * (ks[i] * p.scale_log2) : -INFINITY;
        top = fmaxf(top, x[4 * kt + i]);
      }
    }
    top = fmaxf(m, rows_max(top));
    const float base = top == -INFINITY ? 0.0f : top;
    const float fade = __builtin_amdgcn_exp2f(m - base);
    m = top;
    l *= fade;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const f32x4 vs =
          *(lds_f32x4)static_cast<uintptr_t>(mine + kValues + 128 + 64 * kt + 16 * quad);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& w = x[4 * kt + i];
        w = __builtin_amdgcn_exp2f(w - base);
        l += w;
        // Not 0 times a scale that is no number.
        w = (mask >> (16 * kt + 4 * quad + i)) & 1 ? w * vs[i] : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[j] *= fade;
    s16x8 weights[NW];
    split<NW>(x, weights);
    const int vrow = code_row(r, quad);
    const uint32_t value0 = mine + vrow * kRow + (code_swizzle<kPitch>(vrow) << 4) + (r & 1) * 8;
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    wave_sync();
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (lds_i32x2)static_cast<uintptr_t>(value0 ^ (16u * j)));
      const s16x8 vf = decode8(static_cast<uint32_t>(c[0]), static_cast<uint32_t>(c[1]));
#pragma unroll
      for (int n = 0; n < NW; ++n) acc[j] = product(vf, weights[n], acc[j], bf16{});
    }
    wave_sync();  // the values have been read
  }
  l = rows_sum(l);

  const int64_t row = (b * p.Tq + step) * p.Hq + head;
  T* out = static_cast<T*>(p.out) + row * D;
  auto write = [&](int j, f32x4 v, float inv) {
    const int d = first + 16 * j + 4 * quad;
    if (row_ok && d < D) put4<T>(out + d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  };
  auto write_lse = [&](float base, float total) {
    if (row_ok && quad == 0 && share == 0)
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

template <typename T, int DC, int MAXW, int SHARES>
hipError_t launch(const Params& p, hipStream_t stream) {
  constexpr int DT = 2 * DC / SHARES;
  // Waves of a query: enough to fill the chip, and one tile each at least.
  const int64_t tiles = (p.local_window + p.TOP * p.BS + kKeys - 1) / kKeys;
  int waves = 1;
  while (waves < MAXW && waves < tiles && static_cast<int64_t>(p.items) * waves < 4096) waves *= 2;
  RLM_TRY(check_launch("routed_attention_quantized", int64_t{SHARES} * p.items, kWave * waves));
  const size_t values =
      static_cast<size_t>(waves) * (kKeys * 16 * code_pitch(DT) + 2 * kKeys * 4);
  const size_t merge = waves == 1 ? 0 : static_cast<size_t>(waves) * (DT * kWave * 16 + 16 * 8);
  const size_t lds = std::max(values, merge);
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(&attend_codes_kernel<T, DC, MAXW, SHARES>),
        hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    RLM_REQUIRE(e == hipSuccess, "routed_attention_quantized: %zu bytes of LDS refused: %s", lds,
                hipGetErrorString(e));
  }
  hipLaunchKernelGGL((attend_codes_kernel<T, DC, MAXW, SHARES>), dim3(SHARES * p.items),
                     dim3(kWave * waves), lds, stream, p);
  return launch_status("routed_attention_quantized");
}

// Shares of the value features: as many as leave every workgroup a CU of its own.
constexpr int kUnits = 256;  // compute units
template <typename T, int DC>
hipError_t launch_shares(const Params& p, hipStream_t stream) {
  constexpr int kWaves = DC == 8 || sizeof(T) == 4 ? 8 : 16;
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

template <typename T>
hipError_t launch_type(const Params& p, hipStream_t stream) {
  const int dc = (p.D + 31) / 32;
  if (dc <= 1) return launch_shares<T, 1>(p, stream);
  if (dc <= 2) return launch_shares<T, 2>(p, stream);
  if (dc <= 3) return launch_shares<T, 3>(p, stream);
  if (dc <= 4) return launch_shares<T, 4>(p, stream);
  return launch_shares<T, 8>(p, stream);
}

}  // namespace

namespace attention {

hipError_t quantized_launch(const Params& p, int dtype, hipStream_t stream) {
  if (dtype == RLM_F32) return launch_type<float>(p, stream);
  if (dtype == RLM_BF16) return launch_type<bf16>(p, stream);
  return launch_type<f16>(p, stream);
}

}  // namespace attention
}  // namespace rlm
