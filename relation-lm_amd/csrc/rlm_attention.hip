// Attention of each query over its local window and the blocks picked for it.
//
// A query at position t with window L and picks j_1 .. j_TOP attends to the positions
//   [t - L + 1, t]  and, before them,  [j BS, j BS + BS) of every pick
// that the cache holds (linear: p < T; ring: p > t - T, position p in row p mod T):
//   out = sum_p softmax_p(scale q . k_p) v_p,   lse = log sum_p exp(scale q . k_p).
// A position counts once whichever way it is named; a query that sees none gives 0 and -inf.
#include "rlm_attention.hpp"

namespace rlm {
namespace {

using namespace attention;

// ---------------------------------------------------------------------------
// Up to 16 heads of one query to a wave, fp32 products
// ---------------------------------------------------------------------------
//
// v_mfma_f32_16x16x4_f32 with the keys as rows and the heads as columns, so a lane holds four
// keys' scores of one head, which are the second product's operand as they stand:
//   S^T[key, head]  : lane (head = l % 16, keys 4 (l / 16) + i)
//   O^T[dim, head] += V^T[dim, key] P^T[key, head], four keys (one of each lane group) a step.
// The features are summed in an order that gives a lane four neighbouring ones of a key's row
// (one wide load).  One query's heads share its keys, so a masked key is masked for the whole
// wave; a lane of a masked key reads a key of the same run that is not.
template <typename T, int DT>
__global__ __launch_bounds__(512) void attend_query_kernel(Params p) {
  extern __shared__ __align__(16) float merge[];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r = lane & 15, quad = lane >> 4;
  const int W = p.waves_per_item;
  const uint32_t item = W == 1 ? blockIdx.x * (blockDim.x / kWave) + wave : blockIdx.x;
  const int share = W == 1 ? 0 : wave;
  if (item >= p.items) return;  // W == 1 alone: no barrier follows
  uint32_t chunk, hk, step;
  const uint32_t b = p.by_queries.div(p.by_kv.div(p.by_chunks.div(item, chunk), hk), step);
  const int head_in_group = static_cast<int>(chunk) * 16 + r;
  const bool head_ok = head_in_group < p.G;
  const int head = static_cast<int>(hk) * p.G + (head_ok ? head_in_group : 0);
  const int D = p.D;

  float qf[DT][4];
  {
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + step * p.q_st + head * p.q_sh;
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      const int d = 16 * j + 4 * quad;
      const float4 x = load4(src + (d < D ? d : 0));
      const bool ok = d < D && head_ok;
      qf[j][0] = ok ? x.x : 0.0f;
      qf[j][1] = ok ? x.y : 0.0f;
      qf[j][2] = ok ? x.z : 0.0f;
      qf[j][3] = ok ? x.w : 0.0f;
    }
  }
  const int64_t t = load_any_i(p.pos, p.pos_dtype, b * p.pos_sb + step * p.pos_sq);
  const int32_t* picks = p.blocks + b * p.blk_sb + step * p.blk_st + hk * p.blk_sh;
  const int32_t mine = lane < p.TOP ? picks[lane] : -1;
  // Positions seen: [low, high), of which [start, high) are the window's.
  const int64_t high = p.ring ? t + 1 : (t + 1 < p.T ? t + 1 : p.T);
  const int64_t low = p.ring && t + 1 > p.T ? t + 1 - p.T : 0;
  int64_t start = t - p.local_window + 1;
  start = start > low ? start : low;
  const int64_t near = high > start ? high - start : 0;
  const uint32_t near_tiles = static_cast<uint32_t>((near + 15) / 16);
  const uint32_t tiles = near_tiles + p.TOP * p.by_block_tiles.d;

  const T* kbase = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vbase = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  f32x4 acc[DT] = {};
  float m = -INFINITY, l = 0.0f;

  for (uint32_t tile = share; tile < tiles; tile += W) {
    int64_t first, end;  // this tile's positions [first, end), at most 16
    if (tile < near_tiles) {
      first = start + 16 * static_cast<int64_t>(tile);
      end = first + 16 < high ? first + 16 : high;
    } else {
      uint32_t part;
      const int pick = static_cast<int>(p.by_block_tiles.div(tile - near_tiles, part));
      const int32_t block = __builtin_amdgcn_readlane(mine, pick);
      const uint64_t same = __builtin_amdgcn_ballot_w64(mine == block);
      if (block < 0 || (same & ((uint64_t(1) << pick) - 1)) != 0) continue;
      first = block * p.BS;
      end = first + p.BS < start ? first + p.BS : start;
      end = end < high ? end : high;
      first += 16 * static_cast<int64_t>(part);
      end = first + 16 < end ? first + 16 : end;
      first = first > low ? first : low;
    }
    if (first >= end) continue;
    const int count = static_cast<int>(end - first);
    const int64_t row0 = p.ring ? (first & (p.T - 1)) : first;
    auto row_of = [&](int i) {
      const int64_t row = row0 + (i < count ? i : 0);
      return p.ring && row >= p.T ? row - p.T : row;
    };
    const T* krow = kbase + row_of(r) * p.k_st;
    f32x4 s = {};
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      const int d = 16 * j + 4 * quad;
      const float4 x = load4(krow + (d < D ? d : 0));  // past D: the query's features are 0 ...
      const bool ok = d < D;                           // ... and so is the key's, whatever it holds
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(ok ? x.x : 0.0f, qf[j][0], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(ok ? x.y : 0.0f, qf[j][1], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(ok ? x.z : 0.0f, qf[j][2], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(ok ? x.w : 0.0f, qf[j][3], s, 0, 0, 0);
    }
    float x[4], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = 4 * quad + i < count ? s[i] * p.scale_log2 : -INFINITY;
      top = fmaxf(top, x[i]);
    }
    top = fmaxf(m, rows_max(top));
    const float base = top == -INFINITY ? 0.0f : top;
    const float fade = __builtin_amdgcn_exp2f(m - base);
    m = top;
    l *= fade;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i] - base);
      l += x[i];
    }
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      acc[j] *= fade;
      const int d = 16 * j + r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = to_f32(vbase[row_of(4 * quad + i) * p.v_st + (d < D ? d : 0)]);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[i], acc[j], 0, 0, 0);
      }
    }
  }
  l = rows_sum(l);

  if (W > 1) {
    // The waves' sums into the first wave's, in the waves' order.
    constexpr int kFloats = 4 * DT + 2;
    if (wave != 0) {
      float* to = merge + (wave - 1) * kFloats * kWave + lane;
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(4 * j + i) * kWave] = acc[j][i];
      to[4 * DT * kWave] = m;
      to[(4 * DT + 1) * kWave] = l;
    }
    __syncthreads();
    if (wave != 0) return;
    for (int w = 1; w < W; ++w) {
      const float* from = merge + (w - 1) * kFloats * kWave + lane;
      const float mw = from[4 * DT * kWave], lw = from[(4 * DT + 1) * kWave];
      const float top = fmaxf(m, mw), base = top == -INFINITY ? 0.0f : top;
      const float a = __builtin_amdgcn_exp2f(m - base), c = __builtin_amdgcn_exp2f(mw - base);
      m = top;
      l = l * a + lw * c;
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[j][i] = acc[j][i] * a + from[(4 * j + i) * kWave] * c;
    }
  }
  if (!head_ok) return;
  const int64_t row = (static_cast<int64_t>(b) * p.Tq + step) * p.Hq + head;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(p.out) + row * D;
#pragma unroll
  for (int j = 0; j < DT; ++j) {
    const int d = 16 * j + 4 * quad;
    if (d < D) put4<T>(out + d, acc[j][0] * inv, acc[j][1] * inv, acc[j][2] * inv, acc[j][3] * inv);
  }
  if (quad == 0) p.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T, int DT>
hipError_t launch_query(Params& p, hipStream_t stream) {
  // Waves of an item: one where the items alone fill the chip.
  const int64_t seen = p.local_window + static_cast<int64_t>(p.TOP) * p.BS;
  const int64_t tiles = (seen + 15) / 16;
  int waves = p.items >= 4096 ? 1 : p.items >= 1024 ? 4 : 8;
  if (waves > tiles) waves = static_cast<int>(tiles > 4 ? 4 : 1);
  p.waves_per_item = waves;
  const size_t lds = waves > 1 ? sizeof(float) * (waves - 1) * (4 * DT + 2) * kWave : 0;
  const unsigned grid = waves > 1 ? p.items : (p.items + 3) / 4;
  hipLaunchKernelGGL((attend_query_kernel<T, DT>), dim3(grid),
                     dim3(kWave * (waves > 1 ? waves : 4)), lds, stream, p);
  return launch_status("routed_attention");
}

template <typename T>
hipError_t launch_type(Params& p, hipStream_t stream) {
  if (p.D <= 32) return launch_query<T, 2>(p, stream);
  if (p.D <= 64) return launch_query<T, 4>(p, stream);
  if (p.D <= 96) return launch_query<T, 6>(p, stream);
  if (p.D <= 128) return launch_query<T, 8>(p, stream);
  return launch_query<T, 16>(p, stream);
}

}  // namespace
}  // namespace rlm

using namespace rlm;

extern "C" hipError_t rlm_routed_attention(
    const rlm_tensor* query, const rlm_tensor* key_cache, const rlm_tensor* value_cache,
    const rlm_tensor* blocks, const rlm_tensor* positions, int64_t block_size,
    int64_t local_window, double scale, int32_t ring, const rlm_tensor* out,
    const rlm_tensor* out_lse, hipStream_t stream) {
  clear_error();
  RLM_TRY(check_strided(query, "query", 4));
  RLM_TRY(check_dtype_float(query, "query"));
  const int64_t B = query->shape[0], Tq = query->shape[1], Hq = query->shape[2],
                D = query->shape[3];
  RLM_REQUIRE(D >= 8 && D % 8 == 0 && D <= 256,
              "query: head dim must be a multiple of 8 in [8, 256], got %lld", (long long)D);
  RLM_TRY(check_strided(key_cache, "key_cache", 4));
  RLM_TRY(check_strided(value_cache, "value_cache", 4));
  const int64_t T = key_cache->shape[1], Hk = key_cache->shape[2];
  RLM_REQUIRE(Hk >= 1 && Hq % Hk == 0 && Hq >= 1,
              "query: %lld heads must be a positive multiple of the %lld key heads", (long long)Hq,
              (long long)Hk);
  for (const rlm_tensor* c : {key_cache, value_cache}) {
    const char* name = c == key_cache ? "key_cache" : "value_cache";
    RLM_TRY(check_same_dtype(c, name, query, "query"));
    RLM_TRY(check_dim(c, name, 0, B));
    RLM_TRY(check_dim(c, name, 1, T));
    RLM_TRY(check_dim(c, name, 2, Hk));
    RLM_TRY(check_dim(c, name, 3, D));
  }
  RLM_REQUIRE(block_size >= 1 && block_size <= (int64_t(1) << 24),
              "block_size must be in [1, 2^24], got %lld", (long long)block_size);
  RLM_REQUIRE(local_window >= 0 && local_window <= (int64_t(1) << 30),
              "local_window must be in [0, 2^30], got %lld", (long long)local_window);
  RLM_REQUIRE(T < (int64_t(1) << 31) - (int64_t(1) << 25),
              "caches: at most 2^31 - 2^25 rows, got %lld", (long long)T);
  RLM_REQUIRE(!ring || (T >= 1 && (T & (T - 1)) == 0 && T % block_size == 0),
              "ring-buffer caches need a power-of-two cache length split into whole blocks (cache "
              "length %lld, block_size %lld)",
              (long long)T, (long long)block_size);
  RLM_REQUIRE(blocks != nullptr && (blocks->ndim == 3 || blocks->ndim == 4),
              "blocks: expected [B,Tq,TOP] or [B,Tq,Hk,TOP]");
  RLM_TRY(check_strided(blocks, "blocks", blocks->ndim));
  RLM_TRY(check_dtype_is(blocks, "blocks", RLM_I32));
  RLM_TRY(check_dim(blocks, "blocks", 0, B));
  RLM_TRY(check_dim(blocks, "blocks", 1, Tq));
  if (blocks->ndim == 4) RLM_TRY(check_dim(blocks, "blocks", 2, Hk));
  const int64_t TOP = blocks->shape[blocks->ndim - 1];
  RLM_REQUIRE(TOP <= kMaxTop, "blocks: at most %d picks, got %lld", kMaxTop, (long long)TOP);
  Params p{};
  RLM_TRY(check_positions(positions, "positions", B, Tq, &p.pos_sb, &p.pos_sq));
  RLM_TRY(check_dense(out, "out", 4));
  RLM_TRY(check_same_dtype(out, "out", query, "query"));
  for (int i = 0; i < 4; ++i) RLM_TRY(check_dim(out, "out", i, query->shape[i]));
  RLM_TRY(check_dense(out_lse, "out_lse", 3));
  RLM_TRY(check_dtype_is(out_lse, "out_lse", RLM_F32));
  for (int i = 0; i < 3; ++i) RLM_TRY(check_dim(out_lse, "out_lse", i, query->shape[i]));
  for (const rlm_tensor* t : {query, key_cache, value_cache, out}) {
    bool aligned = (reinterpret_cast<uintptr_t>(t->data) & 15u) == 0;
    for (int i = 0; i < 3; ++i)
      aligned = aligned && (t->shape[i] <= 1 || t->stride[i] % 8 == 0);
    RLM_REQUIRE(aligned,
                "query, key_cache, value_cache and out must be 16-byte aligned with strides that "
                "are multiples of 8 elements");
  }
  p.q = query->data;
  p.q_sb = query->stride[0], p.q_st = query->stride[1], p.q_sh = query->stride[2];
  p.k = key_cache->data;
  p.k_sb = key_cache->stride[0], p.k_st = key_cache->stride[1], p.k_sh = key_cache->stride[2];
  p.v = value_cache->data;
  p.v_sb = value_cache->stride[0], p.v_st = value_cache->stride[1], p.v_sh = value_cache->stride[2];
  p.blocks = static_cast<const int32_t*>(blocks->data);
  p.blk_sb = blocks->stride[0], p.blk_st = blocks->stride[1];
  p.blk_sh = blocks->ndim == 4 ? blocks->stride[2] : 0;
  p.pos = positions->data;
  p.pos_dtype = positions->dtype;
  p.out = out->data;
  p.lse = static_cast<float*>(out_lse->data);
  p.T = T;
  p.BS = block_size;
  p.local_window = local_window;
  p.scale_log2 = static_cast<float>(scale) * kLog2e;
  p.Hq = static_cast<int>(Hq);
  p.Hk = static_cast<int>(Hk);
  p.G = static_cast<int>(Hq / Hk);
  p.D = static_cast<int>(D);
  p.TOP = static_cast<int>(TOP);
  p.ring = ring != 0;
  p.head_chunks = (p.G + 15) / 16;
  RLM_REQUIRE(B * Tq * Hk * p.head_chunks < (int64_t(1) << 31),
              "at most 2^31 - 1 (query, key head, 16 query heads) items");
  p.items = static_cast<uint32_t>(B * Tq * Hk * p.head_chunks);
  if (p.items == 0) return hipSuccess;
  p.B = static_cast<int>(B);
  p.Tq = static_cast<int>(Tq);
  p.by_chunks = FastDiv(static_cast<uint32_t>(p.head_chunks));
  p.by_kv = FastDiv(static_cast<uint32_t>(Hk));
  p.by_queries = FastDiv(static_cast<uint32_t>(Tq));
  p.by_block_tiles = FastDiv(static_cast<uint32_t>((block_size + 15) / 16));
  if (tile_fits(p, query->dtype)) return tile_launch(p, query->dtype, stream);
  switch (query->dtype) {
    case RLM_F32: return launch_type<float>(p, stream);
    case RLM_BF16: return launch_type<bf16>(p, stream);
    default: return launch_type<f16>(p, stream);
  }
}
