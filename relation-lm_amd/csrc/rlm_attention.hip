// Attention of each query over its local window and the blocks picked for it.
//
// A query at position t with window L and picks j_1 .. j_TOP attends to the positions
//   [t - L + 1, t]  and, before them,  [j BS, j BS + BS) of every pick
// that the cache holds (linear: p < T; ring: p > t - T, position p in row p mod T):
//   out = sum_p softmax_p(scale q . k_p) v_p,   lse = log sum_p exp(scale q . k_p).
// Caches of 8 bits hold codes and a scale for each row of a key head: k_p = key_scale_p code_p.
// A position counts once whichever way it is named; a query that sees none gives 0 and -inf.
#include "rlm_attention.hpp"

namespace rlm {
namespace {

using namespace attention;

// Checks a call's descriptors and fills its parameters; key_scale and value_scale come with caches
// of 8 bits.
hipError_t fill(const rlm_tensor* query, const rlm_tensor* key_cache, const rlm_tensor* value_cache,
                const rlm_tensor* key_scale, const rlm_tensor* value_scale, bool quantized,
                const rlm_tensor* blocks, const rlm_tensor* positions, int64_t block_size,
                int64_t local_window, double scale, int32_t ring, const rlm_tensor* out,
                const rlm_tensor* out_lse, Params& p) {
  RLM_TRY(check_strided(query, "query", 4));
  RLM_TRY(check_dtype_float(query, "query"));
  const int64_t B = query->shape[0], Tq = query->shape[1], Hq = query->shape[2],
                D = query->shape[3];
  const int unit = quantized ? 16 : 8;  // features of a 16-byte access
  RLM_REQUIRE(D >= unit && D % unit == 0 && D <= 256,
              "query: head dim must be a multiple of %d in [%d, 256], got %lld", unit, unit,
              (long long)D);
  RLM_TRY(check_strided(key_cache, "key_cache", 4));
  RLM_TRY(check_strided(value_cache, "value_cache", 4));
  const int64_t T = key_cache->shape[1], Hk = key_cache->shape[2];
  RLM_REQUIRE(Hk >= 1 && Hq % Hk == 0 && Hq >= 1,
              "query: %lld heads must be a positive multiple of the %lld key heads", (long long)Hq,
              (long long)Hk);
  for (const rlm_tensor* c : {key_cache, value_cache}) {
    const char* name = c == key_cache ? "key_cache" : "value_cache";
    if (quantized)
      RLM_TRY(check_dtype_is(c, name, RLM_F8E4M3));
    else
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
  RLM_TRY(check_positions(positions, "positions", B, Tq, &p.pos_sb, &p.pos_sq));
  RLM_TRY(check_dense(out, "out", 4));
  RLM_TRY(check_same_dtype(out, "out", query, "query"));
  for (int i = 0; i < 4; ++i) RLM_TRY(check_dim(out, "out", i, query->shape[i]));
  RLM_TRY(check_dense(out_lse, "out_lse", 3));
  RLM_TRY(check_dtype_is(out_lse, "out_lse", RLM_F32));
  for (int i = 0; i < 3; ++i) RLM_TRY(check_dim(out_lse, "out_lse", i, query->shape[i]));
  for (const rlm_tensor* t : {query, key_cache, value_cache, out}) {
    const int64_t step = t->dtype == RLM_F8E4M3 ? 16 : 8;
    bool aligned = (reinterpret_cast<uintptr_t>(t->data) & 15u) == 0;
    for (int i = 0; i < 3; ++i)
      aligned = aligned && (t->shape[i] <= 1 || t->stride[i] % step == 0);
    RLM_REQUIRE(aligned,
                "query, key_cache, value_cache and out must be 16-byte aligned with strides that "
                "are multiples of 8 elements (8-bit caches: 16)");
  }
  if (quantized) {
    RLM_TRY(check_scales(key_scale, "key_scale", B, T, Hk));
    RLM_TRY(check_scales(value_scale, "value_scale", B, T, Hk));
    p.ks = static_cast<const float*>(key_scale->data);
    p.ks_sb = key_scale->stride[0], p.ks_st = key_scale->stride[1], p.ks_sh = key_scale->stride[2];
    p.vs = static_cast<const float*>(value_scale->data);
    p.vs_sb = value_scale->stride[0], p.vs_st = value_scale->stride[1],
    p.vs_sh = value_scale->stride[2];
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
  p.heads_per_chunk = (p.G + p.head_chunks - 1) / p.head_chunks;
  RLM_REQUIRE(B * Tq * Hk * p.head_chunks < (int64_t(1) << 31),
              "at most 2^31 - 1 (query, key head, 16 query heads) items");
  p.items = static_cast<uint32_t>(B * Tq * Hk * p.head_chunks);
  if (p.items == 0) return hipSuccess;
  p.B = static_cast<int>(B);
  p.Tq = static_cast<int>(Tq);
  p.by_chunks = FastDiv(static_cast<uint32_t>(p.head_chunks));
  p.by_kv = FastDiv(static_cast<uint32_t>(Hk));
  p.by_queries = FastDiv(static_cast<uint32_t>(Tq));
  p.by_block = FastDiv(static_cast<uint32_t>(block_size));
  return hipSuccess;
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
  Params p{};
  const hipError_t e = fill(query, key_cache, value_cache, nullptr, nullptr, false, blocks,
                            positions, block_size, local_window, scale, ring, out, out_lse, p);
  if (e != hipSuccess || p.items == 0) return e;
  return tile_fits(p, query->dtype) && tile_faster(p, query->dtype)
             ? tile_launch(p, query->dtype, stream)
             : query_launch(p, query->dtype, stream);
}

extern "C" hipError_t rlm_routed_attention_quantized(
    const rlm_tensor* query, const rlm_tensor* key_cache, const rlm_tensor* value_cache,
    const rlm_tensor* key_scale, const rlm_tensor* value_scale, const rlm_tensor* blocks,
    const rlm_tensor* positions, int64_t block_size, int64_t local_window, double scale,
    int32_t ring, const rlm_tensor* out, const rlm_tensor* out_lse, hipStream_t stream) {
  clear_error();
  Params p{};
  const hipError_t e =
      fill(query, key_cache, value_cache, key_scale, value_scale, true, blocks, positions,
           block_size, local_window, scale, ring, out, out_lse, p);
  if (e != hipSuccess || p.items == 0) return e;
  const int waves = quantized_tile_waves(p, query->dtype);
  return waves != 0 ? quantized_tile_launch(p, query->dtype, waves, stream)
                    : quantized_launch(p, query->dtype, stream);
}
