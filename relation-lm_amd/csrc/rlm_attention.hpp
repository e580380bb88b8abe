// What the attention kernels share: the call's parameters and reductions over a lane's column.
#pragma once

#include "rlm_common.hpp"
#include "rlm_fastdiv.hpp"

namespace rlm {

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace attention {

constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct Params {
  const void *q, *k, *v;   // [B,Tq,Hq,D], [B,T,Hk,D] twice; unit stride in D
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  const float *ks, *vs;    // 8-bit caches: their rows' scales [B,T,Hk]
  int64_t ks_sb, ks_st, ks_sh, vs_sb, vs_st, vs_sh;
  const int32_t* blocks;   // [B,Tq,(Hk),TOP]
  int64_t blk_sb, blk_st, blk_sh;
  const void* pos;
  int pos_dtype;
  int64_t pos_sb, pos_sq;
  void* out;               // [B,Tq,Hq,D]
  float* lse;              // [B,Tq,Hq]
  int64_t T, BS, local_window;
  float scale_log2;        // scale * log2(e): scores are kept in powers of two
  int B, Tq, Hq, Hk, G, D, TOP;
  int head_chunks;         // of a key head's query heads, at most 16 each
  int heads_per_chunk;
  uint32_t items;          // B * Tq * Hk * head_chunks
  FastDiv by_chunks, by_kv, by_queries, by_block;
  bool ring;
};

// A query's position, within what its sums below hold in 64 bits (any negative one sees nothing).
__device__ __forceinline__ int64_t position_of(const Params& p, int64_t b, int64_t step) {
  const int64_t t = load_any_i(p.pos, p.pos_dtype, b * p.pos_sb + step * p.pos_sq);
  constexpr int64_t kMost = INT64_MAX - 1;
  return t < -1 ? -1 : t < kMost ? t : kMost;
}

__device__ __forceinline__ float rows_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float rows_sum(float v) { return swap32_sum(swap16_sum(v)); }

// One query to a workgroup (rlm_attention_query.hip).
hipError_t query_launch(const Params& p, int dtype, hipStream_t stream);
// The same over caches of 8 bits (rlm_attention_quantized.hip).
hipError_t quantized_launch(const Params& p, int dtype, hipStream_t stream);
// And shared tiles over them (rlm_attention_quantized_tile.hip), for workgroups of so many waves (two:
// of one's rows; 0: the kernel above is the faster one).
int quantized_tile_waves(const Params& p, int dtype);
hipError_t quantized_tile_launch(Params& p, int dtype, int waves, hipStream_t stream);
// Key tiles shared by the rows of a workgroup (rlm_attention_tile.hip).
bool tile_fits(const Params& p, int dtype);
bool tile_faster(const Params& p, int dtype);
hipError_t tile_launch(Params& p, int dtype, hipStream_t stream);

}  // namespace attention
}  // namespace rlm
