// Key tiles shared by the rows of a workgroup (rlm_attention_tile.hpp) over caches of the query's type.
#include "rlm_attention_tile.hpp"

namespace rlm {
namespace {

// Tiles and waves of a workgroup, by what was measured (us, 4 x 4096 queries of 12 heads on 4 of 64
// features / 8192 of 16 on 2 of 128; two tiles in LDS, with 128 registers to a lane):
//   keys x waves   64 x 8: 135 / 153   64 x 4: 115 / 277 (two workgroups per CU only)
//                  32 x 8:   - / 161   32 x 4: 124 / 131   32 x 2: 126 / 173
// Fewer waves share a tile's loads with fewer queries but wait for fewer of them: what counts is
// the number of workgroups on a CU (four).  One tile in LDS (seven fit) 120 / 144: registers
// still allow only four.  Three in LDS (two or three workgroups) 179 / 207.
// WHOLE by multiples of 64, the largest tile, whatever the instance's own.  Other blocks take the form
// that looks up the picks per 16 keys and spills registers above 96 features (bf16 and fp16 20, fp32 30;
// 5 at fp32 above 128).  Measured, as many keys in blocks of 64 / 32 / 16 (us, bf16): 4 x 4096 queries of 12
// heads on 4 of 64 features 115 / 164 / 181, 8192 of 16 on 2 of 128 121 / 160 / 230, of 96 - / 123 / -; fp32, 2
// x 4096 of 8 on 4 of 128 535 / 617 / -.  8 x 512 queries of 12 on 4 of 64, blocks of 32: 16.8.  Tiles of 32 keys
// would take blocks of 32 in the WHOLE form as well: 8192 queries 160 -> 119 (128 features), 123 -> 104
// (96), fp32 617 -> 514, 2 x 4096 of 8 on 2 of 256 173 -> 138; fp32 of 64 features 284 -> 275.
template <typename T, bool WHOLE>
hipError_t launch_type(TileParams& tp, hipStream_t stream) {
  constexpr int kSmall = sizeof(T) == 4 ? 32 : 64;
  const int dc = (tp.p.D + 31) / 32;
  if (dc <= 1) return launch_tiles<T, T, 1, WHOLE, 64, 4>(tp, stream);
  if (dc <= 2) return launch_tiles<T, T, 2, WHOLE, kSmall, 4>(tp, stream);
  if (dc <= 3) return launch_tiles<T, T, 3, WHOLE, 32, 4>(tp, stream);
  if (dc <= 4) return launch_tiles<T, T, 4, WHOLE, 32, 4>(tp, stream);
  return launch_tiles<T, T, 8, WHOLE, 32, 4>(tp, stream);
}

}  // namespace

namespace attention {

bool tile_fits(const Params& p, int dtype) {
  const int64_t limit =
      (int64_t(1) << 31) / (dtype_size(dtype) * kMostKeys) - 1;  // a tile below 2 GiB
  return !p.ring && p.Tq > 1 && p.T >= 1 && p.BS % 4 == 0 && p.k_st < limit && p.v_st < limit &&
         static_cast<int64_t>(p.B) * p.Hk * ((p.G + 15) / 16) * p.Tq < (int64_t(1) << 31);
}

// Whether the shared tiles are the faster kernel.  Both times (us) are modelled; measured, with
// picks half of which 64 neighbouring queries share (batch, key heads, group, dim, rows, block,
// window, picks; then queries: one query to a workgroup / shared tiles):
//   bf16  1,4,3,64,4096,64,128,8     64: 9.5 / 33    512: 29 / 41    1024: 52 / 40
//         1,2,8,128,8192,64,256,8    64: 13 / 55     512: 35 / 66    1024: 64 / 63
//         8,4,4,128,4096,64,128,8    16: 22 / 65      64: 59 / 64     128: 106 / 63
//         2,8,1,32,1024,16,32,8     256: 13 / 19     512: 20 / 16    1024: 34 / 12
//         4,8,2,64,16384,64,256,16   64: 53 / 110    128: 111 / 104   256: 213 / 110
//   fp32  1,4,3,64,4096,64,128,8    512: 73 / 149   1024: 137 / 141
//         8,4,4,128,4096,64,128,8    64: 255 / 263   128: 468 / 271   512: 1358 / 649
// One query: 8 us and its keys' products.  Tiles: a chain of the union of a workgroup's keys, which
// grows with about the root of its queries, a step of about 1.1 us (fp32: the slower matrix
// instructions) while the workgroups find room on the chip.
bool tile_faster(const Params& p, int dtype) {
  const bool is32 = dtype == RLM_F32;
  const double keys = static_cast<double>(std::min<int64_t>(p.T, p.local_window + p.TOP * p.BS));
  const double query = 8.0 + p.items * keys * p.D * (is32 ? 8.5e-7 : 2.7e-7);
  const int chunks = (p.G + kRows - 1) / kRows, heads = (p.G + chunks - 1) / chunks;
  const int queries = 4 * (kRows / heads);  // of a workgroup
  const double tile_keys = p.D <= 32 || (!is32 && p.D <= 64) ? 64.0 : 32.0;
  const double alone = keys / tile_keys + 1.0;
  const double steps =
      std::min(p.T / tile_keys + 1.0, alone * (1.0 + 0.45 * std::sqrt(static_cast<double>(queries))));
  const double step = is32 ? 2.2 * std::max(1.0, p.D / 64.0) : 1.1 * std::max(1.0, p.D / 128.0);
  const double groups = static_cast<double>(p.B) * p.Hk * chunks * ((p.Tq + queries - 1) / queries);
  return 5.0 + steps * step * std::max(1.0, groups / 820.0) < query;
}

hipError_t tile_launch(Params& p, int dtype, hipStream_t stream) {
  TileParams tp{};
  tp.p = p;
  tp.negate = p.scale_log2 < 0.0f;
  tp.far = dtype_size(dtype) * p.T * std::max(p.k_st, p.v_st) >= (int64_t(1) << 31) - 4096;
  // A scale of 0 as the smallest number: scores of 0 for the keys, -inf for the masked.
  tp.c = std::max(std::fabs(p.scale_log2), 1e-37f);
  const bool whole = p.BS % kMostKeys == 0;
#define RLM_TILE_TYPE(T) \
  return whole ? launch_type<T, true>(tp, stream) : launch_type<T, false>(tp, stream);
  if (dtype == RLM_F32) RLM_TILE_TYPE(float)
  if (dtype == RLM_BF16) RLM_TILE_TYPE(bf16)
  RLM_TILE_TYPE(f16)
#undef RLM_TILE_TYPE
}

}  // namespace attention
}  // namespace rlm
