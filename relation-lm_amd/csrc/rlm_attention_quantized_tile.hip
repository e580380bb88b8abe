// Key tiles shared by the rows of a workgroup (rlm_attention_tile.hpp) over caches of 8 bits.
//
// Tiles of codes come by DMA as they are, with their rows' scales, a wave's keys' and another's values';
// keys are decoded as they are read from LDS, values by transposing 8-bit reads.  A query is a sum of bf16
// parts, the weights times their values' scales likewise (rlm_attention_quantized.hip says which).
//
// A wave spends about 400 vector instructions on 64 keys of 64 features, 64 of them on decoding and 48 on
// splitting the weights, for 24 products; a third of the weights are of keys that a row did not pick.
//
// Bound, many queries: these instructions.  4 x 4096 queries of 12 heads on 4 of 64 features (a window of
// 128, eight blocks of 64) take 167 to 172 us, in 69% of whose clocks vector instructions issue (matrix cores busy
// 20%), and 8000 of 16 on 2 of 128 (256, eight) 189 to 195; caches of 16 bits, with nothing to decode, take 110
// and 124.  Fewer: rounds of workgroups.  2 x 999 of the first kind, late in 8192 rows, are 1600 workgroups of
// two waves with 38 KB of LDS each, four to a CU: 6.25 to a CU are two rounds of about 26 us, 62 to 64 us with what
// surrounds them (a query to a workgroup 79).  Vector instructions issue in 35% of the clocks and matrix cores are
// busy in 10; 37% of the waves' life is waits for tiles and lists, 17% for their turn to issue.
#include "rlm_attention_tile.hpp"

namespace rlm {
namespace {

// Tiles of 64 keys up to 64 features, of 32 above.  Measured with 32 and one wave where 64 are taken: 76
// against 63 us, and with 64 where 32 are: 189 against 64 (2 x 999 queries of 12 heads on 4 of 64 and of
// 16 on 2 of 128 features).  A third and fourth tile under way bring nothing: what a wave does with a
// tile, about 400 instructions to 64 keys, hides the loads of the next.
// Two waves: the rows of one, whose tiles they share out.  One wave is never asked for up to 64 features
// (quantized_tile_waves), which is why it has no tiles of 64 keys.
template <typename T, bool WHOLE, int kWaves>
hipError_t launch_waves(TileParams& tp, hipStream_t stream) {
  constexpr int kRowWaves = kWaves == 2 ? 1 : kWaves, kShares = kWaves == 2 ? 2 : 1;
  const int dc = (tp.p.D + 31) / 32;
  if constexpr (kWaves != 1) {
    if (dc <= 1) return launch_tiles<T, code8, 1, WHOLE, 64, kRowWaves, kShares>(tp, stream);
    if (dc <= 2) return launch_tiles<T, code8, 2, WHOLE, 64, kRowWaves, kShares>(tp, stream);
  }
  if (dc <= 3) return launch_tiles<T, code8, 3, WHOLE, 32, kRowWaves, kShares>(tp, stream);
  if (dc <= 4) return launch_tiles<T, code8, 4, WHOLE, 32, kRowWaves, kShares>(tp, stream);
  return launch_tiles<T, code8, 8, WHOLE, 32, kRowWaves, kShares>(tp, stream);
}

template <typename T, bool WHOLE>
hipError_t launch_type(TileParams& tp, int waves, hipStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (waves == 4) return launch_waves<T, WHOLE, 4>(tp, stream);
  return waves == 2 ? launch_waves<T, WHOLE, 2>(tp, stream) : launch_waves<T, WHOLE, 1>(tp, stream);
}

bool fits(const Params& p) {
  const int64_t limit = (int64_t(1) << 31) / kMostKeys - 1;  // a tile, and its scales, below 2 GiB
  return !p.ring && p.Tq > 1 && p.T >= 1 && p.BS % 4 == 0 && p.k_st < limit && p.v_st < limit &&
         4 * p.ks_st < limit && 4 * p.vs_st < limit &&
         static_cast<int64_t>(p.B) * p.Hk * ((p.G + 15) / 16) * p.Tq < (int64_t(1) << 31);
}

}  // namespace

namespace attention {

// Shared tiles for workgroups of 4 waves (16-bit queries), of one, of two that share out one's tiles, or (0)
// a query to a workgroup: the fastest of these by modelled times (us).  Measured, with picks half of
// which 64 neighbouring queries share (batch, key heads, group, dim, rows, block, window, picks; then
// queries: one query / 4 waves / one / two):
//   bf16  2,4,3,64,8192,64,128,8    256: 25 / 78 / 49 / 30    512: 45 / 78 / 49 / 33    999: 79 / 90 / 63 / 62
//                                  2000: 145 / 111 / 110 / 96    4000: 279 / 168 / 173 / 170
//         1,2,8,128,8192,64,256,8   512: 24 / 100 / 53 / 33  2000: 74 / 110 / 65 / 73  4000: 132 / 125 / 135 / 126
//         4,4,3,64,4096,64,128,8   4096: 504 / 166 / 211 / 236
//         2,8,1,32,1024,16,32,8    1000: 35 / 26 / 25 / 17
//         2,4,2,96,4096,16,100,8   1000: 49 / 78 / 63 / 37
//         2,4,3,64,8192,8,64,8     1500: 30 / 137 / 124 / 104
//   fp32  2,4,3,64,8192,64,128,8    256: 29 / - / - / 36    999: 93 / 113 / 76 / 75    4000: 329 / 239 / 206 / 207
//         1,2,8,128,8192,64,256,8   512: 35 / 104 / 56 / 41  2000: 99 / 125 / 78 / 91   4000: 171 / 206 / 150 / 160
// One query: its keys' products.  Tiles: a chain of the union of a workgroup's keys, which grows with
// about the root of its queries, while the workgroups find room on the chip; sharing it out helps while
// there are few, beyond 64 features only then.
int quantized_tile_waves(const Params& p, int dtype) {
  if (!fits(p)) return 0;
  const bool is32 = dtype == RLM_F32;
  const double keys = static_cast<double>(std::min<int64_t>(p.T, p.local_window + p.TOP * p.BS));
  const double query = 8.0 + p.items * keys * (6e-6 + 1.2e-7 * p.D) * (is32 ? 1.4 : 1.0);
  const int chunks = (p.G + kRows - 1) / kRows, heads = (p.G + chunks - 1) / chunks;
  const double tile_keys = p.D <= 64 ? 64.0 : 32.0;
  const double alone = std::min(p.T / tile_keys + 1.0,
                                p.local_window / tile_keys + 1.0 + p.TOP * std::max(1.0, p.BS / tile_keys));
  const double step = tile_keys * (0.009 + 2.3e-4 * p.D) * (is32 ? 1.2 : 1.0) *
                      (p.BS % kMostKeys == 0 ? 1.0 : 1.5);
  // `least`: of a chain, however few the workgroups are.
  auto groups = [&](int queries) {
    return static_cast<double>(p.B) * p.Hk * chunks * ((p.Tq + queries - 1) / queries);
  };
  auto tiles = [&](int waves, double cost, double room, double least) {
    const int queries = waves * (kRows / heads);  // of a workgroup
    const double steps =
        std::min(p.T / tile_keys + 1.0, alone * (1.0 + 0.45 * std::sqrt(static_cast<double>(queries))));
    return 5.0 + steps * step * cost * std::max(least, groups(queries) / room);
  };
  const bool split = p.D <= 64 || groups(kRows / heads) <= 1200.0;
  const double one = split ? tiles(1, 1.0, 1300.0, 0.65) : tiles(1, 1.0, 1400.0, 1.0);
  const double four = is32 ? one : tiles(4, 1.6, 1000.0, 1.0);
  if (query <= std::min(one, four)) return 0;
  return one > four ? 4 : split ? 2 : 1;
}

hipError_t quantized_tile_launch(Params& p, int dtype, int waves, hipStream_t stream) {
  TileParams tp{};
  tp.p = p;
  tp.negate = p.scale_log2 < 0.0f;
  tp.far = p.T * std::max(p.k_st, p.v_st) >= (int64_t(1) << 31) - 4096;
  // A scale of 0 as the smallest number: scores of 0 for the keys, -inf for the masked.
  tp.c = std::max(std::fabs(p.scale_log2), 1e-37f);
  // (Instances of 32-key tiles would hold blocks that are multiples of 32 as whole ones.)
  const bool whole = p.BS % kMostKeys == 0;
#define RLM_TILE_TYPE(T)                                \
  return whole ? launch_type<T, true>(tp, waves, stream) \
               : launch_type<T, false>(tp, waves, stream);
  if (dtype == RLM_F32) RLM_TILE_TYPE(float)
  if (dtype == RLM_BF16) RLM_TILE_TYPE(bf16)
  RLM_TILE_TYPE(f16)
#undef RLM_TILE_TYPE
}

}  // namespace attention
}  // namespace rlm
