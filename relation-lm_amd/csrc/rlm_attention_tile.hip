// Attention over a window and picked blocks for many queries: key tiles shared by the rows of a
// workgroup.
//
// A workgroup holds 4 waves of 16 rows, a row being one query head of one query; the rows of a
// wave are whole queries with the heads of one key head, consecutive positions of the sequence.
// It walks the tiles of 64 or 32 keys that any of its queries sees -- its windows' and its picked
// blocks' union, found from the picks in LDS -- and every wave takes part in those that its own
// queries see.  Neighbouring queries share their windows and much of their picks, so a
// tile is read once for all of them; a query's own picks decide only which of its scores count.
//
// Tiles come by DMA (buffer_load ... lds), the next one in flight while one is worked on.  With
// keys as rows and query rows as columns of v_mfma_f32_16x16x32:
//   S^T[key, row]: lane (row = l % 16, keys 16 kt + 4 (l / 16) + i) -- scores of one row, so
//     the softmax needs two lane exchanges for its maximum and none for its weights;
//   O^T[dim, row] += V^T P^T over 32 keys whose order is free: a lane's eight weights of two
//     16-key groups are its operand as they stand, and V^T's operand is two transposing reads
//     (ds_read_b64_tr_b16) of four keys each from the row-major tile.
// LDS rows are swizzled in 16-byte pieces, which spreads the key reads over all banks.  A third of
// the LDS cycles (4 x 4096 queries) still count as conflicts; an exchange that gives the transposing
// reads columns of their own too left that count and the time as they were.
//
// Bound: waits.  4 x 4096 queries of 12 heads on 4 of 64 features (a window of 128, eight blocks of
// 64) take 110 us and 8192 of 16 on 2 of 128 (256, eight) 124 us: 260 and 400 TFLOP/s over the keys
// that each query sees (567 and 730 on average).  A wave's rows see about twice the tiles that one query does, and a
// workgroup's 1.4 times those of a wave; the waves spend half their life at the loads' wait and the
// barrier of each tile, with VALU issuing 61% and the matrix cores busy 24% of the time.  Taking a
// tenth of the VALU instructions out left the time as it was.
//
// The weights are rounded to the 16-bit type for the second product, which takes no other operands
// (half a step, relative to each weight: the measured outputs are 0.0021 off in bf16, where weights of
// 32 bits would leave the output's own rounding, 0.0016); scores, maxima, sums and outputs stay fp32.
//
// A masked key's weight is 0, which is no protection from what its value row holds if that is
// an infinity or NaN (0 x inf): a row whose sums are not finite at the end is computed again,
// position by position, from the rows that it sees alone.
#include <type_traits>

#include "rlm_attention.hpp"
#include "rlm_attention_mfma.hpp"

namespace rlm {
namespace {

using namespace attention;

constexpr int kRows = 16;           // rows of a wave
constexpr int kMostKeys = 64;       // keys of the largest tile
constexpr int kWindowTiles = 256;   // tiles (and blocks) looked at at once
// Sum of a lane's weights of a row in one tile beyond which its base is raised: fp16 weights stay far
// inside the type, and the outputs' rescaling is rare.
constexpr float kLimit = 4096.0f;

struct TileParams {
  Params p;
  int hg;                // heads of a wave's query (a chunk of the group)
  int chunks;            // chunks of a group
  int nqw;               // queries of a wave
  uint32_t pairs;        // (batch row, key head, chunk)
  uint32_t tiles;        // workgroups along the sequence
  FastDiv by_pairs, by_chunks, by_kv, by_heads, by_block, by_picks, by_wave_queries;
  float c;               // |scale| log2(e), above 0
  bool negate;
  bool far;              // rows of a key head reach over 2 GiB: offsets from each tile's first
};

// A workgroup barrier that orders LDS reads and leaves loads into LDS outstanding.
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// One row from the positions that it sees alone, a position at a time: lanes hold features.
template <typename T>
__device__ void attend_row_alone(const Params& p, int64_t b, int64_t step, int64_t hk, int64_t head,
                                 float scale_log2) {
  const int lane = threadIdx.x & (kWave - 1);
  const T* q = static_cast<const T*>(p.q) + b * p.q_sb + step * p.q_st + head * p.q_sh;
  const T* kbase = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vbase = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  const int32_t* picks = p.blocks + b * p.blk_sb + step * p.blk_st + hk * p.blk_sh;
  const int32_t mine = lane < p.TOP ? picks[lane] : -1;
  const int64_t t = position_of(p, b, step);
  const int64_t high = t + 1 < p.T ? t + 1 : p.T;
  int64_t start = t - p.local_window + 1;
  start = start > 0 ? start : 0;
  float qf[4], acc[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + kWave * i;
    qf[i] = d < p.D ? to_f32(q[d]) : 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int run = -1; run < p.TOP; ++run) {
    int64_t first = start, end = high;
    if (run >= 0) {
      const int32_t block = __builtin_amdgcn_readlane(mine, run);
      const uint64_t same = __builtin_amdgcn_ballot_w64(mine == block);
      if (block < 0 || (same & ((uint64_t(1) << run) - 1)) != 0) continue;
      first = block * p.BS;
      end = first + p.BS < start ? first + p.BS : start;
      end = end < high ? end : high;
    }
    for (int64_t at = first; at < end; ++at) {
      float s = 0.0f, v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = lane + kWave * i;
        v[i] = d < p.D ? to_f32(vbase[at * p.v_st + d]) : 0.0f;
        if (d < p.D) s = fmaf(qf[i], to_f32(kbase[at * p.k_st + d]), s);
      }
      s = wave_sum_f32(s) * scale_log2;
      const float top = fmaxf(m, s), base = top == -INFINITY ? 0.0f : top;
      const float fade = __builtin_amdgcn_exp2f(m - base);
      const float w = __builtin_amdgcn_exp2f(s - base);
      m = top;
      l = fmaf(l, fade, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(acc[i], fade, w * v[i]);
    }
  }
  const int64_t row = (b * p.Tq + step) * p.Hq + head;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(p.out) + row * p.D;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + kWave * i;
    if (d < p.D) out[d] = from_f32<T>(acc[i] * inv);
  }
  if (lane == 0)
    p.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// DC: head dim in 32s, WHOLE: a tile lies within one block; tiles of kKeys keys for kWaves waves,
// two of them in LDS.
template <typename T, int DC, bool WHOLE, int kKeys, int kWaves>
__global__ __launch_bounds__(kWaves* kWave, DC <= 4 ? 4 : 2) void attend_tile_kernel(TileParams tp) {
  constexpr int kThreads = kWaves * kWave;
  constexpr int KT = kKeys / 16;                           // 16-key groups of a tile
  constexpr bool k32 = sizeof(T) == 4;
  constexpr int kPitch = pitch<T, DC>();                   // 16-byte pieces of an LDS row
  constexpr int kRow = 16 * kPitch;                        // bytes
  constexpr int kTile = kKeys * kRow;                      // bytes of a key (or value) tile
  constexpr int kDma = kPitch * kKeys / kThreads;          // DMA instructions of a wave per tile
  constexpr int DT = 2 * DC;                               // head dim in 16s
  constexpr int kWords = kWaves / 2;                       // 16 queries of a wave: half a word
  extern __shared__ __align__(1024) char lds[];            // [2][key tile, value tile]
  __shared__ __align__(16) uint32_t sel[(kWindowTiles + 2) * kWords];  // [block]: who picked it
  __shared__ __align__(16) uint32_t act[kWindowTiles * kWords];        // [tile]: who sees it
  __shared__ int32_t s_high[kWaves * kRows], s_start[kWaves * kRows];
  __shared__ uint16_t list[kWindowTiles];
  __shared__ int32_t s_count, s_last;

  const Params& p = tp.p;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, quad = lane >> 4;
  // The longest sequences' ends first; a (batch row, key head)'s workgroups stay on one XCD
  // (or a few) where their number and the XCDs' divide each other.
  uint32_t pair, chunk, hk;
  const uint32_t tile = tp.tiles - 1 - tp.by_pairs.div(blockIdx.x, pair);
  const int64_t b = tp.by_kv.div(tp.by_chunks.div(pair, chunk), hk);
  const int queries = kWaves * tp.nqw;
  const int q0 = static_cast<int>(tile) * queries;

  const T* kbase = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vbase = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;

  // Positions: query i of the workgroup sees [.., high) and its window starts at `start`.
  if (threadIdx.x == 0) s_last = 0;
  __syncthreads();
  if (threadIdx.x < queries) {
    const int q = q0 + threadIdx.x;
    int32_t high = 0, start = 0;
    if (q < p.Tq) {
      const int64_t t = position_of(p, b, q);
      int64_t s = t - p.local_window + 1;
      s = s > 0 ? s : 0;
      high = static_cast<int32_t>(t < 0 ? 0 : t + 1 < p.T ? t + 1 : p.T);
      start = static_cast<int32_t>(s < high ? s : high);
    }
    s_high[threadIdx.x] = high;
    s_start[threadIdx.x] = start;
    atomicMax(&s_last, high);
  }

  // This lane's row.
  uint32_t in_query;
  const uint32_t in_wave = tp.by_heads.div(r, in_query);
  const int q = q0 + wave * tp.nqw + static_cast<int>(in_wave);
  const int h = static_cast<int>(chunk) * tp.hg + static_cast<int>(in_query);
  const bool row_ok = in_wave < static_cast<uint32_t>(tp.nqw) && q < p.Tq && h < p.G;
  const int head = static_cast<int>(hk) * p.G + (row_ok ? h : 0);
  const int step = row_ok ? q : 0;
  const int bit = (row_ok ? static_cast<int>(in_wave) : 0) + 16 * (wave & 1);
  typedef typename std::conditional<k32, float4, s16x8>::type frag_t;
  constexpr int kFrags = k32 ? DT : DC;     // 16-byte pieces of a row that a lane has,
  constexpr int kFeatures = k32 ? 4 : 8;    // of so many features: pieces 4 j + quad
  frag_t qf[kFrags];
  {
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + step * p.q_st + head * p.q_sh;
    const uint32_t flip = !tp.negate ? 0u : k32 ? 0x80000000u : 0x80008000u;
#pragma unroll
    for (int j = 0; j < kFrags; ++j) {
      const int d = kFeatures * (4 * j + quad);
      uint4 x = *reinterpret_cast<const uint4*>(src + (d < p.D ? d : 0));
      x = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
      if (!(d < p.D && row_ok)) x = make_uint4(0, 0, 0, 0);
      qf[j] = __builtin_bit_cast(frag_t, x);
    }
  }
  __syncthreads();
  const int32_t high = row_ok ? s_high[wave * tp.nqw + (bit & 15)] : 0;
  const int32_t start = row_ok ? s_start[wave * tp.nqw + (bit & 15)] : 0;
  const int32_t last = __builtin_amdgcn_readfirstlane(s_last);
  // Tiles that end at `remote` or before lie before every window of the wave's rows: their keys
  // are seen by the picks alone, whole blocks at a time.
  int32_t remote = high > 0 ? start : 0x7fffffff;
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) remote = min(remote, __shfl_xor(remote, off, kWave));
  remote = __builtin_amdgcn_readfirstlane(remote);

  f32x4 acc[DT];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int j = 0; j < DT; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // This lane's pieces of a tile: row and byte in the row, which the swizzle permutes; pieces
  // past the head dim come as zeros.
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const uint32_t k_bytes = static_cast<uint32_t>(p.k_st * sizeof(T));
  const uint32_t v_bytes = static_cast<uint32_t>(p.v_st * sizeof(T));
  uint32_t k_off[kDma], v_off[kDma];
  auto dma_row = [&](int k) {
    return static_cast<uint32_t>(((wave * kDma + k) * kWave + lane) / kPitch);
  };
#pragma unroll
  for (int k = 0; k < kDma; ++k) {
    const uint32_t row = dma_row(k);
    const int from = (lane % kPitch) ^ swizzle<kPitch>(row);
    const bool ok = kFeatures * from < p.D;
    k_off[k] = ok ? row * k_bytes + 16u * from : kNoOffset;
    v_off[k] = ok ? row * v_bytes + 16u * from : kNoOffset;
  }
  const rsrc_t k_rows = make_rsrc(kbase, 0x7ffffff0u), v_rows = make_rsrc(vbase, 0x7ffffff0u);
  auto issue = [&](int buffer, int32_t first) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + buffer * 2 * kTile + wave * kDma * 1024);
    // Rows past the last that a query of the workgroup sees (their keys are masked, and they may
    // hold anything) read that one.
    const uint32_t rows = static_cast<uint32_t>(last - 1 - first);
    if (!tp.far && rows >= kKeys - 1) {
      const uint32_t ks = first * k_bytes, vs = first * v_bytes;
#pragma unroll
      for (int k = 0; k < kDma; ++k) lds_dma16(k_rows, to + 1024u * k, k_off[k], ks);
#pragma unroll
      for (int k = 0; k < kDma; ++k) lds_dma16(v_rows, to + kTile + 1024u * k, v_off[k], vs);
    } else {
      const rsrc_t kr = make_rsrc(kbase + first * p.k_st, 0x7ffffff0u);
      const rsrc_t vr = make_rsrc(vbase + first * p.v_st, 0x7ffffff0u);
#pragma unroll
      for (int k = 0; k < kDma; ++k) {
        const uint32_t row = dma_row(k), over = row > rows ? row - rows : 0;
        const uint32_t ko = k_off[k] - over * k_bytes, vo = v_off[k] - over * v_bytes;
        lds_dma16(kr, to + 1024u * k, k_off[k] == kNoOffset ? kNoOffset : ko);
        lds_dma16(vr, to + kTile + 1024u * k, v_off[k] == kNoOffset ? kNoOffset : vo);
      }
    }
  };

  // Windows of the cache: as many keys as kWindowTiles tiles or blocks hold.
  const int32_t span = kKeys * static_cast<int32_t>(
      min(static_cast<int64_t>(kWindowTiles), max(static_cast<int64_t>(1), kWindowTiles * p.BS / kKeys)));
  for (int32_t w0 = 0; w0 < last; w0 += span) {
    const int32_t w1 = min(w0 + span, last);
    const int32_t block0 = static_cast<int32_t>(tp.by_block.div(w0));
    const int window_tiles = (w1 - w0 + kKeys - 1) / kKeys;
    // What the queries see in this window.
    for (int i = threadIdx.x; i < (kWindowTiles + 2) * kWords; i += kThreads) sel[i] = 0;
    for (int i = threadIdx.x; i < window_tiles * kWords; i += kThreads) act[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < queries * (p.TOP + 1); i += kThreads) {
      uint32_t pick;
      const int query = static_cast<int>(tp.by_picks.div(i, pick));
      if (q0 + query >= p.Tq) continue;
      uint32_t place;
      const uint32_t of = tp.by_wave_queries.div(query, place);
      const uint32_t mine = 1u << (place + 16 * (of & 1));
      int32_t first = s_start[query], end = s_high[query];
      const bool window = pick == static_cast<uint32_t>(p.TOP);
      if (!window) {
        const int32_t block = p.blocks[b * p.blk_sb + static_cast<int64_t>(q0 + query) * p.blk_st +
                                       hk * p.blk_sh + pick];
        const int64_t at = static_cast<int64_t>(block) * p.BS;
        if (block < 0 || at >= min(first, w1) || at + p.BS <= w0) continue;
        if (!WHOLE) atomicOr(&sel[(block - block0) * kWords + of / 2], mine);
        end = static_cast<int32_t>(min(at + p.BS, static_cast<int64_t>(first)));
        first = static_cast<int32_t>(at);
      }
      first = max(first, w0);
      end = min(end, w1);
      for (int32_t t = (first - w0) / kKeys; w0 + t * kKeys < end; ++t) {
        if (first < end) {
          atomicOr(&act[t * kWords + of / 2], mine);
          if (WHOLE && !window) atomicOr(&sel[t * kWords + of / 2], mine);
        }
      }
    }
    __syncthreads();
    if (wave == 0) {
      int count = 0;
      for (int i = 0; i < window_tiles; i += kWave) {
        const int t = i + lane;
        bool any = false;
        if (t < window_tiles) {
          uint32_t a = 0;
#pragma unroll
          for (int w = 0; w < kWords; ++w) a |= act[t * kWords + w];
          any = a != 0;
        }
        const uint64_t mask = __builtin_amdgcn_ballot_w64(any);
        if (any) list[count + __builtin_popcountll(mask & ((uint64_t(1) << lane) - 1))] = t;
        count += __builtin_popcountll(mask);
      }
      if (lane == 0) s_count = count;
    }
    __syncthreads();
    const int count = __builtin_amdgcn_readfirstlane(s_count);
    if (count == 0) continue;
    // Lane i holds the list's entry i of the current 64, and what the wave's queries see of it.
    const int word = wave / 2;
    const uint32_t own = 0xffffu << (16 * (wave & 1));
    int entry = list[min(lane, count - 1)];
    uint32_t seen = act[entry * kWords + word] & own;
    auto tile_of = [&](int i) {
      if ((i & (kWave - 1)) == 0 && i != 0) {
        entry = list[min(i + lane, count - 1)];
        seen = act[entry * kWords + word] & own;
      }
      return __builtin_amdgcn_readlane(entry, i & (kWave - 1));
    };
    // Tile n of the list is in LDS half n mod 2; the next one is on its way while it is worked on.
    int next = tile_of(0);
    uint32_t next_see = __builtin_amdgcn_readlane(seen, 0);
    issue(0, w0 + kKeys * next);
    for (int n = 0; n < count; ++n) {
      const int t = next;
      const uint32_t see = next_see;
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      barrier();  // tile n is in LDS for every wave, tile n - 1 has been read by every wave
      if (n + 1 < count) {
        next = tile_of(n + 1);
        next_see = __builtin_amdgcn_readlane(seen, (n + 1) & (kWave - 1));
        issue((n + 1) & 1, w0 + kKeys * next);
      }
      const uint32_t tile0 = lds0 + (n & 1) * 2 * kTile;
      if (see == 0) continue;
      const int32_t p0 = w0 + t * kKeys;
      const bool near = p0 + kKeys > remote;
      // A lane's first piece of the key and of the value rows that it reads; the swizzle makes
      // later ones an exclusive or away (pieces 4 j + quad of the keys, 2 j + (0 or 1) of the
      // values).
      const uint32_t key0 = tile0 + r * kRow + ((quad ^ swizzle<kPitch>(r)) << 4);
      // Whether the row picked the block of this lane's four keys of 16-key group kt.
      constexpr int kPicked = WHOLE ? 1 : KT;
      bool pick[kPicked];
#pragma unroll
      for (int kt = 0; kt < kPicked; ++kt) {
        const uint32_t who =
            WHOLE ? sel[t * kWords + word]
                  : sel[(tp.by_block.div(p0 + 16 * kt + 4 * quad) - block0) * kWords + word];
        pick[kt] = row_ok & (((who >> bit) & 1) != 0);
      }

      // S^T = K Q^T.
      f32x4 s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        s[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
          const s16x8 kf = *(lds_s16x8)static_cast<uintptr_t>((key0 ^ (64u * j)) + 16 * kt * kRow);
          s[kt] = product(__builtin_bit_cast(frag_t, kf), qf[j], s[kt], T{});
        }
      }
      // 16-bit values: step i of the second product is 32-key half i / DT and feature group
      // i % DT; the first steps' operands come while the weights are computed.
      constexpr int kAhead = 4, kSteps = DT * KT / 2;
      const int vrow = 4 * quad + (r >> 2);
      const uint32_t value0 = tile0 + kTile + vrow * kRow +
                              ((((r & 3) >> 1) ^ swizzle<kPitch>(vrow)) << 4) + (r & 1) * 8;
      auto values = [&](int i) {
        return read_values((value0 ^ (32u * (i % DT))) + i / DT * 32 * kRow, 16 * kRow);
      };
      s16x8 vf[kAhead];
      if constexpr (!k32) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (i < kSteps) vf[i] = values(i);
      }
      __builtin_amdgcn_sched_barrier(0);

      // The weights, as the second product's operand: two 16-key groups to each.
      if (near) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int32_t at = p0 + 16 * kt + 4 * quad;
          const int32_t from = pick[WHOLE ? 0 : kt] ? 0 : start - at;
          const int32_t to = high - at;
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kt][i] = ((i >= from) & (i < to)) ? s[kt][i] : -INFINITY;
        }
      }
      // A row's base m is the maximum of its first tile; past the limit it is raised to a later
      // tile's, where the weights give a lane at most 16.
      bool up = __builtin_amdgcn_ballot_w64((m == -INFINITY) & (((see >> bit) & 1) != 0) &
                                            row_ok) != 0;
      uint4 weights[KT / 2];
      float w32[k32 ? KT : 1][4];
      for (int pass = 0;; ++pass) {
        if (up) {
          float top = -INFINITY;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            float x = fmaxf(fmaxf(s[kt][0], s[kt][1]), fmaxf(s[kt][2], s[kt][3]));
            asm("" : "+v"(x));  // keeps these maxima in this rare branch
            top = (near | pick[WHOLE ? 0 : kt]) ? fmaxf(top, x) : top;
          }
          const float more = fmaxf(m, rows_max(top) * tp.c);
          const float fade = __builtin_amdgcn_exp2f(m - (more == -INFINITY ? 0.0f : more));
          m = more;
          l *= fade;
#pragma unroll
          for (int j = 0; j < DT; ++j) acc[j] *= fade;
        }
        const float base = m == -INFINITY ? 0.0f : -m;
        uint32_t half[2 * KT];
        float sum[4];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const float shift = (near | pick[WHOLE ? 0 : kt]) ? base : -INFINITY;
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], tp.c, shift));
            sum[i] = kt == 0 ? w[i] : sum[i] + w[i];
            if constexpr (k32) w32[kt][i] = w[i];
          }
          if constexpr (!k32) {
            half[2 * kt] = pack2(w[0], w[1], T{});
            half[2 * kt + 1] = pack2(w[2], w[3], T{});
          }
        }
        if constexpr (!k32) {
#pragma unroll
          for (int i = 0; i < KT / 2; ++i)
            weights[i] = make_uint4(half[4 * i], half[4 * i + 1], half[4 * i + 2], half[4 * i + 3]);
        }
        const float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        up = pass == 0 && __builtin_amdgcn_ballot_w64(total > kLimit) != 0;
        if (!up) {
          l += total;
          break;
        }
      }

      // O^T += V^T P^T.
      if constexpr (k32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = 4 * quad + i;  // of each 16-key group; feature 16 j + r
          const uint32_t at = tile0 + kTile + key * kRow + (((r >> 2) ^ swizzle<kPitch>(key)) << 4) +
                              (r & 3) * 4;
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
              const float v = *(lds_f32)static_cast<uintptr_t>((at ^ (64u * j)) + 16 * kt * kRow);
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, w32[kt][i], acc[j], 0, 0, 0);
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          acc[i % DT] = product(vf[i % kAhead], __builtin_bit_cast(s16x8, weights[i / DT]),
                                acc[i % DT], T{});
          if (i + kAhead < kSteps) vf[i % kAhead] = values(i + kAhead);
        }
      }
    }
    __syncthreads();  // the lists and tiles have been read
  }

  const float total = rows_sum(l);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  bool fine = fabsf(total) < INFINITY;
#pragma unroll
  for (int j = 0; j < DT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) fine = fine & (fabsf(acc[j][i]) < INFINITY);
  const uint64_t bad = __builtin_amdgcn_ballot_w64(!fine && row_ok);
  if (row_ok) {
    const int64_t row = (b * p.Tq + step) * p.Hq + head;
    T* out = static_cast<T*>(p.out) + row * p.D;
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      const int d = 16 * j + 4 * quad;
      if (d < p.D)
        put4<T>(out + d, acc[j][0] * inv, acc[j][1] * inv, acc[j][2] * inv, acc[j][3] * inv);
    }
    if (quad == 0)
      p.lse[row] = total == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(total)) * kLn2;
  }
  if (bad != 0) {
    uint32_t rows = static_cast<uint32_t>(bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & 0xffffu;
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the stores above, which these replace
    while (rows != 0) {
      const int from = __builtin_ctz(rows);
      rows &= rows - 1;
      attend_row_alone<T>(p, b, __builtin_amdgcn_readlane(step, from), hk,
                          __builtin_amdgcn_readlane(head, from), tp.negate ? -tp.c : tp.c);
    }
  }
}

template <typename T, int DC, bool WHOLE, int kKeys, int kWaves>
hipError_t launch(TileParams& tp, hipStream_t stream) {
  const Params& p = tp.p;
  // Rows of a wave: whole queries, the heads of one key head each.
  tp.chunks = (p.G + kRows - 1) / kRows;
  tp.hg = (p.G + tp.chunks - 1) / tp.chunks;
  tp.nqw = kRows / tp.hg;
  tp.pairs = static_cast<uint32_t>(p.B * p.Hk * tp.chunks);
  tp.tiles = (static_cast<uint32_t>(p.Tq) + kWaves * tp.nqw - 1) / (kWaves * tp.nqw);
  RLM_TRY(check_launch("routed_attention", static_cast<int64_t>(tp.pairs) * tp.tiles,
                       kWaves * kWave));
  tp.by_pairs = FastDiv(tp.pairs);
  tp.by_chunks = FastDiv(static_cast<uint32_t>(tp.chunks));
  tp.by_kv = FastDiv(static_cast<uint32_t>(p.Hk));
  tp.by_heads = FastDiv(static_cast<uint32_t>(tp.hg));
  tp.by_picks = FastDiv(static_cast<uint32_t>(p.TOP + 1));
  tp.by_wave_queries = FastDiv(static_cast<uint32_t>(tp.nqw));
  tp.by_block = FastDiv(static_cast<uint32_t>(p.BS));
  const size_t lds = 2 * 2 * kKeys * 16 * pitch<T, DC>();  // two tiles of keys and values
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(&attend_tile_kernel<T, DC, WHOLE, kKeys, kWaves>),
        hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    RLM_REQUIRE(e == hipSuccess, "routed_attention: %zu bytes of LDS refused: %s", lds,
                hipGetErrorString(e));
  }
  hipLaunchKernelGGL((attend_tile_kernel<T, DC, WHOLE, kKeys, kWaves>),
                     dim3(tp.pairs * tp.tiles), dim3(kWaves * kWave), lds, stream, tp);
  return launch_status("routed_attention");
}

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
  if (dc <= 1) return launch<T, 1, WHOLE, 64, 4>(tp, stream);
  if (dc <= 2) return launch<T, 2, WHOLE, kSmall, 4>(tp, stream);
  if (dc <= 3) return launch<T, 3, WHOLE, 32, 4>(tp, stream);
  if (dc <= 4) return launch<T, 4, WHOLE, 32, 4>(tp, stream);
  return launch<T, 8, WHOLE, 32, 4>(tp, stream);
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
