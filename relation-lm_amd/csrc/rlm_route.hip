// Block routing by itself: for each query the `top` best blocks of a cache by the block
// router's score, as the routed selection kernels rank them:
//   s_h   = (mean_j,h . q_h + softplus(gamma_h) std_j,h . |q_h|) / sqrt(HD) + bias[h, bucket]
//   score = log sum_h exp(s_h), rounded to fp32
// over the complete blocks j (strict: those wholly before the local window), bucket =
// floor(log2(distance + 1)) of the block's last position, ties to the lowest block.
//
// The score is formed in float64: two blocks are ranked by their fp32 scores, so a score has
// to be right to its rounding or equal inputs would not tie.  Bound: VALU issue, 85% of the time: 4 x
// 4096 queries over up to 64 blocks (router of 4 x 16) take 24.9 us and 2860 instructions a wave.
// Of the some 150 that a head of 64 (query, block) pairs takes, 65 are float64 arithmetic (2 RD products
// and H exponentials per pair); the rest are conversions, the lanes' sums, the selects that give each
// lane its own query, and addresses.  A pick of the first 64 blocks takes about 74 more.  8 queries over
// 16 blocks take 6.1 us, one wave's chain.
// A wave takes Q queries of one batch row over 64 / P blocks at a time, P lanes to a block;
// each statistics access (16 bytes a lane, P lanes together) then serves Q queries.  Where there
// are too few queries to fill the chip, a workgroup's waves share the blocks of its queries
// (SPLIT) and their lists are merged.  After a
// head's products the P lanes share their sums, and each of them carries on the exponentials
// of its own Q / P queries.
#include "rlm_common.hpp"
#include "rlm_fastdiv.hpp"

namespace rlm {
namespace {

constexpr int kMaxTop = 64;

struct RouteParams {
  const void* q;                    // [B,Tq,S,RD]
  int64_t q_sb, q_st, q_ss;
  int q_dtype;
  const float *mean, *std;          // [B,NB,H,HD]
  const void *gamma, *bias;
  int gamma_dtype, bias_dtype;
  const void* pos;
  int pos_dtype;
  int64_t pos_sb, pos_sq;
  int32_t* out_blocks;              // [B,Tq,S,TOP]
  float* out_scores;
  int64_t BS, local_window;
  uint32_t rows_per_batch;          // Tq * S
  uint32_t groups_per_batch, groups;
  FastDiv by_slots, by_groups;
  int NB, H, HD, RB, TOP;
  bool strict, ring;
  double head_scale;
};

// The lane below's value, all ones in lane 0: within a row of 16 lanes for lists up to 16.
__device__ __forceinline__ uint64_t from_below(uint64_t v, bool short_list) {
  if (short_list) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(-1, static_cast<int>(v), 0x111, 0xF, 0xF, false);
    const uint32_t hi =
        __builtin_amdgcn_update_dpp(-1, static_cast<int>(v >> 32), 0x111, 0xF, 0xF, false);
    return static_cast<uint64_t>(lo) | (static_cast<uint64_t>(hi) << 32);
  }
  const uint64_t up = __shfl_up(v, 1, kWave);
  return (threadIdx.x & (kWave - 1)) == 0 ? ~uint64_t(0) : up;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return static_cast<uint64_t>(lo) | (static_cast<uint64_t>(hi) << 32);
}

// Puts the candidates of the wave (key 0: none) into the list whose i-th best lane i holds.
__device__ __forceinline__ void insert_keys(uint64_t& list, uint64_t key, int top, bool short_list) {
  uint64_t worst = lane_u64(list, top - 1);
  uint64_t left = __builtin_amdgcn_ballot_w64(key > worst);
  while (left != 0) {
    const int from = __builtin_ctzll(left);
    left &= left - 1;
    const uint64_t x = lane_u64(key, from);
    if (x <= worst) continue;
    const uint64_t below = from_below(list, short_list);
    list = list > x ? list : (below > x ? x : below);
    worst = lane_u64(list, top - 1);
  }
}

// exp(x) for x <= 0 to 4e-16, NaN for NaN: x = k ln 2 + r with |r| <= ln 2 / 2, the Taylor
// polynomial of degree 12 in r (its remainder is r^13 / 13! < 2e-16).  The score is rounded to fp32
// after it, as the selection's is, whose exponentials are float64 ones: a polynomial that stops at
// 1e-11 rounded some 4e-6 of the scores to another number and picked other blocks than the
// selection where two scores are next to each other.
__device__ __forceinline__ double exp_down(double x) {
  x = x < -700.0 ? -700.0 : x;  // 1e-304: nothing beside a sum of at least 1
  const double k = rint(x * 1.44269504088896340736);
  double r = fma(k, -0x1.62e42fefap-1, x);  // ln 2: its first 36 bits (k takes 10), and the rest
  r = fma(k, -0x1.cf79abc9e3b3ap-40, r);
  double y = 1.0 / 479001600.0;
  y = fma(y, r, 1.0 / 39916800.0);
  y = fma(y, r, 1.0 / 3628800.0);
  y = fma(y, r, 1.0 / 362880.0);
  y = fma(y, r, 1.0 / 40320.0);
  y = fma(y, r, 1.0 / 5040.0);
  y = fma(y, r, 1.0 / 720.0);
  y = fma(y, r, 1.0 / 120.0);
  y = fma(y, r, 1.0 / 24.0);
  y = fma(y, r, 1.0 / 6.0);
  y = fma(y, r, 0.5);
  y = fma(y, r, 1.0);
  y = fma(y, r, 1.0);
  return ldexp(y, static_cast<int>(k));
}
// log(s) for s >= 1 to 8e-16: the fp32 logarithm y, corrected by log(s exp(-y)) = z - z^2 / 2 +
// O(z^3), |z| <= 1e-6.
__device__ __forceinline__ double log_up(double s) {
  const double y = static_cast<double>(__builtin_amdgcn_logf(static_cast<float>(s)) * 0.69314718055994530942f);
  const double z = fma(s, exp_down(-y), -1.0);
  return y + fma(z * z, -0.5, z);
}

// Maximum over the lanes whose number leaves the same remainder by 4 (P = 4), or over all of
// the wave (P = 1), in each of them.
template <int P>
__device__ __forceinline__ uint64_t part_max(uint64_t v) {
  if constexpr (P == 1) {
    v = umax64(v, dpp_u64<kDppXor1>(v));
    v = umax64(v, dpp_u64<kDppXor2>(v));
  }
  v = umax64(v, dpp_u64<0x124>(v));  // row_ror:4, row_ror:8
  v = umax64(v, dpp_u64<0x128>(v));
  auto lo = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(v), static_cast<uint32_t>(v),
                                             false, false);
  auto hi = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(v >> 32),
                                             static_cast<uint32_t>(v >> 32), false, false);
  v = umax64(static_cast<uint64_t>(lo[0]) | (static_cast<uint64_t>(hi[0]) << 32),
             static_cast<uint64_t>(lo[1]) | (static_cast<uint64_t>(hi[1]) << 32));
  lo = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(v), static_cast<uint32_t>(v), false,
                                        false);
  hi = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(v >> 32),
                                        static_cast<uint32_t>(v >> 32), false, false);
  return umax64(static_cast<uint64_t>(lo[0]) | (static_cast<uint64_t>(hi[0]) << 32),
                static_cast<uint64_t>(lo[1]) | (static_cast<uint64_t>(hi[1]) << 32));
}

template <typename TQ, int P, int Q, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 1024 : 256, 4) void route_kernel(RouteParams p) {
  extern __shared__ __align__(16) double lds[];
  constexpr int kPer = (Q + P - 1) / P;  // queries whose exponentials a lane carries on
  constexpr int kBlocks = kWave / P;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int waves = blockDim.x / kWave;
  const int RD = p.H * p.HD;
  double* spread = lds;                       // [H]: softplus(gamma)
  double* bias = spread + p.H;                // [H,RB]
  double* q = bias + p.H * p.RB + (SPLIT ? 0 : wave * Q * RD);
  uint64_t* lists = reinterpret_cast<uint64_t*>(bias + p.H * p.RB + Q * RD);  // SPLIT: [waves,Q,64]

  uint32_t group = SPLIT ? blockIdx.x : blockIdx.x * waves + wave;
  const bool live = group < p.groups;
  if (!live) group = p.groups - 1;
  uint32_t in_batch;
  const uint32_t b = p.by_groups.div(group, in_batch);
  // Later positions have more blocks: every other batch row runs from the end, so that a CU's
  // workgroups (whole rounds of the grid apart) are not all long ones.
  if (!SPLIT && (b & 1)) in_batch = p.groups_per_batch - 1 - in_batch;
  const uint32_t row0 = in_batch * Q;

  for (int i = threadIdx.x; i < p.H; i += blockDim.x)
    spread[i] = log(1.0 + exp(static_cast<double>(load_any_f(p.gamma, p.gamma_dtype, i))));
  for (int i = threadIdx.x; i < p.H * p.RB; i += blockDim.x)
    bias[i] = static_cast<double>(load_any_f(p.bias, p.bias_dtype, i));
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    uint32_t slot;
    const uint32_t row = min(row0 + i, p.rows_per_batch - 1);
    const uint32_t step = p.by_slots.div(row, slot);
    const TQ* src = static_cast<const TQ*>(p.q) + b * p.q_sb + step * p.q_st + slot * p.q_ss;
    for (int d = SPLIT ? threadIdx.x : lane; d < RD; d += SPLIT ? blockDim.x : kWave)
      q[i * RD + d] = static_cast<double>(to_f32(src[d]));
  }
  int64_t t[Q];
  int64_t tmax = -1;
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    uint32_t slot;
    const uint32_t row = min(row0 + i, p.rows_per_batch - 1);
    const uint32_t step = p.by_slots.div(row, slot);
    const int64_t at = load_any_i(p.pos, p.pos_dtype, b * p.pos_sb + step * p.pos_sq);
    // Within what the sums below hold in 64 bits (any negative one has no block).
    t[i] = at < -1 ? -1 : at < INT64_MAX - 1 ? at : INT64_MAX - 1;
    tmax = t[i] > tmax ? t[i] : tmax;
  }
  __syncthreads();

  const int part = lane % P, in_wave = lane / P;
  // This lane's own queries: their position, first position of the window and, in a ring, the
  // lowest absolute block that the slots hold.
  int64_t mine[kPer], start[kPer], lowest[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    mine[k] = t[0];
#pragma unroll
    for (int i = 0; i < Q; ++i)
      if (i == k * P + part) mine[k] = t[i];
    const int64_t s = mine[k] - p.local_window + 1;
    start[k] = s > 0 ? s : 0;
    lowest[k] = p.ring ? mine[k] / p.BS - p.NB + 1 : 0;
  }
  // Slots that can hold an eligible block of any of the queries.
  const int64_t complete = p.ring ? p.NB : (tmax + 1) / p.BS;
  const int slots = static_cast<int>(complete < p.NB ? complete : p.NB);
  const bool short_list = p.TOP <= 16;
  uint64_t list[Q] = {};
  // Four queries, four lanes to a block: the wave's first 64 blocks' keys wait in registers (a lane has
  // its own query's), and the lists start from their TOP largest, found for the four queries
  // at once.  Blocks after those enter one by one where they pass the list's last.
  constexpr bool kFirst = Q == 4 && P == 4;
  uint64_t waiting[kFirst ? P : 1] = {};
  auto start_lists = [&]() {
    if constexpr (kFirst) {
      for (int rank = 0; rank < p.TOP; ++rank) {
        const uint64_t best = part_max<P>(
            umax64(umax64(waiting[0], waiting[1]), umax64(waiting[2], waiting[3])));
#pragma unroll
        for (int i = 0; i < P; ++i) waiting[i] = waiting[i] == best ? 0 : waiting[i];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          const uint64_t x = lane_u64(best, i);
          list[i] = lane == rank ? x : list[i];
        }
      }
    }
  };

  // This lane's statistics of the block that it has in the pass from j0 on (the last block's
  // past the end).
  auto block_at = [&](int j0) {
    return (static_cast<int64_t>(b) * p.NB + min(j0 + in_wave, p.NB - 1)) * RD + 4 * part;
  };
  float4 m, s4;
  {
    const int64_t at = block_at((SPLIT ? wave : 0) * kBlocks);
    m = *reinterpret_cast<const float4*>(p.mean + at);
    s4 = *reinterpret_cast<const float4*>(p.std + at);
  }
  const int stride = (SPLIT ? waves : 1) * kBlocks;
  int pass = 0;
  for (int j0 = (SPLIT ? wave : 0) * kBlocks; j0 < slots; j0 += stride, ++pass) {
    const int j = j0 + in_wave;
    const int64_t at = block_at(j0), next_at = block_at(j0 + stride);
    int64_t block[kPer];
    int bucket[kPer];
    bool ok[kPer];
    double most[kPer], sum[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      // In a ring, slot j holds the block of remainder j among [lowest, lowest + NB).
      block[k] = p.ring ? lowest[k] + ((j - lowest[k]) & (p.NB - 1)) : j;
      const int64_t end = block[k] * p.BS + p.BS - 1;
      // (A ring's block that the picks' type does not hold is no pick.)
      ok[k] = j < slots && block[k] >= 0 && block[k] <= INT32_MAX && end <= mine[k] &&
              (!p.strict || end < start[k]);
      const int64_t away = mine[k] > end ? mine[k] - end : 0;
      const int log2 = 63 - __builtin_clzll(static_cast<uint64_t>(away + 1));
      bucket[k] = log2 < p.RB ? log2 : p.RB - 1;
      most[k] = sum[k] = 0.0;
    }
    for (int h = 0; h < p.H; ++h) {
      double like[Q] = {}, wide[Q] = {};
      for (int d = 0; d < p.HD; d += 4 * P) {
        const double md[4] = {m.x, m.y, m.z, m.w}, sd[4] = {s4.x, s4.y, s4.z, s4.w};
        // The next features of this block, or the first of the next.
        const int after = h * p.HD + d + 4 * P;
        const int64_t load = after < RD ? at + after : next_at;
        m = *reinterpret_cast<const float4*>(p.mean + load);
        s4 = *reinterpret_cast<const float4*>(p.std + load);
        const double* qd = q + h * p.HD + d + 4 * part;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double x = qd[i * RD + e];
            like[i] = fma(md[e], x, like[i]);
            wide[i] = fma(sd[e], fabs(x), wide[i]);
          }
        }
      }
      double s[Q];
#pragma unroll
      for (int i = 0; i < Q; ++i)
        s[i] = group_sum_f64(fma(spread[h], wide[i], like[i]), P) * p.head_scale;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        double x = s[0];
#pragma unroll
        for (int i = 0; i < Q; ++i)
          if (i == k * P + part) x = s[i];
        x += bias[h * p.RB + bucket[k]];
        if (h == 0) {
          most[k] = x;
          sum[k] = 1.0;
        } else {
          // (Equal terms may be infinite: their difference is none, not inf - inf.)
          const double e = exp_down(x == most[k] ? 0.0 : -fabs(x - most[k]));
          sum[k] = x > most[k] ? fma(sum[k], e, 1.0) : sum[k] + e;
          most[k] = x > most[k] ? x : most[k];
        }
      }
    }
    uint64_t key[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const float score = static_cast<float>(most[k] + log_up(sum[k]));
      key[k] = ok[k] && score > -1.0e30f
                   ? select_key(score, static_cast<uint32_t>(block[k] - lowest[k]))
                   : 0;
    }
    if (kFirst && pass < P) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (pass == i) waiting[kFirst ? i : 0] = key[0];
      if (j0 + stride >= slots || pass == P - 1) start_lists();
    } else {
#pragma unroll
      for (int i = 0; i < Q; ++i)
        insert_keys(list[i], part == i % P ? key[i / P] : 0, p.TOP, short_list);
    }
  }

  if constexpr (SPLIT) {
    // The waves' lists into one, each query's by a wave of its own.
#pragma unroll
    for (int i = 0; i < Q; ++i)
      lists[(wave * Q + i) * kWave + lane] = lane < p.TOP ? list[i] : 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Q; ++i)
      if (i % waves == wave)
        for (int w = 0; w < waves; ++w)
          if (w != wave) insert_keys(list[i], lists[(w * Q + i) * kWave + lane], p.TOP, short_list);
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    if (SPLIT && i % waves != wave) continue;
    if (row0 + i >= p.rows_per_batch || lane >= p.TOP) continue;
    const int64_t low = p.ring ? t[i] / p.BS - p.NB + 1 : 0;
    const int64_t at =
        (static_cast<int64_t>(b) * p.rows_per_batch + row0 + i) * p.TOP + lane;
    const bool some = list[i] != 0;
    p.out_blocks[at] = some ? static_cast<int32_t>(low + key_index(list[i])) : -1;
    p.out_scores[at] = some ? key_score(list[i]) : -INFINITY;
  }
}

template <typename TQ, int P, int Q>
hipError_t launch_split(RouteParams& p, int64_t B, int waves, size_t shared, hipStream_t stream) {
  p.groups_per_batch = (p.rows_per_batch + Q - 1) / Q;
  p.groups = static_cast<uint32_t>(B * p.groups_per_batch);
  p.by_groups = FastDiv(p.groups_per_batch);
  RLM_TRY(check_launch("block_route", p.groups, waves * kWave));
  const size_t bytes =
      shared + sizeof(double) * Q * p.H * p.HD + sizeof(uint64_t) * waves * Q * kWave;
  hipLaunchKernelGGL((route_kernel<TQ, P, Q, true>), dim3(p.groups), dim3(waves * kWave), bytes,
                     stream, p);
  return launch_status("block_route");
}

// Waves that the chip holds at this register count, four to a SIMD.  Measured, all queries at the
// caches' end, router of 4 x 16 (us: one query to a workgroup with all its waves / four queries
// with as many waves as are resident / four queries to a wave; with exponentials of degree 9, which
// took 2 to 4% off each):
//     64 blocks    256 queries: 8.4 / 11.0 / 17.0    1024: 12.0 / 11.4 / 17.2    4096: 29 / 18 / 17
//    512 blocks    256: 18.7 / 23 / 107              1024: 52 / 24 / 108         4096: 191 / 57 / 109
//   2048 blocks    256: 38 / 58 / 393                1024: 127 / 60 / 396        4096: 491 / 193 / 398
//   2048 blocks    16384: 1942 / 716 / 717
// Routers wider than 256 take one query to a workgroup at any number of queries, each reading all
// statistics: four queries to each of four waves would take 128 bytes of LDS per feature.  4 x 4096
// queries over up to 64 blocks: router of 4 x 64 46.6 us, of 5 x 64 115.8, of 8 x 64 171; 4096 queries over
// up to 512 blocks, 4 x 64 112 and 8 x 64 525.
constexpr int kResident = 4096;
template <typename TQ, int P>
hipError_t launch_route(RouteParams& p, int64_t B, hipStream_t stream) {
  const int RD = p.H * p.HD;
  const size_t shared = sizeof(double) * (p.H + static_cast<size_t>(p.H) * p.RB);
  const int64_t queries = B * p.rows_per_batch;
  const int passes = (p.NB + kWave / P - 1) / (kWave / P);
  const int most = std::min(16, passes);
  // One query to a workgroup while all its waves are resident: the shortest chain.  Also where a
  // batch row has fewer than the four queries that share its statistics (a decode batch).
  if (queries * most <= kResident || p.rows_per_batch < 4 || RD > 256)
    return launch_split<TQ, P, 1>(p, B, most, shared, stream);
  int waves = 1;
  while (2 * waves <= most && queries / 4 * waves < kResident) waves *= 2;
  if (waves > 1) return launch_split<TQ, P, 4>(p, B, waves, shared, stream);
  constexpr int kWaves = 4, kQueries = 4;
  p.groups_per_batch = (p.rows_per_batch + kQueries - 1) / kQueries;
  p.groups = static_cast<uint32_t>(B * p.groups_per_batch);
  p.by_groups = FastDiv(p.groups_per_batch);
  const size_t bytes = shared + sizeof(double) * kWaves * kQueries * RD;
  const dim3 grid((p.groups + kWaves - 1) / kWaves);
  RLM_TRY(check_launch("block_route", grid.x, kWaves * kWave));
  hipLaunchKernelGGL((route_kernel<TQ, P, kQueries, false>), grid,
                     dim3(kWaves * kWave), bytes, stream, p);
  return launch_status("block_route");
}

// Four lanes to a block where they divide a head in 16-byte pieces, one lane otherwise; that lane has
// four queries' sums and exponentials to itself (24 registers spilled at four queries to a wave) and
// picks enter one by one.  4 x 4096 queries, each asking for itself, over up to 64 blocks: router of 4 x 16
// 27 us, of 8 x 8 58.8, of 4 x 8 41.6; 4096 queries over up to 512: 4 x 16 63.8, 8 x 8 97.0; 256 queries over
// 64: 8.8 and 11.2.
template <typename TQ>
hipError_t launch_route_type(RouteParams& p, int64_t B, hipStream_t stream) {
  if (p.HD % 16 == 0) return launch_route<TQ, 4>(p, B, stream);
  return launch_route<TQ, 1>(p, B, stream);
}

}  // namespace
}  // namespace rlm

using namespace rlm;

extern "C" hipError_t rlm_block_route(const rlm_tensor* router_query, const rlm_tensor* block_mean,
                                      const rlm_tensor* block_std, const rlm_tensor* gamma,
                                      const rlm_tensor* bias, const rlm_tensor* positions,
                                      int64_t block_size, int64_t local_window, int64_t top_blocks,
                                      int32_t strict_valid, int32_t ring,
                                      const rlm_tensor* out_blocks, const rlm_tensor* out_scores,
                                      hipStream_t stream) {
  clear_error();
  RLM_TRY(check_strided(router_query, "router_query", 4));
  RLM_TRY(check_dtype_float(router_query, "router_query"));
  const int64_t B = router_query->shape[0], Tq = router_query->shape[1],
                S = router_query->shape[2], RD = router_query->shape[3];
  RLM_TRY(check_dense(block_mean, "block_mean", 4));
  RLM_TRY(check_dtype_is(block_mean, "block_mean", RLM_F32));
  RLM_TRY(check_dim(block_mean, "block_mean", 0, B));
  const int64_t NB = block_mean->shape[1], H = block_mean->shape[2], HD = block_mean->shape[3];
  RLM_TRY(check_dense(block_std, "block_std", 4));
  RLM_TRY(check_dtype_is(block_std, "block_std", RLM_F32));
  for (int i = 0; i < 4; ++i) RLM_TRY(check_dim(block_std, "block_std", i, block_mean->shape[i]));
  RLM_REQUIRE(NB >= 1 && NB < (int64_t(1) << 30), "block_mean: need between 1 and 2^30 blocks");
  RLM_REQUIRE(H >= 1 && HD >= 4 && HD % 4 == 0 && H * HD <= 1024,
              "block_mean: router heads of a multiple of 4 features, heads * head dim <= 1024, got "
              "%lld x %lld",
              (long long)H, (long long)HD);
  RLM_TRY(check_dim(router_query, "router_query", 3, H * HD));
  RLM_TRY(check_dense(gamma, "gamma", 1));
  RLM_TRY(check_dtype_float(gamma, "gamma"));
  RLM_TRY(check_dim(gamma, "gamma", 0, H));
  RLM_TRY(check_dense(bias, "bias", 2));
  RLM_TRY(check_dtype_float(bias, "bias"));
  RLM_TRY(check_dim(bias, "bias", 0, H));
  const int64_t RB = bias->shape[1];
  RLM_REQUIRE(RB >= 1 && H * RB <= 2048,
              "bias: heads * buckets must be in [1, 2048], got %lld x %lld", (long long)H,
              (long long)RB);
  RLM_REQUIRE(block_size >= 1 && block_size <= (int64_t(1) << 30),
              "block_size must be in [1, 2^30], got %lld", (long long)block_size);
  RLM_REQUIRE(local_window >= 0 && local_window <= (int64_t(1) << 40),
              "local_window must not be negative, got %lld", (long long)local_window);
  RLM_REQUIRE(top_blocks >= 1 && top_blocks <= kMaxTop, "top_blocks must be in [1, %d], got %lld",
              kMaxTop, (long long)top_blocks);
  RLM_REQUIRE(!ring || ((NB & (NB - 1)) == 0 && (block_size & (block_size - 1)) == 0),
              "ring-buffer caches need a power-of-two number of blocks of a power-of-two size, got "
              "%lld blocks of %lld",
              (long long)NB, (long long)block_size);
  RouteParams p{};
  RLM_TRY(check_positions(positions, "positions", B, Tq, &p.pos_sb, &p.pos_sq));
  for (const rlm_tensor* t : {out_blocks, out_scores}) {
    const char* name = t == out_blocks ? "out_blocks" : "out_scores";
    RLM_TRY(check_dense(t, name, 4));
    RLM_TRY(check_dtype_is(t, name, t == out_blocks ? RLM_I32 : RLM_F32));
    for (int i = 0; i < 3; ++i) RLM_TRY(check_dim(t, name, i, router_query->shape[i]));
    RLM_TRY(check_dim(t, name, 3, top_blocks));
  }
  RLM_REQUIRE((reinterpret_cast<uintptr_t>(block_mean->data) & 15u) == 0 &&
                  (reinterpret_cast<uintptr_t>(block_std->data) & 15u) == 0,
              "block_mean and block_std must be 16-byte aligned");
  RLM_REQUIRE(B * Tq * S < (int64_t(1) << 31), "at most 2^31 - 1 queries");
  p.q = router_query->data;
  p.q_sb = router_query->stride[0], p.q_st = router_query->stride[1];
  p.q_ss = router_query->stride[2];
  p.mean = static_cast<const float*>(block_mean->data);
  p.std = static_cast<const float*>(block_std->data);
  p.gamma = gamma->data;
  p.gamma_dtype = gamma->dtype;
  p.bias = bias->data;
  p.bias_dtype = bias->dtype;
  p.pos = positions->data;
  p.pos_dtype = positions->dtype;
  p.out_blocks = static_cast<int32_t*>(out_blocks->data);
  p.out_scores = static_cast<float*>(out_scores->data);
  p.BS = block_size;
  p.local_window = local_window;
  p.rows_per_batch = static_cast<uint32_t>(Tq * S);
  if (B * Tq * S == 0) return hipSuccess;
  p.by_slots = FastDiv(static_cast<uint32_t>(S));
  p.NB = static_cast<int>(NB);
  p.H = static_cast<int>(H);
  p.HD = static_cast<int>(HD);
  p.RB = static_cast<int>(RB);
  p.TOP = static_cast<int>(top_blocks);
  p.strict = strict_valid != 0;
  p.ring = ring != 0;
  p.head_scale = 1.0 / std::sqrt(static_cast<double>(HD));
  switch (router_query->dtype) {
    case RLM_F32: return launch_route_type<float>(p, B, stream);
    case RLM_BF16: return launch_route_type<bf16>(p, B, stream);
    default: return launch_route_type<f16>(p, B, stream);
  }
}
