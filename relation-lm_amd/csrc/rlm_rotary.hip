// Rotary positions of query and key, alone or with the key and value rows' cache writes.
//
// Pair i of a head, at position p with frequency f_i, turns by p f_i:
//   (a, b) -> (a cos - b sin, a sin + b cos) * scale
// with a, b features (i, F + i) of the head, or (2 i, 2 i + 1) when interleaved; features
// from 2 F on pass unchanged.
//
// The angle is reduced in float64 (p f_i reaches 10^6 turns far into a context, where fp32
// has no bits left for the turn's fraction): p f_i / (2 pi) less its nearest whole number,
// then fp32 sine and cosine of pi times that (5.6e-8 off in fp32 outputs, where float64 ones would be
// 4.1e-8 off; half a step of a 16-bit output is 2e-3 or 2e-4).  They depend on the token alone, so a
// workgroup computes them once for its tokens into LDS and every head reads them there.
//
// Bound: memory, every row read once and written once: 4 x 4096 tokens of 12 + 4 + 4 heads of 64
// bf16 features into caches, 63% of the tokens real on average (71.5 MB, which the MALL holds), take
// 13.2 to 14.0 us, 5.1 to 5.4 TB/s.  2 x 1999 of 8 + 8 fp32 heads, 48 of whose 64 features turn, take 9.4
// us (3.5 TB/s) and wait (74% of the waves' life): a wave's lanes turn some pieces and copy
// others, one after the other, each a load, its wait and a store, in seven rounds.  A decode step of 8
// tokens takes 3.1 us, a launch and two round trips.
//
// Accesses are of 16 bytes where pairs, head dim, strides and addresses allow, else of one element: the
// 4 x 4096 tokens with every token real, into caches, take 15.5 us in bf16 (26.5 in fp32), 37.2 (35.4) with
// 31 pairs in place of 32 and 29.5 (28.5) from rows one element off; 8 single tokens 6.0 either way.
#include <type_traits>

#include "rlm_common.hpp"
#include "rlm_fastdiv.hpp"

namespace rlm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 2048;  // per workgroup: 16 KiB of LDS
constexpr int kMaxTokens = 16;    // per workgroup
constexpr int kMaxQuantized = 256;  // head dim of 8-bit caches

struct RotaryParams {
  const void *q, *k, *v;           // [B,Tq,H*,D], unit stride in D
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  void *oq, *ok, *ov;              // ok / ov: [B,Tq,Hk,D], or the caches [B,T,Hk,D]
  int64_t ok_sb, ok_st, ok_sh, ov_sb, ov_st, ov_sh;
  float *ks, *vs;                  // 8-bit caches: their scales [B,T,Hk]
  int64_t ks_sb, ks_st, ks_sh, vs_sb, vs_st, vs_sh;
  const void* pos;
  int pos_dtype;
  int64_t pos_sb, pos_st;
  const void* lengths;             // [B], or null
  int lengths_dtype;
  const float* freq;
  float scale;
  int64_t rows;                    // cache rows T
  uint32_t tokens;                 // B * Tq
  int Hq, Hk, D, F;
  int heads;                       // Hq + Hk (+ Hk value heads)
  int per_group;                   // tokens of a workgroup
  bool to_cache, ring;
  FastDiv by_queries, by_pairs, by_units, by_token_units, by_heads;
};

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

// The turns of a workgroup's `count` tokens and their rows of ok / ov (negative: not written).
__device__ __forceinline__ void set_up(const RotaryParams& p, uint32_t first, uint32_t count,
                                       float2* turn, int64_t* dest) {
  const uint32_t F = p.F;
  for (uint32_t i = threadIdx.x; i < count * F; i += kThreads) {
    uint32_t f, step;
    const uint32_t local = p.by_pairs.div(i, f);
    const uint32_t b = p.by_queries.div(first + local, step);
    // (Sums of float64 numbers do not pass the end of int64; exact up to 2^53.)
    double at = static_cast<double>(
        load_any_i(p.pos, p.pos_dtype, b * p.pos_sb + step * p.pos_st));
    if (p.to_cache) at += step;
    const double turns = at * static_cast<double>(p.freq[f]) *
                         0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    turn[i] = make_float2(c * p.scale, s * p.scale);
  }
  if (threadIdx.x < count) {
    uint32_t step;
    const uint32_t b = p.by_queries.div(first + threadIdx.x, step);
    int64_t row = step;
    if (p.to_cache) {
      // Past the end of int64 the sum wraps to a negative position, which is not written.
      const int64_t at = static_cast<int64_t>(
          static_cast<uint64_t>(load_any_i(p.pos, p.pos_dtype, b * p.pos_sb + step * p.pos_st)) +
          step);
      const bool real =
          p.lengths == nullptr || static_cast<int64_t>(step) < load_any_i(p.lengths, p.lengths_dtype, b);
      row = p.ring ? (at & (p.rows - 1)) : at;
      if (at < 0 || row >= p.rows || !real) row = -1;
    }
    dest[threadIdx.x] = row;
  }
  __syncthreads();
}

// V: elements of one access (16 bytes, or one element for unaligned shapes).
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams p) {
  using raw_t = typename Raw<V * sizeof(T)>::type;
  struct Vec {
    T e[V];
  };
  __shared__ float2 turn[kMaxAngles];
  __shared__ int64_t dest[kMaxTokens];
  const uint32_t first = blockIdx.x * static_cast<uint32_t>(p.per_group);
  const uint32_t count = min(static_cast<uint32_t>(p.per_group), p.tokens - first);
  const uint32_t F = p.F;
  set_up(p, first, count, turn, dest);

  const int D = p.D;
  // Units of a head: one pair of accesses (INTERLEAVED: one access), or one that is copied.
  const uint32_t turned = INTERLEAVED ? 2 * F / V : F / V;
  const uint32_t total = count * p.by_token_units.d;
  for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
    uint32_t in_token, unit, step;
    const uint32_t local = p.by_token_units.div(i, in_token);
    const uint32_t head = p.by_units.div(in_token, unit);
    const uint32_t b = p.by_queries.div(first + local, step);
    const int64_t row = dest[local];
    const bool is_q = head < static_cast<uint32_t>(p.Hq);
    const bool is_v = head >= static_cast<uint32_t>(p.Hq + p.Hk);
    if (!is_q && row < 0) continue;
    const T* src;
    T* dst;
    if (is_q) {
      src = static_cast<const T*>(p.q) + b * p.q_sb + step * p.q_st + head * p.q_sh;
      dst = static_cast<T*>(p.oq) + (static_cast<int64_t>(first + local) * p.Hq + head) * D;
    } else if (!is_v) {
      const int64_t h = head - p.Hq;
      src = static_cast<const T*>(p.k) + b * p.k_sb + step * p.k_st + h * p.k_sh;
      dst = static_cast<T*>(p.ok) + b * p.ok_sb + row * p.ok_st + h * p.ok_sh;
    } else {
      const int64_t h = head - p.Hq - p.Hk;
      src = static_cast<const T*>(p.v) + b * p.v_sb + step * p.v_st + h * p.v_sh;
      dst = static_cast<T*>(p.ov) + b * p.ov_sb + row * p.ov_st + h * p.ov_sh;
    }
    const float2* tr = turn + local * F;
    if (unit < turned) {
      if constexpr (INTERLEAVED) {
        const uint32_t at = unit * V;
        if constexpr (V == 1) {
          // One element: its partner is read as well, only this one is written.
          const uint32_t even = at & ~1u;
          const float a = to_f32(src[even]), bb = to_f32(src[even + 1]);
          const float2 cs = tr[at >> 1];
          const float out = (at & 1) ? fmaf(a, cs.y, bb * cs.x) : fmaf(a, cs.x, -(bb * cs.y));
          dst[at] = is_v ? src[at] : from_f32<T>(out);
        } else {
          Vec x = __builtin_bit_cast(Vec, *reinterpret_cast<const raw_t*>(src + at));
          if (!is_v) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              const float2 cs = tr[(at + e) >> 1];
              const float a = to_f32(x.e[e]), bb = to_f32(x.e[e + 1]);
              x.e[e] = from_f32<T>(fmaf(a, cs.x, -(bb * cs.y)));
              x.e[e + 1] = from_f32<T>(fmaf(a, cs.y, bb * cs.x));
            }
          }
          *reinterpret_cast<raw_t*>(dst + at) = __builtin_bit_cast(raw_t, x);
        }
      } else {
        const uint32_t at = unit * V;
        Vec x = __builtin_bit_cast(Vec, *reinterpret_cast<const raw_t*>(src + at));
        Vec y = __builtin_bit_cast(Vec, *reinterpret_cast<const raw_t*>(src + F + at));
        if (!is_v) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 cs = tr[at + e];
            const float a = to_f32(x.e[e]), bb = to_f32(y.e[e]);
            x.e[e] = from_f32<T>(fmaf(a, cs.x, -(bb * cs.y)));
            y.e[e] = from_f32<T>(fmaf(a, cs.y, bb * cs.x));
          }
        }
        *reinterpret_cast<raw_t*>(dst + at) = __builtin_bit_cast(raw_t, x);
        *reinterpret_cast<raw_t*>(dst + F + at) = __builtin_bit_cast(raw_t, y);
      }
    } else {
      const uint32_t at = (INTERLEAVED ? 0 : F) + unit * V;
      *reinterpret_cast<raw_t*>(dst + at) = *reinterpret_cast<const raw_t*>(src + at);
    }
  }
}

template <typename T, int V>
hipError_t launch_rotary(const RotaryParams& p, bool interleaved, hipStream_t stream) {
  const char* name = p.to_cache ? "rotary_to_caches" : "rotary_positions";
  const dim3 grid((p.tokens + p.per_group - 1) / p.per_group);
  RLM_TRY(check_launch(name, grid.x, kThreads));
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, dim3(kThreads), 0, stream, p);
  return launch_status(name);
}

template <typename T>
hipError_t launch_rotary_type(RotaryParams& p, bool aligned, bool interleaved,
                              hipStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  const int per_vec = aligned ? kWide : 1;
  const uint32_t units = interleaved ? p.D / per_vec : (p.D - p.F) / per_vec;
  p.by_units = FastDiv(units);
  p.by_token_units = FastDiv(units * p.heads);
  return aligned ? launch_rotary<T, kWide>(p, interleaved, stream)
                 : launch_rotary<T, 1>(p, interleaved, stream);
}

// Eight elements from `src`, of which `count` are read (WIDE: whole 16-byte accesses).
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* src, int count, float (&x)[8]) {
  if constexpr (WIDE) {
    struct Raws {
      uint4 part[sizeof(T) / 2];
    };
    struct Vec {
      T e[8];
    };
    Raws raw;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      raw.part[i] = reinterpret_cast<const uint4*>(src)[i];
    const Vec v = __builtin_bit_cast(Vec, raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32(v.e[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < count ? to_f32(src[e]) : 0.0f;
  }
}

// Eight features of a row whose L lanes each have eight: its scale, and these features' codes.
template <int L>
__device__ __forceinline__ float quantize8(const float (&x)[8], uint32_t (&codes)[2]) {
  // The largest magnitude as bits: NaN above infinity above every number.
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
  for (int off = 1; off < L; off <<= 1)
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), off, kWave)));
  const bool finite = most < 0x7f800000u;
  // Not below the smallest normal number, whose reciprocal is finite.
  const float least = fmaxf(__uint_as_float(most) / 448.0f, 1.17549435e-38f);
  const float inv = 1.0f / least;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // x / s as the correctly rounded reciprocal and one correction give it: values that are
      // few-bit fractions of the largest fall on or beside the codes' ties.
      const float q = x[4 * w + e] * inv;
      y[e] = fmaf(fmaf(-q, least, x[4 * w + e]), inv, q);
    }
    const int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    codes[w] = finite ? static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true))
                      : 0u;
  }
  return !finite ? __uint_as_float(0x7fc00000u) : most == 0 ? 0.0f : least;
}

// Rotation with the key and value rows written as e4m3 codes and a scale each.  L lanes have a
// row, eight features each, so that its largest magnitude is a few lane exchanges; a pair's
// other half is read a second time (from L1) by the lane that has it not.
// Bound: few tokens wait, a launch and two round trips (8 tokens of 9 + 3 + 3 heads of 64 take 4.0 us);
// for many the kernel below is the faster one where accesses are whole (else 53 us where it takes 16).
template <typename T, int L, bool WIDE, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_quantize_kernel(RotaryParams p) {
  __shared__ float2 turn[kMaxAngles];
  __shared__ int64_t dest[kMaxTokens];
  const uint32_t first = blockIdx.x * static_cast<uint32_t>(p.per_group);
  const uint32_t count = min(static_cast<uint32_t>(p.per_group), p.tokens - first);
  set_up(p, first, count, turn, dest);

  const int D = p.D, F = p.F;
  const int at = 8 * (threadIdx.x % L);
  const int mine = min(8, D - at);  // features of this lane, none where negative
  const uint32_t total = count * p.by_heads.d;
  for (uint32_t i = threadIdx.x / L; i < total; i += kThreads / L) {
    uint32_t head, step;
    const uint32_t local = p.by_heads.div(i, head);
    const uint32_t b = p.by_queries.div(first + local, step);
    const int64_t row = dest[local];
    const bool is_q = head < static_cast<uint32_t>(p.Hq);
    const bool is_v = head >= static_cast<uint32_t>(p.Hq + p.Hk);
    if (!is_q && row < 0) continue;  // all of a row's lanes
    const int64_t h = is_q ? head : is_v ? head - p.Hq - p.Hk : head - p.Hq;
    const T* src = is_q ? static_cast<const T*>(p.q) + b * p.q_sb + step * p.q_st + h * p.q_sh
                   : is_v ? static_cast<const T*>(p.v) + b * p.v_sb + step * p.v_st + h * p.v_sh
                          : static_cast<const T*>(p.k) + b * p.k_sb + step * p.k_st + h * p.k_sh;
    const float2* tr = turn + local * F;
    float x[8] = {};
    if (mine > 0) {
      load8<T, WIDE>(src + at, mine, x);
      if (!is_v && at < 2 * F) {
        if constexpr (INTERLEAVED) {
          // Pairs do not straddle lanes.
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            if (WIDE || at + e < 2 * F) {
              const float2 cs = tr[(at + e) >> 1];
              const float a = x[e], bb = x[e + 1];
              x[e] = fmaf(a, cs.x, -(bb * cs.y));
              x[e + 1] = fmaf(a, cs.y, bb * cs.x);
            }
          }
        } else if constexpr (WIDE) {
          // F is a multiple of 8: a lane's features are all of one half.
          const bool low = at < F;
          float y[8];
          load8<T, true>(src + (low ? at + F : at - F), 8, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 cs = tr[(low ? at : at - F) + e];
            x[e] = low ? fmaf(x[e], cs.x, -(y[e] * cs.y)) : fmaf(y[e], cs.y, x[e] * cs.x);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int d = at + e;
            if (d < 2 * F) {  // 2 F <= D
              const bool low = d < F;
              const float2 cs = tr[low ? d : d - F];
              const float y = to_f32(src[low ? d + F : d - F]);
              x[e] = low ? fmaf(x[e], cs.x, -(y * cs.y)) : fmaf(y, cs.y, x[e] * cs.x);
            }
          }
        }
      }
    }
    if (is_q) {
      T* dst = static_cast<T*>(p.oq) + (static_cast<int64_t>(first + local) * p.Hq + h) * D + at;
      if constexpr (WIDE) {
        if (mine > 0) {
          put4<T>(dst, x[0], x[1], x[2], x[3]);
          put4<T>(dst + 4, x[4], x[5], x[6], x[7]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < mine) dst[e] = from_f32<T>(x[e]);
      }
      continue;
    }
    uint32_t codes[2];
    const float scale = quantize8<L>(x, codes);
    uint8_t* dst = is_v ? static_cast<uint8_t*>(p.ov) + b * p.ov_sb + row * p.ov_st + h * p.ov_sh
                        : static_cast<uint8_t*>(p.ok) + b * p.ok_sb + row * p.ok_st + h * p.ok_sh;
    if constexpr (WIDE) {
      if (mine > 0) *reinterpret_cast<uint2*>(dst + at) = make_uint2(codes[0], codes[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < mine) dst[at + e] = static_cast<uint8_t>(codes[e / 4] >> (8 * (e % 4)));
    }
    if (at == 0) {
      float* to = is_v ? p.vs + b * p.vs_sb + row * p.vs_st + h * p.vs_sh
                       : p.ks + b * p.ks_sb + row * p.ks_st + h * p.ks_sh;
      *to = scale;
    }
  }
}

// The same for workgroups of several tokens: a wave has one head of 64 / L tokens at a time, the next one's
// rows on their way, so that what depends on the head is scalar and what depends on the token comes
// from LDS.  A lane has both halves of four pairs (interleaved: four pairs), or eight features that do not
// turn.  With every address from 64-bit products per row, as above, instructions bound it: 4 x 4096 tokens
// of 12 + 4 + 4 heads of 64 take 16.1 us (84 MB, 5.2 TB/s) where they took 22.0.  (Rows of tokens that are not
// real are read with the others, and not written.)
template <typename T, int L, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_quantize_tokens_kernel(RotaryParams p) {
  __shared__ float2 turn[kMaxAngles];
  __shared__ int64_t dest[kMaxTokens];
  __shared__ int64_t from[3][kMaxTokens], to[2][kMaxTokens], scale_to[2][kMaxTokens];
  const uint32_t first = blockIdx.x * static_cast<uint32_t>(p.per_group);
  const uint32_t count = min(static_cast<uint32_t>(p.per_group), p.tokens - first);
  if (threadIdx.x < count) {
    uint32_t step;
    const uint32_t b = p.by_queries.div(first + threadIdx.x, step);
    from[0][threadIdx.x] = b * p.q_sb + step * p.q_st;
    from[1][threadIdx.x] = b * p.k_sb + step * p.k_st;
    from[2][threadIdx.x] = b * p.v_sb + step * p.v_st;
  }
  set_up(p, first, count, turn, dest);
  if (threadIdx.x < count) {
    const int64_t b = p.by_queries.div(first + threadIdx.x), row = dest[threadIdx.x];
    to[0][threadIdx.x] = b * p.ok_sb + row * p.ok_st;
    to[1][threadIdx.x] = b * p.ov_sb + row * p.ov_st;
    scale_to[0][threadIdx.x] = b * p.ks_sb + row * p.ks_st;
    scale_to[1][threadIdx.x] = b * p.vs_sb + row * p.vs_st;
  }
  __syncthreads();

  constexpr int kTokens = kWave / L, kWaves = kThreads / kWave;
  typedef typename std::conditional<sizeof(T) == 4, uint4, uint2>::type raw_t;  // four features
  struct Four {
    T e[4];
  };
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1), part = lane % L;
  const int D = p.D, F = p.F;
  const bool inside = 8 * part < D;
  const bool turns = INTERLEAVED ? 8 * part < 2 * F : 4 * part < F;
  // A lane's first and second four features.
  const int one = !INTERLEAVED && turns ? 4 * part : inside ? 8 * part : 0;
  const int two = !INTERLEAVED && turns ? F + 4 * part : one + 4;
  const int chunks = (count + kTokens - 1) / kTokens;
  const int total = p.heads * chunks;  // (head, chunk of tokens), the waves' in turn
  auto kind_of = [&](int head) { return head < p.Hq ? 0 : head < p.Hq + p.Hk ? 1 : 2; };
  auto token_of = [&](int chunk) {
    return min(chunk * kTokens + lane / L, static_cast<int>(count) - 1);
  };
  raw_t next[2];
  auto fetch = [&](int head, int chunk) {
    const int kind = kind_of(head);
    const T* base = kind == 0   ? static_cast<const T*>(p.q) + head * p.q_sh
                    : kind == 1 ? static_cast<const T*>(p.k) + (head - p.Hq) * p.k_sh
                                : static_cast<const T*>(p.v) + (head - p.Hq - p.Hk) * p.v_sh;
    const T* src = base + from[kind][token_of(chunk)];
    next[0] = *reinterpret_cast<const raw_t*>(src + one);
    next[1] = *reinterpret_cast<const raw_t*>(src + two);
  };
  int head = wave % p.heads, chunk = wave / p.heads;
  auto advance = [&](int& h, int& c) {
    h += kWaves;
    while (h >= p.heads) {
      h -= p.heads;
      ++c;
    }
  };
  if (wave < total) fetch(head, chunk);
  for (int i = wave; i < total; i += kWaves) {
    const Four low = __builtin_bit_cast(Four, next[0]), high = __builtin_bit_cast(Four, next[1]);
    int next_head = head, next_chunk = chunk;
    advance(next_head, next_chunk);
    if (i + kWaves < total) fetch(next_head, next_chunk);
    const int kind = kind_of(head);
    const int token = token_of(chunk);
    const bool here = inside && chunk * kTokens + lane / L < static_cast<int>(count);
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = inside ? to_f32(low.e[e]) : 0.0f;
      x[4 + e] = inside ? to_f32(high.e[e]) : 0.0f;
    }
    if (kind != 2 && turns) {
      const float2* tr = turn + token * F + 4 * part;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 cs = tr[e];
        float &a = INTERLEAVED ? x[2 * e] : x[e], &b = INTERLEAVED ? x[2 * e + 1] : x[4 + e];
        const float a0 = a;
        a = fmaf(a0, cs.x, -(b * cs.y));
        b = fmaf(a0, cs.y, b * cs.x);
      }
    }
    if (kind == 0) {
      T* dst = static_cast<T*>(p.oq) + (static_cast<int64_t>(first + token) * p.Hq + head) * D;
      if (here) {
        put4<T>(dst + one, x[0], x[1], x[2], x[3]);
        put4<T>(dst + two, x[4], x[5], x[6], x[7]);
      }
    } else {
      uint32_t codes[2];
      const float scale = quantize8<L>(x, codes);
      const int h = kind == 1 ? head - p.Hq : head - p.Hq - p.Hk;
      uint8_t* dst = (kind == 1 ? static_cast<uint8_t*>(p.ok) + h * p.ok_sh
                                : static_cast<uint8_t*>(p.ov) + h * p.ov_sh) + to[kind - 1][token];
      float* sc = (kind == 1 ? p.ks + h * p.ks_sh : p.vs + h * p.vs_sh) + scale_to[kind - 1][token];
      if (here && dest[token] >= 0) {
        *reinterpret_cast<uint32_t*>(dst + one) = codes[0];
        *reinterpret_cast<uint32_t*>(dst + two) = codes[1];
        if (part == 0) *sc = scale;
      }
    }
    head = next_head;
    chunk = next_chunk;
  }
}

template <typename T, int L, bool WIDE>
hipError_t launch_quantize(const RotaryParams& p, bool interleaved, hipStream_t stream) {
  const dim3 grid((p.tokens + p.per_group - 1) / p.per_group);
  RLM_TRY(check_launch("rotary_to_quantized_caches", grid.x, kThreads));
  if constexpr (WIDE) {
    if (p.per_group * L >= kWave) {
      if (interleaved)
        hipLaunchKernelGGL((rotary_quantize_tokens_kernel<T, L, true>), grid, dim3(kThreads), 0,
                           stream, p);
      else
        hipLaunchKernelGGL((rotary_quantize_tokens_kernel<T, L, false>), grid, dim3(kThreads), 0,
                           stream, p);
      return launch_status("rotary_to_quantized_caches");
    }
  }
  if (interleaved)
    hipLaunchKernelGGL((rotary_quantize_kernel<T, L, WIDE, true>), grid, dim3(kThreads), 0, stream,
                       p);
  else
    hipLaunchKernelGGL((rotary_quantize_kernel<T, L, WIDE, false>), grid, dim3(kThreads), 0, stream,
                       p);
  return launch_status("rotary_to_quantized_caches");
}

template <typename T, bool WIDE>
hipError_t launch_quantize_lanes(const RotaryParams& p, int lanes, bool interleaved,
                                 hipStream_t stream) {
  if (lanes <= 4) return launch_quantize<T, 4, WIDE>(p, interleaved, stream);
  if (lanes <= 8) return launch_quantize<T, 8, WIDE>(p, interleaved, stream);
  if (lanes <= 16) return launch_quantize<T, 16, WIDE>(p, interleaved, stream);
  return launch_quantize<T, 32, WIDE>(p, interleaved, stream);
}

// A 4-d tensor of unit stride in its last dim (the others as they come, 0 included: they
// are read only).
bool check_view(const rlm_tensor* t, const char* name, int64_t heads, int64_t B, int64_t Tq,
                int64_t D) {
  return check_strided(t, name, 4) && check_dim(t, name, 0, B) && check_dim(t, name, 1, Tq) &&
         (heads < 0 || check_dim(t, name, 2, heads)) && check_dim(t, name, 3, D);
}

bool wide_access(const rlm_tensor* t, int64_t per_vec, uintptr_t bytes = 16) {
  if ((reinterpret_cast<uintptr_t>(t->data) & (bytes - 1)) != 0) return false;
  for (int i = 0; i + 1 < t->ndim; ++i)
    if (t->shape[i] > 1 && t->stride[i] % per_vec != 0) return false;
  return true;
}

hipError_t rotary_common(const rlm_tensor* query, const rlm_tensor* key, const rlm_tensor* value,
                         const rlm_tensor* position, const rlm_tensor* frequencies,
                         const rlm_tensor* out_key, const rlm_tensor* out_value,
                         const rlm_tensor* key_scale, const rlm_tensor* value_scale,
                         bool quantized, const rlm_tensor* lengths, int32_t interleaved,
                         double scale, int32_t ring, const rlm_tensor* out_query,
                         hipStream_t stream) {
  const bool to_cache = value != nullptr;
  RLM_TRY(check_strided(query, "query", 4));
  RLM_TRY(check_dtype_float(query, "query"));
  const int64_t B = query->shape[0], Tq = query->shape[1], Hq = query->shape[2],
                D = query->shape[3];
  const int most = quantized ? kMaxQuantized : 1024;
  RLM_REQUIRE(D >= 1 && D <= most, "query: head dim must be in [1, %d], got %lld", most,
              (long long)D);
  RLM_TRY(check_view(key, "key", -1, B, Tq, D));
  RLM_TRY(check_same_dtype(key, "key", query, "query"));
  const int64_t Hk = key->shape[2];
  RLM_REQUIRE(Hq <= 4096 && Hk <= 4096, "at most 4096 heads (got %lld and %lld)", (long long)Hq,
              (long long)Hk);
  RLM_TRY(check_dense(frequencies, "frequencies", 1));
  RLM_TRY(check_dtype_is(frequencies, "frequencies", RLM_F32));
  const int64_t F = frequencies->shape[0];
  RLM_REQUIRE(F >= 1 && 2 * F <= D,
              "frequencies: one per pair, at least one and at most head dim / 2 = %lld, got %lld",
              (long long)(D / 2), (long long)F);
  RLM_TRY(check_dense(out_query, "out_query", 4));
  for (int i = 0; i < 4; ++i) RLM_TRY(check_dim(out_query, "out_query", i, query->shape[i]));
  RLM_TRY(check_same_dtype(out_query, "out_query", query, "query"));
  RLM_REQUIRE(B * Tq < (int64_t(1) << 31), "at most 2^31 - 1 tokens");

  RotaryParams p{};
  if (to_cache) {
    RLM_REQUIRE(position != nullptr && is_index_dtype(position->dtype),
                "position: expected an int32/int64 tensor");
    RLM_TRY(check_view(value, "value", Hk, B, Tq, D));
    RLM_TRY(check_same_dtype(value, "value", query, "query"));
    for (const rlm_tensor* c : {out_key, out_value}) {
      const char* name = c == out_key ? "key_cache" : "value_cache";
      RLM_TRY(check_strided(c, name, 4));
      RLM_TRY(check_no_overlap(c, name));
      if (quantized)
        RLM_TRY(check_dtype_is(c, name, RLM_F8E4M3));
      else
        RLM_TRY(check_same_dtype(c, name, query, "query"));
      RLM_TRY(check_dim(c, name, 0, B));
      RLM_TRY(check_dim(c, name, 2, Hk));
      RLM_TRY(check_dim(c, name, 3, D));
    }
    p.rows = out_key->shape[1];
    RLM_TRY(check_dim(out_value, "value_cache", 1, p.rows));
    if (quantized) {
      for (const rlm_tensor* s : {key_scale, value_scale}) {
        const char* name = s == key_scale ? "key_scale" : "value_scale";
        RLM_TRY(check_scales(s, name, B, p.rows, Hk));
        RLM_TRY(check_no_overlap(s, name));
      }
      p.ks = static_cast<float*>(key_scale->data);
      p.ks_sb = key_scale->stride[0], p.ks_st = key_scale->stride[1], p.ks_sh = key_scale->stride[2];
      p.vs = static_cast<float*>(value_scale->data);
      p.vs_sb = value_scale->stride[0], p.vs_st = value_scale->stride[1],
      p.vs_sh = value_scale->stride[2];
    }
    RLM_REQUIRE(!ring || (p.rows >= 1 && (p.rows & (p.rows - 1)) == 0),
                "ring-buffer caches need a power-of-two cache length, got %lld",
                (long long)p.rows);
    RLM_REQUIRE(!ring || Tq <= p.rows,
                "ring-buffer caches: %lld tokens at once would overwrite each other in %lld rows",
                (long long)Tq, (long long)p.rows);
    if (position->ndim == 0) {
      RLM_TRY(check_dense(position, "position", 0));
    } else {
      RLM_TRY(check_dense(position, "position", 1));
      RLM_TRY(check_dim(position, "position", 0, B));
      p.pos_sb = 1;
    }
    if (lengths != nullptr) {
      RLM_TRY(check_dense(lengths, "lengths", 1));
      RLM_TRY(check_dim(lengths, "lengths", 0, B));
      RLM_REQUIRE(is_index_dtype(lengths->dtype), "lengths: expected an int32/int64 tensor");
      p.lengths = lengths->data;
      p.lengths_dtype = lengths->dtype;
    }
    p.v = value->data;
    p.v_sb = value->stride[0], p.v_st = value->stride[1], p.v_sh = value->stride[2];
    p.ov = out_value->data;
    p.ov_sb = out_value->stride[0], p.ov_st = out_value->stride[1], p.ov_sh = out_value->stride[2];
  } else {
    RLM_TRY(check_dense(out_key, "out_key", 4));
    for (int i = 0; i < 4; ++i) RLM_TRY(check_dim(out_key, "out_key", i, key->shape[i]));
    RLM_TRY(check_same_dtype(out_key, "out_key", query, "query"));
    RLM_TRY(check_positions(position, "positions", B, Tq, &p.pos_sb, &p.pos_st));
  }
  p.q = query->data;
  p.q_sb = query->stride[0], p.q_st = query->stride[1], p.q_sh = query->stride[2];
  p.k = key->data;
  p.k_sb = key->stride[0], p.k_st = key->stride[1], p.k_sh = key->stride[2];
  p.oq = out_query->data;
  p.ok = out_key->data;
  p.ok_sb = out_key->stride[0], p.ok_st = out_key->stride[1], p.ok_sh = out_key->stride[2];
  p.pos = position->data;
  p.pos_dtype = position->dtype;
  p.freq = static_cast<const float*>(frequencies->data);
  p.scale = static_cast<float>(scale);
  p.tokens = static_cast<uint32_t>(B * Tq);
  p.Hq = static_cast<int>(Hq);
  p.Hk = static_cast<int>(Hk);
  p.D = static_cast<int>(D);
  p.F = static_cast<int>(F);
  p.heads = static_cast<int>(Hq + (to_cache ? 2 : 1) * Hk);
  p.to_cache = to_cache;
  p.ring = ring != 0;
  if (p.tokens == 0 || p.heads == 0) return hipSuccess;
  p.by_queries = FastDiv(static_cast<uint32_t>(Tq));
  p.by_pairs = FastDiv(static_cast<uint32_t>(F));
  const int elem = static_cast<int>(dtype_size(query->dtype));
  const int per_vec = 16 / elem;
  // Tokens of a workgroup: enough 16-byte accesses for eight rounds of its threads, so that
  // the angles' set-up is shared, but at least two workgroups per CU (a decode batch: one
  // token each).  Measured, one / four / sixteen tokens / this rule (us, bf16):
  //   16384 tokens of 12 + 4 heads of 64    17.4 / 12.4 / 12.7 / 12.6
  //    4096 tokens of the same               5.9 /  4.4 /  5.8 /  4.7
  //       8 tokens of 32 + 8 heads of 128    3.0 /  4.6 /  7.3 /  3.0
  const int lanes = static_cast<int>(D + 7) / 8;
  const int64_t work = static_cast<int64_t>(p.heads) *
                       (quantized ? lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32
                                  : (D + per_vec - 1) / per_vec);
  int64_t group = (8 * kThreads) / work;
  group = std::min<int64_t>(group, p.tokens / 512);
  group = std::min<int64_t>(group, std::min<int64_t>(kMaxTokens, kMaxAngles / F));
  p.per_group = static_cast<int>(std::max<int64_t>(group, 1));
  bool aligned = D % per_vec == 0 && (interleaved ? (2 * F) % per_vec == 0 : F % per_vec == 0);
  aligned = aligned && wide_access(query, per_vec) && wide_access(key, per_vec) &&
            wide_access(out_query, per_vec) && wide_access(out_key, per_vec) &&
            (!to_cache || (wide_access(value, per_vec) && wide_access(out_value, per_vec)));
  if (quantized) {
    p.by_heads = FastDiv(static_cast<uint32_t>(p.heads));
    // Eight features to a lane: whole accesses of them, and of their codes.
    const bool wide = D % 8 == 0 && (interleaved ? (2 * F) % 8 == 0 : F % 8 == 0) &&
                      wide_access(query, per_vec) && wide_access(key, per_vec) &&
                      wide_access(value, per_vec) && wide_access(out_query, per_vec) &&
                      wide_access(out_key, 8, 8) && wide_access(out_value, 8, 8);
    const int row_lanes = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32;
    const int together = kWave / row_lanes;
    // Many tokens: as many to a workgroup as a wave has at a time.  Measured, the rule above / these (us,
    // bf16; tokens of 12 + 4 + 4 heads of 64): 4096 8.6 / 8.7, 8192 14.9 / 10.6, 16384 20.1 / 16.1; of 32 + 8 + 8
    // of 128: 2048 13.2 / 14.7, 4096 22.4 / 19.4, 8000 45.3 / 35.8.
    if (wide && p.tokens / together >= 1024 && together * F <= kMaxAngles) p.per_group = together;
#define RLM_QUANTIZE(T)                                                          \
  return wide ? launch_quantize_lanes<T, true>(p, lanes, interleaved != 0, stream) \
              : launch_quantize_lanes<T, false>(p, lanes, interleaved != 0, stream);
    switch (query->dtype) {
      case RLM_F32: RLM_QUANTIZE(float)
      case RLM_BF16: RLM_QUANTIZE(bf16)
      default: RLM_QUANTIZE(f16)
    }
#undef RLM_QUANTIZE
  }
  switch (query->dtype) {
    case RLM_F32: return launch_rotary_type<float>(p, aligned, interleaved != 0, stream);
    case RLM_BF16: return launch_rotary_type<bf16>(p, aligned, interleaved != 0, stream);
    default: return launch_rotary_type<f16>(p, aligned, interleaved != 0, stream);
  }
}

}  // namespace
}  // namespace rlm

using namespace rlm;

extern "C" hipError_t rlm_rotary_positions(const rlm_tensor* query, const rlm_tensor* key,
                                           const rlm_tensor* positions,
                                           const rlm_tensor* frequencies, int32_t interleaved,
                                           double scale, const rlm_tensor* out_query,
                                           const rlm_tensor* out_key, hipStream_t stream) {
  clear_error();
  return rotary_common(query, key, nullptr, positions, frequencies, out_key, nullptr, nullptr,
                       nullptr, false, nullptr, interleaved, scale, 0, out_query, stream);
}

extern "C" hipError_t rlm_rotary_to_caches(
    const rlm_tensor* query, const rlm_tensor* key, const rlm_tensor* value,
    const rlm_tensor* position, const rlm_tensor* frequencies, const rlm_tensor* key_cache,
    const rlm_tensor* value_cache, const rlm_tensor* lengths, int32_t interleaved, double scale,
    int32_t ring, const rlm_tensor* out_query, hipStream_t stream) {
  clear_error();
  RLM_REQUIRE(value != nullptr, "value: missing tensor");
  return rotary_common(query, key, value, position, frequencies, key_cache, value_cache, nullptr,
                       nullptr, false, lengths, interleaved, scale, ring, out_query, stream);
}

extern "C" hipError_t rlm_rotary_to_quantized_caches(
    const rlm_tensor* query, const rlm_tensor* key, const rlm_tensor* value,
    const rlm_tensor* position, const rlm_tensor* frequencies, const rlm_tensor* key_cache,
    const rlm_tensor* value_cache, const rlm_tensor* key_scale, const rlm_tensor* value_scale,
    const rlm_tensor* lengths, int32_t interleaved, double scale, int32_t ring,
    const rlm_tensor* out_query, hipStream_t stream) {
  clear_error();
  RLM_REQUIRE(value != nullptr, "value: missing tensor");
  return rotary_common(query, key, value, position, frequencies, key_cache, value_cache, key_scale,
                       value_scale, true, lengths, interleaved, scale, ring, out_query, stream);
}
