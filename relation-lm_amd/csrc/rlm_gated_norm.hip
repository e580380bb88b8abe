// What stands between two blocks of a layer stack, in one pass over the rows:
//   hidden     = residual_scale * residual + sigmoid(gate) * post(branch)
//   normalized = norm(hidden)
// post is the norm after a block (or nothing), norm the next block's: LayerNorm
// (x - mean) / sqrt(var + eps) * w + b, or the root-mean-square norm x / sqrt(mean x^2 + eps)
// * w + b.  The second norm reads the fp32 sums, not the rounded hidden.
//
// Bound: memory, two rows read and two written for each row: 16384 rows of 768 bf16 features take
// 22.2 us, 4.5 TB/s, where a large copy reaches 4.7; few rows take the chain of their reads and four
// sums, 4.3 to 4.6 us for 8 of 576 by the profiler (3.9 at least).  The statistics are wave reductions over a row held in registers, the
// variance in a second sweep of those registers (no cancellation between mean x^2 and mean^2).
#include "rlm_common.hpp"

namespace rlm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxWidth = 8192;

enum GateForm { kGateOne = 0, kGateColumns = 1, kGateRows = 2 };

struct GatedNormParams {
  const void *branch, *residual, *gate;
  int64_t branch_s, residual_s, gate_s;  // row strides
  int gate_form, gate_dtype;
  const void *pw, *pb, *w, *b;           // pw, pb, b may be null
  int pw_dtype, pb_dtype, w_dtype, b_dtype;
  void *hidden, *normalized;
  int64_t rows;
  int D;
  float post_eps, eps, residual_scale;
  bool rms;
};

template <int BYTES>
struct Raw;
template <>
struct Raw<32> {
  struct type {
    uint4 lo, hi;
  };
};
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

template <typename T, int V>
struct Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[V]) {
  using raw_t = typename Raw<V * sizeof(T)>::type;
  const Vec<T, V> x = __builtin_bit_cast(Vec<T, V>, *reinterpret_cast<const raw_t*>(p));
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = to_f32(x.e[e]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  using raw_t = typename Raw<V * sizeof(T)>::type;
  Vec<T, V> x;
#pragma unroll
  for (int e = 0; e < V; ++e) x.e[e] = from_f32<T>(in[e]);
  *reinterpret_cast<raw_t*>(p) = __builtin_bit_cast(raw_t, x);
}

// Parameter vectors of any element type (W: their common type, or void where they differ).
template <typename W, int V>
__device__ __forceinline__ void load_param(const void* p, int dtype, int at, float (&out)[V]) {
  if constexpr (__is_same(W, void)) {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = load_any_f(p, dtype, at + e);
  } else {
    load_vec<W, V>(static_cast<const W*>(p) + at, out);
  }
}

// Sum over the R threads of a row, in every one of them and in one order for every launch.
template <int R>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  v = wave_sum_f32(v);
  if constexpr (R > kWave) {
    __syncthreads();  // the scratch of the sum before has been read
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
  }
  return v;
}

template <int R, int NV, int V>
__device__ __forceinline__ void normalize(float (&x)[NV][V], int D, int lane, bool rms, float eps,
                                          float* scratch) {
  float mean = 0.0f;
  if (!rms) {
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) sum += x[v][e];  // 0 past the row's end
    mean = row_sum<R>(sum, scratch) / static_cast<float>(D);
  }
  float square = 0.0f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if ((v * R + lane) * V < D) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[v][e] -= mean;
        square = fmaf(x[v][e], x[v][e], square);
      }
    }
  }
  const float inv = 1.0f / sqrtf(row_sum<R>(square, scratch) / static_cast<float>(D) + eps);
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < V; ++e) x[v][e] *= inv;
}

// R threads hold a row, NV accesses of V elements each; kThreads / R rows to a workgroup.
template <typename T, typename W, int V, int R, int NV>
__global__ __launch_bounds__(kThreads) void gated_norm_kernel(GatedNormParams p) {
  __shared__ float scratch[kThreads / kWave];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / R) + threadIdx.x / R;
  const int lane = threadIdx.x % R;
  if (row >= p.rows) return;  // whole rows: R == kThreads leaves with its whole workgroup
  const int D = p.D;
  const T* branch = static_cast<const T*>(p.branch) + row * p.branch_s;
  const T* residual = static_cast<const T*>(p.residual) + row * p.residual_s;
  float x[NV][V], res[NV][V];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * R + lane) * V;
    if (at < D) {
      load_vec<T, V>(branch + at, x[v]);
      load_vec<T, V>(residual + at, res[v]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x[v][e] = res[v][e] = 0.0f;
    }
  }
  const bool post = p.pw != nullptr;
  if (post) normalize<R, NV, V>(x, D, lane, p.rms, p.post_eps, scratch);
  float one = 0.0f;
  if (p.gate_form == kGateOne)
    one = 1.0f / (1.0f + expf(-load_any_f(p.gate, p.gate_dtype, 0)));
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * R + lane) * V;
    if (at >= D) continue;
    if (post) {
      float w[V];
      load_param<W, V>(p.pw, p.pw_dtype, at, w);
#pragma unroll
      for (int e = 0; e < V; ++e) x[v][e] *= w[e];
      if (p.pb != nullptr) {
        load_param<W, V>(p.pb, p.pb_dtype, at, w);
#pragma unroll
        for (int e = 0; e < V; ++e) x[v][e] += w[e];
      }
    }
    float g[V];
    if (p.gate_form == kGateOne) {
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = one;
    } else {
      if (p.gate_form == kGateRows)
        load_vec<T, V>(static_cast<const T*>(p.gate) + row * p.gate_s + at, g);
      else
        load_param<W, V>(p.gate, p.gate_dtype, at, g);
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = 1.0f / (1.0f + expf(-g[e]));
    }
#pragma unroll
    for (int e = 0; e < V; ++e) x[v][e] = fmaf(g[e], x[v][e], p.residual_scale * res[v][e]);
    store_vec<T, V>(static_cast<T*>(p.hidden) + row * D + at, x[v]);
  }
  normalize<R, NV, V>(x, D, lane, p.rms, p.eps, scratch);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * R + lane) * V;
    if (at >= D) continue;
    float w[V];
    load_param<W, V>(p.w, p.w_dtype, at, w);
#pragma unroll
    for (int e = 0; e < V; ++e) x[v][e] *= w[e];
    if (p.b != nullptr) {
      load_param<W, V>(p.b, p.b_dtype, at, w);
#pragma unroll
      for (int e = 0; e < V; ++e) x[v][e] += w[e];
    }
    store_vec<T, V>(static_cast<T*>(p.normalized) + row * D + at, x[v]);
  }
}

template <typename T, typename W, int V, int R, int NV>
hipError_t launch(const GatedNormParams& p, hipStream_t stream) {
  constexpr int kRows = kThreads / R;
  const dim3 grid(static_cast<unsigned>((p.rows + kRows - 1) / kRows));
  RLM_TRY(check_launch("gated_residual_norm", grid.x, kThreads));
  hipLaunchKernelGGL((gated_norm_kernel<T, W, V, R, NV>), grid, dim3(kThreads), 0, stream, p);
  return launch_status("gated_residual_norm");
}

// A row on one wave up to 4 accesses of each lane (a row's statistics then need no LDS), on the
// workgroup's four waves beyond, and already from 64 accesses on where there are few rows, each a
// chain of its own.  Measured, a row on a wave / on four (us, bf16, both norms):
//    576 features    8 rows: 4.5 / 3.5    512: 4.7 / 4.0    1024: 4.9 / 4.7    4096: 7.3 / 11.0
//   2048 features    8 rows: 6.1 / 3.6    512: 6.9 / 4.4    1024: 7.6 / 6.0    4096: 15.7 / 16.3
//   4096 features    8 rows: 9.7 / 4.8    512: 11.3 / 6.4   4096: 31.9 / 26.7  16384: 133 / 111
constexpr int kFewRows = 1024;
template <typename T, typename W>
hipError_t launch_wide(const GatedNormParams& p, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int accesses = p.D / V;
  if (accesses <= 1 * kWave) return launch<T, W, V, kWave, 1>(p, stream);
  if (p.rows <= kFewRows && accesses <= kThreads) return launch<T, W, V, kThreads, 1>(p, stream);
  if (accesses <= 2 * kWave) return launch<T, W, V, kWave, 2>(p, stream);
  if (accesses <= 4 * kWave) return launch<T, W, V, kWave, 4>(p, stream);
  if (accesses <= 2 * kThreads) return launch<T, W, V, kThreads, 2>(p, stream);
  if (accesses <= 4 * kThreads) return launch<T, W, V, kThreads, 4>(p, stream);
  return launch<T, W, V, kThreads, 8>(p, stream);
}
// Widths, strides or addresses that are not whole 16-byte accesses: an element each, with a switch on
// each parameter's type.  Measured (us, bf16 rows, both norms, parameters bf16 or fp32 / some of each):
//   16384 rows of 768 features: 22.8 / 77    of 767: 57    4096 of 2048: 17.5 / 54    of 2047: 32
// so parameters of one type are what whole accesses want: with some of each they still read the rows
// whole, but switch for every element of every parameter.
template <typename T>
hipError_t launch_narrow(const GatedNormParams& p, hipStream_t stream) {
  if (p.D <= 8 * kWave) return launch<T, void, 1, kWave, 8>(p, stream);
  if (p.D <= 8 * kThreads) return launch<T, void, 1, kThreads, 8>(p, stream);
  return launch<T, void, 1, kThreads, 32>(p, stream);
}

template <typename T>
hipError_t launch_type(const GatedNormParams& p, int dtype, int param_dtype, bool aligned,
                       hipStream_t stream) {
  if (!aligned) return launch_narrow<T>(p, stream);
  if (param_dtype == dtype) return launch_wide<T, T>(p, stream);
  if (param_dtype == RLM_F32) return launch_wide<T, float>(p, stream);
  return launch_wide<T, void>(p, stream);
}

}  // namespace
}  // namespace rlm

using namespace rlm;

extern "C" hipError_t rlm_gated_residual_norm(
    const rlm_tensor* branch, const rlm_tensor* residual, const rlm_tensor* gate,
    const rlm_tensor* norm_weight, const rlm_tensor* norm_bias, double norm_eps,
    const rlm_tensor* post_weight, const rlm_tensor* post_bias, double post_eps,
    double residual_scale, int32_t rms, const rlm_tensor* out_hidden,
    const rlm_tensor* out_normalized, hipStream_t stream) {
  clear_error();
  RLM_TRY(check_rows(branch, "branch"));
  RLM_TRY(check_dtype_float(branch, "branch"));
  const int64_t N = branch->shape[0], D = branch->shape[1];
  RLM_REQUIRE(D >= 1 && D <= kMaxWidth, "branch: width must be in [1, %d], got %lld", kMaxWidth,
              (long long)D);
  RLM_TRY(check_rows(residual, "residual"));
  RLM_TRY(check_same_dtype(residual, "residual", branch, "branch"));
  for (const rlm_tensor* t : {residual, out_hidden, out_normalized}) {
    const char* name = t == residual ? "residual" : t == out_hidden ? "out_hidden"
                                                                    : "out_normalized";
    if (t != residual) {
      RLM_TRY(check_dense(t, name, 2));
      RLM_TRY(check_same_dtype(t, name, branch, "branch"));
    }
    RLM_TRY(check_dim(t, name, 0, N));
    RLM_TRY(check_dim(t, name, 1, D));
  }
  GatedNormParams p{};
  const int elem = static_cast<int>(dtype_size(branch->dtype));
  const int per_vec = 16 / elem;
  bool aligned = D % per_vec == 0;
  auto aligned_rows = [&](const rlm_tensor* t) {
    return (reinterpret_cast<uintptr_t>(t->data) & 15u) == 0 &&
           (N <= 1 || t->stride[0] % per_vec == 0);
  };
  for (const rlm_tensor* t : {branch, residual, out_hidden, out_normalized})
    aligned = aligned && aligned_rows(t);

  // Parameter vectors: any element type each; one common type (that of the rows, or fp32) is
  // read with whole accesses.
  int param_dtype = -1;
  auto take = [&](const rlm_tensor* t, const char* name, const void** data, int* dtype) {
    if (!check_dense(t, name, 1) || !check_dtype_float(t, name) || !check_dim(t, name, 0, D))
      return false;
    *data = t->data;
    *dtype = t->dtype;
    param_dtype = param_dtype == -1 || param_dtype == t->dtype ? t->dtype : -2;
    if ((reinterpret_cast<uintptr_t>(t->data) & 15u) != 0) param_dtype = -2;
    return true;
  };
  RLM_TRY(take(norm_weight, "norm_weight", &p.w, &p.w_dtype));
  if (norm_bias != nullptr) RLM_TRY(take(norm_bias, "norm_bias", &p.b, &p.b_dtype));
  RLM_REQUIRE(post_weight != nullptr || post_bias == nullptr,
              "post_bias: needs a post_weight beside it");
  if (post_weight != nullptr) RLM_TRY(take(post_weight, "post_weight", &p.pw, &p.pw_dtype));
  if (post_bias != nullptr) RLM_TRY(take(post_bias, "post_bias", &p.pb, &p.pb_dtype));
  RLM_REQUIRE(gate != nullptr, "gate: missing tensor");
  if (gate->ndim == 0) {
    RLM_TRY(check_dense(gate, "gate", 0));
    RLM_TRY(check_dtype_float(gate, "gate"));
    p.gate_form = kGateOne;
    p.gate = gate->data;
    p.gate_dtype = gate->dtype;
  } else if (gate->ndim == 1) {
    p.gate_form = kGateColumns;
    RLM_TRY(take(gate, "gate", &p.gate, &p.gate_dtype));
  } else {
    RLM_TRY(check_rows(gate, "gate"));
    RLM_TRY(check_same_dtype(gate, "gate", branch, "branch"));
    RLM_TRY(check_dim(gate, "gate", 0, N));
    RLM_TRY(check_dim(gate, "gate", 1, D));
    p.gate_form = kGateRows;
    p.gate = gate->data;
    p.gate_s = gate->stride[0];
    aligned = aligned && aligned_rows(gate);
  }
  RLM_REQUIRE((N + 3) / 4 < (int64_t(1) << 31) && N < (int64_t(1) << 31), "at most 2^31 - 1 rows");
  p.branch = branch->data;
  p.branch_s = branch->stride[0];
  p.residual = residual->data;
  p.residual_s = residual->stride[0];
  p.hidden = out_hidden->data;
  p.normalized = out_normalized->data;
  p.rows = N;
  p.D = static_cast<int>(D);
  p.post_eps = static_cast<float>(post_eps);
  p.eps = static_cast<float>(norm_eps);
  p.residual_scale = static_cast<float>(residual_scale);
  p.rms = rms != 0;
  if (N == 0) return hipSuccess;
  switch (branch->dtype) {
    case RLM_F32: return launch_type<float>(p, RLM_F32, param_dtype, aligned, stream);
    case RLM_BF16: return launch_type<bf16>(p, RLM_BF16, param_dtype, aligned, stream);
    default: return launch_type<f16>(p, RLM_F16, param_dtype, aligned, stream);
  }
}
