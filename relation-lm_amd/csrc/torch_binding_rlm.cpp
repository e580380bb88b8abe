// PyTorch-ROCm registration of the routed attention layer's operators, in the namespace `rlm`,
// and of its forms for caches of 8 bits and weights of 4, in `rlm_quantized` (operators that the
// reference has no counterpart of; its own names and schemas are relation_lm:: and
// relationlex::).  Outputs come from the caching allocator on the input
// device, every kernel goes on the current HIP stream.
#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "torch_binding_util.hpp"

namespace {

// The descriptor of `t` with a dim of size 1 put in before dim `at` (decode forms take the
// sequence forms' entry points with one query).
rlm_tensor with_dim(const at::Tensor& t, const char* name, int64_t at) {
  TORCH_CHECK(t.defined() && t.dim() >= at && t.dim() < RLM_MAX_DIMS, name,
              ": expected a tensor of ", at, " to ", RLM_MAX_DIMS - 1, " dims");
  rlm_tensor d = desc(t, name);
  for (int64_t i = d.ndim; i > at; --i) {
    d.shape[i] = d.shape[i - 1];
    d.stride[i] = d.stride[i - 1];
  }
  d.shape[at] = 1;
  d.stride[at] = 1;
  ++d.ndim;
  return d;
}

// Positions of a decode form: 0-d, or one per batch row ([B] read as [B,1]).
rlm_tensor decode_position(const at::Tensor& t, const char* name) {
  return t.dim() == 0 ? desc(t, name) : with_dim(t, name, 1);
}

std::tuple<at::Tensor, at::Tensor> rotary_positions(const at::Tensor& query, const at::Tensor& key,
                                                    const at::Tensor& positions,
                                                    const at::Tensor& frequencies,
                                                    bool interleaved, double scale) {
  const char* op = "rlm::rotary_positions";
  c10::DeviceGuard guard(query.device());
  hipStream_t stream = device_stream(op, {&query, &key, &positions, &frequencies});
  at::Tensor out_query = at::empty(query.sizes(), query.options());
  at::Tensor out_key = at::empty(key.sizes(), key.options());
  const rlm_tensor d[6] = {desc(query, "query"),           desc(key, "key"),
                           desc(positions, "positions"),   desc(frequencies, "frequencies"),
                           desc(out_query, "out_query"),   desc(out_key, "out_key")};
  check(rlm_rotary_positions(&d[0], &d[1], &d[2], &d[3], interleaved ? 1 : 0, scale, &d[4], &d[5],
                             stream),
        op);
  return {out_query, out_key};
}

at::Tensor rotary_to_caches(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
                            const at::Tensor& position, const at::Tensor& frequencies,
                            const at::Tensor& key_cache, const at::Tensor& value_cache,
                            bool interleaved, double scale, bool ring,
                            const std::optional<at::Tensor>& lengths) {
  const char* op = "rlm::rotary_to_caches";
  c10::DeviceGuard guard(query.device());
  const at::Tensor none;
  const at::Tensor& len = lengths.has_value() ? *lengths : none;
  hipStream_t stream = device_stream(
      op, {&query, &key, &value, &position, &frequencies, &key_cache, &value_cache, &len});
  at::Tensor out_query = at::empty(query.sizes(), query.options());
  const rlm_tensor d[8] = {desc(query, "query"),         desc(key, "key"),
                           desc(value, "value"),         desc(position, "position"),
                           desc(frequencies, "frequencies"), desc(key_cache, "key_cache"),
                           desc(value_cache, "value_cache"), desc(out_query, "out_query")};
  rlm_tensor dl{};
  if (len.defined()) dl = desc(len, "lengths");
  check(rlm_rotary_to_caches(&d[0], &d[1], &d[2], &d[3], &d[4], &d[5], &d[6],
                             len.defined() ? &dl : nullptr, interleaved ? 1 : 0, scale,
                             ring ? 1 : 0, &d[7], stream),
        op);
  return out_query;
}

at::Tensor rotary_to_quantized_caches(
    const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
    const at::Tensor& position, const at::Tensor& frequencies, const at::Tensor& key_cache,
    const at::Tensor& value_cache, const at::Tensor& key_scale, const at::Tensor& value_scale,
    bool interleaved, double scale, bool ring, const std::optional<at::Tensor>& lengths) {
  const char* op = "rlm_quantized::rotary_to_quantized_caches";
  c10::DeviceGuard guard(query.device());
  const at::Tensor none;
  const at::Tensor& len = lengths.has_value() ? *lengths : none;
  hipStream_t stream =
      device_stream(op, {&query, &key, &value, &position, &frequencies, &key_cache, &value_cache,
                         &key_scale, &value_scale, &len});
  at::Tensor out_query = at::empty(query.sizes(), query.options());
  const rlm_tensor d[10] = {desc(query, "query"),
                            desc(key, "key"),
                            desc(value, "value"),
                            desc(position, "position"),
                            desc(frequencies, "frequencies"),
                            codes_desc(key_cache, "key_cache"),
                            codes_desc(value_cache, "value_cache"),
                            desc(key_scale, "key_scale"),
                            desc(value_scale, "value_scale"),
                            desc(out_query, "out_query")};
  rlm_tensor dl{};
  if (len.defined()) dl = desc(len, "lengths");
  check(rlm_rotary_to_quantized_caches(&d[0], &d[1], &d[2], &d[3], &d[4], &d[5], &d[6], &d[7], &d[8],
                                       len.defined() ? &dl : nullptr, interleaved ? 1 : 0, scale,
                                       ring ? 1 : 0, &d[9], stream),
        op);
  return out_query;
}

at::Tensor quantized_rows(const at::Tensor& cache, const at::Tensor& scale,
                          const std::optional<at::Tensor>& rows, at::ScalarType dtype) {
  const char* op = "rlm_quantized::quantized_rows";
  c10::DeviceGuard guard(cache.device());
  const at::Tensor none;
  const at::Tensor& named = rows.has_value() ? *rows : none;
  hipStream_t stream = device_stream(op, {&cache, &scale, &named});
  TORCH_CHECK(cache.dim() == 4, op, ": cache must be [B,T,Hk,D]");
  TORCH_CHECK(!named.defined() || named.dim() == 2, op, ": rows must be [B,N]");
  TORCH_CHECK(dtype == at::kFloat || dtype == at::kBFloat16 || dtype == at::kHalf, op,
              ": dtype must be float32, bfloat16 or float16, got ", dtype);
  at::Tensor out = at::empty({cache.size(0), named.defined() ? named.size(1) : cache.size(1),
                              cache.size(2), cache.size(3)},
                             cache.options().dtype(dtype));
  const rlm_tensor d[3] = {codes_desc(cache, "cache"), desc(scale, "scale"), desc(out, "out")};
  rlm_tensor dr{};
  if (named.defined()) dr = desc(named, "rows");
  check(rlm_quantized_rows(&d[0], &d[1], named.defined() ? &dr : nullptr, &d[2], stream), op);
  return out;
}

std::tuple<at::Tensor, at::Tensor> block_route_common(
    const char* op, bool seq, const at::Tensor& router_query, const at::Tensor& block_mean,
    const at::Tensor& block_std, const at::Tensor& gamma, const at::Tensor& bias,
    const at::Tensor& positions, int64_t block_size, int64_t local_window, int64_t top_blocks,
    bool strict_valid, bool ring) {
  c10::DeviceGuard guard(router_query.device());
  hipStream_t stream = device_stream(
      op, {&router_query, &block_mean, &block_std, &gamma, &bias, &positions});
  const int64_t lead = seq ? 2 : 1;
  TORCH_CHECK(router_query.dim() == lead + 1 || router_query.dim() == lead + 2, op,
              ": router_query must be ", seq ? "[B,Tq,RD] or [B,Tq,S,RD]" : "[B,RD] or [B,S,RD]");
  TORCH_CHECK(top_blocks >= 1, op, ": top_blocks must be positive");
  std::vector<int64_t> shape(router_query.sizes().begin(), router_query.sizes().end());
  shape.back() = top_blocks;
  at::Tensor blocks = at::empty(shape, i32(router_query));
  at::Tensor scores = at::empty(shape, f32(router_query));
  const bool slots = router_query.dim() == lead + 2;
  auto full = [&](const at::Tensor& t, const char* name) {
    rlm_tensor d = seq ? desc(t, name) : with_dim(t, name, 1);
    if (!slots) {  // [B,Tq,n] -> [B,Tq,1,n]
      d.shape[3] = d.shape[2];
      d.stride[3] = d.stride[2];
      d.shape[2] = d.stride[2] = 1;
      d.ndim = 4;
    }
    return d;
  };
  const rlm_tensor d[8] = {
      full(router_query, "router_query"), desc(block_mean, "block_mean"),
      desc(block_std, "block_std"),       desc(gamma, "gamma"),
      desc(bias, "bias"),
      seq ? desc(positions, "positions") : decode_position(positions, "position"),
      full(blocks, "blocks"),             full(scores, "scores")};
  check(rlm_block_route(&d[0], &d[1], &d[2], &d[3], &d[4], &d[5], block_size, local_window,
                        top_blocks, strict_valid ? 1 : 0, ring ? 1 : 0, &d[6], &d[7], stream),
        op);
  return {blocks, scores};
}

std::tuple<at::Tensor, at::Tensor> block_route(
    const at::Tensor& router_query, const at::Tensor& block_mean, const at::Tensor& block_std,
    const at::Tensor& gamma, const at::Tensor& bias, const at::Tensor& position,
    int64_t block_size, int64_t local_window, int64_t top_blocks, bool strict_valid, bool ring) {
  return block_route_common("rlm::block_route", false, router_query, block_mean, block_std, gamma,
                            bias, position, block_size, local_window, top_blocks, strict_valid,
                            ring);
}

std::tuple<at::Tensor, at::Tensor> block_route_seq(
    const at::Tensor& router_query, const at::Tensor& block_mean, const at::Tensor& block_std,
    const at::Tensor& gamma, const at::Tensor& bias, const at::Tensor& positions,
    int64_t block_size, int64_t local_window, int64_t top_blocks, bool strict_valid) {
  return block_route_common("rlm::block_route_seq", true, router_query, block_mean, block_std,
                            gamma, bias, positions, block_size, local_window, top_blocks,
                            strict_valid, false);
}

// key_scale and value_scale: undefined, or those of 8-bit caches.
std::tuple<at::Tensor, at::Tensor> routed_attention_common(
    const char* op, bool seq, const at::Tensor& query, const at::Tensor& key_cache,
    const at::Tensor& value_cache, const at::Tensor& key_scale, const at::Tensor& value_scale,
    const at::Tensor& blocks, const at::Tensor& positions, int64_t block_size,
    int64_t local_window, std::optional<double> scale, bool ring) {
  c10::DeviceGuard guard(query.device());
  hipStream_t stream = device_stream(
      op, {&query, &key_cache, &value_cache, &key_scale, &value_scale, &blocks, &positions});
  const int64_t lead = seq ? 2 : 1;
  TORCH_CHECK(query.dim() == lead + 2, op, ": query must be ",
              seq ? "[B,Tq,Hq,D]" : "[B,Hq,D]");
  TORCH_CHECK(blocks.dim() == lead + 1 || blocks.dim() == lead + 2, op, ": blocks must be ",
              seq ? "[B,Tq,TOP] or [B,Tq,Hk,TOP]" : "[B,TOP] or [B,Hk,TOP]");
  at::Tensor out = at::empty(query.sizes(), query.options());
  at::Tensor lse = at::empty(query.sizes().slice(0, lead + 1), f32(query));
  const int64_t width = query.size(-1);
  auto full = [&](const at::Tensor& t, const char* name) {
    return seq ? desc(t, name) : with_dim(t, name, 1);
  };
  const bool quantized = key_scale.defined();
  auto cache = [&](const at::Tensor& t, const char* name) {
    return quantized ? codes_desc(t, name) : desc(t, name);
  };
  const rlm_tensor d[7] = {
      full(query, "query"),   cache(key_cache, "key_cache"), cache(value_cache, "value_cache"),
      full(blocks, "blocks"), seq ? desc(positions, "positions") : decode_position(positions, "position"),
      full(out, "out"),       full(lse, "lse")};
  const double factor =
      scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(width, 1)));
  if (quantized) {
    const rlm_tensor s[2] = {desc(key_scale, "key_scale"), desc(value_scale, "value_scale")};
    check(rlm_routed_attention_quantized(&d[0], &d[1], &d[2], &s[0], &s[1], &d[3], &d[4], block_size,
                                         local_window, factor, ring ? 1 : 0, &d[5], &d[6], stream),
          op);
  } else {
    check(rlm_routed_attention(&d[0], &d[1], &d[2], &d[3], &d[4], block_size, local_window, factor,
                               ring ? 1 : 0, &d[5], &d[6], stream),
          op);
  }
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> routed_attention(
    const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
    const at::Tensor& blocks, const at::Tensor& position, int64_t block_size, int64_t local_window,
    std::optional<double> scale, bool ring) {
  return routed_attention_common("rlm::routed_attention", false, query, key_cache, value_cache, {},
                                 {}, blocks, position, block_size, local_window, scale, ring);
}

std::tuple<at::Tensor, at::Tensor> routed_attention_seq(
    const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
    const at::Tensor& blocks, const at::Tensor& positions, int64_t block_size,
    int64_t local_window, std::optional<double> scale) {
  return routed_attention_common("rlm::routed_attention_seq", true, query, key_cache, value_cache,
                                 {}, {}, blocks, positions, block_size, local_window, scale, false);
}

std::tuple<at::Tensor, at::Tensor> routed_attention_quantized(
    const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
    const at::Tensor& key_scale, const at::Tensor& value_scale, const at::Tensor& blocks,
    const at::Tensor& position, int64_t block_size, int64_t local_window,
    std::optional<double> scale, bool ring) {
  return routed_attention_common("rlm_quantized::routed_attention_quantized", false, query, key_cache,
                                 value_cache, key_scale, value_scale, blocks, position, block_size,
                                 local_window, scale, ring);
}

std::tuple<at::Tensor, at::Tensor> routed_attention_quantized_seq(
    const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
    const at::Tensor& key_scale, const at::Tensor& value_scale, const at::Tensor& blocks,
    const at::Tensor& positions, int64_t block_size, int64_t local_window,
    std::optional<double> scale) {
  return routed_attention_common("rlm_quantized::routed_attention_quantized_seq", true, query, key_cache,
                                 value_cache, key_scale, value_scale, blocks, positions, block_size,
                                 local_window, scale, false);
}

// Any leading dims as rows: a view where the strides allow one, else a copy.
at::Tensor as_rows(const at::Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

std::tuple<at::Tensor, at::Tensor> gated_residual_norm(
    const at::Tensor& branch, const at::Tensor& residual, const at::Tensor& gate,
    const at::Tensor& norm_weight, const std::optional<at::Tensor>& norm_bias, double norm_eps,
    const std::optional<at::Tensor>& post_weight, const std::optional<at::Tensor>& post_bias,
    double residual_scale, bool rms, std::optional<double> post_eps) {
  const char* op = "rlm::gated_residual_norm";
  c10::DeviceGuard guard(branch.device());
  const at::Tensor none;
  auto given = [&](const std::optional<at::Tensor>& t) -> const at::Tensor& {
    return t.has_value() ? *t : none;
  };
  const at::Tensor &nb = given(norm_bias), &pw = given(post_weight), &pb = given(post_bias);
  hipStream_t stream =
      device_stream(op, {&branch, &residual, &gate, &norm_weight, &nb, &pw, &pb});
  TORCH_CHECK(branch.dim() >= 1 && branch.size(-1) >= 1, op,
              ": branch must have at least one dimension, of at least one element");
  TORCH_CHECK(residual.sizes() == branch.sizes(), op, ": residual must have branch's shape");
  TORCH_CHECK(gate.dim() <= 1 || gate.sizes() == branch.sizes(), op,
              ": gate must be 0-d, [D] or of branch's shape");
  at::Tensor hidden = at::empty(branch.sizes(), branch.options());
  at::Tensor normalized = at::empty(branch.sizes(), branch.options());
  const at::Tensor x = as_rows(branch), r = as_rows(residual);
  const at::Tensor g = gate.dim() > 1 ? as_rows(gate) : gate;
  const at::Tensor h = as_rows(hidden), n = as_rows(normalized);
  const rlm_tensor d[6] = {desc(x, "branch"),           desc(r, "residual"),
                           desc(g, "gate"),             desc(norm_weight, "norm_weight"),
                           desc(h, "hidden"),           desc(n, "normalized")};
  rlm_tensor dn{}, dw{}, db{};
  if (nb.defined()) dn = desc(nb, "norm_bias");
  if (pw.defined()) dw = desc(pw, "post_weight");
  if (pb.defined()) db = desc(pb, "post_bias");
  check(rlm_gated_residual_norm(&d[0], &d[1], &d[2], &d[3], nb.defined() ? &dn : nullptr, norm_eps,
                                pw.defined() ? &dw : nullptr, pb.defined() ? &db : nullptr,
                                post_eps.value_or(norm_eps), residual_scale, rms ? 1 : 0, &d[4],
                                &d[5], stream),
        op);
  return {hidden, normalized};
}

// Leading dims of a product's input, with N outputs as the last.
std::vector<int64_t> product_shape(const char* op, const at::Tensor& input, const at::Tensor& scales,
                                   const char* scales_name) {
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) >= 1, op,
              ": input must have at least one dimension, of at least one element");
  TORCH_CHECK(scales.dim() == 2, op, ": ", scales_name, " must be [groups, N]");
  std::vector<int64_t> shape(input.sizes().begin(), input.sizes().end());
  shape.back() = scales.size(1);
  return shape;
}

at::Tensor linear_4bit(const at::Tensor& input, const at::Tensor& codes, const at::Tensor& scales,
                       const std::optional<at::Tensor>& zeros, int64_t group_size,
                       const std::optional<at::Tensor>& bias) {
  const char* op = "rlm_quantized::linear_4bit";
  c10::DeviceGuard guard(input.device());
  const at::Tensor none;
  const at::Tensor &z = zeros.has_value() ? *zeros : none, &add = bias.has_value() ? *bias : none;
  hipStream_t stream = device_stream(op, {&input, &codes, &scales, &z, &add});
  at::Tensor out = at::empty(product_shape(op, input, scales, "scales"), input.options());
  const at::Tensor x = as_rows(input), y = as_rows(out);
  const rlm_tensor d[4] = {desc(x, "input"), desc(codes, "codes"), desc(scales, "scales"),
                           desc(y, "out")};
  rlm_tensor dz{}, db{};
  if (z.defined()) dz = desc(z, "zeros");
  if (add.defined()) db = desc(add, "bias");
  check(rlm_linear_4bit(&d[0], &d[1], &d[2], z.defined() ? &dz : nullptr, group_size,
                        add.defined() ? &db : nullptr, &d[3], stream),
        op);
  return out;
}

at::Tensor gated_linear_4bit(const at::Tensor& input, const at::Tensor& gate_codes,
                             const at::Tensor& gate_scales, const at::Tensor& up_codes,
                             const at::Tensor& up_scales,
                             const std::optional<at::Tensor>& gate_zeros,
                             const std::optional<at::Tensor>& up_zeros, int64_t group_size,
                             c10::string_view activation) {
  const char* op = "rlm_quantized::gated_linear_4bit";
  c10::DeviceGuard guard(input.device());
  const at::Tensor none;
  const at::Tensor& gz = gate_zeros.has_value() ? *gate_zeros : none;
  const at::Tensor& uz = up_zeros.has_value() ? *up_zeros : none;
  hipStream_t stream = device_stream(
      op, {&input, &gate_codes, &gate_scales, &up_codes, &up_scales, &gz, &uz});
  TORCH_CHECK(activation == "silu" || activation == "gelu", op,
              ": activation must be \"silu\" or \"gelu\", got \"", activation, "\"");
  at::Tensor out = at::empty(product_shape(op, input, gate_scales, "gate_scales"), input.options());
  const at::Tensor x = as_rows(input), y = as_rows(out);
  const rlm_tensor d[6] = {desc(x, "input"),
                           desc(gate_codes, "gate_codes"),
                           desc(gate_scales, "gate_scales"),
                           desc(up_codes, "up_codes"),
                           desc(up_scales, "up_scales"),
                           desc(y, "out")};
  rlm_tensor dg{}, du{};
  if (gz.defined()) dg = desc(gz, "gate_zeros");
  if (uz.defined()) du = desc(uz, "up_zeros");
  check(rlm_gated_linear_4bit(&d[0], &d[1], &d[2], gz.defined() ? &dg : nullptr, &d[3], &d[4],
                              uz.defined() ? &du : nullptr, group_size, activation == "silu" ? 0 : 1,
                              &d[5], stream),
        op);
  return out;
}

}  // namespace

TORCH_LIBRARY(rlm, m) {
  m.def(
      "rotary_positions(Tensor query, Tensor key, Tensor positions, Tensor frequencies, bool "
      "interleaved=False, float scale=1.0) -> (Tensor, Tensor)");
  m.def(
      "rotary_to_caches(Tensor query, Tensor key, Tensor value, Tensor position, Tensor "
      "frequencies, Tensor(a!) key_cache, Tensor(b!) value_cache, bool interleaved=False, float "
      "scale=1.0, bool ring=False, Tensor? lengths=None) -> Tensor");
  m.def(
      "block_route(Tensor router_query, Tensor block_mean, Tensor block_std, Tensor gamma, Tensor "
      "bias, Tensor position, SymInt block_size, SymInt local_window, SymInt top_blocks, bool "
      "strict_valid, bool ring=False) -> (Tensor, Tensor)");
  m.def(
      "block_route_seq(Tensor router_query, Tensor block_mean, Tensor block_std, Tensor gamma, "
      "Tensor bias, Tensor positions, SymInt block_size, SymInt local_window, SymInt top_blocks, "
      "bool strict_valid) -> (Tensor, Tensor)");
  m.def(
      "routed_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor blocks, Tensor "
      "position, SymInt block_size, SymInt local_window, float? scale=None, bool ring=False) -> "
      "(Tensor, Tensor)");
  m.def(
      "routed_attention_seq(Tensor query, Tensor key_cache, Tensor value_cache, Tensor blocks, "
      "Tensor positions, SymInt block_size, SymInt local_window, float? scale=None) -> (Tensor, "
      "Tensor)");
  m.def(
      "gated_residual_norm(Tensor branch, Tensor residual, Tensor gate, Tensor norm_weight, Tensor? "
      "norm_bias, float norm_eps, Tensor? post_weight=None, Tensor? post_bias=None, float "
      "residual_scale=1.0, bool rms=False, float? post_eps=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(rlm, CUDA, m) {
  m.impl("rotary_positions", TORCH_FN(rotary_positions));
  m.impl("rotary_to_caches", TORCH_FN(rotary_to_caches));
  m.impl("block_route", TORCH_FN(block_route));
  m.impl("block_route_seq", TORCH_FN(block_route_seq));
  m.impl("routed_attention", TORCH_FN(routed_attention));
  m.impl("routed_attention_seq", TORCH_FN(routed_attention_seq));
  m.impl("gated_residual_norm", TORCH_FN(gated_residual_norm));
}

TORCH_LIBRARY(rlm_quantized, m) {
  m.def(
      "rotary_to_quantized_caches(Tensor query, Tensor key, Tensor value, Tensor position, Tensor "
      "frequencies, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor(c!) key_scale, Tensor(d!) "
      "value_scale, bool interleaved=False, float scale=1.0, bool ring=False, Tensor? lengths=None) "
      "-> Tensor");
  m.def(
      "quantized_rows(Tensor cache, Tensor scale, Tensor? rows=None, ScalarType dtype=bfloat16) -> "
      "Tensor");
  m.def(
      "routed_attention_quantized(Tensor query, Tensor key_cache, Tensor value_cache, Tensor "
      "key_scale, Tensor value_scale, Tensor blocks, Tensor position, SymInt block_size, SymInt "
      "local_window, float? scale=None, bool ring=False) -> (Tensor, Tensor)");
  m.def(
      "routed_attention_quantized_seq(Tensor query, Tensor key_cache, Tensor value_cache, Tensor "
      "key_scale, Tensor value_scale, Tensor blocks, Tensor positions, SymInt block_size, SymInt "
      "local_window, float? scale=None) -> (Tensor, Tensor)");
  m.def(
      "linear_4bit(Tensor input, Tensor codes, Tensor scales, Tensor? zeros=None, SymInt "
      "group_size=128, Tensor? bias=None) -> Tensor");
  m.def(
      "gated_linear_4bit(Tensor input, Tensor gate_codes, Tensor gate_scales, Tensor up_codes, "
      "Tensor up_scales, Tensor? gate_zeros=None, Tensor? up_zeros=None, SymInt group_size=128, str "
      "activation=\"silu\") -> Tensor");
}

TORCH_LIBRARY_IMPL(rlm_quantized, CUDA, m) {
  m.impl("rotary_to_quantized_caches", TORCH_FN(rotary_to_quantized_caches));
  m.impl("quantized_rows", TORCH_FN(quantized_rows));
  m.impl("routed_attention_quantized", TORCH_FN(routed_attention_quantized));
  m.impl("routed_attention_quantized_seq", TORCH_FN(routed_attention_quantized_seq));
  m.impl("linear_4bit", TORCH_FN(linear_4bit));
  m.impl("gated_linear_4bit", TORCH_FN(gated_linear_4bit));
}
