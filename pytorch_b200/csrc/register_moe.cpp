// PyTorch registration of the mixture-of-experts block operators, in the same way as register.cpp: schemas, CUDA and
// Meta implementations over the C ABI, and autograd functions whose backward passes are operators of their own
// (npu_moe_token_permute_grad, npu_moe_token_unpermute_grad).  A call that needs no gradient goes straight to the
// CUDA implementation.
#include <torch/csrc/autograd/custom_function.h>

#include "register_common.h"

namespace {

using namespace b200q_torch;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// npu_moe_token_permute takes indices below this and sorts for all of them, as it is not told how many experts there are: the routing of
// 8192 x 8 indices, which is told, takes 19.8 us for 8 experts and 21.0 for 1024.
constexpr int64_t kPermuteExperts = 1024;

bool is_float_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

// A gradient that would itself be differentiated.
void no_second_derivative(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": second derivatives (create_graph=True) are not supported");
}

// ---------------------------------------------------------------------------------------------
// npu_moe_init_routing_v2
struct RoutingSpec {
  int64_t n, hidden, begin, end;
  bool quant;
};

RoutingSpec routing_check(const Tensor& x, const Tensor& expert_idx, const optional<Tensor>& scale, const optional<Tensor>& offset,
                          int64_t active_num, int64_t expert_num, int64_t drop_pad_mode, int64_t tokens_type, int64_t quant_mode,
                          at::OptionalIntArrayRef range, int64_t row_idx_type) {
  constexpr const char* op = "npu_moe_init_routing_v2";
  TORCH_CHECK(x.dim() == 2 && expert_idx.dim() == 2 && expert_idx.size(0) == x.size(0), op,
              ": x must be [tokens, hidden] and expert_idx [tokens, topk], got ", x.sizes(), " and ", expert_idx.sizes());
  TORCH_CHECK(expert_idx.scalar_type() == at::kInt || expert_idx.scalar_type() == at::kLong, op,
              ": expert_idx must be int32 or int64, got ", expert_idx.scalar_type());
  TORCH_CHECK(drop_pad_mode == 0, op, ": only drop_pad_mode=0 (every token keeps its rows) is implemented, got ", drop_pad_mode);
  TORCH_CHECK(tokens_type == 0 || tokens_type == 1, op, ": expert_tokens_num_type must be 0 (cumulative) or 1 (counts), got ", tokens_type);
  TORCH_CHECK(quant_mode == -1 || quant_mode == 1, op, ": only quant_mode=-1 (none) and 1 (dynamic, per row) are implemented, got ", quant_mode);
  TORCH_CHECK(row_idx_type == 0 || row_idx_type == 1, op, ": row_idx_type must be 0 or 1, got ", row_idx_type);
  TORCH_CHECK(!offset.has_value(), op, ": offset belongs to static quantisation, which is not implemented");
  TORCH_CHECK(expert_num >= 1, op, ": expert_num must be given, got ", expert_num);
  RoutingSpec s;
  s.n = expert_idx.numel();
  s.hidden = x.size(1);
  s.quant = quant_mode == 1;
  TORCH_CHECK(active_num <= 0 || active_num == s.n, op, ": active_num must be tokens * topk (or not positive), got ", active_num);
  s.begin = 0;
  s.end = expert_num;
  if (range.has_value() && !range->empty()) {
    TORCH_CHECK(range->size() == 2 && (*range)[0] >= 0 && (*range)[0] < (*range)[1] && (*range)[1] <= expert_num, op,
                ": active_expert_range must be [start, end) within [0, ", expert_num, ")");
    s.begin = (*range)[0];
    s.end = (*range)[1];
  }
  TORCH_CHECK(s.end - s.begin <= kPermuteExperts, op, ": at most ", kPermuteExperts, " experts, got ", s.end - s.begin);
  if (s.quant) {
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, op, ": quant_mode=1 takes a float16 or bfloat16 x, got ",
                x.scalar_type());
    if (scale.has_value()) {
      TORCH_CHECK(scale->dim() == 2 && scale->size(1) == s.hidden && (scale->size(0) == 1 || scale->size(0) == s.end - s.begin), op,
                  ": smooth scales must be [1, ", s.hidden, "] or [", s.end - s.begin, ", ", s.hidden, "], got ", scale->sizes());
      TORCH_CHECK(scale->scalar_type() == at::kFloat || scale->scalar_type() == x.scalar_type(), op,
                  ": smooth scales must be float32 or x's dtype");
    }
  } else {
    TORCH_CHECK(is_float_type(x.scalar_type()) || x.scalar_type() == at::kChar, op, ": x must be float16, bfloat16, float32 or int8, got ",
                x.scalar_type());
    if (scale.has_value())
      TORCH_CHECK(scale->scalar_type() == at::kFloat && scale->dim() == 1 && scale->size(0) == x.size(0), op,
                  ": without quantisation, scale must be float32 [tokens]");
  }
  return s;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> routing_outputs(const RoutingSpec& s, const Tensor& x, bool with_scale) {
  return {at::empty({s.n, s.hidden}, x.options().dtype(s.quant ? at::kChar : x.scalar_type())), at::empty({s.n}, x.options().dtype(at::kInt)),
          at::empty({s.end - s.begin}, x.options().dtype(at::kLong)),
          at::empty({s.quant || with_scale ? s.n : 0}, x.options().dtype(at::kFloat))};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> init_routing_cuda(const Tensor& x, const Tensor& expert_idx, const optional<Tensor>& scale,
                                                             const optional<Tensor>& offset, int64_t active_num, int64_t /*expert_capacity*/,
                                                             int64_t expert_num, int64_t drop_pad_mode, int64_t tokens_type, bool /*tokens_flag*/,
                                                             int64_t quant_mode, at::OptionalIntArrayRef range, int64_t row_idx_type) {
  constexpr const char* op = "npu_moe_init_routing_v2";
  const optional<Tensor> eo(expert_idx);
  check_same_device(op, x, {&eo, &scale, &offset});
  c10::cuda::CUDAGuard guard(x.device());
  surface_device_error(op, x);
  const RoutingSpec s = routing_check(x, expert_idx, scale, offset, active_num, expert_num, drop_pad_mode, tokens_type, quant_mode, range, row_idx_type);
  auto [rows, row_idx, expert_tokens, row_scale] = routing_outputs(s, x, scale.has_value());
  Tensor xc = x.contiguous(), ids = expert_idx.contiguous();
  Tensor sc = scale.has_value() ? scale->contiguous() : Tensor();
  Tensor row_src = row_idx_type == 1 ? at::empty({s.n}, row_idx.options()) : Tensor();
  Tensor ws = scratch(b200q_moe_route_workspace_bytes(s.n, s.quant ? 1 : 0), x);
  b200q_moe_route_args a{};
  a.x = xc.data_ptr(); a.x_dtype = dtype_enum(x.scalar_type());
  a.expert_idx = ids.data_ptr(); a.idx_dtype = dtype_enum(ids.scalar_type());
  a.tokens = x.size(0); a.topk = ids.size(1); a.hidden = s.hidden;
  a.expert_begin = s.begin; a.expert_end = s.end;
  a.quantise = s.quant ? 1 : 0;
  if (sc.defined()) { a.scale = sc.data_ptr(); a.scale_dtype = dtype_enum(sc.scalar_type()); a.scale_rows = s.quant ? sc.size(0) : 0; }
  a.out = rows.data_ptr(); a.out_rows = s.n;
  a.out_scale = row_scale.numel() ? static_cast<float*>(row_scale.data_ptr()) : nullptr;
  if (!s.quant && a.out_scale == nullptr) a.scale = nullptr;
  a.row_idx = static_cast<int32_t*>(row_idx.data_ptr());
  a.row_src = row_src.defined() ? static_cast<int32_t*>(row_src.data_ptr()) : nullptr;
  a.expert_tokens = static_cast<int64_t*>(expert_tokens.data_ptr());
  a.cumulative = tokens_type == 0 ? 1 : 0;
  if (ws.defined()) { a.workspace = ws.data_ptr(); a.workspace_bytes = ws.numel(); }
  check_status(b200q_moe_route(&a, stream_of(x)), op);
  return {rows, row_src.defined() ? row_src : row_idx, expert_tokens, row_scale};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> init_routing_meta(const Tensor& x, const Tensor& expert_idx, const optional<Tensor>& scale,
                                                             const optional<Tensor>& offset, int64_t active_num, int64_t, int64_t expert_num,
                                                             int64_t drop_pad_mode, int64_t tokens_type, bool, int64_t quant_mode,
                                                             at::OptionalIntArrayRef range, int64_t row_idx_type) {
  return routing_outputs(
      routing_check(x, expert_idx, scale, offset, active_num, expert_num, drop_pad_mode, tokens_type, quant_mode, range, row_idx_type), x,
      scale.has_value());
}

// ---------------------------------------------------------------------------------------------
// npu_moe_token_permute(tokens, indices, num_out_tokens=None, padded_mode=False) -> (permuted_tokens, sorted_indices)
std::tuple<Tensor, Tensor> permute_check(const Tensor& tokens, const Tensor& indices, optional<int64_t> num_out, bool padded_mode) {
  constexpr const char* op = "npu_moe_token_permute";
  TORCH_CHECK(!padded_mode, op, ": padded_mode=True is not implemented");
  TORCH_CHECK(tokens.dim() == 2, op, ": tokens must be [num_tokens, hidden], got ", tokens.sizes());
  TORCH_CHECK(is_float_type(tokens.scalar_type()) || tokens.scalar_type() == at::kChar, op,
              ": tokens must be float16, bfloat16, float32 or int8, got ", tokens.scalar_type());
  TORCH_CHECK((indices.dim() == 1 || indices.dim() == 2) && indices.size(0) == tokens.size(0), op,
              ": indices must be [num_tokens] or [num_tokens, topk] with num_tokens ", tokens.size(0), ", got ", indices.sizes());
  TORCH_CHECK(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong, op, ": indices must be int32 or int64, got ",
              indices.scalar_type());
  const int64_t n = indices.numel(), asked = num_out.value_or(0);
  const int64_t rows = asked > 0 ? std::min(n, asked) : std::max<int64_t>(0, n + asked);
  return {at::empty({rows, tokens.size(1)}, tokens.options()), at::empty({n}, tokens.options().dtype(at::kInt))};
}

std::tuple<Tensor, Tensor> permute_cuda(const Tensor& tokens, const Tensor& indices, optional<int64_t> num_out, bool padded_mode) {
  constexpr const char* op = "npu_moe_token_permute";
  const optional<Tensor> io(indices);
  check_same_device(op, tokens, {&io});
  c10::cuda::CUDAGuard guard(tokens.device());
  surface_device_error(op, tokens);
  auto [rows, sorted] = permute_check(tokens, indices, num_out, padded_mode);
  Tensor xc = tokens.contiguous(), ids = indices.contiguous();
  Tensor ws = scratch(b200q_moe_route_workspace_bytes(ids.numel(), 0), tokens);
  b200q_moe_route_args a{};
  a.x = xc.data_ptr(); a.x_dtype = dtype_enum(tokens.scalar_type());
  a.expert_idx = ids.data_ptr(); a.idx_dtype = dtype_enum(ids.scalar_type());
  a.tokens = tokens.size(0); a.topk = ids.dim() == 2 ? ids.size(1) : 1; a.hidden = tokens.size(1);
  a.expert_begin = 0; a.expert_end = kPermuteExperts; a.strict = 1;
  a.out = rows.data_ptr(); a.out_rows = rows.size(0);
  a.row_idx = static_cast<int32_t*>(sorted.data_ptr());
  if (ws.defined()) { a.workspace = ws.data_ptr(); a.workspace_bytes = ws.numel(); }
  check_status(b200q_moe_route(&a, stream_of(tokens)), op);
  return {rows, sorted};
}

// ---------------------------------------------------------------------------------------------
// npu_moe_token_unpermute(permuted_tokens, sorted_indices, probs=None, padded_mode=False, restore_shape=None) -> Tensor
struct UnpermuteSpec {
  int64_t tokens, topk, hidden, rows;
};

UnpermuteSpec unpermute_check(const char* op, const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode,
                              at::OptionalIntArrayRef restore_shape) {
  TORCH_CHECK(!padded_mode && (!restore_shape.has_value() || restore_shape->empty()), op, ": padded_mode=True and restore_shape are not implemented");
  TORCH_CHECK(rows.dim() == 2 && is_float_type(rows.scalar_type()), op, ": permuted_tokens must be a float16, bfloat16 or float32 matrix, got ",
              rows.scalar_type(), " ", rows.sizes());
  TORCH_CHECK(sorted.dim() == 1 && sorted.scalar_type() == at::kInt, op, ": sorted_indices must be a 1-D int32 tensor, got ", sorted.scalar_type(),
              " ", sorted.sizes());
  UnpermuteSpec s{sorted.size(0), 1, rows.size(1), rows.size(0)};
  if (probs.has_value()) {
    TORCH_CHECK(probs->dim() == 2 && is_float_type(probs->scalar_type()), op, ": probs must be a float16, bfloat16 or float32 [num_tokens, topk], got ",
                probs->scalar_type(), " ", probs->sizes());
    TORCH_CHECK(probs->numel() == sorted.numel() && probs->size(1) >= 1, op, ": probs ", probs->sizes(), " and sorted_indices ", sorted.sizes(),
                " do not match");
    s.tokens = probs->size(0);
    s.topk = probs->size(1);
  }
  return s;
}

Tensor combine_cuda(const char* op, const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, int64_t tokens, int64_t topk) {
  Tensor out = at::empty({tokens, rows.size(1)}, rows.options());
  Tensor rc = rows.contiguous(), sc = sorted.contiguous();
  Tensor pc = probs.has_value() ? probs->contiguous() : Tensor();
  check_status(b200q_moe_combine(rc.data_ptr(), dtype_enum(rc.scalar_type()), rc.size(0), static_cast<const int32_t*>(sc.data_ptr()),
                                 pc.defined() ? pc.data_ptr() : nullptr, pc.defined() ? dtype_enum(pc.scalar_type()) : B200Q_NONE, out.data_ptr(),
                                 tokens, topk, rc.size(1), stream_of(rows)),
               op);
  return out;
}

Tensor unpermute_cuda(const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode, at::OptionalIntArrayRef restore_shape) {
  constexpr const char* op = "npu_moe_token_unpermute";
  const optional<Tensor> so(sorted);
  check_same_device(op, rows, {&so, &probs});
  c10::cuda::CUDAGuard guard(rows.device());
  surface_device_error(op, rows);
  const UnpermuteSpec s = unpermute_check(op, rows, sorted, probs, padded_mode, restore_shape);
  return combine_cuda(op, rows, sorted, probs, s.tokens, s.topk);
}

Tensor unpermute_meta(const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode, at::OptionalIntArrayRef restore_shape) {
  const UnpermuteSpec s = unpermute_check("npu_moe_token_unpermute", rows, sorted, probs, padded_mode, restore_shape);
  return at::empty({s.tokens, s.hidden}, rows.options());
}

// npu_moe_token_permute_grad(tokens, grad_permuted_tokens, indices, sorted_indices, padded_mode=False) -> Tensor
// The gradient of a token is the sum of its rows' gradients; `tokens` and `indices` give shapes only.
void permute_grad_check(const Tensor& tokens, const Tensor& grad, const Tensor& indices, const Tensor& sorted, bool padded_mode) {
  constexpr const char* op = "npu_moe_token_permute_grad";
  TORCH_CHECK(!padded_mode, op, ": padded_mode=True is not implemented");
  TORCH_CHECK(tokens.dim() == 2 && grad.dim() == 2 && grad.size(1) == tokens.size(1) && is_float_type(grad.scalar_type()) &&
                  grad.scalar_type() == tokens.scalar_type(),
              op, ": tokens and grad_permuted_tokens must be float16, bfloat16 or float32 matrices of one dtype and width, got ", tokens.scalar_type(),
              " ", tokens.sizes(), " and ", grad.scalar_type(), " ", grad.sizes());
  TORCH_CHECK((indices.dim() == 1 || indices.dim() == 2) && indices.size(0) == tokens.size(0) && sorted.dim() == 1 &&
                  sorted.scalar_type() == at::kInt && sorted.numel() == indices.numel(),
              op, ": indices ", indices.sizes(), " and sorted_indices (int32) ", sorted.sizes(), " do not match ", tokens.size(0), " tokens");
}

Tensor permute_grad_cuda(const Tensor& tokens, const Tensor& grad, const Tensor& indices, const Tensor& sorted, bool padded_mode) {
  constexpr const char* op = "npu_moe_token_permute_grad";
  const optional<Tensor> go(grad), io(indices), so(sorted);
  check_same_device(op, tokens, {&go, &io, &so});
  c10::cuda::CUDAGuard guard(tokens.device());
  surface_device_error(op, tokens);
  permute_grad_check(tokens, grad, indices, sorted, padded_mode);
  const int64_t topk = indices.dim() == 2 ? indices.size(1) : 1;
  if (topk == 0) return at::zeros(tokens.sizes(), tokens.options());
  return combine_cuda(op, grad, sorted, {}, tokens.size(0), topk);
}

Tensor permute_grad_meta(const Tensor& tokens, const Tensor& grad, const Tensor& indices, const Tensor& sorted, bool padded_mode) {
  permute_grad_check(tokens, grad, indices, sorted, padded_mode);
  return at::empty(tokens.sizes(), tokens.options());
}

// npu_moe_token_unpermute_grad(permuted_tokens, grad_unpermuted_tokens, sorted_indices, probs=None, padded_mode=False,
//                              restore_shape=None) -> (grad_permuted_tokens, grad_probs); grad_probs is empty without probs.
UnpermuteSpec unpermute_grad_check(const Tensor& rows, const Tensor& grad, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode,
                                   at::OptionalIntArrayRef restore_shape) {
  constexpr const char* op = "npu_moe_token_unpermute_grad";
  const UnpermuteSpec s = unpermute_check(op, rows, sorted, probs, padded_mode, restore_shape);
  TORCH_CHECK(grad.dim() == 2 && grad.size(0) == s.tokens && grad.size(1) == s.hidden && grad.scalar_type() == rows.scalar_type(), op,
              ": grad_unpermuted_tokens must be [", s.tokens, ", ", s.hidden, "] in permuted_tokens' dtype, got ", grad.scalar_type(), " ", grad.sizes());
  return s;
}

std::tuple<Tensor, Tensor> unpermute_grad_cuda(const Tensor& rows, const Tensor& grad, const Tensor& sorted, const optional<Tensor>& probs,
                                               bool padded_mode, at::OptionalIntArrayRef restore_shape) {
  constexpr const char* op = "npu_moe_token_unpermute_grad";
  const optional<Tensor> go(grad), so(sorted);
  check_same_device(op, rows, {&go, &so, &probs});
  c10::cuda::CUDAGuard guard(rows.device());
  surface_device_error(op, rows);
  const UnpermuteSpec s = unpermute_grad_check(rows, grad, sorted, probs, padded_mode, restore_shape);
  Tensor drows = at::empty(rows.sizes(), rows.options());
  Tensor dprobs = probs.has_value() ? at::empty(probs->sizes(), probs->options()) : at::empty({0}, rows.options());
  Tensor rc = rows.contiguous(), gc = grad.contiguous(), sc = sorted.contiguous();
  Tensor pc = probs.has_value() ? probs->contiguous() : Tensor();
  Tensor ws = scratch(b200q_moe_combine_grad_workspace_bytes(s.rows), rows);
  b200q_moe_combine_grad_args a{};
  a.dy = gc.data_ptr(); a.dtype = dtype_enum(rows.scalar_type());
  a.rows = rc.data_ptr(); a.num_rows = s.rows;
  a.row_idx = static_cast<const int32_t*>(sc.data_ptr());
  a.weight_dtype = B200Q_NONE;
  if (pc.defined()) { a.weights = pc.data_ptr(); a.weight_dtype = dtype_enum(pc.scalar_type()); a.dweights = dprobs.data_ptr(); }
  a.tokens = s.tokens; a.topk = s.topk; a.hidden = s.hidden;
  a.drows = drows.data_ptr();
  if (ws.defined()) { a.workspace = ws.data_ptr(); a.workspace_bytes = ws.numel(); }
  check_status(b200q_moe_combine_grad(&a, stream_of(rows)), op);
  return {drows, dprobs};
}

std::tuple<Tensor, Tensor> unpermute_grad_meta(const Tensor& rows, const Tensor& grad, const Tensor& sorted, const optional<Tensor>& probs,
                                               bool padded_mode, at::OptionalIntArrayRef restore_shape) {
  unpermute_grad_check(rows, grad, sorted, probs, padded_mode, restore_shape);
  return {at::empty(rows.sizes(), rows.options()), probs.has_value() ? at::empty(probs->sizes(), probs->options()) : at::empty({0}, rows.options())};
}

// ---------------------------------------------------------------------------------------------
// npu_gated_add_rms_norm(x, residual, gamma, *, post_gamma, gate, residual_scale, epsilon) -> (y, rstd, h, post_rstd)
struct GateSpec {
  bool per_row = false;
  int64_t rows = 1;            // rows that share a gate
};

GateSpec gate_spec(const char* op, const Tensor& x, const Tensor& gate) {
  const int64_t width = x.size(-1), rows = width ? x.numel() / width : 0, d = x.dim();
  GateSpec s;
  TORCH_CHECK(is_float_type(gate.scalar_type()), op, ": gate must be float16, bfloat16 or float32, got ", gate.scalar_type());
  if (gate.dim() == 1 && gate.size(0) == width) {
    s.rows = std::max<int64_t>(1, rows);
    return s;
  }
  TORCH_CHECK(gate.dim() == d && (gate.size(-1) == width || gate.size(-1) == 1), op, ": gate ", gate.sizes(), " does not fit x ", x.sizes(),
              " (one value a channel, a row or an element, or a row of channels for each leading index)");
  // The leading sizes are x's up to some dimension and 1 from there on.
  int64_t i = 0;
  while (i + 1 < d && gate.size(i) == x.size(i)) ++i;
  int64_t shared = 1;
  for (int64_t j = i; j + 1 < d; ++j) {
    TORCH_CHECK(gate.size(j) == 1, op, ": gate ", gate.sizes(), " does not fit x ", x.sizes());
    shared *= x.size(j);
  }
  s.rows = std::max<int64_t>(1, shared);
  s.per_row = gate.size(-1) == 1 && width != 1;
  TORCH_CHECK(!s.per_row || s.rows == 1, op, ": a gate of one value a row needs x's leading sizes, got ", gate.sizes(), " for x ", x.sizes());
  return s;
}

// Fills the arguments that both directions share; the tensors must be contiguous.
b200q_gated_norm_args norm_args(const char* op, const Tensor& x, const Tensor& residual, const Tensor& gamma, const Tensor& post, const Tensor& gate,
                                double residual_scale, double epsilon) {
  b200q_gated_norm_args a{};
  a.x = x.data_ptr(); a.residual = residual.data_ptr(); a.dtype = dtype_enum(x.scalar_type());
  a.gamma = gamma.data_ptr(); a.param_dtype = dtype_enum(gamma.scalar_type());
  if (post.defined()) a.post_gamma = post.data_ptr();
  a.gate_rows = 1;
  if (gate.defined()) {
    const GateSpec g = gate_spec(op, x, gate);
    a.gate = gate.data_ptr();
    a.gate_per_row = g.per_row ? 1 : 0;
    a.gate_rows = g.rows;
  }
  a.residual_scale = static_cast<float>(residual_scale);
  a.epsilon = static_cast<float>(epsilon);
  a.width = x.size(-1);
  a.rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) a.rows *= x.size(i);   // rows without columns have statistics too
  return a;
}

void norm_check(const char* op, const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post, const optional<Tensor>& gate) {
  TORCH_CHECK(x.dim() >= 1 && is_float_type(x.scalar_type()), op, ": x must be float16, bfloat16 or float32, got ", x.scalar_type());
  TORCH_CHECK(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(), op, ": residual must have x's shape and dtype, got ",
              residual.scalar_type(), " ", residual.sizes(), " for ", x.scalar_type(), " ", x.sizes());
  auto vector = [&](const Tensor& v, const char* name) {
    TORCH_CHECK(v.dim() == 1 && v.size(0) == x.size(-1) && is_float_type(v.scalar_type()), op, ": ", name, " must be a float16, bfloat16 or float32 [",
                x.size(-1), "], got ", v.scalar_type(), " ", v.sizes());
  };
  vector(gamma, "gamma");
  if (post.has_value()) vector(*post, "post_gamma");
  if (gate.has_value()) gate_spec(op, x, *gate);
}

// The kernels take the parameters all in x's dtype or all in float32: any mix is brought to float32 first.
at::ScalarType param_type(const Tensor& x, const Tensor& gamma, const optional<Tensor>& post, const optional<Tensor>& gate) {
  auto differs = [&](const optional<Tensor>& t) { return t.has_value() && t->scalar_type() != gamma.scalar_type(); };
  const bool one_type = !differs(post) && !differs(gate);
  return one_type && gamma.scalar_type() == x.scalar_type() ? x.scalar_type() : at::kFloat;
}
Tensor as_param(const optional<Tensor>& t, at::ScalarType type) { return t.has_value() ? t->to(type).contiguous() : Tensor(); }

Tensor contiguous_or_none(const optional<Tensor>& t) { return t.has_value() ? t->contiguous() : Tensor(); }

std::vector<int64_t> row_sizes(const Tensor& x) {
  auto s = x.sizes().vec();
  s.pop_back();
  return s;
}

using NormOutputs = std::tuple<Tensor, Tensor, Tensor, Tensor>;

NormOutputs norm_meta(const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post, const optional<Tensor>& gate,
                      double, double) {
  norm_check("npu_gated_add_rms_norm", x, residual, gamma, post, gate);
  const auto rows = row_sizes(x);
  const auto f32 = x.options().dtype(at::kFloat);
  return {at::empty(x.sizes(), x.options()), at::empty(rows, f32), at::empty(x.sizes(), x.options()),
          post.has_value() ? at::empty(rows, f32) : at::empty({0}, f32)};
}

NormOutputs norm_cuda(const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post, const optional<Tensor>& gate,
                      double residual_scale, double epsilon) {
  constexpr const char* op = "npu_gated_add_rms_norm";
  const optional<Tensor> ro(residual), go(gamma);
  check_same_device(op, x, {&ro, &go, &post, &gate});
  c10::cuda::CUDAGuard guard(x.device());
  surface_device_error(op, x);
  auto [y, rstd, h, post_rstd] = norm_meta(x, residual, gamma, post, gate, residual_scale, epsilon);
  const at::ScalarType pt = param_type(x, gamma, post, gate);
  Tensor xc = x.contiguous(), rc = residual.contiguous(), wc = as_param(gamma, pt), pc = as_param(post, pt), gc = as_param(gate, pt);
  b200q_gated_norm_args a = norm_args(op, xc, rc, wc, pc, gc, residual_scale, epsilon);
  a.y = y.data_ptr(); a.h = h.data_ptr();
  a.rstd = static_cast<float*>(rstd.data_ptr());
  if (post.has_value()) a.post_rstd = static_cast<float*>(post_rstd.data_ptr());
  check_status(b200q_gated_norm(&a, stream_of(x)), op);
  return {y, rstd, h, post_rstd};
}

// npu_gated_add_rms_norm_dynamic_quant(x, residual, gamma, *, post_gamma, gate, smooth_scales, residual_scale, epsilon) -> (y int8, scale, h)
std::tuple<Tensor, Tensor, Tensor> norm_quant_meta(const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post,
                                                   const optional<Tensor>& gate, const optional<Tensor>& smooth, double, double) {
  constexpr const char* op = "npu_gated_add_rms_norm_dynamic_quant";
  norm_check(op, x, residual, gamma, post, gate);
  if (smooth.has_value())
    TORCH_CHECK(smooth->dim() == 1 && smooth->size(0) == x.size(-1) && is_float_type(smooth->scalar_type()), op,
                ": smooth_scales must be a float16, bfloat16 or float32 [", x.size(-1), "], got ", smooth->scalar_type(), " ", smooth->sizes());
  return {at::empty(x.sizes(), x.options().dtype(at::kChar)), at::empty(row_sizes(x), x.options().dtype(at::kFloat)),
          at::empty(x.sizes(), x.options())};
}

std::tuple<Tensor, Tensor, Tensor> norm_quant_cuda(const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post,
                                                   const optional<Tensor>& gate, const optional<Tensor>& smooth, double residual_scale,
                                                   double epsilon) {
  constexpr const char* op = "npu_gated_add_rms_norm_dynamic_quant";
  const optional<Tensor> ro(residual), go(gamma);
  check_same_device(op, x, {&ro, &go, &post, &gate, &smooth});
  c10::cuda::CUDAGuard guard(x.device());
  surface_device_error(op, x);
  auto [y, scale, h] = norm_quant_meta(x, residual, gamma, post, gate, smooth, residual_scale, epsilon);
  if (x.size(-1) == 0) return {y, scale.zero_(), h};
  const at::ScalarType pt = param_type(x, gamma, post, gate);
  Tensor xc = x.contiguous(), rc = residual.contiguous(), wc = as_param(gamma, pt), pc = as_param(post, pt), gc = as_param(gate, pt);
  Tensor sc = as_param(smooth, smooth.has_value() && smooth->scalar_type() == x.scalar_type() ? x.scalar_type() : at::kFloat);
  b200q_gated_norm_args a = norm_args(op, xc, rc, wc, pc, gc, residual_scale, epsilon);
  a.y = y.data_ptr(); a.h = h.data_ptr();
  a.scale = static_cast<float*>(scale.data_ptr());
  if (sc.defined()) { a.smooth = sc.data_ptr(); a.smooth_dtype = dtype_enum(sc.scalar_type()); }
  if (a.rows > 0) check_status(b200q_gated_norm(&a, stream_of(x)), op);
  return {y, scale, h};
}

// npu_gated_add_rms_norm_grad(grad_y, grad_h, x, residual, gamma, rstd, *, post_gamma, gate, post_rstd, residual_scale)
//   -> (grad_x, grad_residual, grad_gamma, grad_post_gamma, grad_gate); what there is no parameter for is empty.
using NormGrads = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

NormGrads norm_grad_meta(const Tensor& dy, const optional<Tensor>& dh, const Tensor& x, const Tensor& residual, const Tensor& gamma, const Tensor& rstd,
                         const optional<Tensor>& post, const optional<Tensor>& gate, const optional<Tensor>& post_rstd, double) {
  constexpr const char* op = "npu_gated_add_rms_norm_grad";
  norm_check(op, x, residual, gamma, post, gate);
  const int64_t rows = x.size(-1) ? x.numel() / x.size(-1) : rstd.numel();
  auto like_x = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type(), op, ": ", name, " must have x's shape and dtype, got ", t.scalar_type(), " ",
                t.sizes());
  };
  auto stat = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == rows, op, ": ", name, " must be float32 with one value a row (", rows, "), got ",
                t.scalar_type(), " ", t.sizes());
  };
  like_x(dy, "grad_y");
  if (dh.has_value()) like_x(*dh, "grad_h");
  stat(rstd, "rstd");
  TORCH_CHECK(!post.has_value() || post_rstd.has_value(), op, ": post_gamma needs post_rstd");
  if (post.has_value()) stat(*post_rstd, "post_rstd");
  auto like = [&](const optional<Tensor>& t) { return t.has_value() ? at::empty(t->sizes(), t->options()) : at::empty({0}, x.options()); };
  return {at::empty(x.sizes(), x.options()), at::empty(x.sizes(), x.options()), at::empty(gamma.sizes(), gamma.options()), like(post), like(gate)};
}

NormGrads norm_grad_cuda(const Tensor& dy, const optional<Tensor>& dh, const Tensor& x, const Tensor& residual, const Tensor& gamma, const Tensor& rstd,
                         const optional<Tensor>& post, const optional<Tensor>& gate, const optional<Tensor>& post_rstd, double residual_scale) {
  constexpr const char* op = "npu_gated_add_rms_norm_grad";
  const optional<Tensor> xo(x), ro(residual), go(gamma), so(rstd);
  check_same_device(op, dy, {&dh, &xo, &ro, &go, &so, &post, &gate, &post_rstd});
  c10::cuda::CUDAGuard guard(x.device());
  surface_device_error(op, x);
  auto [dx, dres, dgamma, dpost, dgate] = norm_grad_meta(dy, dh, x, residual, gamma, rstd, post, gate, post_rstd, residual_scale);
  const at::ScalarType pt = param_type(x, gamma, post, gate);
  Tensor xc = x.contiguous(), rc = residual.contiguous(), wc = as_param(gamma, pt), pc = as_param(post, pt), gc = as_param(gate, pt);
  Tensor yc = dy.contiguous(), hc = contiguous_or_none(dh), sc = rstd.contiguous(), qc = contiguous_or_none(post_rstd);
  if (x.numel() == 0 && gate.has_value()) dgate.zero_();
  // Gradients of parameters that had to change their type are computed in float32 and rounded afterwards.
  auto as_grad = [&](const Tensor& t) { return t.scalar_type() == pt ? t : at::empty(t.sizes(), t.options().dtype(pt)); };
  Tensor gw = as_grad(dgamma), gp = post.has_value() ? as_grad(dpost) : dpost, gg = gate.has_value() ? as_grad(dgate) : dgate;
  b200q_gated_norm_args a = norm_args(op, xc, rc, wc, pc, gc, residual_scale, 0.0);
  a.rstd = static_cast<float*>(sc.data_ptr());
  if (post.has_value()) a.post_rstd = static_cast<float*>(qc.data_ptr());
  Tensor ws = scratch(b200q_gated_norm_grad_workspace_bytes(&a), x);
  b200q_gated_norm_grads g{};
  g.dy = yc.data_ptr();
  if (hc.defined()) g.dh = hc.data_ptr();
  g.dx = dx.data_ptr(); g.dresidual = dres.data_ptr(); g.dgamma = gw.data_ptr();
  if (post.has_value()) g.dpost_gamma = gp.data_ptr();
  if (gate.has_value()) g.dgate = gg.data_ptr();
  if (ws.defined()) { g.workspace = ws.data_ptr(); g.workspace_bytes = ws.numel(); }
  check_status(b200q_gated_norm_grad(&a, &g, stream_of(x)), op);
  if (!gw.is_same(dgamma)) dgamma.copy_(gw);
  if (!gp.is_same(dpost)) dpost.copy_(gp);
  if (!gg.is_same(dgate) && x.numel() > 0) dgate.copy_(gg);
  return {dx, dres, dgamma, dpost, dgate};
}

// ---------------------------------------------------------------------------------------------
// npu_grouped_matmul(x, weight, *, bias, scale, per_token_scale, group_list, split_item, group_type, group_list_type, output_dtype)
// One x, one weight [groups, k, n] and one output (split_item 2 or 3, group_type 0), int8 operands.
struct GroupedSpec {
  int64_t m, k, n, groups;
  at::ScalarType out;
};

GroupedSpec grouped_check(at::TensorList x, at::TensorList weight, const c10::optional<std::vector<Tensor>>& bias,
                          const c10::optional<std::vector<Tensor>>& scale, bool others, const c10::optional<std::vector<Tensor>>& row_scale,
                          const optional<Tensor>& group_list, int64_t split_item, int64_t group_type, int64_t list_type, int64_t act_type,
                          optional<at::ScalarType> output_dtype) {
  constexpr const char* op = "npu_grouped_matmul";
  TORCH_CHECK(x.size() == 1 && weight.size() == 1, op, ": one x and one weight [groups, k, n] are implemented, got ", x.size(), " and ", weight.size(),
              " tensors");
  TORCH_CHECK(!others, op, ": offset, antiquant_scale, antiquant_offset and activation inputs are not implemented (the int8 form takes scale, ",
              "per_token_scale and bias)");
  TORCH_CHECK(split_item == 2 || split_item == 3, op, ": split_item must be 2 or 3 (one output), got ", split_item);
  TORCH_CHECK(group_type == 0, op, ": group_type must be 0 (rows of x are grouped), got ", group_type);
  TORCH_CHECK(list_type == 0 || list_type == 1, op, ": group_list_type must be 0 (cumulative) or 1 (counts), got ", list_type);
  TORCH_CHECK(act_type == 0, op, ": act_type must be 0, got ", act_type);
  const Tensor &a = x[0], &w = weight[0];
  TORCH_CHECK(a.dim() == 2 && a.scalar_type() == at::kChar && w.dim() == 3 && w.scalar_type() == at::kChar, op,
              ": x must be int8 [m, k] and weight int8 [groups, k, n], got ", a.scalar_type(), " ", a.sizes(), " and ", w.scalar_type(), " ", w.sizes());
  TORCH_CHECK(w.size(1) == a.size(1), op, ": inner dimensions differ: x ", a.sizes(), " and weight ", w.sizes());
  GroupedSpec s{a.size(0), a.size(1), w.size(2), w.size(0), output_dtype.value_or(at::kBFloat16)};
  TORCH_CHECK(s.groups >= 1 && s.groups <= 1024, op, ": 1 to 1024 groups, got ", s.groups);
  TORCH_CHECK(s.out == at::kBFloat16 || s.out == at::kHalf || s.out == at::kInt, op, ": output_dtype must be bfloat16, float16 or int32, got ", s.out);
  TORCH_CHECK(group_list.has_value() && group_list->dim() == 1 && group_list->size(0) == s.groups &&
                  (group_list->scalar_type() == at::kLong || group_list->scalar_type() == at::kInt),
              op, ": group_list must be an int64 tensor with one entry for each of the ", s.groups, " groups");
  auto one = [&](const c10::optional<std::vector<Tensor>>& list, const char* name) -> const Tensor* {
    if (!list.has_value() || list->empty()) return nullptr;
    TORCH_CHECK(list->size() == 1, op, ": ", name, " must hold one tensor, got ", list->size());
    return &(*list)[0];
  };
  if (const Tensor* t = one(scale, "scale")) {
    TORCH_CHECK(t->numel() == s.groups * s.n && t->size(-1) == s.n &&
                    (t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kLong),
                op, ": scale must be float32, bfloat16 or int64 [", s.groups, ", ", s.n, "], got ", t->scalar_type(), " ", t->sizes());
  } else {
    TORCH_CHECK(s.out == at::kInt, op, ": scale is needed unless output_dtype is int32");
  }
  if (const Tensor* t = one(row_scale, "per_token_scale"))
    TORCH_CHECK(t->numel() == s.m && t->scalar_type() == at::kFloat, op, ": per_token_scale must be float32 [", s.m, "], got ", t->scalar_type(), " ",
                t->sizes());
  if (const Tensor* t = one(bias, "bias"))
    TORCH_CHECK(t->numel() == s.groups * s.n && t->size(-1) == s.n && (t->scalar_type() == at::kInt || (s.out != at::kInt && is_float_type(t->scalar_type()))),
                op, ": bias must be int32 or (not for int32 output) a float type, [", s.groups, ", ", s.n, "], got ", t->scalar_type(), " ", t->sizes());
  return s;
}

bool given(const c10::optional<std::vector<Tensor>>& list) { return list.has_value() && !list->empty(); }

std::vector<Tensor> grouped_matmul_cuda(at::TensorList x, at::TensorList weight, const c10::optional<std::vector<Tensor>>& bias,
                                        const c10::optional<std::vector<Tensor>>& scale, const c10::optional<std::vector<Tensor>>& offset,
                                        const c10::optional<std::vector<Tensor>>& antiquant_scale,
                                        const c10::optional<std::vector<Tensor>>& antiquant_offset,
                                        const c10::optional<std::vector<Tensor>>& row_scale, const optional<Tensor>& group_list,
                                        const c10::optional<std::vector<Tensor>>& act_input, const c10::optional<std::vector<Tensor>>& act_quant_scale,
                                        const c10::optional<std::vector<Tensor>>& act_quant_offset, int64_t split_item, int64_t group_type,
                                        int64_t list_type, int64_t act_type, at::OptionalIntArrayRef /*tuning_config*/,
                                        optional<at::ScalarType> output_dtype) {
  constexpr const char* op = "npu_grouped_matmul";
  const GroupedSpec s = grouped_check(x, weight, bias, scale,
                                      given(offset) || given(antiquant_scale) || given(antiquant_offset) || given(act_input) || given(act_quant_scale) ||
                                          given(act_quant_offset),
                                      row_scale, group_list, split_item, group_type, list_type, act_type, output_dtype);
  auto first = [](const c10::optional<std::vector<Tensor>>& list) { return given(list) ? optional<Tensor>((*list)[0]) : optional<Tensor>(); };
  const Tensor& a = x[0];
  const optional<Tensor> wo(weight[0]), bo = first(bias), so = first(scale), ro = first(row_scale);
  check_same_device(op, a, {&wo, &bo, &so, &ro, &group_list});
  c10::cuda::CUDAGuard guard(a.device());
  surface_device_error(op, a);
  Tensor out = at::empty({s.m, s.n}, a.options().dtype(s.out));
  Tensor xc = a.contiguous(), list = group_list->to(at::kLong).contiguous();
  Tensor bc = contiguous_or_none(bo), sc = contiguous_or_none(so), rc = contiguous_or_none(ro);
  const Tensor& w = weight[0];
  b200q_grouped_matmul_args g{};
  g.x = static_cast<const int8_t*>(xc.data_ptr()); g.weight = static_cast<const int8_t*>(w.data_ptr());
  g.m = s.m; g.k = s.k; g.n = s.n; g.groups = s.groups;
  g.w_stride_g = w.stride(0); g.w_stride_k = w.stride(1); g.w_stride_n = w.stride(2);
  g.group_list = static_cast<const int64_t*>(list.data_ptr()); g.counts = list_type == 1 ? 1 : 0;
  if (sc.defined()) { g.scale = sc.data_ptr(); g.scale_dtype = dtype_enum(sc.scalar_type()); }
  if (rc.defined()) g.row_scale = static_cast<const float*>(rc.data_ptr());
  g.bias_dtype = B200Q_NONE;
  if (bc.defined()) { g.bias = bc.data_ptr(); g.bias_dtype = dtype_enum(bc.scalar_type()); }
  g.out = out.data_ptr(); g.out_dtype = dtype_enum(s.out);
  check_status(b200q_grouped_matmul(&g, stream_of(a)), op);
  return {out};
}

std::vector<Tensor> grouped_matmul_meta(at::TensorList x, at::TensorList weight, const c10::optional<std::vector<Tensor>>& bias,
                                        const c10::optional<std::vector<Tensor>>& scale, const c10::optional<std::vector<Tensor>>& offset,
                                        const c10::optional<std::vector<Tensor>>& antiquant_scale,
                                        const c10::optional<std::vector<Tensor>>& antiquant_offset,
                                        const c10::optional<std::vector<Tensor>>& row_scale, const optional<Tensor>& group_list,
                                        const c10::optional<std::vector<Tensor>>& act_input, const c10::optional<std::vector<Tensor>>& act_quant_scale,
                                        const c10::optional<std::vector<Tensor>>& act_quant_offset, int64_t split_item, int64_t group_type,
                                        int64_t list_type, int64_t act_type, at::OptionalIntArrayRef, optional<at::ScalarType> output_dtype) {
  const GroupedSpec s = grouped_check(x, weight, bias, scale,
                                      given(offset) || given(antiquant_scale) || given(antiquant_offset) || given(act_input) || given(act_quant_scale) ||
                                          given(act_quant_offset),
                                      row_scale, group_list, split_item, group_type, list_type, act_type, output_dtype);
  return {at::empty({s.m, s.n}, x[0].options().dtype(s.out))};
}

// ---------------------------------------------------------------------------------------------
// Autograd.  Both directions go through the dispatcher below the autograd keys, so that a dispatch mode (fake tensors, a profiler of
// operators) sees the operators that run, the gradients among them.
template <typename F>
c10::TypedOperatorHandle<F> operator_handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

std::tuple<Tensor, Tensor> permute_below(const Tensor& tokens, const Tensor& indices, optional<int64_t> num_out, bool padded_mode) {
  static const auto op = operator_handle<decltype(permute_cuda)>("npu::npu_moe_token_permute");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(tokens, indices, num_out, padded_mode);
}

Tensor unpermute_below(const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode, at::OptionalIntArrayRef restore_shape) {
  static const auto op = operator_handle<decltype(unpermute_cuda)>("npu::npu_moe_token_unpermute");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(rows, sorted, probs, padded_mode, restore_shape);
}

NormOutputs norm_below(const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post, const optional<Tensor>& gate,
                       double residual_scale, double epsilon) {
  static const auto op = operator_handle<decltype(norm_cuda)>("npu::npu_gated_add_rms_norm");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, residual, gamma, post, gate, residual_scale, epsilon);
}

// A dual tensor's tangent (forward-mode differentiation) would be lost below autograd: it is refused, as PyTorch refuses it for an
// autograd function without a jvp.
void no_forward_mode(const char* op, std::initializer_list<const optional<Tensor>*> inputs) {
  for (const optional<Tensor>* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!(t->has_value() && (*t)->defined() && (*t)->_fw_grad(/*level=*/0).defined()), op,
                                ": forward-mode differentiation is not supported");
}

class PermuteFunction : public torch::autograd::Function<PermuteFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& indices, optional<int64_t> num_out, bool padded_mode) {
    auto [rows, sorted] = permute_below(tokens, indices, num_out, padded_mode);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({sorted});
    ctx->save_for_backward({sorted});
    ctx->saved_data["tokens"] = tokens.size(0);
    ctx->saved_data["topk"] = indices.dim() == 2 ? indices.size(1) : int64_t(1);
    return {rows, sorted};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    no_second_derivative("npu_moe_token_permute_grad");
    static const auto op = operator_handle<decltype(permute_grad_cuda)>("npu::npu_moe_token_permute_grad");
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor sorted = ctx->get_saved_variables()[0];
    const int64_t tokens = ctx->saved_data["tokens"].toInt(), topk = ctx->saved_data["topk"].toInt();
    // The operator takes the shapes of tokens and indices only: neither is kept for it.
    const Tensor shape = at::empty({1, 1}, grads[0].options()).expand({tokens, grads[0].size(1)});
    Tensor g = op.call(shape, grads[0], sorted.view({tokens, topk}), sorted, false);
    return {g, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> permute_autograd(const Tensor& tokens, const Tensor& indices, optional<int64_t> num_out, bool padded_mode) {
  const optional<Tensor> to(tokens);
  no_forward_mode("npu_moe_token_permute", {&to});
  if (!(at::GradMode::is_enabled() && tokens.requires_grad())) {
    return permute_below(tokens, indices, num_out, padded_mode);
  }
  auto out = PermuteFunction::apply(tokens, indices, num_out, padded_mode);
  return {out[0], out[1]};
}

class UnpermuteFunction : public torch::autograd::Function<UnpermuteFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode,
                               at::OptionalIntArrayRef restore_shape) {
    Tensor out = unpermute_below(rows, sorted, probs, padded_mode, restore_shape);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({rows, sorted, probs.value_or(Tensor())});
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    no_second_derivative("npu_moe_token_unpermute_grad");
    static const auto op = operator_handle<decltype(unpermute_grad_cuda)>("npu::npu_moe_token_unpermute_grad");
    at::AutoDispatchBelowADInplaceOrView below;
    auto saved = ctx->get_saved_variables();
    const optional<Tensor> probs = saved[2].defined() ? optional<Tensor>(saved[2]) : optional<Tensor>();
    auto [drows, dprobs] = op.call(saved[0], grads[0], saved[1], probs, false, c10::nullopt);
    return {drows, Tensor(), probs.has_value() ? dprobs : Tensor(), Tensor(), Tensor()};
  }
};

Tensor unpermute_autograd(const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode,
                          at::OptionalIntArrayRef restore_shape) {
  const optional<Tensor> ro(rows);
  no_forward_mode("npu_moe_token_unpermute", {&ro, &probs});
  if (!(at::GradMode::is_enabled() && (rows.requires_grad() || (probs.has_value() && probs->requires_grad())))) {
    return unpermute_below(rows, sorted, probs, padded_mode, restore_shape);
  }
  return UnpermuteFunction::apply(rows, sorted, probs, padded_mode, restore_shape)[0];
}

class NormFunction : public torch::autograd::Function<NormFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post,
                               const optional<Tensor>& gate, double residual_scale, double epsilon) {
    auto [y, rstd, h, post_rstd] = norm_below(x, residual, gamma, post, gate, residual_scale, epsilon);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({rstd, post_rstd});
    ctx->save_for_backward({x, residual, gamma, post.value_or(Tensor()), gate.value_or(Tensor()), rstd, post_rstd});
    ctx->saved_data["residual_scale"] = residual_scale;
    return {y, rstd, h, post_rstd};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined() && !grads[2].defined()) return out;
    no_second_derivative("npu_gated_add_rms_norm_grad");
    static const auto op = operator_handle<decltype(norm_grad_cuda)>("npu::npu_gated_add_rms_norm_grad");
    at::AutoDispatchBelowADInplaceOrView below;
    auto s = ctx->get_saved_variables();
    auto opt = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); };
    const Tensor dy = grads[0].defined() ? grads[0] : at::zeros(s[0].sizes(), s[0].options());
    auto [dx, dres, dgamma, dpost, dgate] = op.call(dy, opt(grads[2]), s[0], s[1], s[2], s[5], opt(s[3]), opt(s[4]), opt(s[6]),
                                                   ctx->saved_data["residual_scale"].toDouble());
    out[0] = dx;
    out[1] = dres;
    out[2] = dgamma;
    if (s[3].defined()) out[3] = dpost;
    if (s[4].defined()) out[4] = dgate;
    return out;
  }
};

NormOutputs norm_autograd(const Tensor& x, const Tensor& residual, const Tensor& gamma, const optional<Tensor>& post, const optional<Tensor>& gate,
                          double residual_scale, double epsilon) {
  const optional<Tensor> xo(x), ro(residual), go(gamma);
  no_forward_mode("npu_gated_add_rms_norm", {&xo, &ro, &go, &post, &gate});
  const bool wanted = x.requires_grad() || residual.requires_grad() || gamma.requires_grad() || (post.has_value() && post->requires_grad()) ||
                      (gate.has_value() && gate->requires_grad());
  if (!(at::GradMode::is_enabled() && wanted)) {
    return norm_below(x, residual, gamma, post, gate, residual_scale, epsilon);
  }
  auto o = NormFunction::apply(x, residual, gamma, post, gate, residual_scale, epsilon);
  return {o[0], o[1], o[2], o[3]};
}

// The same for the operators without an autograd kernel, below PyTorch's default one for them.
void no_forward_mode_boxed(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const char* name = op.schema().name().c_str();
  auto check = [&](const optional<Tensor>& t) { no_forward_mode(name, {&t}); };
  for (const c10::IValue& v : torch::jit::last(*stack, op.schema().arguments().size())) {
    if (v.isTensor()) check(v.toTensor());
    else if (v.isTensorList())
      for (const Tensor& t : v.toTensorVector()) check(t);
  }
  op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(npu, m) {
  m.def("npu_moe_init_routing_v2(Tensor x, Tensor expert_idx, *, Tensor? scale=None, Tensor? offset=None, int active_num=-1, "
        "int expert_capacity=-1, int expert_num=-1, int drop_pad_mode=0, int expert_tokens_num_type=0, bool expert_tokens_num_flag=False, "
        "int quant_mode=-1, int[]? active_expert_range=None, int row_idx_type=0) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("npu_moe_token_permute(Tensor tokens, Tensor indices, int? num_out_tokens=None, bool padded_mode=False) -> (Tensor, Tensor)");
  m.def("npu_moe_token_permute_grad(Tensor tokens, Tensor grad_permuted_tokens, Tensor indices, Tensor sorted_indices, "
        "bool padded_mode=False) -> Tensor");
  m.def("npu_moe_token_unpermute(Tensor permuted_tokens, Tensor sorted_indices, Tensor? probs=None, bool padded_mode=False, "
        "int[]? restore_shape=None) -> Tensor");
  m.def("npu_moe_token_unpermute_grad(Tensor permuted_tokens, Tensor grad_unpermuted_tokens, Tensor sorted_indices, Tensor? probs=None, "
        "bool padded_mode=False, int[]? restore_shape=None) -> (Tensor, Tensor)");
  m.def("npu_gated_add_rms_norm(Tensor x, Tensor residual, Tensor gamma, *, Tensor? post_gamma=None, Tensor? gate=None, "
        "float residual_scale=1.0, float epsilon=1e-06) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("npu_gated_add_rms_norm_dynamic_quant(Tensor x, Tensor residual, Tensor gamma, *, Tensor? post_gamma=None, Tensor? gate=None, "
        "Tensor? smooth_scales=None, float residual_scale=1.0, float epsilon=1e-06) -> (Tensor, Tensor, Tensor)");
  m.def("npu_gated_add_rms_norm_grad(Tensor grad_y, Tensor? grad_h, Tensor x, Tensor residual, Tensor gamma, Tensor rstd, *, "
        "Tensor? post_gamma=None, Tensor? gate=None, Tensor? post_rstd=None, float residual_scale=1.0) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("npu_grouped_matmul(Tensor[] x, Tensor[] weight, *, Tensor[]? bias=None, Tensor[]? scale=None, Tensor[]? offset=None, "
        "Tensor[]? antiquant_scale=None, Tensor[]? antiquant_offset=None, Tensor[]? per_token_scale=None, Tensor? group_list=None, "
        "Tensor[]? activation_input=None, Tensor[]? activation_quant_scale=None, Tensor[]? activation_quant_offset=None, int split_item=0, "
        "int group_type=0, int group_list_type=0, int act_type=0, int[]? tuning_config=None, ScalarType? output_dtype=None) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
  m.impl("npu_moe_init_routing_v2", TORCH_FN(init_routing_cuda));
  m.impl("npu_moe_token_permute", TORCH_FN(permute_cuda));
  m.impl("npu_moe_token_permute_grad", TORCH_FN(permute_grad_cuda));
  m.impl("npu_moe_token_unpermute", TORCH_FN(unpermute_cuda));
  m.impl("npu_moe_token_unpermute_grad", TORCH_FN(unpermute_grad_cuda));
  m.impl("npu_gated_add_rms_norm", TORCH_FN(norm_cuda));
  m.impl("npu_gated_add_rms_norm_dynamic_quant", TORCH_FN(norm_quant_cuda));
  m.impl("npu_gated_add_rms_norm_grad", TORCH_FN(norm_grad_cuda));
  m.impl("npu_grouped_matmul", TORCH_FN(grouped_matmul_cuda));
}

TORCH_LIBRARY_IMPL(npu, AutogradCUDA, m) {
  m.impl("npu_moe_token_permute", TORCH_FN(permute_autograd));
  m.impl("npu_moe_token_unpermute", TORCH_FN(unpermute_autograd));
  m.impl("npu_gated_add_rms_norm", TORCH_FN(norm_autograd));
}

// No derivative of their own, although some of their outputs are floats.  PyTorch's default autograd kernel warns of that in a backward
// pass, but loses a tangent without a word.
TORCH_LIBRARY_IMPL(npu, ADInplaceOrView, m) {
  for (const char* op : {"npu_moe_init_routing_v2", "npu_moe_token_permute_grad", "npu_moe_token_unpermute_grad", "npu_gated_add_rms_norm_grad",
                         "npu_gated_add_rms_norm_dynamic_quant", "npu_grouped_matmul"})
    m.impl(op, torch::CppFunction::makeFromBoxedFunction<&no_forward_mode_boxed>());
}

TORCH_LIBRARY_IMPL(npu, Meta, m) {
  m.impl("npu_moe_init_routing_v2", TORCH_FN(init_routing_meta));
  m.impl("npu_moe_token_permute", TORCH_FN(permute_check));
  m.impl("npu_moe_token_permute_grad", TORCH_FN(permute_grad_meta));
  m.impl("npu_moe_token_unpermute", TORCH_FN(unpermute_meta));
  m.impl("npu_moe_token_unpermute_grad", TORCH_FN(unpermute_grad_meta));
  m.impl("npu_gated_add_rms_norm", TORCH_FN(norm_meta));
  m.impl("npu_gated_add_rms_norm_dynamic_quant", TORCH_FN(norm_quant_meta));
  m.impl("npu_gated_add_rms_norm_grad", TORCH_FN(norm_grad_meta));
  m.impl("npu_grouped_matmul", TORCH_FN(grouped_matmul_meta));
}
