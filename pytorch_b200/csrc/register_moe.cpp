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

constexpr int64_t kPermuteExperts = 1024;      // npu_moe_token_permute takes indices below this

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
// Autograd
class PermuteFunction : public torch::autograd::Function<PermuteFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& indices, optional<int64_t> num_out, bool padded_mode) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [rows, sorted] = permute_cuda(tokens, indices, num_out, padded_mode);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({sorted});
    ctx->save_for_backward({sorted});
    ctx->saved_data["tokens"] = tokens.size(0);
    ctx->saved_data["topk"] = indices.dim() == 2 ? indices.size(1) : int64_t(1);
    return {rows, sorted};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    constexpr const char* op = "npu_moe_token_permute_grad";
    no_second_derivative(op);
    const Tensor sorted = ctx->get_saved_variables()[0];
    const int64_t tokens = ctx->saved_data["tokens"].toInt(), topk = ctx->saved_data["topk"].toInt();
    c10::cuda::CUDAGuard guard(grads[0].device());
    surface_device_error(op, grads[0]);
    Tensor g = topk == 0 ? at::zeros({tokens, grads[0].size(1)}, grads[0].options()) : combine_cuda(op, grads[0], sorted, {}, tokens, topk);
    return {g, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> permute_autograd(const Tensor& tokens, const Tensor& indices, optional<int64_t> num_out, bool padded_mode) {
  if (!(at::GradMode::is_enabled() && tokens.requires_grad())) {
    at::AutoDispatchBelowADInplaceOrView below;
    return permute_cuda(tokens, indices, num_out, padded_mode);
  }
  auto out = PermuteFunction::apply(tokens, indices, num_out, padded_mode);
  return {out[0], out[1]};
}

class UnpermuteFunction : public torch::autograd::Function<UnpermuteFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode,
                               at::OptionalIntArrayRef restore_shape) {
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor out = unpermute_cuda(rows, sorted, probs, padded_mode, restore_shape);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({rows, sorted, probs.value_or(Tensor())});
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    no_second_derivative("npu_moe_token_unpermute_grad");
    auto saved = ctx->get_saved_variables();
    const optional<Tensor> probs = saved[2].defined() ? optional<Tensor>(saved[2]) : optional<Tensor>();
    auto [drows, dprobs] = unpermute_grad_cuda(saved[0], grads[0], saved[1], probs, false, c10::nullopt);
    return {drows, Tensor(), probs.has_value() ? dprobs : Tensor(), Tensor(), Tensor()};
  }
};

Tensor unpermute_autograd(const Tensor& rows, const Tensor& sorted, const optional<Tensor>& probs, bool padded_mode,
                          at::OptionalIntArrayRef restore_shape) {
  if (!(at::GradMode::is_enabled() && (rows.requires_grad() || (probs.has_value() && probs->requires_grad())))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return unpermute_cuda(rows, sorted, probs, padded_mode, restore_shape);
  }
  return UnpermuteFunction::apply(rows, sorted, probs, padded_mode, restore_shape)[0];
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
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
  m.impl("npu_moe_init_routing_v2", TORCH_FN(init_routing_cuda));
  m.impl("npu_moe_token_permute", TORCH_FN(permute_cuda));
  m.impl("npu_moe_token_permute_grad", TORCH_FN(permute_grad_cuda));
  m.impl("npu_moe_token_unpermute", TORCH_FN(unpermute_cuda));
  m.impl("npu_moe_token_unpermute_grad", TORCH_FN(unpermute_grad_cuda));
}

TORCH_LIBRARY_IMPL(npu, AutogradCUDA, m) {
  m.impl("npu_moe_token_permute", TORCH_FN(permute_autograd));
  m.impl("npu_moe_token_unpermute", TORCH_FN(unpermute_autograd));
}

TORCH_LIBRARY_IMPL(npu, Meta, m) {
  m.impl("npu_moe_init_routing_v2", TORCH_FN(init_routing_meta));
  m.impl("npu_moe_token_permute", TORCH_FN(permute_check));
  m.impl("npu_moe_token_permute_grad", TORCH_FN(permute_grad_meta));
  m.impl("npu_moe_token_unpermute", TORCH_FN(unpermute_meta));
  m.impl("npu_moe_token_unpermute_grad", TORCH_FN(unpermute_grad_meta));
}
