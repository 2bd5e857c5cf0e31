// The operators around a layer's experts for torch: their outputs, workspaces and launches, and
// the backward passes of those that have gradients as nodes of torch's autograd engine.
//
// The engine runs a backward pass on a thread of its own, where a node in Python runs at half
// the pace of the caller's thread: 515 FP32 rows with a gate and a norm and their gradients
// took 137 us of host time so and take 89 with these nodes, which need no interpreter (18 us of
// them are the card's). Forward calls made from Python took a token's order, rows and sum 24.5
// us, from here 15.5. Tensors are checked by the functions' callers in Python; every launch goes
// through the C entry points, on the current stream of the tensors' device.

#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include "cfmoe_reader.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using Optional = std::optional<Tensor>;

Tensor given(const Optional &t) { return t ? *t : Tensor(); }

void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

cfmoe_stream stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int status) {
  if (status == 0) return;
  TORCH_CHECK_VALUE(status != CFMOE_EINVAL, cfmoe_last_error());
  TORCH_CHECK(false, cfmoe_last_error());
}

bool dual(const Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
bool dual(const Optional &t) { return t && dual(*t); }

// What would be answered wrongly without a word: the kernels read values alone and have no
// derivative forwards, so that a tensor's tangent would be lost, which stands for zero; and a
// trace holds torch's own calls, so that of an operator it would have the output's allocation.
template <typename... T>
void check_mode(const char *name, const T &...tensors) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  const bool traced = at::tracer::impl::is_dispatch_enabled() ||
                      (TorchDispatchModeTLS::any_modes_set() && TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY));
  TORCH_CHECK_VALUE(!traced, name, " cannot be recorded by torch.jit.trace or torch.fx");
  TORCH_CHECK_VALUE(!(dual(tensors) || ...), name, " has no forward-mode derivative: call it with tensors without a tangent");
}

Tensor contiguous(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

// A workspace of the call's own, undefined where it needs none.
Tensor bytes(int64_t size, const Tensor &like) {
  if (size < 0) check(static_cast<int>(-size));
  if (size == 0) return {};
  return at::empty({size}, like.options().dtype(at::kByte));
}

// Gradients of a pass whose own graph is asked for: the kernels leave none, and who
// differentiates them gets an error.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor &grad : grads) {
    if (!grad.defined()) continue;
    Tensor leaf = grad.detach();
    leaf.set_requires_grad(true);
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that has first derivatives only", 1);
    grad = (*node)({leaf})[0];
  }
  return grads;
}

uint32_t rows_flags(const Tensor &rows, const Tensor &weights) {
  return (rows.scalar_type() == at::kFloat ? CFMOE_FP32 : 0) |
         (weights.defined() && weights.scalar_type() == at::kBFloat16 ? CFMOE_WEIGHTS_BF16 : 0);
}

int32_t narrow(int64_t v) { return static_cast<int32_t>(v); }

Tensor combined(const Tensor &rows, const Tensor &places, const Tensor &weights) {
  c10::DeviceGuard guard(rows.device());
  Tensor out = at::empty({places.size(0), rows.size(1)}, rows.options());
  check(cfmoe_combine_rows(narrow(rows.size(1)), narrow(places.size(1)), rows_flags(rows, weights), pointer(rows),
                           places.const_data_ptr<int32_t>(), pointer(weights), pointer(out), narrow(places.size(0)),
                           stream_of(rows)));
  return out;
}

Tensor gathered(const Tensor &hidden, const Tensor &places) {
  c10::DeviceGuard guard(hidden.device());
  Tensor rows = at::empty({places.numel(), hidden.size(1)}, hidden.options());
  check(cfmoe_gather_rows(narrow(hidden.size(1)), narrow(places.size(1)), rows_flags(hidden, {}), pointer(hidden),
                          places.const_data_ptr<int32_t>(), pointer(rows), narrow(places.size(0)), stream_of(hidden)));
  return rows;
}

struct Gather : torch::autograd::Function<Gather> {
  static Tensor forward(AutogradContext *ctx, const Tensor &hidden, const Tensor &places) {
    ctx->save_for_backward({places});
    return gathered(hidden, places);
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const Tensor places = ctx->get_saved_variables()[0];
    Tensor grad;
    {
      at::NoGradGuard none;
      grad = combined(grads[0].contiguous(), places, {});
    }
    return once({grad, {}});
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext *ctx, const Tensor &rows, const Tensor &places, const Optional &weights) {
    // (rows are read again for the weights' gradient only)
    const bool again = weights && weights->requires_grad();
    ctx->save_for_backward({again ? rows : Tensor(), places, given(weights)});
    return combined(rows, places, given(weights));
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &places = saved[1], &weights = saved[2];
    Tensor grad_rows, grad_weights;
    {
      at::NoGradGuard none;
      c10::DeviceGuard guard(grads[0].device());
      const Tensor grad = grads[0].contiguous();
      if (ctx->needs_input_grad(0)) grad_rows = at::empty({places.numel(), grad.size(1)}, grad.options());
      if (rows.defined() && ctx->needs_input_grad(2)) grad_weights = at::empty_like(weights);
      check(cfmoe_combine_rows_backward(narrow(grad.size(1)), narrow(places.size(1)), rows_flags(grad, weights),
                                        pointer(grad), pointer(rows), places.const_data_ptr<int32_t>(), pointer(weights),
                                        pointer(grad_rows), pointer(grad_weights), narrow(places.size(0)),
                                        stream_of(grad)));
    }
    return once({grad_rows, {}, grad_weights});
  }
};

// joined and next, those that are asked for.
variable_list joined_block(const Tensor &hidden, const Tensor &block, const Tensor &post, const Tensor &gate,
                           const Tensor &next, double scale, double epsilon, int64_t flags, const Tensor &statistics) {
  c10::DeviceGuard guard(hidden.device());
  variable_list made;
  if (block.defined()) made.push_back(at::empty_like(hidden));
  if (next.defined()) made.push_back(at::empty_like(hidden));
  check(cfmoe_join_block(narrow(hidden.size(1)), static_cast<uint32_t>(flags), pointer(hidden), pointer(block),
                         pointer(post), pointer(gate), static_cast<float>(scale), pointer(next),
                         static_cast<float>(epsilon), block.defined() ? pointer(made.front()) : nullptr,
                         next.defined() ? pointer(made.back()) : nullptr, static_cast<float *>(pointer(statistics)),
                         narrow(hidden.size(0)), stream_of(hidden)));
  return made;
}

struct Join : torch::autograd::Function<Join> {
  static variable_list forward(AutogradContext *ctx, const Tensor &hidden, const Optional &given_block,
                               const Optional &given_post, const Optional &given_gate, const Optional &given_next,
                               double scale, double epsilon, int64_t flags) {
    const Tensor block = given(given_block), post = given(given_post), gate = given(given_gate), next = given(given_next);
    const Tensor statistics = at::empty({hidden.size(0), 2}, hidden.options().dtype(at::kFloat));
    ctx->save_for_backward({hidden, block, post, gate, next, statistics});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["flags"] = flags;
    ctx->set_materialize_grads(false);
    return joined_block(hidden, block, post, gate, next, scale, epsilon, flags, statistics);
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &hidden = saved[0], &block = saved[1], &post = saved[2], &gate = saved[3], &next = saved[4];
    Tensor grad_joined, grad_out;
    if (block.defined()) grad_joined = grads.front();
    if (next.defined()) grad_out = grads.back();
    variable_list made(8);
    if (!grad_joined.defined() && !grad_out.defined()) return made;
    const double scale = ctx->saved_data["scale"].toDouble();
    {
      at::NoGradGuard none;
      c10::DeviceGuard guard(hidden.device());
      grad_joined = contiguous(grad_joined);
      grad_out = contiguous(grad_out);
      bool needed[5];
      int edge = 0;  // (tensors that are not given have none)
      for (int i = 0; i < 5; ++i) needed[i] = saved[i].defined() && ctx->needs_input_grad(edge++);
      // a weight of an output that nothing was made of has no gradient
      needed[4] = needed[4] && grad_out.defined();
      // both terms of a plain sum have one gradient, written once as by torch's own sum
      const bool shared = needed[0] && needed[1] && !post.defined() && !gate.defined() && scale == 1.0;
      for (int i = 0; i < 5; ++i)
        if (needed[i] && !(i == 1 && shared)) made[i] = at::empty_like(saved[i]);
      const int sums = made[2].defined() + made[4].defined() + (made[3].defined() && gate.dim() == 1);
      const int32_t tokens = narrow(hidden.size(0)), size = narrow(hidden.size(1));
      Tensor scratch;
      if (sums) scratch = bytes(cfmoe_join_block_backward_scratch_bytes(size, sums, tokens), hidden);
      check(cfmoe_join_block_backward(size, static_cast<uint32_t>(ctx->saved_data["flags"].toInt()), pointer(hidden),
                                      pointer(block), pointer(post), pointer(gate), static_cast<float>(scale),
                                      pointer(next), saved[5].const_data_ptr<float>(), pointer(grad_joined),
                                      pointer(grad_out), pointer(made[0]), pointer(made[1]), pointer(made[2]),
                                      pointer(made[3]), pointer(made[4]), pointer(scratch), tokens, stream_of(hidden)));
      if (shared) made[1] = made[0];
    }
    return once(std::move(made));
  }
};

// offsets, places and pairs of the batch's order.
std::tuple<Tensor, Tensor, Tensor> sort_by_expert(const Tensor &ids, int64_t experts, const Optional &padding) {
  check_mode("sort_by_expert");
  c10::DeviceGuard guard(ids.device());
  const int32_t tokens = narrow(ids.size(0)), top_k = narrow(ids.size(1));
  const auto options = ids.options().dtype(at::kInt);
  Tensor offsets = at::empty({experts + 1}, options), places = at::empty({tokens, top_k}, options);
  Tensor pairs = at::empty({ids.numel()}, options);
  const Tensor scratch = bytes(cfmoe_sort_by_expert_scratch_bytes(tokens, top_k, narrow(experts)), ids);
  check(cfmoe_sort_by_expert(narrow(experts), top_k, ids.scalar_type() == at::kLong ? CFMOE_IDS_INT64 : 0, pointer(ids),
                             static_cast<const uint8_t *>(pointer(given(padding))), offsets.data_ptr<int32_t>(),
                             places.data_ptr<int32_t>(), pairs.data_ptr<int32_t>(), pointer(scratch), tokens,
                             stream_of(ids)));
  return {offsets, places, pairs};
}

// Values from one row to the next; of a single row, which has none, its length.
int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Whether out's rows [tokens, O] and a contiguous tensor have memory in common.
bool overlaps(const Tensor &out, const Tensor &t) {
  if (!t.defined() || t.numel() == 0 || out.numel() == 0) return false;
  const int64_t size = out.element_size(), step = row_stride(out) * size, row = out.size(1) * size;
  const int64_t at = static_cast<const char *>(t.const_data_ptr()) - static_cast<const char *>(out.const_data_ptr());
  // the first of out's rows that ends behind t's begin, if it begins before t's end
  const int64_t first = at < row ? 0 : (at - row) / step + 1;
  return first < out.size(0) && first * step < at + static_cast<int64_t>(t.nbytes());
}

Tensor apply_adapters(const Tensor &base, const Tensor &hidden, const Tensor &encoder, const Tensor &decoder,
                      const Tensor &slots, const Optional &scales, const Optional &to) {
  check_mode("apply_adapters", base, hidden, encoder, decoder, scales, to);
  c10::DeviceGuard guard(hidden.device());
  const int32_t tokens = narrow(hidden.size(0)), size = narrow(hidden.size(1)), outputs = narrow(base.size(1));
  const int32_t adapters = narrow(encoder.size(0)), rank = narrow(encoder.size(1));
  Tensor out = to ? *to : at::empty({tokens, outputs}, hidden.options());
  if (to)
    for (const Tensor &t : {encoder, decoder, slots, given(scales)})
      TORCH_CHECK_VALUE(!overlaps(out, t), "out overlaps the adapters, their slots or their scales");
  const Tensor scratch = bytes(cfmoe_apply_adapters_scratch_bytes(size, outputs, rank, adapters, tokens,
                                                                  out.data_ptr() == hidden.data_ptr()), hidden);
  check(cfmoe_apply_adapters(size, outputs, rank, adapters, slots.scalar_type() == at::kLong ? CFMOE_IDS_INT64 : 0,
                             pointer(base), row_stride(base), pointer(hidden), row_stride(hidden), pointer(encoder),
                             pointer(decoder), pointer(slots), static_cast<const float *>(pointer(given(scales))),
                             pointer(out), row_stride(out), pointer(scratch), tokens, stream_of(hidden)));
  // (what saved the tensor for a backward pass is to see that it changed)
  if (to && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  return out;
}

bool trained(const Tensor &t) { return t.requires_grad(); }
bool trained(const Optional &t) { return t && t->requires_grad(); }

// The module's functions: a node in the graph where a gradient is asked for.

Tensor gather_rows(const Tensor &hidden, const Tensor &places) {
  check_mode("gather_rows", hidden);
  if (at::GradMode::is_enabled() && trained(hidden)) return Gather::apply(hidden, places);
  return gathered(hidden, places);
}

Tensor combine_rows(const Tensor &rows, const Tensor &places, const Optional &weights) {
  check_mode("combine_rows", rows, weights);
  if (at::GradMode::is_enabled() && (trained(rows) || trained(weights))) return Combine::apply(rows, places, weights);
  return combined(rows, places, given(weights));
}

variable_list join_block(const Tensor &hidden, const Optional &block, const Optional &post, const Optional &gate,
                         const Optional &next, double scale, double epsilon, int64_t flags) {
  check_mode(block ? "join_block" : "norm_rows", hidden, block, post, gate, next);
  if (at::GradMode::is_enabled() &&
      (trained(hidden) || trained(block) || trained(post) || trained(gate) || trained(next)))
    return Join::apply(hidden, block, post, gate, next, scale, epsilon, flags);
  return joined_block(hidden, given(block), given(post), given(gate), given(next), scale, epsilon, flags, {});
}

}  // namespace

PYBIND11_MODULE(_torch, m) {
  using release = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.attr("ABI_VERSION") = CFMOE_ABI_VERSION;
  m.def("sort_by_expert", &sort_by_expert, release());
  m.def("apply_adapters", &apply_adapters, release());
  m.def("gather_rows", &gather_rows, release());
  m.def("combine_rows", &combine_rows, release());
  m.def("join_block", &join_block, release());
}
