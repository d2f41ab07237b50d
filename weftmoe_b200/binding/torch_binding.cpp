// Autograd edges of the router operators and of the FP8 projection: allocation of results, the C ABI calls
// (include/weftmoe_b200.h) and their backward passes.  In C++ because a training call of these is a few short kernels:
// as Python autograd functions the calls took 98 (router), 130 (balance loss) and 160 us (router step) on the host,
// several times what the GPU needs.  Arguments are checked by router.py and fp8.py before they get here.
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "../../include/weftmoe_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Status -> the exception the Python layer raises for it (ValueError for contract violations).
void check(int code) {
  if (code == WM_OK) return;
  const char* message = wm_last_error();
  if (code == WM_ERR_INVALID || code == WM_ERR_CAPACITY || code == WM_ERR_ROUTE) TORCH_CHECK_VALUE(false, message);
  TORCH_CHECK(false, message);
}

// The current stream of the tensors' device, made current; storage of tensors from another stream that the call uses
// (reads or, where the caller gives a result, writes) is kept for it.
struct Launch {
  c10::cuda::CUDAGuard guard;
  c10::cuda::CUDAStream stream;
  explicit Launch(const Tensor& like) : guard(like.device()), stream(c10::cuda::getCurrentCUDAStream()) {}
  void uses(const Tensor& t) {
    if (t.defined() && t.numel() > 0) c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), stream);
  }
  operator void*() const { return static_cast<void*>(stream.stream()); }
};

void refuse_second_derivative(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " cannot be differentiated again");
}

// Inputs of forward-mode differentiation need not require a gradient, so they would pass as constants and the
// results would lack their tangents.
void refuse_tangent(const char* what, const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), what, " has no derivative in forward mode");
}

// In a backward pass under capture: gradients that go on to a node of the legacy default stream, as to a leaf whose
// gradient an eager graph, still alive, accumulates there.  That stream cannot join a capture; autograd would have it wait
// for this one, which fails and can take the process along, so this is refused before anything is enqueued.
void refuse_uncaptured_gradient(const char* what, const Tensor& like) {
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const c10::Stream outside = c10::cuda::getDefaultCUDAStream(like.device().index()).unwrap();
  for (uint32_t i = 0; i < node->num_outputs(); ++i) {
    const torch::autograd::Edge& edge = node->next_edge(i);
    if (!edge.is_valid() || !node->task_should_compute_output(i)) continue;
    const optional<c10::Stream> stream = edge.function->stream();
    if (!stream.has_value() || *stream != outside) continue;
    const c10::cuda::CUDAGuard guard(like.device());
    TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None, what,
                " cannot be captured: one goes to a leaf or a node of an eager graph on the default stream; drop that "
                "graph before the capture, or make it on a side stream");
    return;
  }
}

template <class T>
T* data(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor or_none(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// ------------------------------------------------------------------ router
struct Choice {
  int64_t top_k = 1, score = 0;
  bool renormalize = false;
  double scale = 1.0;
};

wm_router describe(const Tensor& logits, const Choice& c, const Tensor& bias, const Tensor& padding,
                   const Tensor& sequences) {
  wm_router r{};
  r.logits = logits.data_ptr();
  r.row_stride = logits.size(0) > 1 ? logits.stride(0) : logits.size(1);
  r.dtype = logits.scalar_type() == at::kBFloat16 ? 0 : logits.scalar_type() == at::kFloat ? 1 : 2;
  r.tokens = static_cast<int32_t>(logits.size(0));
  r.experts = static_cast<int32_t>(logits.size(1));
  r.top_k = static_cast<int32_t>(c.top_k);
  r.score = static_cast<int32_t>(c.score);
  r.renormalize = c.renormalize;
  r.scale = static_cast<float>(c.scale);
  r.num_sequences = sequences.defined() ? static_cast<int32_t>(sequences.numel() - 1) : 0;
  r.bias = data<float>(bias);
  r.padding = data<uint8_t>(padding);
  r.sequences = data<int32_t>(sequences);
  return r;
}

// Rows of unit column stride (copied only if they are not).
Tensor rows_of(const Tensor& logits) {
  const bool plain = (logits.size(1) == 1 || logits.stride(1) == 1) &&
                     (logits.size(0) <= 1 || logits.stride(0) >= logits.size(1));
  return plain ? logits : logits.contiguous();
}

struct Loss {
  Tensor loss, table, workspace;
  Loss(const Tensor& logits, const wm_router& r) {
    int64_t bytes = 0;
    check(wm_router_workspace(&r, &bytes));
    loss = at::empty({}, logits.options().dtype(at::kFloat));
    table = at::empty({static_cast<int64_t>(std::max(1, r.num_sequences)) * r.experts + 1}, loss.options());
    workspace = at::empty({bytes}, logits.options().dtype(at::kByte));
  }
};

Tensor empty_counts(const Tensor& like, int64_t experts, const Tensor& sequences) {
  const auto options = like.options().dtype(at::kInt);
  return sequences.defined() ? at::empty({sequences.numel() - 1, experts}, options) : at::empty({experts}, options);
}

// routes, gates, and with the loss counts, loss, table
variable_list route_forward(const Tensor& rows, const Choice& c, const Tensor& bias, const Tensor& padding,
                            const Tensor& sequences, bool balance) {
  Launch launch(rows);
  const wm_router r = describe(rows, c, bias, padding, sequences);
  Tensor routes = at::empty({rows.size(0), c.top_k}, rows.options().dtype(at::kInt));
  Tensor gates = at::empty({rows.size(0), c.top_k}, rows.options().dtype(at::kFloat));
  for (const Tensor& t : {rows, bias, padding, sequences}) launch.uses(t);
  if (!balance) {
    check(wm_router_forward(&r, data<int32_t>(routes), data<float>(gates), nullptr, nullptr, nullptr, nullptr, 0, launch));
    return {routes, gates};
  }
  Loss l(rows, r);
  Tensor counts = empty_counts(rows, rows.size(1), sequences);
  check(wm_router_forward(&r, data<int32_t>(routes), data<float>(gates), data<int32_t>(counts), data<float>(l.loss),
                          data<float>(l.table), l.workspace.data_ptr(), l.workspace.numel(), launch));
  return {routes, gates, counts, l.loss, l.table};
}

std::pair<Tensor, Tensor> balance_forward(const Tensor& rows, const Tensor& counts, int64_t score, const Tensor& padding,
                                          const Tensor& sequences) {
  Launch launch(rows);
  Choice c;
  c.score = score;
  const wm_router r = describe(rows, c, Tensor(), padding, sequences);
  Loss l(rows, r);
  for (const Tensor& t : {rows, counts, padding, sequences}) launch.uses(t);
  check(wm_balance_forward(&r, data<int32_t>(counts), data<float>(l.loss), data<float>(l.table), l.workspace.data_ptr(),
                           l.workspace.numel(), launch));
  return {l.loss, l.table};
}

Tensor router_backward(const Tensor& rows, const Choice& c, const Tensor& padding, const Tensor& sequences,
                       const Tensor& routes, Tensor dgates, const Tensor& table, Tensor dloss) {
  refuse_second_derivative("The router's gradients");
  const bool gates_part = dgates.defined(), loss_part = dloss.defined();
  if (!gates_part && !loss_part) return Tensor();
  refuse_uncaptured_gradient("The router's gradients", rows);
  Launch launch(rows);
  if (gates_part) dgates = dgates.to(at::kFloat).contiguous();   // broadcast gradients are expanded
  if (loss_part) dloss = dloss.to(at::kFloat).contiguous();
  const wm_router r = describe(rows, c, Tensor(), padding, sequences);
  Tensor dlogits = at::empty(rows.sizes(), rows.options());
  for (const Tensor& t : {rows, padding, sequences, routes, dgates, table, dloss}) launch.uses(t);
  check(wm_router_backward(&r, gates_part ? data<int32_t>(routes) : nullptr, data<float>(dgates),
                           loss_part ? data<float>(table) : nullptr, data<float>(dloss), dlogits.data_ptr(), launch));
  return dlogits;
}

void keep_choice(AutogradContext* ctx, const Choice& c) {
  ctx->saved_data["top_k"] = c.top_k;
  ctx->saved_data["score"] = c.score;
  ctx->saved_data["renormalize"] = c.renormalize;
  ctx->saved_data["scale"] = c.scale;
}
Choice kept_choice(AutogradContext* ctx) {
  Choice c;
  c.top_k = ctx->saved_data["top_k"].toInt();
  c.score = ctx->saved_data["score"].toInt();
  c.renormalize = ctx->saved_data["renormalize"].toBool();
  c.scale = ctx->saved_data["scale"].toDouble();
  return c;
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Choice& c, const optional<Tensor>& bias,
                               const optional<Tensor>& padding_, const optional<Tensor>& sequences_, bool balance) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor rows = rows_of(logits), padding = or_none(padding_), sequences = or_none(sequences_);
    variable_list out = route_forward(rows, c, or_none(bias), padding, sequences, balance);
    keep_choice(ctx, c);
    ctx->save_for_backward({rows, padding, sequences, out[0], balance ? out[4] : Tensor()});
    ctx->set_materialize_grads(false);
    if (balance) {
      out.pop_back();
      ctx->mark_non_differentiable({out[0], out[2]});
    } else {
      ctx->mark_non_differentiable({out[0]});
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    Tensor dlogits = router_backward(s[0], kept_choice(ctx), s[1], s[2], s[3], grads[1], s[4],
                                     grads.size() > 3 ? grads[3] : Tensor());
    return {dlogits, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct Balance : torch::autograd::Function<Balance> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& counts, int64_t score,
                        const optional<Tensor>& padding_, const optional<Tensor>& sequences_) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor rows = rows_of(logits), padding = or_none(padding_), sequences = or_none(sequences_);
    auto [loss, table] = balance_forward(rows, counts, score, padding, sequences);
    ctx->saved_data["score"] = score;
    ctx->save_for_backward({rows, padding, sequences, table});
    ctx->set_materialize_grads(false);
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    Choice c;
    c.score = ctx->saved_data["score"].toInt();
    return {router_backward(s[0], c, s[1], s[2], Tensor(), Tensor(), s[3], grads[0]), Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

bool wants_gradient(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

variable_list route(const Tensor& logits, int64_t top_k, int64_t score, bool renormalize, double scale,
                    const optional<Tensor>& bias, const optional<Tensor>& padding, const optional<Tensor>& sequences,
                    bool balance) {
  refuse_tangent("The router", logits);
  const Choice c{top_k, score, renormalize, scale};
  if (wants_gradient(logits))
    return Route::apply(logits, c, bias, padding, sequences, balance);
  variable_list out = route_forward(rows_of(logits), c, or_none(bias), or_none(padding), or_none(sequences), balance);
  if (balance) out.pop_back();
  return out;
}

Tensor balance(const Tensor& logits, const Tensor& counts, int64_t score, const optional<Tensor>& padding,
               const optional<Tensor>& sequences) {
  refuse_tangent("balance_loss", logits);
  if (wants_gradient(logits)) return Balance::apply(logits, counts, score, padding, sequences);
  return balance_forward(rows_of(logits), counts, score, or_none(padding), or_none(sequences)).first;
}

Tensor expert_counts(const Tensor& routes, int64_t experts, const optional<Tensor>& sequences) {
  Launch launch(routes);
  const Tensor seq = or_none(sequences);
  Tensor counts = empty_counts(routes, experts, seq);
  launch.uses(routes);
  launch.uses(seq);
  check(wm_expert_counts(data<int32_t>(routes), static_cast<int32_t>(routes.size(0)), static_cast<int32_t>(routes.size(1)),
                         static_cast<int32_t>(experts), data<int32_t>(seq),
                         seq.defined() ? static_cast<int32_t>(seq.numel() - 1) : 0, data<int32_t>(counts), launch));
  return counts;
}

// ------------------------------------------------------------------ FP8
struct Quantised {
  Tensor values, scales;   // [rows][ceil128(k)] E4M3, [rows][ceil(k / 128)] FP32
  Quantised() = default;
  Quantised(const Tensor& like, int64_t rows, int64_t k)
      : values(at::empty({rows, (k + 127) / 128 * 128}, like.options().dtype(at::kFloat8_e4m3fn))),
        scales(at::empty({rows, (k + 127) / 128}, like.options().dtype(at::kFloat))) {}
};

// The C ABI takes sizes in 32 bits.
void check_sizes(std::initializer_list<int64_t> sizes) {
  for (const int64_t n : sizes)
    TORCH_CHECK_VALUE(n >= 0 && n < (int64_t{1} << 31), "FP8 matrices must have fewer than 2^31 rows and columns");
}

int is_f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }

// out[m][n] (+)= A[m][k] B[n][k]^T on the current device and stream
void matmul_into(Launch& launch, const Tensor& a, const Tensor& as, int64_t a_block_rows, const Tensor& b, const Tensor& bs,
                 int64_t b_block_rows, const Tensor& out, int64_t ld, int64_t m, int64_t n, int64_t k, bool accumulate) {
  int64_t bytes = 0;
  check(wm_fp8_matmul_workspace(static_cast<int32_t>(m), static_cast<int32_t>(n), static_cast<int32_t>(k), &bytes));
  Tensor workspace;
  if (bytes) workspace = at::empty({bytes}, as.options().dtype(at::kByte));
  for (const Tensor& t : {a, as, b, bs}) launch.uses(t);
  check(wm_fp8_matmul(a.data_ptr(), data<float>(as), b.data_ptr(), data<float>(bs), out.data_ptr(), ld,
                      static_cast<int32_t>(m), static_cast<int32_t>(n), static_cast<int32_t>(k),
                      static_cast<int32_t>(a_block_rows), static_cast<int32_t>(b_block_rows), is_f32(out), accumulate,
                      data<void>(workspace), bytes, launch));
}

Tensor fp8_matmul(const Tensor& a, const Tensor& as, int64_t a_block_rows, const Tensor& b, const Tensor& bs,
                  int64_t b_block_rows, int64_t m, int64_t n, int64_t k, bool out_is_f32, const optional<Tensor>& given,
                  bool accumulate) {
  for (const Tensor& t : {as, bs, or_none(given)})
    if (t.defined()) refuse_tangent("fp8_matmul", t);
  check_sizes({m, n, k});
  Launch launch(as);
  Tensor out = given.has_value() ? *given : at::empty({m, n}, as.options().dtype(out_is_f32 ? at::kFloat : at::kBFloat16));
  if (given.has_value()) launch.uses(out);
  matmul_into(launch, a, as, a_block_rows, b, bs, b_block_rows, out, m > 1 ? out.stride(0) : std::max<int64_t>(n, 1), m, n,
              k, accumulate);
  if (given.has_value() && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  return out;
}

void quantise_both(Launch& launch, const Tensor& x, Quantised& rows, Quantised& columns) {
  const int64_t m = x.size(0), k = x.size(1);
  rows = Quantised(x, m, k);
  columns = Quantised(x, k, m);
  launch.uses(x);
  check(wm_fp8_quantize_both(x.data_ptr(), is_f32(x), 1, static_cast<int32_t>(m), static_cast<int32_t>(k),
                             rows.values.data_ptr(), data<float>(rows.scales), columns.values.data_ptr(),
                             data<float>(columns.scales), launch));
}
Quantised quantise(Launch& launch, const Tensor& x, bool transpose) {
  Quantised q(x, x.size(transpose ? 1 : 0), x.size(transpose ? 0 : 1));
  launch.uses(x);
  check(wm_fp8_quantize(x.data_ptr(), is_f32(x), 1, static_cast<int32_t>(x.size(0)), static_cast<int32_t>(x.size(1)), 1,
                        transpose, q.values.data_ptr(), data<float>(q.scales), launch));
  return q;
}

// y = x W^T, quantising x on the way
Tensor linear_forward(const Tensor& x, const Tensor& wq, const Tensor& ws, int64_t n) {
  Launch launch(x);
  const int32_t rows = static_cast<int32_t>(x.size(0)), k = static_cast<int32_t>(x.size(1));
  int64_t bytes = 0;
  check(wm_fp8_linear_workspace(rows, static_cast<int32_t>(n), k, &bytes));
  Tensor y = at::empty({x.size(0), n}, x.options());
  Tensor workspace = at::empty({bytes}, x.options().dtype(at::kByte));
  for (const Tensor& t : {x, wq, ws}) launch.uses(t);
  check(wm_fp8_linear(x.data_ptr(), is_f32(x), rows, k, wq.data_ptr(), data<float>(ws), static_cast<int32_t>(n),
                      y.data_ptr(), workspace.data_ptr(), bytes, launch));
  return y;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& wq, const Tensor& ws,
                        const optional<Tensor>& wtq_, const optional<Tensor>& wts_, bool to_weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor wtq = or_none(wtq_), wts = or_none(wts_);
    const int64_t n = weight.size(0);
    ctx->saved_data["x_type"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["tokens"] = x.size(0);
    if (!to_weight) {
      ctx->save_for_backward({weight, wtq, wts});   // the weight: detects optimizer updates before backward
      return linear_forward(x, wq, ws, n);
    }
    Launch launch(x);
    Quantised rows, columns;   // the blocks along the tokens, a byte each, are kept for dW instead of x
    quantise_both(launch, x, rows, columns);
    Tensor y = at::empty({x.size(0), n}, x.options());
    matmul_into(launch, rows.values, rows.scales, 1, wq, ws, 128, y, n, x.size(0), n, x.size(1), false);
    ctx->save_for_backward({weight, wtq, wts, columns.values, columns.scales});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_second_derivative("The gradients of fp8_linear");
    const variable_list s = ctx->get_saved_variables();
    variable_list out(7);
    if (!grads[0].defined()) return out;
    refuse_uncaptured_gradient("The gradients of fp8_linear", grads[0]);
    const Tensor& weight = s[0];
    const Tensor dy = grads[0].contiguous();
    const bool to_x = ctx->needs_input_grad(0), to_weight = ctx->needs_input_grad(1);
    const int64_t tokens = ctx->saved_data["tokens"].toInt(), n = weight.size(0), k = weight.size(1);
    Launch launch(dy);
    Quantised rows, columns;
    if (to_x && to_weight) quantise_both(launch, dy, rows, columns);
    else if (to_x) rows = quantise(launch, dy, false);
    else if (to_weight) columns = quantise(launch, dy, true);
    if (to_x) {
      const auto type = static_cast<at::ScalarType>(ctx->saved_data["x_type"].toInt());
      out[0] = at::empty({tokens, k}, dy.options().dtype(type));
      matmul_into(launch, rows.values, rows.scales, 1, s[1], s[2], 128, out[0], k, tokens, k, n, false);
    }
    if (to_weight) {
      out[1] = at::empty({n, k}, weight.options());
      matmul_into(launch, columns.values, columns.scales, 1, s[3], s[4], 1, out[1], k, n, k, tokens, false);
    }
    return out;
  }
};

Tensor fp8_linear(const Tensor& x, const Tensor& weight, const Tensor& wq, const Tensor& ws, const optional<Tensor>& wtq,
                  const optional<Tensor>& wts) {
  refuse_tangent("fp8_linear", x);
  refuse_tangent("fp8_linear", weight);
  check_sizes({x.size(0), x.size(1), weight.size(0)});
  const bool to_weight = wants_gradient(weight);
  if (wants_gradient(x) || to_weight) return Linear::apply(x, weight, wq, ws, wtq, wts, to_weight);
  return linear_forward(x, wq, ws, weight.size(0));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("route", &route);
  m.def("balance", &balance);
  m.def("expert_counts", &expert_counts);
  m.def("fp8_matmul", &fp8_matmul);
  m.def("fp8_linear", &fp8_linear);
}
