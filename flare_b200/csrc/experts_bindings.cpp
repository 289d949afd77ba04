// The routed-expert operators as autograd functions, and their Python bindings.
// They take tensors and allocate their outputs and scratch from the caching
// allocator on the current stream: scratch that belongs to one call cannot be
// shared by two captured graphs.  For a few tokens the call itself is what
// counts, so the graph nodes are C++ (a Python node costs some 40 us a step) and
// arguments are checked here (in Python the checks alone took 8 us).  The entry
// points at the end check what a caller may get wrong; the functions above them
// check again what a wrong pointer or size would cost.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "experts.cuh"

namespace py = pybind11;
using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

int code_of(at::ScalarType t) {
  if (t == at::kFloat) return flare::kF32;
  if (t == at::kBFloat16) return flare::kBF16;
  TORCH_CHECK(t == at::kHalf, "expected float32, bfloat16 or float16");
  return flare::kF16;
}

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType t) {
  return at::empty(sizes, like.options().dtype(t));
}

// 2-D rows of unit inner stride
void check_rows(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1), what, ": rows of unit inner stride on a CUDA device");
}
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

const int* ints(const Tensor& t, const Tensor& like, int64_t n, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == like.device() && t.numel() == n, what,
              ": int32, contiguous, on the same device, with as many values as expected");
  return t.data_ptr<int>();
}

// logits [S, B, E] of unit inner stride
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route_topk(const Tensor& logits, int64_t k) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 3, "route_topk: logits [slots, tokens, experts] on a CUDA device");
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t S = logits.size(0), B = logits.size(1), E = logits.size(2);
  TORCH_CHECK(E >= 1 && E <= flare::kRouteMaxExperts, "route_topk: 1 to 512 experts");
  TORCH_CHECK(k >= 1 && k <= E && k <= flare::kRouteMaxTopK, "route_topk: top_k from 1 to the number of experts and 32");
  TORCH_CHECK(S * E < (1ll << 31) - 1 && S * B * k < (1ll << 31) - 512, "route_topk: too many rows");
  TORCH_CHECK(E == 1 || logits.stride(2) == 1, "route_topk: logits need unit inner stride");
  Tensor experts = empty({S, B, k}, logits, at::kInt), weights = empty({S, B, k}, logits, at::kFloat);
  Tensor offsets = empty({S * E + 1}, logits, at::kInt), rows = empty({S * B * k}, logits, at::kInt);
  Tensor row_of = empty({S, B, k}, logits, at::kInt);
  if (S * B == 0) {
    offsets.zero_();
    return {experts, weights, offsets, rows, row_of};
  }
  flare::RouteParams p{};
  p.logits = logits.data_ptr();
  p.stride_slot = logits.stride(0);
  p.stride_token = logits.stride(1);
  p.dtype = code_of(logits.scalar_type());
  p.S = static_cast<int>(S);
  p.B = static_cast<int>(B);
  p.E = static_cast<int>(E);
  p.k = static_cast<int>(k);
  p.experts = experts.data_ptr<int>();
  p.weights = weights.data_ptr<float>();
  p.offsets = offsets.data_ptr<int>();
  p.rows = rows.data_ptr<int>();
  p.row_of = row_of.data_ptr<int>();
  const int64_t ints_needed = flare::route_work_ints(p.S, p.B, p.E);
  Tensor work;
  if (ints_needed > 0) {
    work = empty({ints_needed}, logits, at::kInt);
    p.work = work.data_ptr<int>();
  }
  flare::route_topk(p, stream());
  return {experts, weights, offsets, rows, row_of};
}

Tensor route_topk_backward(const Tensor& experts, const Tensor& weights, const Tensor& dweights, int64_t E, at::ScalarType dtype) {
  const c10::cuda::CUDAGuard guard(experts.device());
  const int64_t k = experts.size(2), T = experts.size(0) * experts.size(1);
  TORCH_CHECK(weights.is_contiguous() && dweights.is_contiguous() && dweights.scalar_type() == at::kFloat && dweights.numel() == T * k,
              "route_topk: gradient of the weights");
  Tensor d = empty({experts.size(0), experts.size(1), E}, experts, dtype);
  flare::RouteBwdParams p{};
  p.experts = ints(experts, experts, T * k, "experts");
  p.weights = weights.data_ptr<float>();
  p.dweights = dweights.data_ptr<float>();
  p.T = T;
  p.E = static_cast<int>(E);
  p.k = static_cast<int>(k);
  p.dlogits = d.data_ptr();
  p.dtype = code_of(dtype);
  flare::route_topk_backward(p, stream());
  return d;
}

flare::SwigluParams swiglu_params(const Tensor& x) {
  check_rows(x, "swiglu");
  TORCH_CHECK(x.size(1) % 2 == 0, "swiglu: an even number of columns [up | gate]");
  flare::SwigluParams p{};
  p.x = x.data_ptr();
  p.ldx = pitch(x);
  p.R = x.size(0);
  p.h = x.size(1) / 2;
  p.dtype = code_of(x.scalar_type());
  return p;
}

// (y, q, scale); q and scale are empty without a checkpoint
std::tuple<Tensor, Tensor, Tensor> swiglu_forward(const Tensor& x, bool keep) {
  flare::SwigluParams p = swiglu_params(x);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = empty({p.R, p.h}, x, x.scalar_type()), q, scale;
  p.y = y.data_ptr();
  if (keep) {
    q = empty({p.R, 2 * p.h}, x, at::kByte);
    scale = empty({p.R, 2 * ((p.h + 31) / 32)}, x, at::kByte);
    p.q = q.data_ptr<uint8_t>();
    p.scale = scale.data_ptr<uint8_t>();
  }
  flare::swiglu_forward(p, stream());
  return {y, q, scale};
}

// from x, or from the checkpoint (q, scale) that the forward pass kept
Tensor swiglu_backward(const optional<Tensor>& x, const optional<Tensor>& q, const optional<Tensor>& scale, const Tensor& dy) {
  check_rows(dy, "swiglu gradient");
  const c10::cuda::CUDAGuard guard(dy.device());
  flare::SwigluParams p{};
  if (x.has_value()) {
    p = swiglu_params(*x);
    TORCH_CHECK(x->scalar_type() == dy.scalar_type(), "swiglu: type of the gradient");
  } else {
    p.R = dy.size(0);
    p.h = dy.size(1);
    p.dtype = code_of(dy.scalar_type());
    TORCH_CHECK(q.has_value() && scale.has_value() && q->is_contiguous() && scale->is_contiguous() && q->numel() == 2 * p.R * p.h &&
                    scale->numel() == p.R * 2 * ((p.h + 31) / 32),
                "swiglu: checkpoint of another size");
    p.q = q->data_ptr<uint8_t>();
    p.scale = scale->data_ptr<uint8_t>();
  }
  TORCH_CHECK(dy.size(0) == p.R && dy.size(1) == p.h, "swiglu: gradient of another size");
  Tensor dx = empty({p.R, 2 * p.h}, dy, dy.scalar_type());
  p.dy = dy.data_ptr();
  p.lddy = pitch(dy);
  p.dx = dx.data_ptr();
  flare::swiglu_backward(p, stream());
  return dx;
}

// y [T, N] from z [R, N]; row_of [T, k]; weights fp32 [T, k] or none (plain sum)
Tensor combine_forward(const Tensor& z, const Tensor& row_of, const optional<Tensor>& weights, int64_t T, int64_t k, at::ScalarType out) {
  check_rows(z, "combine_rows");
  const c10::cuda::CUDAGuard guard(z.device());
  flare::CombineParams p{};
  p.z = z.data_ptr();
  p.ldz = pitch(z);
  p.row_of = ints(row_of, z, T * k, "row_of");
  if (weights.has_value()) {
    TORCH_CHECK(weights->scalar_type() == at::kFloat && weights->is_contiguous() && weights->numel() == T * k && weights->device() == z.device(),
                "combine_rows: weights are float32, contiguous, one for each choice");
    p.weights = weights->data_ptr<float>();
  }
  p.T = T;
  p.R = z.size(0);
  TORCH_CHECK(z.size(1) < (1ll << 31) - 4096, "combine_rows: too wide");
  p.N = static_cast<int>(z.size(1));
  p.k = static_cast<int>(k);
  p.dtype = code_of(z.scalar_type());
  TORCH_CHECK(out == z.scalar_type() || z.scalar_type() == at::kFloat, "combine_rows: type of the result");
  p.out_dtype = code_of(out);
  Tensor y = empty({T, z.size(1)}, z, out);
  p.y = y.data_ptr();
  flare::combine_forward(p, stream());
  return y;
}

// (dz, dw); without weights every row's gradient is its token's, and dw is none
std::tuple<Tensor, optional<Tensor>> combine_backward(const optional<Tensor>& z, const Tensor& row_of, const optional<Tensor>& weights,
                                                      const Tensor& offsets, const Tensor& dy, int64_t R, int64_t T, int64_t k) {
  check_rows(dy, "combine_rows gradient");
  const c10::cuda::CUDAGuard guard(dy.device());
  const int64_t N = dy.size(1);
  TORCH_CHECK(dy.size(0) == T && N < (1ll << 31) - 4096, "combine_rows: gradient of another size");
  flare::CombineParams p{};
  p.row_of = ints(row_of, dy, T * k, "row_of");
  p.T = T;
  p.R = R;
  p.N = static_cast<int>(N);
  p.k = static_cast<int>(k);
  p.dtype = code_of(dy.scalar_type());
  p.dy = dy.data_ptr();
  p.lddy = pitch(dy);
  Tensor dz = empty({R, N}, dy, dy.scalar_type());
  p.dz = dz.data_ptr();
  TORCH_CHECK(offsets.numel() >= 1, "combine_rows: offsets without a value");
  p.total = ints(offsets, dy, offsets.numel(), "offsets") + offsets.numel() - 1;
  optional<Tensor> dw;
  if (weights.has_value()) {
    TORCH_CHECK(z.has_value(), "combine_rows: the weights' gradient needs the rows");
    check_rows(*z, "combine_rows");
    TORCH_CHECK(z->size(0) == R && z->size(1) == N && z->scalar_type() == dy.scalar_type() && weights->is_contiguous() &&
                    weights->scalar_type() == at::kFloat && weights->numel() == T * k,
                "combine_rows: gradient of another size or type");
    p.z = z->data_ptr();
    p.ldz = pitch(*z);
    p.weights = weights->data_ptr<float>();
    dw = empty({T * k}, dy, at::kFloat);
    p.dw = dw->data_ptr<float>();
    if (N == 0) dw->zero_();
  }
  flare::combine_backward(p, stream());
  return {dz, dw};
}

void fill(flare::GroupedArgs& a, const Tensor& offsets, const Tensor& like, int64_t G, int64_t status, int64_t timeout_ns) {
  a.offsets = ints(offsets, like, G + 1, "offsets");
  a.G = static_cast<int>(G);
  a.status = reinterpret_cast<int*>(status);
  a.timeout_ns = static_cast<uint64_t>(timeout_ns);
}

// The tokens' rows in group order (rows behind the last group: zeros)
Tensor gather_rows(const Tensor& x, const Tensor& offsets, const Tensor& row_of) {
  return std::get<0>(combine_backward(std::nullopt, row_of, std::nullopt, offsets, x, row_of.numel(), x.size(0), row_of.size(-1)));
}

// y [R, N]: rows of x (or, for few of them, x[rows]) times their group's weight [G, K, N], plus its bias
Tensor grouped_forward(const Tensor& x, const Tensor& w, const optional<Tensor>& bias, const Tensor& offsets, const optional<Tensor>& rows,
                       int64_t status, int64_t timeout_ns) {
  check_rows(x, "grouped_linear");
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(w.dim() == 3 && w.is_contiguous() && w.scalar_type() == x.scalar_type() && w.device() == x.device() && w.size(1) == x.size(1),
              "grouped_linear: weight [groups, in, out] of x's type");
  flare::GroupedArgs a{};
  a.mode = flare::kGroupedFwd;
  a.dtype = code_of(x.scalar_type());
  a.x = x.data_ptr();
  a.ldx = pitch(x);
  a.x_rows = x.size(0);
  a.R = rows.has_value() ? rows->numel() : x.size(0);
  if (rows.has_value()) a.rows = ints(*rows, x, a.R, "rows");
  a.w = w.data_ptr();
  a.K = static_cast<int>(w.size(1));
  a.N = static_cast<int>(w.size(2));
  fill(a, offsets, x, w.size(0), status, timeout_ns);
  if (bias.has_value()) {
    TORCH_CHECK(bias->is_contiguous() && bias->numel() == w.size(0) * w.size(2) && bias->device() == x.device(), "grouped_linear: bias [groups, out]");
    a.bias = bias->data_ptr();
    a.bias_dtype = code_of(bias->scalar_type());
  }
  Tensor y = empty({a.R, w.size(2)}, x, x.scalar_type());
  if (a.x_rows == 0 || a.R == 0) return y.zero_();
  a.out = y.data_ptr();
  a.out_dtype = a.dtype;
  flare::grouped_gemm(a, stream());
  return y;
}

// dX of the rows [R, K], in dy's type or float32
Tensor grouped_input_grad(const Tensor& dy, const Tensor& w, const Tensor& offsets, at::ScalarType out, int64_t status, int64_t timeout_ns) {
  check_rows(dy, "grouped_linear gradient");
  const c10::cuda::CUDAGuard guard(dy.device());
  TORCH_CHECK(w.dim() == 3 && w.is_contiguous() && w.scalar_type() == dy.scalar_type() && w.device() == dy.device() && w.size(2) == dy.size(1),
              "grouped_linear: gradient of another size or type");
  flare::GroupedArgs a{};
  a.mode = flare::kGroupedDgrad;
  a.dtype = code_of(dy.scalar_type());
  a.dy = dy.data_ptr();
  a.lddy = pitch(dy);
  a.R = dy.size(0);
  a.w = w.data_ptr();
  a.K = static_cast<int>(w.size(1));
  a.N = static_cast<int>(w.size(2));
  fill(a, offsets, dy, w.size(0), status, timeout_ns);
  Tensor dx = empty({a.R, w.size(1)}, dy, out);
  if (a.R == 0) return dx;
  a.out = dx.data_ptr();
  a.out_dtype = code_of(out);
  flare::grouped_gemm(a, stream());
  return dx;
}

// dW [G, K, N], written or (fp32 only) added to.  x is in group order.
void grouped_weight_grad(const Tensor& x, const Tensor& dy, const Tensor& offsets, const Tensor& dw, bool accumulate, int64_t G,
                         int64_t status, int64_t timeout_ns) {
  check_rows(x, "grouped_linear");
  check_rows(dy, "grouped_linear gradient");
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.scalar_type() == dy.scalar_type() && x.device() == dy.device() && x.size(0) == dy.size(0),
              "grouped_linear: gradient of another type or size");
  TORCH_CHECK(dw.is_contiguous() && dw.device() == x.device() && dw.numel() == G * x.size(1) * dy.size(1) &&
                  reinterpret_cast<uintptr_t>(dw.data_ptr()) % 16 == 0 && (!accumulate || dw.scalar_type() == at::kFloat),
              "grouped_linear: weight gradient [groups, in, out], 16-byte aligned, accumulated in float32");
  flare::GroupedArgs a{};
  a.mode = flare::kGroupedWgrad;
  a.dtype = code_of(x.scalar_type());
  a.x = x.data_ptr();
  a.ldx = pitch(x);
  a.x_rows = x.size(0);
  a.dy = dy.data_ptr();
  a.lddy = pitch(dy);
  a.R = dy.size(0);
  a.K = static_cast<int>(x.size(1));
  a.N = static_cast<int>(dy.size(1));
  fill(a, offsets, x, G, status, timeout_ns);
  a.out = dw.data_ptr();
  a.out_dtype = code_of(dw.scalar_type());
  a.accumulate = accumulate ? 1 : 0;
  const int64_t scratch = flare::grouped_work_floats(a.G, a.R, a.K, a.N);
  Tensor work;
  if (scratch > 0) {
    work = empty({scratch}, x, at::kFloat);
    a.work = work.data_ptr<float>();
  }
  if (a.R > 0) flare::grouped_gemm(a, stream());
  else if (!accumulate) dw.zero_();
}

// db [G, N], written or (fp32 only) added to
void group_sums(const Tensor& dy, const Tensor& offsets, const Tensor& db, bool accumulate, int64_t G) {
  const c10::cuda::CUDAGuard guard(dy.device());
  TORCH_CHECK(db.is_contiguous() && db.device() == dy.device() && db.numel() == G * dy.size(1) && (!accumulate || db.scalar_type() == at::kFloat),
              "grouped_linear: bias gradient [groups, out], accumulated in float32");
  flare::GroupSumArgs b{};
  b.y = dy.data_ptr();
  b.ldy = pitch(dy);
  b.R = dy.size(0);
  b.dtype = code_of(dy.scalar_type());
  b.offsets = ints(offsets, dy, G + 1, "offsets");
  b.G = static_cast<int>(G);
  b.N = static_cast<int>(dy.size(1));
  b.out = db.data_ptr();
  b.out_dtype = code_of(db.scalar_type());
  b.accumulate = accumulate ? 1 : 0;
  const int64_t scratch = flare::group_sum_work_floats(b.G, b.R, b.N);
  Tensor work;
  if (scratch > 0) {
    work = empty({scratch}, dy, at::kFloat);
    b.work = work.data_ptr<float>();
  }
  if (b.R > 0) flare::group_colsum(b, stream());
  else if (!accumulate) db.zero_();
}

// ------------------------------------------------------------ graph nodes
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative");
}
// A forward-mode tangent would be lost: the kernels see values only, and the result would have none.
void no_tangent(const char* what, const Tensor& t) {
  if (t._fw_grad(0).defined()) throw std::runtime_error(std::string(what) + " has no forward-mode derivative");
}
bool wants(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}
optional<Tensor> some(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }
Tensor unit_rows(const Tensor& t) { return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous(); }

// Rows that the tiled loads can address: unit inner stride, 16-byte aligned rows.  Others are copied.
Tensor tma_rows(const Tensor& t) {
  const bool aligned = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (aligned && t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1)))) return t;
  return t.is_contiguous() ? t.clone() : t.contiguous();
}

struct RouteFn : torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k) {
    ctx->set_materialize_grads(false);
    auto [experts, weights, offsets, rows, row_of] = route_topk(logits, k);
    ctx->save_for_backward({experts, weights});
    ctx->saved_data["n"] = logits.size(2);
    ctx->saved_data["type"] = static_cast<int64_t>(logits.scalar_type());
    ctx->mark_non_differentiable({experts, offsets, rows, row_of});
    return {experts, weights, offsets, rows, row_of};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("route_topk");
    const auto saved = ctx->get_saved_variables();
    if (!g[1].defined()) return {Tensor(), Tensor()};
    return {route_topk_backward(saved[0], saved[1], g[1].to(at::kFloat).contiguous(), ctx->saved_data["n"].toInt(),
                                static_cast<at::ScalarType>(ctx->saved_data["type"].toInt())),
            Tensor()};
  }
};

struct SwigluFn : torch::autograd::Function<SwigluFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, bool keep) {
    auto [y, q, scale] = swiglu_forward(x, keep);
    if (keep) ctx->save_for_backward({q, scale});
    else ctx->save_for_backward({x});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("swiglu");
    const auto saved = ctx->get_saved_variables();
    if (!g[0].defined()) return {Tensor(), Tensor()};
    const Tensor dy = unit_rows(g[0]);
    return {saved.size() == 2 ? swiglu_backward(std::nullopt, saved[0], saved[1], dy) : swiglu_backward(saved[0], std::nullopt, std::nullopt, dy),
            Tensor()};
  }
};

struct CombineFn : torch::autograd::Function<CombineFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const optional<Tensor>& weights, const Tensor& offsets, const Tensor& row_of) {
    const int64_t k = row_of.size(-1);
    Tensor y = combine_forward(z, row_of, weights, row_of.numel() / k, k, z.scalar_type());
    ctx->save_for_backward({weights.has_value() ? z : Tensor(), weights.value_or(Tensor()), offsets, row_of});
    ctx->saved_data["R"] = z.size(0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("combine_rows");
    const auto saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &weights = saved[1], &offsets = saved[2], &row_of = saved[3];
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const int64_t k = row_of.size(-1);
    auto [dz, dw] = combine_backward(some(z), row_of, some(weights), offsets, unit_rows(g[0]), ctx->saved_data["R"].toInt(), row_of.numel() / k, k);
    return {dz, dw.has_value() ? dw->view(weights.sizes()) : Tensor(), Tensor(), Tensor()};
  }
};

// A weight (or bias) bound to a flat fused optimizer (flat_w, flat_b: its fp32 view of the gradient
// buffer) gets its gradient added there by the kernel; others get a gradient of their own type.
struct GroupedLinearFn : torch::autograd::Function<GroupedLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const Tensor& offsets,
                        const optional<Tensor>& row_of, const optional<Tensor>& flat_w, const optional<Tensor>& flat_b, const Tensor& w,
                        int64_t status, int64_t timeout_ns) {
    // The gathered rows are kept for the weight gradient: they are a small part of what a block keeps
    // (in against 2h + h values a row), and gathering them again costs as much as the first time.
    const Tensor xr = row_of.has_value() ? gather_rows(x, offsets, *row_of) : x;
    Tensor y = grouped_forward(xr, w, bias, offsets, std::nullopt, status, timeout_ns);
    auto& d = ctx->saved_data;
    d["x?"] = x.requires_grad();
    d["w?"] = weight.requires_grad();
    d["b?"] = bias.has_value() && bias->requires_grad();
    ctx->save_for_backward({weight.requires_grad() ? xr : Tensor(), x.requires_grad() ? w : Tensor(), offsets, row_of.value_or(Tensor())});
    d["tokens"] = x.size(0);
    d["flat_w"] = flat_w;
    d["flat_b"] = flat_b;
    d["groups"] = w.sizes();
    d["wshape"] = weight.sizes();
    d["wtype"] = static_cast<int64_t>(weight.scalar_type());
    if (bias.has_value()) {
      d["bshape"] = bias->sizes();
      d["btype"] = static_cast<int64_t>(bias->scalar_type());
    }
    d["status"] = status;
    d["timeout"] = timeout_ns;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("grouped_linear");
    variable_list out(10);
    if (!g[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &offsets = saved[2], &row_of = saved[3];
    auto& d = ctx->saved_data;
    const int64_t status = d["status"].toInt(), timeout = d["timeout"].toInt();
    const Tensor dy = tma_rows(g[0]);
    if (d["x?"].toBool() && ctx->needs_input_grad(0)) {
      if (row_of.defined()) {  // a token's gradient is the sum over its rows: kept in fp32 until it is complete
        const Tensor dr = grouped_input_grad(dy, w, offsets, at::kFloat, status, timeout);
        out[0] = combine_forward(dr, row_of, std::nullopt, d["tokens"].toInt(), row_of.size(-1), dy.scalar_type());
      } else {
        out[0] = grouped_input_grad(dy, w, offsets, dy.scalar_type(), status, timeout);
      }
    }
    const bool need_w = d["w?"].toBool() && ctx->needs_input_grad(1), need_b = d["b?"].toBool() && ctx->needs_input_grad(2);
    if (!need_w && !need_b) return out;
    const auto groups = d["groups"].toIntVector();
    const optional<Tensor> flat_w = d["flat_w"].toOptional<Tensor>(), flat_b = d["flat_b"].toOptional<Tensor>();
    Tensor dw, db;
    if (need_w) {
      dw = flat_w.has_value() ? flat_w->view(groups) : empty(groups, dy, static_cast<at::ScalarType>(d["wtype"].toInt()));
      grouped_weight_grad(x, dy, offsets, dw, flat_w.has_value(), groups[0], status, timeout);
      if (!flat_w.has_value()) out[1] = dw.view(d["wshape"].toIntVector());
    }
    if (need_b) {
      db = flat_b.has_value() ? flat_b->view({-1}) : empty(d["bshape"].toIntVector(), dy, static_cast<at::ScalarType>(d["btype"].toInt()));
      group_sums(dy, offsets, db, flat_b.has_value(), groups[0]);
      if (!flat_b.has_value()) out[2] = db;
    }
    return out;
  }
};

// ------------------------------------------------------------ entry points
// Messages are put together from strings: formatting numbers through a stream here crashes (the
// extension's and torch's C++ runtimes are not the same).
std::string text(const char* v) { return v; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(at::Device d) { return d.str(); }
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <typename... A>
void value_check(bool ok, const A&... what) {
  if (!ok) throw py::value_error((text(what) + ...));
}
template <typename... A>
void type_check(bool ok, const A&... what) {
  if (!ok) throw py::type_error((text(what) + ...));
}
bool is_half(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool is_float(at::ScalarType t) { return is_half(t) || t == at::kFloat; }
void same_device(const Tensor& a, const Tensor& b) {
  value_check(a.device() == b.device(), "all tensors of one op must be on the same device, got ", a.device(), " and ", b.device());
}

py::tuple route_topk_op(const Tensor& logits, int64_t k) {
  value_check(logits.dim() == 2 || logits.dim() == 3, "logits must be [tokens, experts] or [slots, tokens, experts], got ", logits.sizes());
  const int64_t E = logits.size(-1);
  value_check(k >= 1 && k <= E && k <= flare::kRouteMaxTopK, "top_k must be from 1 to the number of experts (", E, ") and ",
              flare::kRouteMaxTopK, ", got ", k);
  value_check(E <= flare::kRouteMaxExperts, "at most ", flare::kRouteMaxExperts, " experts a slot, got ", E);
  type_check(is_float(logits.scalar_type()), "logits must be float32, bfloat16 or float16, got ", logits.scalar_type());
  no_tangent("route_topk", logits);
  const bool flat = logits.dim() == 2;
  Tensor lg = flat ? logits.unsqueeze(0) : logits;
  if (lg.stride(2) != 1 && E > 1) lg = lg.contiguous();
  value_check(lg.size(0) * E <= flare::kRouteMaxGroups, "at most ", flare::kRouteMaxGroups, " groups (slots * experts), got ", lg.size(0) * E);
  value_check(lg.size(0) * lg.size(1) * k < (1ll << 31) - 512, "too many rows: 2^31 - 513 at most");
  Tensor experts, weights, offsets, rows, row_of;
  if (wants({&lg})) {
    const auto o = RouteFn::apply(lg, k);
    experts = o[0], weights = o[1], offsets = o[2], rows = o[3], row_of = o[4];
  } else {
    std::tie(experts, weights, offsets, rows, row_of) = route_topk(lg, k);
  }
  if (flat) experts = experts.squeeze(0), weights = weights.squeeze(0), row_of = row_of.squeeze(0);
  return py::make_tuple(experts, weights, offsets, rows, row_of);
}

Tensor swiglu_op(const Tensor& x, bool keep) {
  value_check(x.dim() == 2 && x.size(1) % 2 == 0, "x must be [rows, 2h], got ", x.sizes());
  type_check(is_float(x.scalar_type()), "x must be float32, bfloat16 or float16, got ", x.scalar_type());
  no_tangent("swiglu", x);
  const Tensor v = unit_rows(x);
  if (wants({&v})) return SwigluFn::apply(v, keep);
  return std::get<0>(swiglu_forward(v, false));
}

Tensor combine_rows_op(const Tensor& z, const optional<Tensor>& weights, const Tensor& offsets, const Tensor& row_of) {
  value_check(row_of.dim() >= 2 && row_of.size(-1) >= 1, "row_of must be [.., tokens, choices], got ", row_of.sizes());
  value_check(z.dim() == 2 && z.size(0) == row_of.numel(), "z must be [", row_of.numel(), ", n] for this route, got ", z.sizes());
  type_check(is_float(z.scalar_type()), "z must be float32, bfloat16 or float16, got ", z.scalar_type());
  same_device(z, row_of);
  // the gradient of z reads the last offset
  value_check(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.size(0) >= 1 && offsets.is_contiguous(),
              "offsets must be int32 [groups + 1], got ", offsets.scalar_type(), " ", offsets.sizes());
  same_device(z, offsets);
  value_check(row_of.scalar_type() == at::kInt && row_of.is_contiguous(), "row_of must be int32 and contiguous, got ", row_of.scalar_type());
  no_tangent("combine_rows", z);
  if (weights.has_value()) no_tangent("combine_rows", *weights);
  const Tensor v = unit_rows(z);
  optional<Tensor> w;
  if (weights.has_value()) {
    value_check(weights->numel() == row_of.numel() && weights->dim() >= 1 && weights->size(-1) == row_of.size(-1), "weights must have the shape ", row_of.sizes(), ", got ", weights->sizes());
    same_device(z, *weights);
    w = weights->to(at::kFloat).contiguous();
  }
  if (wants({&v}) || (w.has_value() && wants({&*w}))) return CombineFn::apply(v, w, offsets, row_of);
  const int64_t k = row_of.size(-1);
  return combine_forward(v, row_of, w, row_of.numel() / k, k, v.scalar_type());
}

Tensor grouped_linear_op(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const Tensor& offsets, const optional<Tensor>& rows,
                         const optional<Tensor>& row_of, const optional<Tensor>& flat_w, const optional<Tensor>& flat_b, int64_t status,
                         int64_t timeout_ns) {
  value_check(x.dim() == 2 && weight.dim() >= 3 && weight.size(-2) == x.size(1), "x must be [rows, in] and weight [.., in, out], got ", x.sizes(),
              " and ", weight.sizes());
  const int64_t K = weight.size(-2), N = weight.size(-1);
  type_check(is_half(x.scalar_type()) && (weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat),
             "x must be bfloat16 or float16 and weight of the same type or float32, got ", x.scalar_type(), " and ", weight.scalar_type());
  value_check(K > 0 && N > 0 && K % 8 == 0 && N % 8 == 0, "in and out must be multiples of 8, got ", K, " and ", N);
  const int64_t groups = weight.numel() / (K * N);
  value_check(groups >= 1 && groups <= flare::kGroupedMaxGroups, "1 to ", flare::kGroupedMaxGroups, " groups, got ", groups);
  same_device(x, weight);
  same_device(x, offsets);
  value_check(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.size(0) == groups + 1 && offsets.is_contiguous(), "offsets must be int32 [",
              groups + 1, "] for ", groups, " groups, got ", offsets.scalar_type(), " ", offsets.sizes());
  if (rows.has_value()) {
    value_check(row_of.has_value() && row_of->dim() >= 1 && row_of->size(-1) >= 1 && row_of->numel() == rows->numel() && row_of->numel() == x.size(0) * row_of->size(-1), "route of ",
                rows->numel(), " rows does not fit ", x.size(0), " tokens");
    same_device(x, *rows);
    same_device(x, *row_of);
  }
  value_check((rows.has_value() ? rows->numel() : x.size(0)) < (1ll << 31) - 512, "too many rows: 2^31 - 513 at most");
  if (bias.has_value()) {
    value_check(bias->dim() >= 1 && bias->size(-1) == N && bias->numel() == groups * N, "bias must be [.., ", N, "] for ", groups, " groups, got ", bias->sizes());
    type_check(is_float(bias->scalar_type()), "bias must be float32, bfloat16 or float16, got ", bias->scalar_type());
    same_device(x, *bias);
  }
  no_tangent("grouped_linear", x);
  no_tangent("grouped_linear", weight);
  if (bias.has_value()) no_tangent("grouped_linear", *bias);
  const Tensor v = tma_rows(x);
  optional<Tensor> b;
  if (bias.has_value()) b = bias->contiguous();
  // A float32 weight is rounded in every call, whichever groups have rows: nothing is kept from one call
  // to the next, since the parameter may have changed in between.
  Tensor w = weight.detach().reshape({groups, K, N}).to(x.scalar_type()).contiguous();
  if (reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 != 0) w = w.clone();
  if (wants({&v, &weight}) || (b.has_value() && wants({&*b})))
    return GroupedLinearFn::apply(v, weight, b, offsets, row_of, flat_w, flat_b, w, status, timeout_ns);
  if (rows.has_value() && !flare::grouped_few_rows(rows->numel()))
    return grouped_forward(gather_rows(v, offsets, *row_of), w, b, offsets, std::nullopt, status, timeout_ns);
  return grouped_forward(v, w, b, offsets, rows, status, timeout_ns);
}

}  // namespace

void register_experts(py::module_& m) {
  m.def("route_topk", &route_topk_op);
  m.def("swiglu", &swiglu_op);
  m.def("combine_rows", &combine_rows_op);
  m.def("grouped_linear", &grouped_linear_op);
}
