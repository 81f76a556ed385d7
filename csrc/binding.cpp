// Torch registration: torch.classes.flashoverlap_class.{OverlapImpl,BaselineImpl} and
// torch.ops.flashoverlap_op.*, with the reference's method names and argument orders
// (src/pybind.cpp:114-150) plus the additions this library makes (marked below).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/custom_class.h>
#include <torch/library.h>

#include "common/fo_check.h"
#include "comm/nccl_utils.h"
#include "elementwise/fo_elementwise.h"
#include "flags/fo_wait.h"
#include "moe/fo_moe.h"
#include "norm/fo_norm.h"
#include "norm/fo_norm_block.h"
#include "runtime/baseline_impl.h"
#include "runtime/fused_common.h"
#include "runtime/loopback.h"
#include "runtime/overlap_impl.h"

namespace {

using fo::BaselineImpl;
using fo::OverlapImpl;

int sm_count_of_current_device() {
  return at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
}

bool is_bf16(const at::Tensor& t, const char* name) {
  FO_CHECK(t.is_cuda() && t.is_contiguous(), name, " must be a contiguous CUDA tensor");
  FO_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name,
              " must be bfloat16 or float16");
  return t.scalar_type() == at::kBFloat16;
}

std::vector<int64_t> generate_nccl_id() { return fo::generate_nccl_id(); }

// X: tile-contiguous [rows*dim]; RX: row-major output [rows, dim]; RW: [dim].
void reorder_rmsnorm_eps(at::Tensor X, at::Tensor RX, at::Tensor RW, int64_t BM, int64_t BN,
                         int64_t rldn, at::Tensor RA, double eps) {
  const bool bf = is_bf16(X, "X");
  FO_CHECK(RX.scalar_type() == X.scalar_type() && RW.scalar_type() == X.scalar_type(),
              "X, RX and RW must share a dtype");
  FO_CHECK(RX.dim() == 2 && RX.is_contiguous() && RX.is_cuda(), "RX must be [rows, dim]");
  const int rows = static_cast<int>(RX.size(0));
  const int dim = static_cast<int>(RX.size(1));
  FO_CHECK(X.numel() >= RX.numel() && RW.numel() == dim, "shape mismatch");
  FO_CHECK(RA.is_cuda() && RA.scalar_type() == at::kInt && RA.is_contiguous() &&
                  RA.numel() >= static_cast<int64_t>(rows / BM) * (dim / BN),
              "RA must be an int32 CUDA tensor with one entry per tile");
  c10::cuda::CUDAGuard guard(X.device());
  fo::cuda_check(fo::reorder_rmsnorm_launch(X.data_ptr(), RX.data_ptr(), RW.data_ptr(), rows, dim,
                                            static_cast<int>(BM), static_cast<int>(BN),
                                            static_cast<int>(rldn), RA.data_ptr<int>(),
                                            static_cast<float>(eps), bf, sm_count_of_current_device(),
                                            c10::cuda::getCurrentCUDAStream().stream()),
                 "reorder_rmsnorm");
}

// Reference signature (src/pybind.cpp:149): eps fixed at 1e-5 as in src/rmsnorm/rmsnorm.cuh:102.
void reorder_rmsnorm(at::Tensor X, at::Tensor RX, at::Tensor RW, int64_t BM, int64_t BN,
                     int64_t rldn, at::Tensor RA) {
  reorder_rmsnorm_eps(X, RX, RW, BM, BN, rldn, RA, 1e-5);
}

void rmsnorm(at::Tensor X, at::Tensor RX, at::Tensor RW, double eps) {
  const bool bf = is_bf16(X, "X");
  FO_CHECK(RX.scalar_type() == X.scalar_type() && RW.scalar_type() == X.scalar_type(),
              "X, RX and RW must share a dtype");
  FO_CHECK(X.dim() == 2 && RX.sizes() == X.sizes() && RX.is_contiguous() && RX.is_cuda(),
              "X and RX must be [rows, dim]");
  const int rows = static_cast<int>(X.size(0));
  const int dim = static_cast<int>(X.size(1));
  FO_CHECK(RW.numel() == dim, "RW must have dim elements");
  c10::cuda::CUDAGuard guard(X.device());
  fo::cuda_check(fo::rmsnorm_launch(X.data_ptr(), RX.data_ptr(), RW.data_ptr(), rows, dim,
                                    static_cast<float>(eps), bf, sm_count_of_current_device(),
                                    c10::cuda::getCurrentCUDAStream().stream()),
                 "rmsnorm");
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Whether output `o` shares memory with `t` other than by being it (equal sizes): the row kernels read an
// element and store it in the same thread.
bool clashes(const at::Tensor& o, const at::Tensor& t) {
  return o.data_ptr() != t.data_ptr() && fo::overlaps(o, o.numel(), t, t.numel());
}

// H = X + T, RX = rmsnorm(H) * RW; H and RX may be X or T, not the same one.
void add_rmsnorm(at::Tensor X, at::Tensor T, at::Tensor H, at::Tensor RX, at::Tensor RW, double eps) {
  const bool bf = is_bf16(X, "X");
  is_bf16(T, "T");
  is_bf16(H, "H");
  is_bf16(RX, "RX");
  is_bf16(RW, "RW");
  FO_CHECK(T.scalar_type() == X.scalar_type() && H.scalar_type() == X.scalar_type() &&
               RX.scalar_type() == X.scalar_type() && RW.scalar_type() == X.scalar_type(),
           "X, T, H, RX and RW must share a dtype");
  FO_CHECK(X.dim() == 2 && T.sizes() == X.sizes() && H.sizes() == X.sizes() && RX.sizes() == X.sizes(),
           "X, T, H and RX must be [rows, dim]");
  FO_CHECK(RW.numel() == X.size(1), "RW must have dim elements");
  for (const at::Tensor& t : {T, H, RX, RW}) fo::check_device(t, X, "an operand of add_rmsnorm");
  FO_CHECK(!fo::overlaps(H, H.numel(), RX, RX.numel()), "H and RX must not alias");
  FO_CHECK(!clashes(H, X) && !clashes(H, T) && !clashes(RX, X) && !clashes(RX, T),
           "H and RX must each be X, T or memory of their own");
  FO_CHECK(!fo::overlaps(RW, RW.numel(), H, H.numel()) && !fo::overlaps(RW, RW.numel(), RX, RX.numel()),
           "RW must not alias H or RX");
  FO_CHECK(aligned16(X) && aligned16(T) && aligned16(H) && aligned16(RX) && aligned16(RW),
           "all tensors must be 16-byte aligned");
  c10::cuda::CUDAGuard guard(X.device());
  fo::cuda_check(fo::add_rmsnorm_launch(X.data_ptr(), T.data_ptr(), H.data_ptr(), RX.data_ptr(), RW.data_ptr(),
                                        static_cast<int>(X.size(0)), static_cast<int>(X.size(1)),
                                        static_cast<float>(eps), bf, sm_count_of_current_device(),
                                        c10::cuda::getCurrentCUDAStream().stream()),
                 "add_rmsnorm");
}

// What the ops that return new tensors read from: contiguous and 16-byte aligned, copied if it is not.
at::Tensor dense(const at::Tensor& t) {
  at::Tensor d = t.contiguous();
  return aligned16(d) ? d : d.clone();
}

void check_16bit(const at::Tensor& t, const char* name) {
  FO_CHECK(t.is_cuda() && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf), name,
           " must be a bfloat16 or float16 CUDA tensor");
}

bool given(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined(); }
at::Tensor or_undefined(const c10::optional<at::Tensor>& t) { return given(t) ? *t : at::Tensor(); }
c10::optional<at::Tensor> or_none(const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; }

// The operators with gradients.  They are functions of their own on torch's tape, in C++: a step through a pair of them
// from Python (two calls and one backward pass of few rows) is bound by the host, and the interpreter would be most of that.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A leaf's gradient is accumulated on the stream of the first live graph that it is part of.  A backward pass that is being
// captured would pull that stream into the capture, which ends the process inside the engine: refused here, in the forward pass.
void check_leaf_in_capture(const at::Tensor& t) {
  if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
  if (accumulator == nullptr) return;
  const auto stream = accumulator->stream();
  FO_CHECK(!stream.has_value() || *stream == c10::cuda::getCurrentCUDAStream(t.get_device()).unwrap(),
           "a tensor that requires a gradient is part of a live graph of another stream than the one being captured: ",
           "release that graph (its loss and outputs) before the capture");
}

// Forward-mode derivatives do not exist either, and would get lost without a word.
template <typename... T>
void check_no_tangent(const T&... t) {
  FO_CHECK(!((t.defined() && t._fw_grad(/*level=*/0).defined()) || ...), "this operator has no forward-mode derivative");
}

// Whether a call has a gradient to record.
template <typename... T>
bool records(const T&... t) {
  check_no_tangent(t...);
  if (!at::GradMode::is_enabled() || !((t.defined() && t.requires_grad()) || ...)) return false;
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) (check_leaf_in_capture(t), ...);
  return true;
}

template <typename... T>
void check_no_gradient(const char* what, const T&... t) {
  check_no_tangent(t...);
  FO_CHECK(!at::GradMode::is_enabled() || !((t.defined() && t.requires_grad()) || ...), what,
           " has no gradient: call it under no_grad, or detach its inputs");
}

// Gradients whose own derivatives do not exist: with a graph being recorded for them, differentiating it raises.
variable_list once(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative",
                                                               static_cast<int64_t>(grads.size()));
  for (at::Tensor& g : grads) {
    if (g.defined()) g = g.detach().requires_grad_();
  }
  return (*error)(std::move(grads));
}

// The operands of rmsnorm_add_rmsnorm and of its backward pass, checked.
struct NormBlockOperands {
  at::Tensor X, T, PW, W, G;
  fo::NormBlock p;
};
NormBlockOperands norm_block_operands(const at::Tensor& X, const at::Tensor& T, const at::Tensor& PW, const at::Tensor& W,
                                      const c10::optional<at::Tensor>& G, double alpha, double eps) {
  check_16bit(X, "X");
  FO_CHECK(X.dim() == 2 && T.sizes() == X.sizes(), "X and T must be [rows, dim]");
  const int64_t rows = X.size(0), dim = X.size(1);
  FO_CHECK(dim >= 8 && dim % 8 == 0 && dim <= 16384, "dim must be a multiple of 8 from 8 to 16384 (", dim, ")");
  FO_CHECK(rows <= fo::kMaxNormBlockRows, "too many rows");
  FO_CHECK(PW.dim() == 1 && PW.size(0) == dim && W.dim() == 1 && W.size(0) == dim, "PW and W must be [dim]");
  int64_t lines = 1;
  if (given(G)) {
    FO_CHECK((G->dim() == 1 || G->dim() == 2) && G->size(-1) == dim, "G must be [dim] or [lines, dim]");
    if (G->dim() == 2) lines = G->size(0);
    FO_CHECK(rows == 0 || (lines >= 1 && rows % lines == 0), "rows must be a multiple of G's lines (", rows, ", ", lines, ")");
    fo::check_device(*G, X, "G");
    FO_CHECK(G->scalar_type() == X.scalar_type(), "X, T, PW, W and G must share a dtype");
  }
  for (const at::Tensor& t : {T, PW, W}) {
    fo::check_device(t, X, "an operand");
    FO_CHECK(t.scalar_type() == X.scalar_type(), "X, T, PW, W and G must share a dtype");
  }
  NormBlockOperands o{dense(X), dense(T), dense(PW), dense(W), given(G) ? dense(*G) : at::Tensor(), {}};
  o.p.X = o.X.data_ptr();
  o.p.T = o.T.data_ptr();
  o.p.PW = o.PW.data_ptr();
  o.p.W = o.W.data_ptr();
  o.p.G = o.G.defined() ? o.G.data_ptr() : nullptr;
  o.p.rows = static_cast<int>(rows);
  o.p.dim = static_cast<int>(dim);
  o.p.lines = static_cast<int>(lines);
  o.p.alpha = static_cast<float>(alpha);
  o.p.eps = static_cast<float>(eps);
  o.p.bf16 = X.scalar_type() == at::kBFloat16;
  return o;
}

// (H, Y, stats): u = rmsnorm(T) * PW, H = alpha * X + G * u, Y = rmsnorm(H) * W; stats [rows, 2] fp32 (1 / rms of T and of H),
// what the backward pass needs, if asked for, else None.
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_block_forward(at::Tensor X, at::Tensor T, at::Tensor PW, at::Tensor W,
                                                                  c10::optional<at::Tensor> G, double alpha, double eps,
                                                                  bool with_stats) {
  check_16bit(X, "X");
  c10::cuda::CUDAGuard guard(X.device());
  const NormBlockOperands o = norm_block_operands(X, T, PW, W, G, alpha, eps);
  const at::ScalarType type = o.X.scalar_type();
  at::Tensor H = fo::fresh(X.sizes(), type, X), Y = fo::fresh(X.sizes(), type, X);
  at::Tensor stats;
  if (with_stats) stats = fo::fresh({X.size(0), 2}, at::kFloat, X);
  if (o.p.rows > 0) {
    fo::cuda_check(fo::norm_block_launch(o.p, H.data_ptr(), Y.data_ptr(), with_stats ? stats.data_ptr<float>() : nullptr,
                                         sm_count_of_current_device(), c10::cuda::getCurrentCUDAStream().stream()),
                   "rmsnorm_add_rmsnorm");
  }
  return {H, Y, stats};
}

// Gradients of X, T, PW, W and G (empty without G) from those of H and Y (either may be absent: zero).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> rmsnorm_add_rmsnorm_backward(
    c10::optional<at::Tensor> GH, c10::optional<at::Tensor> GY, at::Tensor X, at::Tensor T, at::Tensor PW, at::Tensor W,
    c10::optional<at::Tensor> G, at::Tensor stats, double alpha) {
  check_16bit(X, "X");
  c10::cuda::CUDAGuard guard(X.device());
  const NormBlockOperands o = norm_block_operands(X, T, PW, W, G, alpha, 0.);
  at::Tensor gh, gy;
  for (const auto& [from, to] : {std::pair{&GH, &gh}, std::pair{&GY, &gy}}) {
    if (!given(*from)) continue;
    const at::Tensor& g = **from;
    FO_CHECK(g.sizes() == X.sizes() && g.scalar_type() == X.scalar_type(), "GH and GY must be like X");
    fo::check_device(g, X, "a gradient");
    *to = dense(g);
  }
  FO_CHECK(stats.is_cuda() && stats.is_contiguous() && stats.scalar_type() == at::kFloat && stats.dim() == 2 &&
               stats.size(0) == X.size(0) && stats.size(1) == 2 && reinterpret_cast<uintptr_t>(stats.data_ptr()) % 8 == 0,
           "stats must be what the forward pass returned");
  fo::check_device(stats, X, "stats");
  const at::ScalarType type = o.X.scalar_type();
  at::Tensor DX = fo::fresh(X.sizes(), type, X), DT = fo::fresh(X.sizes(), type, X);
  const bool none = o.p.rows == 0;
  at::Tensor DPW = none ? at::zeros_like(o.PW) : fo::fresh(PW.sizes(), type, X), DW = none ? at::zeros_like(o.W) : fo::fresh(W.sizes(), type, X);
  at::Tensor DG = !o.G.defined() ? fo::fresh({0}, type, X) : (none ? at::zeros_like(o.G) : fo::fresh(o.G.sizes(), type, X));
  if (!none) {
    const fo::NormBlockPlan plan = fo::norm_block_plan(o.p, sm_count_of_current_device());
    at::Tensor workspace = fo::fresh({static_cast<int64_t>(plan.workspace)}, at::kFloat, X);
    fo::cuda_check(fo::norm_block_backward_launch(o.p, stats.data_ptr<float>(), gh.defined() ? gh.data_ptr() : nullptr,
                                                  gy.defined() ? gy.data_ptr() : nullptr, DX.data_ptr(), DT.data_ptr(),
                                                  DPW.data_ptr(), DW.data_ptr(), DG.data_ptr(), workspace.data_ptr<float>(),
                                                  plan, c10::cuda::getCurrentCUDAStream().stream()),
                   "rmsnorm_add_rmsnorm_backward");
  }
  return {DX, DT, DPW, DW, DG};
}

// As an operator of its own the backward pass has no derivative, and says so.  (On torch's tape `once` does.)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> rmsnorm_add_rmsnorm_backward_op(
    c10::optional<at::Tensor> GH, c10::optional<at::Tensor> GY, at::Tensor X, at::Tensor T, at::Tensor PW, at::Tensor W,
    c10::optional<at::Tensor> G, at::Tensor stats, double alpha) {
  check_no_gradient("rmsnorm_add_rmsnorm_backward", or_undefined(GH), or_undefined(GY), X, T, PW, W, or_undefined(G), stats);
  return rmsnorm_add_rmsnorm_backward(GH, GY, X, T, PW, W, G, stats, alpha);
}

struct NormBlockFunction : public torch::autograd::Function<NormBlockFunction> {
  static variable_list forward(AutogradContext* ctx, at::Tensor X, at::Tensor T, at::Tensor PW, at::Tensor W,
                               c10::optional<at::Tensor> G, double alpha, double eps) {
    auto [H, Y, stats] = norm_block_forward(X, T, PW, W, G, alpha, eps, true);
    ctx->save_for_backward({X, T, PW, W, or_undefined(G), stats});
    ctx->saved_data["alpha"] = alpha;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({stats});
    return {H, Y, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list v = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    auto [DX, DT, DPW, DW, DG] = rmsnorm_add_rmsnorm_backward(or_none(grads[0]), or_none(grads[1]), v[0], v[1], v[2], v[3],
                                                              or_none(v[4]), v[5], ctx->saved_data["alpha"].toDouble());
    const at::Tensor all[5] = {DX, DT, DPW, DW, DG};
    for (int i = 0; i < 5; ++i) {
      if (v[i].defined() && ctx->needs_input_grad(i)) out[i] = all[i];
    }
    return once("rmsnorm_add_rmsnorm", std::move(out));
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> rmsnorm_add_rmsnorm(at::Tensor X, at::Tensor T, at::Tensor PW, at::Tensor W,
                                                                    c10::optional<at::Tensor> G, double alpha, double eps,
                                                                    bool with_stats) {
  const at::Tensor g = or_undefined(G);
  if (!records(X, T, PW, W, g)) return norm_block_forward(X, T, PW, W, G, alpha, eps, with_stats);
  const variable_list out = NormBlockFunction::apply(X, T, PW, W, or_none(g), alpha, eps);
  return {out[0], out[1], out[2]};
}

// (slot [tokens, top_k], source [tokens * top_k], offsets [experts + 1]) of the experts `ids` [tokens, top_k] chosen for each token.
std::tuple<at::Tensor, at::Tensor, at::Tensor> moe_sort(at::Tensor ids, int64_t experts, int64_t most_ctas) {
  FO_CHECK(ids.is_cuda() && ids.dim() == 2 && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong),
           "ids must be an int32 or int64 CUDA tensor [tokens, top_k]");
  FO_CHECK(experts >= 1 && experts <= fo::kMaxExperts, "experts must be from 1 to ", fo::kMaxExperts, " (", experts, ")");
  FO_CHECK(ids.size(1) >= 1 && ids.size(1) <= fo::kMaxTopK, "top_k must be from 1 to ", fo::kMaxTopK, " (", ids.size(1), ")");
  FO_CHECK(ids.numel() <= INT32_MAX, "too many choices");
  FO_CHECK(most_ctas >= 1 && most_ctas <= 16, "most_ctas must be from 1 to 16 (", most_ctas, ")");
  c10::cuda::CUDAGuard guard(ids.device());
  const at::Tensor c = ids.contiguous();
  at::Tensor slot = fo::fresh(ids.sizes(), at::kInt, ids), source = fo::fresh({ids.numel()}, at::kInt, ids);
  at::Tensor offsets = fo::fresh({experts + 1}, at::kInt, ids);
  fo::cuda_check(fo::moe_sort_launch(c.data_ptr(), c.scalar_type() == at::kLong, c.numel(), static_cast<int>(experts),
                                     static_cast<int>(most_ctas), slot.data_ptr<int>(), source.data_ptr<int>(), offsets.data_ptr<int>(),
                                     c10::cuda::getCurrentCUDAStream().stream()),
                 "moe_sort");
  return {slot, source, offsets};
}

// Shape of a call over rows of `like`, with the order's tensors checked.
fo::MoeShape moe_shape(const at::Tensor& like, int64_t dim, const at::Tensor& slot, const at::Tensor* offsets) {
  FO_CHECK(slot.is_cuda() && slot.is_contiguous() && slot.scalar_type() == at::kInt && slot.dim() == 2,
           "slot must be a contiguous int32 CUDA tensor [tokens, top_k]");
  fo::check_device(slot, like, "slot");
  FO_CHECK(slot.size(1) >= 1 && slot.size(1) <= fo::kMaxTopK && slot.numel() <= INT32_MAX, "top_k must be from 1 to ", fo::kMaxTopK);
  FO_CHECK(dim >= 8 && dim % 8 == 0 && dim <= INT32_MAX, "dim must be a multiple of 8 (", dim, ")");
  fo::MoeShape s{static_cast<int>(slot.size(0)), static_cast<int>(slot.size(1)), static_cast<int>(dim), 1,
                 like.scalar_type() == at::kBFloat16};
  if (offsets != nullptr) {
    FO_CHECK(offsets->is_cuda() && offsets->is_contiguous() && offsets->scalar_type() == at::kInt && offsets->dim() == 1 &&
                 offsets->numel() >= 2 && offsets->numel() <= fo::kMaxExperts + 1,
             "offsets must be a contiguous int32 CUDA tensor [experts + 1]");
    fo::check_device(*offsets, like, "offsets");
    s.experts = static_cast<int>(offsets->numel()) - 1;
  }
  return s;
}

// What tells which rows no slot names: the order's sources if they are of its choices, else (or beyond them) a scratch.
struct MoeSourceTensors {
  at::Tensor source, scratch;
  fo::MoeSources arg() const {
    return {source.defined() ? source.data_ptr<int>() : nullptr, scratch.defined() ? scratch.data_ptr<int>() : nullptr};
  }
};
MoeSourceTensors moe_sources(const fo::MoeShape& s, const c10::optional<at::Tensor>& source, const at::Tensor& slot) {
  MoeSourceTensors t;
  if (given(source) && source->device() == slot.device() && source->scalar_type() == at::kInt && source->is_contiguous() &&
      source->numel() == slot.numel()) {
    t.source = *source;
  }
  const int64_t words = fo::moe_scratch_words(s, t.source.defined());
  if (words > 0) t.scratch = fo::fresh({words}, at::kInt, slot);
  return t;
}

// The router's weights, contiguous; none: undefined.
at::Tensor moe_weights(const c10::optional<at::Tensor>& weights, const at::Tensor& like, const at::Tensor& slot) {
  if (!given(weights)) return {};
  FO_CHECK(weights->sizes() == slot.sizes() && (weights->scalar_type() == at::kFloat || weights->scalar_type() == like.scalar_type()),
           "weights must be [tokens, top_k], float32 or of the rows' dtype");
  fo::check_device(*weights, like, "weights");
  return weights->contiguous();
}

fo::MoeWeights weights_arg(const at::Tensor& w) {
  return w.defined() ? fo::MoeWeights{w.data_ptr(), w.scalar_type() == at::kFloat} : fo::MoeWeights{nullptr, false};
}

// R [tokens * top_k, dim]: R[slot[t, k]] = X[t], every other row zero.
at::Tensor dispatch_rows(at::Tensor X, at::Tensor slot, at::Tensor offsets, const c10::optional<at::Tensor>& source) {
  check_16bit(X, "X");
  FO_CHECK(X.dim() == 2 && slot.dim() == 2 && X.size(0) == slot.size(0), "X must be [tokens, dim] and slot [tokens, top_k]");
  c10::cuda::CUDAGuard guard(X.device());
  const fo::MoeShape s = moe_shape(X, X.size(1), slot, &offsets);
  const at::Tensor x = dense(X);
  at::Tensor R = fo::fresh({slot.numel(), X.size(1)}, X.scalar_type(), X);
  if (s.tokens > 0) {
    const MoeSourceTensors from = moe_sources(s, source, slot);
    fo::cuda_check(fo::moe_dispatch_launch(s, x.data_ptr(), slot.data_ptr<int>(), offsets.data_ptr<int>(), from.arg(), R.data_ptr(),
                                           c10::cuda::getCurrentCUDAStream().stream()),
                   "moe_dispatch");
  }
  return R;
}

// O [tokens, dim]: the sum over k of weights[t, k] * R[slot[t, k]] (no weights: 1).
at::Tensor combine_rows(at::Tensor R, c10::optional<at::Tensor> weights, at::Tensor slot, const at::Tensor* offsets) {
  check_16bit(R, "R");
  FO_CHECK(R.dim() == 2 && R.size(0) == slot.numel(), "R must be [tokens * top_k, dim] and slot [tokens, top_k]");
  c10::cuda::CUDAGuard guard(R.device());
  const fo::MoeShape s = moe_shape(R, R.size(1), slot, offsets);
  const at::Tensor r = dense(R), w = moe_weights(weights, R, slot);
  at::Tensor O = fo::fresh({slot.size(0), R.size(1)}, R.scalar_type(), R);
  if (s.tokens > 0) {
    fo::cuda_check(fo::moe_combine_launch(s, r.data_ptr(), weights_arg(w), slot.data_ptr<int>(), O.data_ptr(),
                                          c10::cuda::getCurrentCUDAStream().stream()),
                   "moe_combine");
  }
  return O;
}

// (gradient of R, gradient of weights) from that of O; one that is not asked for comes back empty.
std::tuple<at::Tensor, at::Tensor> moe_combine_backward(at::Tensor GO, c10::optional<at::Tensor> R,
                                                        c10::optional<at::Tensor> weights, at::Tensor slot,
                                                        at::Tensor offsets, bool for_rows, bool for_weights,
                                                        c10::optional<at::Tensor> source) {
  check_16bit(GO, "GO");
  FO_CHECK(GO.dim() == 2 && slot.dim() == 2 && GO.size(0) == slot.size(0), "GO must be [tokens, dim] and slot [tokens, top_k]");
  FO_CHECK(for_rows || for_weights, "no gradient is asked for");
  c10::cuda::CUDAGuard guard(GO.device());
  const fo::MoeShape s = moe_shape(GO, GO.size(1), slot, &offsets);
  const at::Tensor go = dense(GO), w = moe_weights(weights, GO, slot);
  at::Tensor r, DR, DW;
  if (for_weights) {
    FO_CHECK(w.defined() && given(R), "the weights' gradient needs R and weights");
    FO_CHECK(R->dim() == 2 && R->size(0) == slot.numel() && R->size(1) == GO.size(1) && R->scalar_type() == GO.scalar_type(),
             "R must be [tokens * top_k, dim] of GO's dtype");
    fo::check_device(*R, GO, "R");
    r = dense(*R);
  }
  DR = fo::fresh({for_rows ? slot.numel() : 0, GO.size(1)}, GO.scalar_type(), GO);
  DW = for_weights ? fo::fresh(slot.sizes(), w.scalar_type(), GO) : fo::fresh({0}, GO.scalar_type(), GO);
  if (s.tokens > 0) {
    const MoeSourceTensors from = for_rows ? moe_sources(s, source, slot) : MoeSourceTensors{};
    fo::cuda_check(fo::moe_combine_backward_launch(s, go.data_ptr(), r.defined() ? r.data_ptr() : nullptr, weights_arg(w),
                                                   slot.data_ptr<int>(), offsets.data_ptr<int>(), from.arg(),
                                                   for_rows ? DR.data_ptr() : nullptr, for_weights ? DW.data_ptr() : nullptr,
                                                   c10::cuda::getCurrentCUDAStream().stream()),
                   "moe_combine_backward");
  }
  return {DR, DW};
}

std::tuple<at::Tensor, at::Tensor> moe_combine_backward_op(at::Tensor GO, c10::optional<at::Tensor> R,
                                                           c10::optional<at::Tensor> weights, at::Tensor slot,
                                                           at::Tensor offsets, bool for_rows, bool for_weights,
                                                           c10::optional<at::Tensor> source) {
  check_no_gradient("moe_combine_backward", GO, or_undefined(R), or_undefined(weights));
  return moe_combine_backward(GO, R, weights, slot, offsets, for_rows, for_weights, source);
}

struct DispatchFunction : public torch::autograd::Function<DispatchFunction> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor X, at::Tensor slot, at::Tensor offsets, c10::optional<at::Tensor> source) {
    ctx->save_for_backward({slot});
    return dispatch_rows(X, slot, offsets, source);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    return once("moe_dispatch", {combine_rows(grads[0], c10::nullopt, v[0], nullptr), at::Tensor(), at::Tensor(), at::Tensor()});
  }
};

at::Tensor moe_dispatch(at::Tensor X, at::Tensor slot, at::Tensor offsets, c10::optional<at::Tensor> source) {
  return records(X) ? DispatchFunction::apply(X, slot, offsets, source) : dispatch_rows(X, slot, offsets, source);
}

struct CombineFunction : public torch::autograd::Function<CombineFunction> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor R, c10::optional<at::Tensor> weights, at::Tensor slot,
                            at::Tensor offsets, c10::optional<at::Tensor> source) {
    const at::Tensor w = or_undefined(weights);
    // the rows are kept only for the weights' gradient
    ctx->save_for_backward({w.defined() && w.requires_grad() ? R : at::Tensor(), w, slot, offsets, or_undefined(source)});
    return combine_rows(R, weights, slot, &offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const bool rows = ctx->needs_input_grad(0), weights = v[0].defined() && ctx->needs_input_grad(1);
    variable_list out(5);
    if (!rows && !weights) return out;
    at::AutoDispatchBelowADInplaceOrView below;
    auto [DR, DW] = moe_combine_backward(grads[0], or_none(v[0]), or_none(v[1]), v[2], v[3], rows, weights, or_none(v[4]));
    if (rows) out[0] = DR;
    if (weights) out[1] = DW;
    return once("moe_combine", std::move(out));
  }
};

at::Tensor moe_combine(at::Tensor R, c10::optional<at::Tensor> weights, at::Tensor slot, at::Tensor offsets,
                       c10::optional<at::Tensor> source) {
  const at::Tensor w = or_undefined(weights);
  return records(R, w) ? CombineFunction::apply(R, or_none(w), slot, offsets, source) : combine_rows(R, weights, slot, &offsets);
}

// (Q int8, S fp32 [rows]) of X [rows, dim].
std::tuple<at::Tensor, at::Tensor> quantize_rows(at::Tensor X) {
  check_no_gradient("quantize_rows", X);
  check_16bit(X, "X");
  FO_CHECK(X.dim() == 2 && X.size(0) <= INT32_MAX, "X must be [rows, dim]");
  FO_CHECK(X.size(1) >= 8 && X.size(1) % 8 == 0 && X.size(1) <= fo::kMaxQuantizeDim, "dim must be a multiple of 8 from 8 to ",
           fo::kMaxQuantizeDim, " (", X.size(1), ")");
  c10::cuda::CUDAGuard guard(X.device());
  const at::Tensor x = dense(X);
  at::Tensor Q = fo::fresh(X.sizes(), at::kChar, X), S = fo::fresh({X.size(0)}, at::kFloat, X);
  fo::cuda_check(fo::quantize_rows_launch(x.data_ptr(), Q.data_ptr(), S.data_ptr<float>(), static_cast<int>(X.size(0)),
                                          static_cast<int>(X.size(1)), x.scalar_type() == at::kBFloat16,
                                          c10::cuda::getCurrentCUDAStream().stream()),
                 "quantize_rows");
  return {Q, S};
}

// Rotary embedding, in place, of the first `heads` heads of every row of QKV [tokens, row_elems].
void rope_(at::Tensor QKV, int64_t seq, int64_t heads, int64_t head_dim, double theta) {
  const bool bf = is_bf16(QKV, "QKV");
  FO_CHECK(QKV.dim() == 2 && heads >= 0 && head_dim > 0 && heads * head_dim <= QKV.size(1),
           "QKV must be [tokens, at least heads * head_dim]");
  FO_CHECK(seq > 0 && head_dim % 8 == 0 && QKV.size(1) % 8 == 0, "head_dim and the row length must be multiples of 8");
  FO_CHECK(aligned16(QKV), "QKV must be 16-byte aligned");
  c10::cuda::CUDAGuard guard(QKV.device());
  fo::cuda_check(fo::rope_launch(QKV.data_ptr(), static_cast<int>(QKV.size(0)), static_cast<int>(seq),
                                 static_cast<int>(heads), static_cast<int>(head_dim), static_cast<int>(QKV.size(1)),
                                 static_cast<float>(theta), bf, c10::cuda::getCurrentCUDAStream().stream()),
                 "rope");
}

// Y [rows, f] = silu(GU[:, :f]) * GU[:, f:].
void swiglu(at::Tensor GU, at::Tensor Y) {
  const bool bf = is_bf16(GU, "GU");
  is_bf16(Y, "Y");
  FO_CHECK(Y.scalar_type() == GU.scalar_type(), "GU and Y must share a dtype");
  FO_CHECK(GU.dim() == 2 && Y.dim() == 2 && Y.size(0) == GU.size(0) && GU.size(1) == 2 * Y.size(1),
           "GU must be [rows, 2 f] and Y [rows, f]");
  FO_CHECK(Y.size(1) % 8 == 0, "f must be a multiple of 8");
  FO_CHECK(aligned16(GU) && aligned16(Y), "GU and Y must be 16-byte aligned");
  fo::check_device(Y, GU, "Y");
  FO_CHECK(!fo::overlaps(Y, Y.numel(), GU, GU.numel()), "Y must not alias GU");
  c10::cuda::CUDAGuard guard(GU.device());
  fo::cuda_check(fo::swiglu_launch(GU.data_ptr(), Y.data_ptr(), static_cast<int>(GU.size(0)),
                                   static_cast<int>(Y.size(1)), bf, sm_count_of_current_device(),
                                   c10::cuda::getCurrentCUDAStream().stream()),
                 "swiglu");
}

void reorder_impl(at::Tensor X, at::Tensor Y, int64_t rows, int64_t dim, int64_t BM, int64_t BN,
                  int64_t rldn, at::Tensor RA, bool to_reordered) {
  is_bf16(X, "X");
  FO_CHECK(Y.scalar_type() == X.scalar_type() && Y.is_cuda() && Y.is_contiguous(),
              "Y must match X's dtype");
  FO_CHECK(X.numel() == rows * dim && Y.numel() == rows * dim, "X and Y must hold rows*dim elements");
  FO_CHECK(RA.is_cuda() && RA.scalar_type() == at::kInt && RA.is_contiguous() &&
                  RA.numel() >= (rows / BM) * (dim / BN),
              "RA must be an int32 CUDA tensor with one entry per tile");
  c10::cuda::CUDAGuard guard(X.device());
  fo::cuda_check(fo::reorder_launch(X.data_ptr(), Y.data_ptr(), static_cast<int>(rows),
                                    static_cast<int>(dim), static_cast<int>(BM), static_cast<int>(BN),
                                    static_cast<int>(rldn), RA.data_ptr<int>(), to_reordered,
                                    sm_count_of_current_device(),
                                    c10::cuda::getCurrentCUDAStream().stream()),
                 "reorder");
}

// Y (tile-contiguous) <- X (row-major [rows, dim]).
void reorder(at::Tensor X, at::Tensor Y, int64_t BM, int64_t BN, int64_t rldn, at::Tensor RA) {
  FO_CHECK(X.dim() == 2, "X must be [rows, dim]");
  reorder_impl(X, Y, X.size(0), X.size(1), BM, BN, rldn, RA, true);
}

// Y (row-major [rows, dim]) <- X (tile-contiguous).
void unreorder(at::Tensor X, at::Tensor Y, int64_t BM, int64_t BN, int64_t rldn, at::Tensor RA) {
  FO_CHECK(Y.dim() == 2, "Y must be [rows, dim]");
  reorder_impl(X, Y, Y.size(0), Y.size(1), BM, BN, rldn, RA, false);
}

// Bounded counting wait on MM[index] (see flags/fo_wait.h); status: int32[8] CUDA tensor.
void wait_flag(int64_t target, at::Tensor MM, int64_t index, int64_t timeout_ms, at::Tensor status) {
  FO_CHECK(MM.is_cuda() && MM.scalar_type() == at::kInt && MM.is_contiguous() &&
                  index >= 0 && index < MM.numel(),
              "MM must be an int32 CUDA tensor and index in range");
  FO_CHECK(status.is_cuda() && status.scalar_type() == at::kInt &&
                  status.numel() >= fo::kStatusWords,
              "status must be an int32 CUDA tensor with 8 words");
  c10::cuda::CUDAGuard guard(MM.device());
  fo::cuda_check(fo::wait_flag_launch(static_cast<int>(target), MM.data_ptr<int>() + index,
                                      static_cast<int>(index),
                                      static_cast<uint64_t>(timeout_ms) * 1000000ull,
                                      status.data_ptr<int>(),
                                      c10::cuda::getCurrentCUDAStream().stream()),
                 "wait_flag");
}

// Flattened Algo table: for each Algo index (BM, BN, BK, stages, raster strip width, CTA pair,
// row halves per CTA).
std::vector<int64_t> algo_table() {
  std::vector<int64_t> t;
  for (int a = 0; a < fo::kNumAlgos; ++a) {
    const fo::AlgoConfig c = fo::algo_config(a);
    t.insert(t.end(), {c.bm, c.bn, c.bk, c.stages, c.raster_sw, c.cta2, c.mt});
  }
  return t;
}

// Row tables of the fused all-to-all for one rank: row_end[8], dst_row[8], rows sent, rows
// received (see all2all_plan in runtime/fused_common.h).  Host only.
std::vector<int64_t> all2all_plan(at::Tensor mLen_CPU, int64_t rank) {
  FO_CHECK(!mLen_CPU.is_cuda() && mLen_CPU.scalar_type() == at::kInt && mLen_CPU.is_contiguous() &&
               mLen_CPU.dim() == 2 && mLen_CPU.size(0) == mLen_CPU.size(1) &&
               mLen_CPU.size(0) <= fo::kMaxRanks,
           "mLen_CPU must be a contiguous square int32 host tensor of at most 8 x 8");
  const int ws = static_cast<int>(mLen_CPU.size(0));
  FO_CHECK(rank >= 0 && rank < ws, "rank out of range");
  const fo::All2AllPlan plan = fo::all2all_plan(mLen_CPU.data_ptr<int>(), ws, static_cast<int>(rank));
  std::vector<int64_t> out;
  for (int d = 0; d < fo::kMaxRanks; ++d) out.push_back(plan.row_end[d]);
  for (int d = 0; d < fo::kMaxRanks; ++d) out.push_back(plan.dst_row[d]);
  out.push_back(plan.send_rows);
  out.push_back(plan.recv_rows);
  return out;
}

// The exception text check_status() produces for a block of status words (host only).
std::string status_message(std::vector<int64_t> words, int64_t rank) {
  FO_CHECK(static_cast<int>(words.size()) >= fo::kStatusWords, "a status block has ", fo::kStatusWords, " words");
  if (words[fo::kStatusWordCode] == fo::kStatusOk) return "";
  return fo::status_message(words.data(), static_cast<int>(rank));
}

}  // namespace

TORCH_LIBRARY(flashoverlap_class, m) {
  m.class_<BaselineImpl>("BaselineImpl")
      .def(torch::init())
      .def("nccl_init", &BaselineImpl::NcclInit)
      .def("cublas_init", &BaselineImpl::CublasInit)
      .def("gemm_allreduce", &BaselineImpl::GemmAllReduce)
      .def("gemm_reducescatter", &BaselineImpl::GemmReduceScatter)
      .def("gemm_all2all", &BaselineImpl::GemmAll2All)
      .def("cublas_gemm", &BaselineImpl::Gemm)
      .def("nccl_allreduce", &BaselineImpl::NcclAllReduce)
      .def("nccl_reducescatter", &BaselineImpl::NcclReduceScatter)
      .def("nccl_all2all", &BaselineImpl::NcclAll2All);
  m.class_<OverlapImpl>("OverlapImpl")
      .def(torch::init())
      .def("cutlass_init", &OverlapImpl::CutlassInit)
      .def("cutlass_gemm", &OverlapImpl::Gemm)
      .def("gemm_allreduce_overlap", &OverlapImpl::GemmAllReduceOverlap)
      .def("gemm_reducescatter_overlap", &OverlapImpl::GemmReduceScatterOverlap)
      .def("nccl_init", &OverlapImpl::NcclInit)
      .def("gemm_allreduce", &OverlapImpl::GemmAllReduce)
      .def("gemm_reducescatter", &OverlapImpl::GemmReduceScatter)
      .def("gemm_all2all", &OverlapImpl::GemmAll2All)
      .def("overlap_init", &OverlapImpl::OverlapInit)
      .def("nccl_allreduce", &OverlapImpl::NcclAllReduce)
      .def("nccl_reducescatter", &OverlapImpl::NcclReduceScatter)
      .def("nccl_all2all", &OverlapImpl::NcclAll2All)
      .def("seg_allreduce", &OverlapImpl::SegAllReduce)
      // additions
      .def("gemm_allreduce_fused", &OverlapImpl::GemmAllReduceFused)
      .def("gemm_reducescatter_fused", &OverlapImpl::GemmReduceScatterFused)
      .def("gemm_all2all_fused", &OverlapImpl::GemmAll2AllFused)
      .def("gemm_reducescatter_rmsnorm_fused", &OverlapImpl::GemmReduceScatterRmsNormFused)
      .def("gemm_reducescatter_add_rmsnorm_fused", &OverlapImpl::GemmReduceScatterAddRmsNormFused)
      .def("gemm_add", &OverlapImpl::GemmAdd)
      .def("gemm_swiglu", &OverlapImpl::GemmSwiGLU)
      .def("gemm_i8", &OverlapImpl::GemmI8)
      .def("linear_i8", &OverlapImpl::LinearI8)
      .def("set_option", &OverlapImpl::SetOption)
      .def("get_option", &OverlapImpl::GetOption)
      .def("symm_empty", &OverlapImpl::SymmEmpty)
      .def("register_symmetric", &OverlapImpl::RegisterSymmetric)
      .def("use_stage", &OverlapImpl::UseStage)
      .def("set_trace", &OverlapImpl::SetTrace)
      .def("read_status", &OverlapImpl::ReadStatus)
      .def("check_status", &OverlapImpl::CheckStatus)
      .def("reset_status", &OverlapImpl::ResetStatus)
      .def("resync", &OverlapImpl::Resync)
      .def("wait_flag", &OverlapImpl::WaitFlag);
}

TORCH_LIBRARY(flashoverlap_op, m) {
  m.def("generate_nccl_id", &generate_nccl_id);
  m.def("reorder_rmsnorm", &reorder_rmsnorm);
  // additions
  m.def("reorder_rmsnorm_eps", &reorder_rmsnorm_eps);
  m.def("rmsnorm", &rmsnorm);
  m.def("add_rmsnorm", &add_rmsnorm);
  m.def("rope_", &rope_);
  m.def("swiglu", &swiglu);
  m.def("rmsnorm_add_rmsnorm", &rmsnorm_add_rmsnorm);
  m.def("rmsnorm_add_rmsnorm_backward", &rmsnorm_add_rmsnorm_backward_op);
  m.def("moe_sort(Tensor ids, int experts, int most_ctas=16) -> (Tensor, Tensor, Tensor)", &moe_sort);
  m.def("moe_sort_ctas", [](int64_t choices, int64_t most) { return static_cast<int64_t>(fo::moe_sort_ctas(choices, static_cast<int>(most))); });
  // (source: of the sort; without it the call finds out by itself which rows no slot names, with a launch more)
  m.def("moe_dispatch(Tensor X, Tensor slot, Tensor offsets, Tensor? source=None) -> Tensor", &moe_dispatch);
  m.def("moe_combine(Tensor R, Tensor? weights, Tensor slot, Tensor offsets, Tensor? source=None) -> Tensor", &moe_combine);
  m.def("moe_combine_backward(Tensor GO, Tensor? R, Tensor? weights, Tensor slot, Tensor offsets, bool for_rows, bool for_weights, "
        "Tensor? source=None) -> (Tensor, Tensor)", &moe_combine_backward_op);
  m.def("quantize_rows", &quantize_rows);
  m.def("reorder", &reorder);
  m.def("unreorder", &unreorder);
  m.def("wait_flag", &wait_flag);
  m.def("algo_table", &algo_table);
  m.def("fused_loopback", &fo::fused_loopback);
  m.def("all2all_plan", &all2all_plan);
  m.def("status_message", &status_message);
}
