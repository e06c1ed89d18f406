// Bindings of the operators that work on torch tensors: checks of arguments, allocation, autograd, the call into the C API.
//
// Their kernels take a few microseconds for a few tokens, so what a call costs on the host counts: the same checks and
// allocations in Python took 17 us for one norm and 170 us for a training step of it (an autograd function in Python crosses
// the interpreter lock between two threads).  Every kernel is launched on the current stream of its tensors' device, and
// workspaces belong to one call.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <initializer_list>
#include <optional>
#include <tuple>
#include <vector>

#include "rbv/moe.h"
#include "rbv/norm.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor value(const Maybe& t) { return t ? *t : Tensor(); }
bool misaligned(const Tensor& t, uintptr_t to = 16) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % to != 0; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void launched(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " launch failed (CUDA error ", rc, ")"); }
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::empty(sizes, like.options().dtype(type)); }

// Rows of a matrix as the kernels read them: packed elements, starts at 16-byte boundaries.
Tensor packed_rows(const Tensor& x, int64_t step) {
  const bool many = x.size(0) > 1;
  if (x.stride(1) != 1 || misaligned(x) || (many && (x.stride(0) % step || x.stride(0) < x.size(1)))) return x.clone(at::MemoryFormat::Contiguous);
  return x;
}
int64_t row_step(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// Results over an operand that other CTAs still read would be a race.
void apart(const Tensor& out, std::initializer_list<const Tensor*> operands, const char* what) {
  auto span = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); i++) last += (t.size(i) - 1) * t.stride(i);
    const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
    return std::pair<uintptr_t, uintptr_t>(at, at + (last + 1) * t.element_size());
  };
  const auto [begin, end] = span(out);
  for (const Tensor* t : operands) {
    if (t->numel() == 0) continue;
    const auto [from, to] = span(*t);
    TORCH_CHECK_VALUE(to <= begin || end <= from, "out must not share memory with ", what);
  }
}

// A kernel's error flag, if the caller wants to know.
int* error_flag(const Maybe& error, const Tensor& like) {
  if (!error) return nullptr;
  TORCH_CHECK_VALUE(error->scalar_type() == at::kInt && error->numel() >= 1 && error->device() == like.device(),
                    "error must be an int32 tensor on the same GPU");
  return error->data_ptr<int>();
}

// Nothing here has a forward-mode derivative: a tangent is refused rather than dropped.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(!t._fw_grad(/*level=*/0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), what,
                    " has no forward-mode derivative");
}

// The operators without a backward pass refuse inputs that want one (rather than cut the graph without a word).
void no_gradient(const Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(!x.requires_grad() || !at::GradMode::is_enabled(), what, " has no backward pass: call it under torch.no_grad()");
  no_tangent(x, what);
}

// A result's tensor that the caller gave: not one that wants a gradient, and autograd learns that it was written.
void written(const Tensor& out, const char* what) {
  no_gradient(out, what);
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

// ---- norms around a block ----------------------------------------------------------------------------------------------
int norm_type(at::ScalarType t) {
  return t == at::kBFloat16 ? RBV_NORM_BF16 : t == at::kHalf ? RBV_NORM_FP16 : t == at::kFloat ? RBV_NORM_FP32 : -1;
}

// `t` as rows of H packed elements, and the distance between the rows.
std::pair<Tensor, int64_t> norm_rows(const Tensor& t, int64_t H) {
  if (t.is_contiguous()) return {t, H};
  Tensor m = t.dim() == 2 ? t : t.reshape({-1, H});
  if (m.stride(1) != 1 && H > 1) m = m.contiguous();
  return {m, m.size(0) > 1 ? m.stride(0) : H};
}

struct NormCall {
  rbv_norm_t c{};
  std::vector<Tensor> held;               // what the pointers point into
  NormCall(const Tensor& residual, const Tensor& branch, const Tensor& post_weight, const Tensor& gate, int64_t kind, double scale,
           const Tensor& pre_weight, double eps) {
    const int64_t H = residual.size(-1);
    auto keep = [&](const Tensor& t) { held.push_back(t); return t.data_ptr(); };
    auto rows = [&](const Tensor& t, long long* ld) {
      auto [m, step] = norm_rows(t, H);
      *ld = step;
      return keep(m);
    };
    c.T = residual.numel() / H;
    c.H = (int)H;
    c.z_type = norm_type(branch.defined() ? branch.scalar_type() : residual.scalar_type());
    c.r_type = norm_type(residual.scalar_type());
    c.gate_kind = (int)kind;
    c.scale = (float)scale;
    c.eps = (float)eps;
    c.r = rows(residual, &c.r_ld);
    if (branch.defined()) {
      c.z = rows(branch, &c.z_ld);
      c.w1 = keep(post_weight.contiguous());
      c.w1_f32 = post_weight.scalar_type() == at::kFloat;
    }
    if (gate.defined()) {
      c.gate = kind == RBV_GATE_FULL ? rows(gate, &c.gate_ld) : keep(gate.contiguous());
      c.gate_f32 = gate.scalar_type() == at::kFloat;
    }
    if (pre_weight.defined()) {
      c.w2 = keep(pre_weight.contiguous());
      c.w2_f32 = pre_weight.scalar_type() == at::kFloat;
    }
  }
};

// r2, u and the rows' reciprocal norms (each undefined if there is none, or none is wanted).
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& residual, const Tensor& branch, const Tensor& post_weight, const Tensor& gate,
                                                int64_t kind, double scale, const Tensor& pre_weight, double eps, bool stats) {
  const c10::cuda::CUDAGuard guard(residual.device());
  NormCall call(residual, branch, post_weight, gate, kind, scale, pre_weight, eps);
  Tensor r2, u, rstd;
  if (branch.defined()) r2 = empty(residual.sizes(), residual.scalar_type(), residual);
  if (pre_weight.defined()) u = empty(residual.sizes(), (branch.defined() ? branch : residual).scalar_type(), residual);
  if (stats) {
    rstd = empty({2 * call.c.T}, at::kFloat, residual);
    call.c.rstd1 = rstd.data_ptr<float>();
    call.c.rstd2 = call.c.rstd1 + call.c.T;
  }
  call.c.r2 = ptr(r2);
  call.c.u = ptr(u);
  if (call.c.T) launched(rbv_block_norm(&call.c, stream_of(residual)), "block norm");
  return {r2, u, rstd};
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& residual, const Maybe& branch,
                                                const Maybe& post_weight, const Maybe& gate, const Maybe& pre_weight, int64_t kind,
                                                double scale, double eps) {
    const Tensor z = value(branch), w1 = value(post_weight), g = value(gate), w2 = value(pre_weight);
    auto [r2, u, rstd] = norm_forward(residual, z, w1, g, kind, scale, w2, eps, true);
    ctx->save_for_backward({residual, z, w1, g, w2, rstd});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    torch::autograd::variable_list out;    // what there is, in this order
    if (r2.defined()) out.push_back(r2);
    if (u.defined()) out.push_back(u);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &residual = saved[0], &branch = saved[1], &post_weight = saved[2], &gate = saved[3], &pre_weight = saved[4], &rstd = saved[5];
    const int64_t kind = ctx->saved_data["kind"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble(), eps = ctx->saved_data["eps"].toDouble();
    size_t next = 0;
    const Tensor d_r2 = branch.defined() ? grads[next++] : Tensor(), d_u = pre_weight.defined() ? grads[next++] : Tensor();
    torch::autograd::variable_list out(8);
    if (!d_r2.defined() && !d_u.defined()) return out;
    {
      at::AutoGradMode no_graph(false);
      const c10::cuda::CUDAGuard guard(residual.device());
      NormCall call(residual, branch, post_weight, gate, kind, scale, pre_weight, eps);
      rbv_norm_t& c = call.c;
      size_t edge = 0;                     // only tensors that were given have one, in the order of the arguments
      auto grad = [&](const Tensor& t, bool there) {
        if (!t.defined() || !ctx->needs_input_grad(edge++) || !there) return Tensor();
        return c.T ? empty(t.sizes(), t.scalar_type(), t) : at::zeros(t.sizes(), t.options());
      };
      out[0] = grad(residual, true);
      out[1] = grad(branch, true);
      out[2] = grad(post_weight, true);
      out[3] = grad(gate, true);
      out[4] = grad(pre_weight, d_u.defined());
      if (c.T) {
        auto rows = [&](const Tensor& t, long long* ld) -> const void* {
          if (!t.defined()) return nullptr;
          auto [m, step] = norm_rows(t, c.H);
          *ld = step;
          call.held.push_back(m);
          return m.data_ptr();
        };
        c.dr2 = rows(d_r2, &c.dr2_ld);
        c.du = rows(d_u, &c.du_ld);
        c.rstd1 = rstd.data_ptr<float>();
        c.rstd2 = c.rstd1 + c.T;
        c.dr = ptr(out[0]);
        c.dz = ptr(out[1]);
        c.dw1 = ptr(out[2]);
        c.dgate = ptr(out[3]);
        c.dw2 = ptr(out[4]);
        Tensor partial;
        if (c.dw1 || c.dw2 || (c.dgate && kind == RBV_GATE_CHANNEL)) {
          partial = empty({rbv_block_norm_parts(c.T, c.H, c.z_type), 2, c.H}, at::kFloat, residual);
          c.partial = partial.data_ptr<float>();
        }
        launched(rbv_block_norm_backward(&c, stream_of(residual)), "block norm backward");
      }
    }
    if (at::GradMode::is_enabled()) {      // a graph of the backward pass is asked for: there is none through these
      for (Tensor& t : out)
        if (t.defined()) t.requires_grad_(true);
      out = torch::autograd::DelayedError("block_norm is differentiable once", (int64_t)out.size()).apply(std::move(out));
    }
    return out;
  }
};

std::tuple<Tensor, Maybe> block_norm(const Tensor& residual, const Maybe& branch, const Maybe& post_weight, const Maybe& gate, double scale,
                                     const Maybe& pre_weight, double eps) {
  TORCH_CHECK_VALUE(residual.dim() >= 1, "the residual must be a tensor [..., hidden]");
  TORCH_CHECK_VALUE(norm_type(residual.scalar_type()) >= 0, "the residual must be bf16, fp16 or fp32, not ", residual.scalar_type());
  const int64_t H = residual.size(-1);
  TORCH_CHECK_VALUE(H >= 1 && H <= RBV_NORM_MAX_HIDDEN, "hidden sizes of 1 to ", RBV_NORM_MAX_HIDDEN, " are supported, not ", H);
  TORCH_CHECK_VALUE(branch || pre_weight, "neither a block output nor the weight of a norm in front of the next block: nothing to do");
  TORCH_CHECK_VALUE(branch || (!post_weight && !gate), "post_weight and gate belong to a block output");
  TORCH_CHECK_VALUE(!branch || post_weight, "a block output needs its norm's weight (post_weight)");
  const at::ScalarType kind = branch ? branch->scalar_type() : residual.scalar_type();
  auto fits = [&](const Tensor& t) { return t.scalar_type() == kind || t.scalar_type() == at::kFloat; };
  if (branch) {
    TORCH_CHECK_VALUE(branch->sizes() == residual.sizes(), "block output ", branch->sizes(), " and residual ", residual.sizes(), " differ in shape");
    TORCH_CHECK_VALUE(norm_type(kind) >= 0 && fits(residual), "the residual must have the block output's type (", kind, ") or fp32, not ",
                      residual.scalar_type());
  }
  auto weight = [&](const Maybe& w, const char* name) {
    TORCH_CHECK_VALUE(!w || (w->dim() == 1 && w->size(0) == H && fits(*w)), name, " must be [", H, "] in ", kind, " or fp32, not ", w->sizes(), " in ",
                      w->scalar_type());
  };
  weight(post_weight, "post_weight");
  weight(pre_weight, "pre_weight");
  for (const Maybe* t : {&branch, &post_weight, &gate, &pre_weight})
    TORCH_CHECK_VALUE(!*t || (*t)->device() == residual.device(), "all tensors must be on one device");
  int64_t gate_kind = RBV_GATE_NONE;
  Maybe g = gate;
  if (gate) {
    TORCH_CHECK_VALUE(fits(*gate), "the gate must be ", kind, " or fp32, not ", gate->scalar_type());
    const int64_t n = gate->dim(), m = residual.dim();
    bool broadcasts = n <= m;
    for (int64_t i = 1; i <= n && broadcasts; i++) broadcasts = gate->size(n - i) == 1 || gate->size(n - i) == residual.size(m - i);
    TORCH_CHECK_VALUE(broadcasts, "a gate ", gate->sizes(), " does not broadcast to ", residual.sizes());
    if (n == 1 && gate->size(0) == H) {
      gate_kind = RBV_GATE_CHANNEL;
    } else if (n == m && gate->size(-1) == 1 && gate->sizes().slice(0, n - 1) == residual.sizes().slice(0, m - 1)) {
      gate_kind = RBV_GATE_TOKEN;
    } else {
      gate_kind = RBV_GATE_FULL;
      // The gradient of an expanded gate is written element by element and then summed: in 32 bits, so that it is rounded once.
      if (gate->sizes() != residual.sizes())
        g = (gate->requires_grad() && at::GradMode::is_enabled() ? gate->to(at::kFloat) : *gate).expand(residual.sizes());
    }
  }
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative");
  no_tangent(residual, "block_norm");
  for (const Maybe* t : {&branch, &post_weight, &gate, &pre_weight})
    if (*t) no_tangent(**t, "block_norm");
  TORCH_CHECK_VALUE(residual.is_cuda(), "block_norm runs on a GPU: the tensors are on the host");
  bool graph = residual.requires_grad();
  for (const Maybe* t : {&branch, &post_weight, &gate, &pre_weight}) graph = graph || (*t && (*t)->requires_grad());
  Tensor r2, u;
  if (graph && at::GradMode::is_enabled()) {
    const auto out = BlockNorm::apply(residual, branch, post_weight, g, pre_weight, gate_kind, scale, eps);
    size_t next = 0;
    if (branch) r2 = out[next++];
    if (pre_weight) u = out[next++];
  } else {
    std::tie(r2, u, std::ignore) = norm_forward(residual, value(branch), value(post_weight), value(g), gate_kind, scale, value(pre_weight), eps, false);
  }
  return {branch ? r2 : residual, u.defined() ? Maybe(u) : Maybe()};
}

// ---- 8-bit integers ------------------------------------------------------------------------------------------------------
Tensor int8_rows(const Tensor& x) {
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && x.dim() == 2, "rows must be a bf16 matrix, not ", x.sizes(), " in ", x.scalar_type());
  no_gradient(x, "quantising rows to int8");
  const int64_t K = x.size(1);
  TORCH_CHECK_VALUE(K >= 16 && K % 16 == 0 && K <= RBV_INT8_MAX_DEPTH, "depths of 16 to ", RBV_INT8_MAX_DEPTH, " in steps of 16 are supported, not ", K);
  TORCH_CHECK_VALUE(x.is_cuda(), "the rows must be on a GPU");
  return packed_rows(x, 8);
}

void int8_weight(const Tensor& w, const Tensor& scale, int64_t dim) {
  TORCH_CHECK_VALUE(w.dim() == dim && w.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat &&
                        scale.sizes() == w.sizes().slice(0, dim - 1),
                    "weights must be int8 with ", dim, " dimensions and one fp32 scale per channel, not ", w.sizes(), " in ", w.scalar_type(),
                    " with scales ", scale.sizes(), " in ", scale.scalar_type());
  const int64_t N = w.size(-2), K = w.size(-1);
  TORCH_CHECK_VALUE(N >= 8 && N % 8 == 0 && K >= 16 && K % 16 == 0 && K <= RBV_INT8_MAX_DEPTH, "channels in steps of 8 and depths of 16 to ",
                    RBV_INT8_MAX_DEPTH, " in steps of 16 are supported, not ", N, " x ", K);
  TORCH_CHECK_VALUE(w.numel() / K <= RBV_INT8_MAX_CHANNELS, "at most ", RBV_INT8_MAX_CHANNELS, " channels in all groups, not ", w.numel() / K);
  TORCH_CHECK_VALUE(w.is_contiguous() && scale.is_contiguous() && !misaligned(w) && !misaligned(scale),
                    "weights and scales must be contiguous and 16-byte aligned");
  no_gradient(scale, "an int8 product");
}

std::tuple<Tensor, Tensor> quantize_rows_int8(const Tensor& rows, const Maybe& used) {
  const Tensor x = int8_rows(rows);
  TORCH_CHECK_VALUE(!used || (used->scalar_type() == at::kInt && used->numel() >= 1 && used->device() == x.device()),
                    "used must be an int32 tensor on the rows' GPU");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor q = empty(x.sizes(), at::kChar, x), scale = empty({x.size(0)}, at::kFloat, x);
  if (x.size(0))
    launched(rbv_quantize_rows_int8(x.data_ptr(), x.size(0), used ? used->data_ptr<int>() : nullptr, (int)x.size(1), row_step(x), q.data_ptr(),
                                    scale.data_ptr<float>(), stream_of(x)),
             "int8 quantisation");
  return {q, scale};
}

Tensor grouped_gemm_int8(const Tensor& Aq, const Tensor& a_scale, const Tensor& Bq, const Tensor& b_scale, const Tensor& group_start,
                         const Tensor& group_rows, const Maybe& out_, bool swiglu, const Maybe& error, int64_t max_ctas) {
  int8_weight(Bq, b_scale, 3);
  const int64_t G = Bq.size(0), N = Bq.size(1), K = Bq.size(2);
  TORCH_CHECK_VALUE(Aq.dim() == 2 && Aq.scalar_type() == at::kChar && Aq.size(1) == K && a_scale.dim() == 1 && a_scale.size(0) == Aq.size(0) &&
                        a_scale.scalar_type() == at::kFloat,
                    "rows must be int8 [M, ", K, "] with fp32 scales [M], not ", Aq.sizes(), " in ", Aq.scalar_type(), " with ", a_scale.sizes());
  TORCH_CHECK_VALUE(Aq.is_contiguous() && a_scale.is_contiguous() && !misaligned(Aq), "rows and scales must be contiguous and 16-byte aligned");
  no_gradient(a_scale, "grouped_gemm_int8");
  TORCH_CHECK_VALUE(G >= 1 && G <= 64, "at most 64 groups, not ", G);
  for (const Tensor* t : {&group_start, &group_rows})
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == G && t->scalar_type() == at::kInt && t->is_contiguous(),
                      "group_start and group_rows must be int32 [", G, "]");
  const int64_t M = Aq.size(0), n_out = swiglu ? N / 2 : N;
  TORCH_CHECK_VALUE(M <= RBV_INT8_MAX_ROWS, "at most ", RBV_INT8_MAX_ROWS, " rows, not ", M);
  TORCH_CHECK_VALUE(Aq.is_cuda(), "all tensors must be on one GPU");
  for (const Tensor* t : {&a_scale, &Bq, &b_scale, &group_start, &group_rows})
    TORCH_CHECK_VALUE(t->device() == Aq.device(), "all tensors must be on one GPU");
  const c10::cuda::CUDAGuard guard(Aq.device());
  Tensor out = value(out_);
  if (!out.defined()) out = empty({M, n_out}, at::kBFloat16, Aq);
  else
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == M && out.size(1) == n_out && out.scalar_type() == at::kBFloat16 &&
                          out.device() == Aq.device() && out.stride(1) == 1 && !misaligned(out, 4) &&
                          (M <= 1 || (out.stride(0) % 2 == 0 && out.stride(0) >= n_out && out.stride(0) <= 0x7fffffff)),
                      "out must be a bf16 tensor [", M, ", ", n_out, "] with packed, 4-byte aligned rows on the same GPU");
  if (out_ && M) {
    apart(out, {&Aq, &a_scale, &Bq, &b_scale, &group_start, &group_rows}, "an operand");
    written(out, "grouped_gemm_int8");
  }
  if (M)
    launched(rbv_grouped_gemm_int8(Aq.data_ptr(), a_scale.data_ptr<float>(), M, Bq.data_ptr(), b_scale.data_ptr<float>(), out.data_ptr(),
                                   group_start.data_ptr<int>(), group_rows.data_ptr<int>(), (int)G, (int)N, (int)K, (int)row_step(out), swiglu ? 1 : 0,
                                   error_flag(error, Aq), (int)max_ctas, stream_of(Aq)),
             "int8 grouped GEMM");
  return out;
}

Tensor linear_int8(const Tensor& rows, const Tensor& weight, const Tensor& scale, const Maybe& out_, const Maybe& error) {
  int8_weight(weight, scale, 2);
  const Tensor x = int8_rows(rows);
  const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
  TORCH_CHECK_VALUE(weight.size(1) == K, "rows of ", K, " do not fit weights ", weight.sizes());
  TORCH_CHECK_VALUE(weight.device() == x.device() && scale.device() == x.device(), "all tensors must be on one GPU");
  TORCH_CHECK_VALUE(M <= RBV_INT8_MAX_ROWS, "at most ", RBV_INT8_MAX_ROWS, " rows, not ", M);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor out = value(out_);
  if (!out.defined()) out = empty({M, N}, at::kBFloat16, x);
  else
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == M && out.size(1) == N && out.scalar_type() == at::kBFloat16 && out.device() == x.device() &&
                          out.is_contiguous() && !misaligned(out),
                      "out must be a contiguous, 16-byte aligned bf16 tensor [", M, ", ", N, "] on the same GPU");
  if (M == 0) return out;
  if (out_) {
    apart(out, {&weight, &scale}, "the weights or their scales");
    written(out, "linear_int8");
  }
  int* err = error_flag(error, x);
  if (M <= RBV_FEW_ROWS) {
    const long long bytes = rbv_linear_int8_few_workspace((int)M, (int)N, (int)K);
    TORCH_CHECK_VALUE(bytes >= 0, "weights of ", N, " x ", K, " are too large for a few rows");
    Tensor ws = empty({bytes}, at::kByte, x);
    launched(rbv_linear_int8_few(x.data_ptr(), row_step(x), (int)M, weight.data_ptr(), scale.data_ptr<float>(), (int)N, (int)K, out.data_ptr(),
                                 ws.data_ptr(), err, stream_of(x)),
             "int8 linear");
  } else {
    Tensor q = empty({M, K}, at::kChar, x), s = empty({M}, at::kFloat, x);
    launched(rbv_quantize_rows_int8(x.data_ptr(), M, nullptr, (int)K, row_step(x), q.data_ptr(), s.data_ptr<float>(), stream_of(x)),
             "int8 quantisation");
    launched(rbv_grouped_gemm_int8(q.data_ptr(), s.data_ptr<float>(), M, weight.data_ptr(), scale.data_ptr<float>(), out.data_ptr(), nullptr, nullptr, 1,
                                   (int)N, (int)K, (int)N, 0, err, 0, stream_of(x)),
             "int8 linear");
  }
  return out;
}

// ---- a routed layer for a few tokens -------------------------------------------------------------------------------------
Tensor moe_few_tokens(const Tensor& x_, const Tensor& logits_, const Tensor& w13, const Tensor& w2, int64_t top_k, const Maybe& out_,
                      const Maybe& error) {
  TORCH_CHECK_VALUE(x_.dim() == 2 && logits_.dim() == 2 && w13.dim() == 3 && w2.dim() == 3,
                    "x [T, H], logits [T, E], w13 [E, 2 I, H] and w2 [E, H, I] are wanted");
  for (const Tensor* t : {&x_, &logits_, &w13, &w2}) no_gradient(*t, "moe_few_tokens");
  const int64_t T = x_.size(0), H = x_.size(1), E = w2.size(0), I = w2.size(2);
  TORCH_CHECK_VALUE(x_.scalar_type() == at::kBFloat16 && w13.scalar_type() == at::kBFloat16 && w2.scalar_type() == at::kBFloat16 &&
                        logits_.scalar_type() == at::kFloat,
                    "x and the weights must be bf16, the logits fp32");
  TORCH_CHECK_VALUE(logits_.size(0) == T && logits_.size(1) == E && w13.size(0) == E && w13.size(1) == 2 * I && w13.size(2) == H && w2.size(1) == H,
                    "shapes do not fit: x ", x_.sizes(), ", logits ", logits_.sizes(), ", w13 ", w13.sizes(), ", w2 ", w2.sizes());
  TORCH_CHECK_VALUE(T <= RBV_FEW_ROWS, T, " tokens: moe_few_tokens takes at most ", RBV_FEW_ROWS, "; MoEExpertParallel.forward is for more");
  TORCH_CHECK_VALUE(H >= 8 && I >= 8 && H % 8 == 0 && I % 8 == 0 && E >= 1 && E <= 256 && top_k >= 1 && top_k <= RBV_FEW_MAX_TOP_K && top_k <= E,
                    "hidden ", H, " and FFN width ", I, " must be multiples of 8, experts ", E, " at most 256, top_k ", top_k, " at most ",
                    RBV_FEW_MAX_TOP_K, " and the experts");
  TORCH_CHECK_VALUE(w13.is_contiguous() && w2.is_contiguous() && !misaligned(w13) && !misaligned(w2),
                    "the weights must be contiguous and 16-byte aligned");
  TORCH_CHECK_VALUE(x_.is_cuda() && logits_.device() == x_.device() && w13.device() == x_.device() && w2.device() == x_.device(),
                    "all tensors must be on one GPU");
  const c10::cuda::CUDAGuard guard(x_.device());
  Tensor out = value(out_);
  if (!out.defined()) out = empty({T, H}, at::kBFloat16, x_);
  else
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == T && out.size(1) == H && out.scalar_type() == at::kBFloat16 && out.device() == x_.device() &&
                          out.is_contiguous() && !misaligned(out),
                      "out must be a contiguous, 16-byte aligned bf16 tensor [T, H] on the same GPU");
  if (T == 0) return out;
  if (out_) {
    apart(out, {&logits_, &w13, &w2}, "the logits or the weights");              // (the tokens are read before)
    written(out, "moe_few_tokens");
  }
  const Tensor x = packed_rows(x_, 8);
  Tensor logits = logits_;
  if ((E > 1 && logits.stride(1) != 1) || (T > 1 && logits.stride(0) < E)) logits = logits.contiguous();
  const long long bytes = rbv_moe_few_workspace((int)T, (int)H, (int)I, (int)E, (int)top_k);
  TORCH_CHECK_VALUE(bytes >= 0, "a layer of ", E, " experts, hidden ", H, " and FFN width ", I, " is too large");
  Tensor ws = empty({bytes}, at::kByte, x);
  launched(rbv_moe_few_tokens(x.data_ptr(), row_step(x), logits.data_ptr<float>(), row_step(logits), (int)T, (int)H, (int)I, (int)E, (int)top_k,
                              w13.data_ptr(), w2.data_ptr(), out.data_ptr(), ws.data_ptr(), error_flag(error, x), stream_of(x)),
           "few-token MoE");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("block_norm", &block_norm);
  m.def("quantize_rows_int8", &quantize_rows_int8);
  m.def("grouped_gemm_int8", &grouped_gemm_int8);
  m.def("linear_int8", &linear_int8);
  m.def("moe_few_tokens", &moe_few_tokens);
}
