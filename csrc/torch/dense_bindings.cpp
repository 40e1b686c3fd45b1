// Bindings of the dense side of a block: row norm, balance loss, linear layers. Their kernels run on the current stream of the
// tensors' own device, whichever device is current.
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "py_types.h"

namespace py = pybind11;
using namespace fastb;
using namespace fastb_py;

namespace {

using OptTensor = c10::optional<torch::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const torch::Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
template <class... T> bool recorded(const T&... t) { return c10::GradMode::is_enabled() && (wants_grad(t) || ...); }

// Gradients that came from kernels have no graph behind them: one that is asked for a gradient of its own says so.
variable_list once(const char* op, const variable_list& incoming, variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  bool any = false;
  for (const auto& t : incoming) any = any || (t.defined() && t.requires_grad());
  if (!any) return grads;
  variable_list defined;
  for (auto& g : grads)
    if (g.defined()) { g = g.detach(); g.set_requires_grad(true); defined.push_back(g); }
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(op) + ": its backward pass has no gradient", static_cast<int>(defined.size()));
  defined = (*err)(std::move(defined));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = defined[k++];
  return grads;
}

bool row_type(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32; }

// Rows of t as a matrix whose rows are contiguous; only what cannot be seen as one is copied.
torch::Tensor as_rows(const torch::Tensor& t, int64_t cols) {
  torch::Tensor m = t.dim() == 2 ? t : t.reshape({-1, cols});
  return m.stride(1) == 1 || cols == 1 ? m : m.contiguous();
}
int rows_of(const torch::Tensor& m, const char* what) {
  TORCH_CHECK(m.size(0) <= 0x7fffffff, what, ": more than 2^31 - 1 rows");
  return static_cast<int>(m.size(0));
}
int sm_count(const torch::Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }

struct Norm { torch::Tensor y, h, q, scales, rstd; };   // h undefined without residual, q and scales without quantise, rstd without keep
Norm row_norm(const torch::Tensor& x, const torch::Tensor& weight, double eps, const OptTensor& residual, bool quantise, bool keep) {
  TORCH_CHECK(x.is_cuda() && row_type(x) && x.dim() >= 1, "add_rms_norm: x must be a bf16 or fp32 CUDA tensor [..., hidden]");
  const int64_t H = x.size(-1);
  TORCH_CHECK(H >= 1 && H <= kRowNormMaxHidden, "add_rms_norm: hidden size must be 1 to ", kRowNormMaxHidden, ", got ", H);
  TORCH_CHECK(weight.device() == x.device() && weight.dim() == 1 && weight.size(0) == H && weight.is_contiguous() && row_type(weight), "add_rms_norm: weight must be contiguous bf16 or fp32 [hidden] on x's device");
  TORCH_CHECK(!residual.has_value() || (residual->device() == x.device() && residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes()),
              "add_rms_norm: residual must have x's shape, type and device");
  TORCH_CHECK(!quantise || H % 128 == 0, "add_rms_norm: e4m3 rows have a scale per 128 columns, hidden must be a multiple of 128, got ", H);
  TORCH_CHECK(eps >= 0, "add_rms_norm: eps must not be negative");
  c10::cuda::CUDAGuard guard(x.device());
  const torch::Tensor xm = as_rows(x, H);
  RowNormArgs a{};
  a.x = xm.data_ptr(); a.x_stride = xm.stride(0);
  a.T = rows_of(xm, "add_rms_norm"); a.H = static_cast<int>(H);
  a.weight = weight.data_ptr();
  a.rows_bf16 = x.scalar_type() == torch::kBFloat16; a.weight_bf16 = weight.scalar_type() == torch::kBFloat16;
  a.eps = static_cast<float>(eps);
  torch::Tensor y = torch::empty(x.sizes(), x.options()), rm;
  torch::Tensor h, q, scales, rstd;
  a.y = y.data_ptr();
  if (residual.has_value()) {
    rm = as_rows(*residual, H);
    a.residual = rm.data_ptr(); a.residual_stride = rm.stride(0);
    h = torch::empty(x.sizes(), x.options());
    a.h = h.data_ptr();
  }
  if (quantise) {
    q = torch::empty(x.sizes(), x.options().dtype(torch::kUInt8));
    auto shape = x.sizes().vec();
    shape.back() = H / 128;
    scales = torch::empty(shape, x.options().dtype(torch::kFloat32));
    a.q = q.data_ptr<uint8_t>(); a.scales = scales.data_ptr<float>();
  }
  if (keep) {
    rstd = torch::empty({xm.size(0)}, x.options().dtype(torch::kFloat32));
    a.rstd = rstd.data_ptr<float>();
  }
  cuda_check(launch_row_norm(a, cur_stream()), "add_rms_norm");
  return {y, h, q, scales, rstd};
}

// (dx, dweight) from what the forward pass normalised, its rstd, dy and optionally dh.
std::tuple<torch::Tensor, torch::Tensor> row_norm_bwd(const torch::Tensor& h, const torch::Tensor& weight, const torch::Tensor& rstd, const torch::Tensor& dy, const OptTensor& dh) {
  TORCH_CHECK(h.is_cuda() && row_type(h) && row_type(weight) && dy.sizes() == h.sizes() && dy.scalar_type() == h.scalar_type() && dy.device() == h.device(), "add_rms_norm backward: gradient of y");
  TORCH_CHECK(!dh.has_value() || (dh->sizes() == h.sizes() && dh->scalar_type() == h.scalar_type() && dh->device() == h.device()), "add_rms_norm backward: gradient of the sum");
  const int64_t H = h.size(-1);
  c10::cuda::CUDAGuard guard(h.device());
  const torch::Tensor hm = as_rows(h, H), ym = dy.contiguous(), dm = dh.has_value() ? dh->contiguous() : torch::Tensor();
  RowNormBwdArgs a{};
  a.h = hm.data_ptr(); a.h_stride = hm.stride(0);
  a.weight = weight.data_ptr(); a.rstd = rstd.data_ptr<float>();
  a.dy = ym.data_ptr(); a.dh = dm.defined() ? dm.data_ptr() : nullptr;
  a.T = rows_of(hm, "add_rms_norm"); a.H = static_cast<int>(H);
  a.rows_bf16 = h.scalar_type() == torch::kBFloat16; a.weight_bf16 = weight.scalar_type() == torch::kBFloat16;
  auto dx = torch::empty(h.sizes(), h.options());
  if (a.T == 0) return {dx, torch::zeros({H}, weight.options())};
  auto dweight = torch::empty({H}, weight.options());
  const int blocks = row_norm_bwd_blocks(a, sm_count(h));
  auto partials = torch::empty({blocks, H}, h.options().dtype(torch::kFloat32));
  a.dx = dx.data_ptr(); a.dweight = dweight.data_ptr(); a.partials = partials.data_ptr<float>();
  cuda_check(launch_row_norm_bwd(a, blocks, cur_stream()), "add_rms_norm backward");
  return {dx, dweight};
}

torch::Tensor dequantise_rows(const torch::Tensor& q, const torch::Tensor& scales) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kUInt8 && q.dim() >= 1 && q.is_contiguous() && q.size(-1) % 128 == 0 && q.size(-1) > 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 8 == 0,
              "dequantise_rows: q must be contiguous e4m3 bytes [..., hidden], hidden a multiple of 128");
  TORCH_CHECK(scales.device() == q.device() && scales.scalar_type() == torch::kFloat32 && scales.is_contiguous() && scales.dim() == q.dim() && scales.numel() * 128 == q.numel() &&
              scales.size(-1) * 128 == q.size(-1), "dequantise_rows: scales must be contiguous fp32 [..., hidden / 128] on q's device");
  c10::cuda::CUDAGuard guard(q.device());
  auto out = torch::empty(q.sizes(), q.options().dtype(torch::kBFloat16));
  const int H = static_cast<int>(q.size(-1));
  cuda_check(launch_dequant_fp8(q.data_ptr<uint8_t>(), scales.data_ptr<float>(), reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), q.numel() / H, H, nullptr, cur_stream()), "dequantise_rows");
  return out;
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& weight, const OptTensor& residual, double eps, bool quantise) {
    Norm n = row_norm(x, weight, eps, residual, quantise, true);
    ctx->set_materialize_grads(false);
    ctx->saved_data["residual"] = residual.has_value();
    ctx->save_for_backward({residual.has_value() ? n.h : x, weight, n.rstd});
    variable_list out{n.y};
    if (residual.has_value()) out.push_back(n.h);
    if (quantise) { out.push_back(n.q); out.push_back(n.scales); ctx->mark_non_differentiable({n.q, n.scales}); }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    const torch::Tensor dh = residual ? grads[1] : torch::Tensor();
    torch::Tensor dx, dw;
    {
      torch::NoGradGuard no_grad;
      if (grads[0].defined()) {
        std::tie(dx, dw) = row_norm_bwd(saved[0], saved[1], saved[2], grads[0], dh.defined() ? OptTensor(dh) : OptTensor());
      } else {   // only the sum was used
        dx = dh;
        if (ctx->needs_input_grad(1)) dw = torch::zeros_like(saved[1]);
      }
    }
    variable_list in = grads;
    in.insert(in.end(), saved.begin(), saved.end());
    return once("add_rms_norm", in, {ctx->needs_input_grad(0) ? dx : torch::Tensor(), ctx->needs_input_grad(1) ? dw : torch::Tensor(),
                                     residual && ctx->needs_input_grad(2) ? dx : torch::Tensor(), torch::Tensor(), torch::Tensor()});
  }
};
// (y, h, q, scales); h is x without a residual, q and scales are there with quantise.
std::tuple<torch::Tensor, torch::Tensor, OptTensor, OptTensor> add_rms_norm(const torch::Tensor& x, const torch::Tensor& weight, double eps, const OptTensor& residual, bool quantise) {
  const auto some = [](const torch::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  if (!recorded(x, weight, residual)) {
    Norm n = row_norm(x, weight, eps, residual, quantise, false);
    return {n.y, residual.has_value() ? n.h : x, some(n.q), some(n.scales)};
  }
  variable_list out = AddRmsNorm::apply(x, weight, residual, eps, quantise);
  const size_t at = residual.has_value() ? 2 : 1;
  return {out[0], residual.has_value() ? out[1] : x, quantise ? OptTensor(out[at]) : OptTensor(), quantise ? OptTensor(out[at + 1]) : OptTensor()};
}

// ---- balance loss -----------------------------------------------------------------------------------------
struct Balance { torch::Tensor loss, counts, live; };
// logits as rows [T, E], and what the mask is read from.
torch::Tensor mask_bytes(const OptTensor& mask) { return mask.has_value() ? mask->contiguous() : torch::Tensor(); }

Balance balance(const torch::Tensor& logits, const torch::Tensor& topk_idx, const OptTensor& mask, bool sigmoid) {
  TORCH_CHECK(logits.is_cuda() && row_type(logits) && logits.dim() >= 1, "balance_loss: logits must be a bf16 or fp32 CUDA tensor [..., experts]");
  const int64_t E = logits.size(-1);
  TORCH_CHECK(E >= 1 && E <= kBalanceMaxExperts, "balance_loss: 1 to ", kBalanceMaxExperts, " experts, got ", E);
  TORCH_CHECK(topk_idx.device() == logits.device() && topk_idx.scalar_type() == torch::kInt32 && topk_idx.dim() == logits.dim() && topk_idx.sizes().slice(0, topk_idx.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1) &&
              topk_idx.size(-1) >= 1 && topk_idx.size(-1) <= 0x7fffffff, "balance_loss: topk_idx must be int32 [..., k] on the device of logits, a row per token");
  TORCH_CHECK(!mask.has_value() || (mask->device() == logits.device() && mask->scalar_type() == torch::kBool && mask->sizes() == logits.sizes().slice(0, logits.dim() - 1)),
              "balance_loss: mask must be bool [...] on the device of logits, one value per token");
  c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor lm = as_rows(logits, E), im = topk_idx.contiguous(), mm = mask_bytes(mask);
  BalanceArgs a{};
  a.logits = lm.data_ptr(); a.stride = lm.stride(0); a.logits_bf16 = logits.scalar_type() == torch::kBFloat16;
  a.topk_idx = im.data_ptr<int>();
  a.mask = mm.defined() ? reinterpret_cast<const unsigned char*>(mm.data_ptr()) : nullptr;
  a.T = rows_of(lm, "balance_loss"); a.E = static_cast<int>(E); a.K = static_cast<int>(topk_idx.size(-1)); a.sigmoid = sigmoid;
  TORCH_CHECK(static_cast<int64_t>(a.T) * a.K <= 0x7fffffff, "balance_loss: more than 2^31 - 1 choices");
  const auto f32 = logits.options().dtype(torch::kFloat32), i32 = logits.options().dtype(torch::kInt32);
  Balance b{torch::empty({}, f32), torch::empty({E}, i32), torch::empty({}, i32)};
  a.loss = b.loss.data_ptr<float>(); a.counts = b.counts.data_ptr<int>(); a.live = b.live.data_ptr<int>();
  const int blocks = balance_blocks(a, sm_count(logits));
  torch::Tensor scratch;
  if (blocks > 1) {
    scratch = torch::empty({blocks, 2 * E + 1}, i32);
    a.chosen = scratch.data_ptr<int>();
    a.sums = reinterpret_cast<float*>(a.chosen + blocks * (E + 1));
  }
  cuda_check(launch_balance(a, blocks, cur_stream()), "balance_loss");
  return b;
}

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logits, const torch::Tensor& topk_idx, const OptTensor& mask, bool sigmoid) {
    Balance b = balance(logits, topk_idx, mask, sigmoid);
    ctx->set_materialize_grads(false);
    ctx->saved_data["k"] = topk_idx.size(-1);
    ctx->saved_data["sigmoid"] = sigmoid;
    ctx->save_for_backward({logits, mask_bytes(mask), b.counts, b.live});
    ctx->mark_non_differentiable({b.counts});
    return {b.loss, b.counts};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor& logits = saved[0];
    torch::Tensor dlogits;
    {
      torch::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(logits.device());
      const torch::Tensor lm = as_rows(logits, logits.size(-1)), dloss = grads[0].to(torch::kFloat32);
      dlogits = torch::empty(logits.sizes(), logits.options());
      BalanceBwdArgs a{};
      a.logits = lm.data_ptr(); a.stride = lm.stride(0); a.logits_bf16 = logits.scalar_type() == torch::kBFloat16;
      a.mask = saved[1].defined() ? reinterpret_cast<const unsigned char*>(saved[1].data_ptr()) : nullptr;
      a.T = static_cast<int>(lm.size(0)); a.E = static_cast<int>(logits.size(-1)); a.K = static_cast<int>(ctx->saved_data["k"].toInt()); a.sigmoid = ctx->saved_data["sigmoid"].toBool();
      a.counts = saved[2].data_ptr<int>(); a.live = saved[3].data_ptr<int>(); a.dloss = dloss.data_ptr<float>(); a.dlogits = dlogits.data_ptr();
      cuda_check(launch_balance_bwd(a, sm_count(logits), cur_stream()), "balance_loss backward");
    }
    variable_list in = grads;
    in.push_back(logits);
    return once("balance_loss", in, {dlogits, torch::Tensor(), torch::Tensor(), torch::Tensor()});
  }
};
std::tuple<torch::Tensor, torch::Tensor> balance_loss(const torch::Tensor& logits, const torch::Tensor& topk_idx, const OptTensor& mask, bool sigmoid) {
  if (!recorded(logits)) {
    Balance b = balance(logits, topk_idx, mask, sigmoid);
    return {b.loss, b.counts};
  }
  variable_list out = BalanceLoss::apply(logits, topk_idx, mask, sigmoid);
  return {out[0], out[1]};
}

}  // namespace

void bind_dense(py::module_& m) {
  m.def("add_rms_norm", &add_rms_norm, py::arg("x"), py::arg("weight"), py::arg("eps"), py::arg("residual"), py::arg("quantise"));
  m.def("balance_loss", &balance_loss, py::arg("logits"), py::arg("topk_idx"), py::arg("mask"), py::arg("sigmoid"));
  m.def("dequantise_rows", &dequantise_rows, py::arg("q"), py::arg("scales"));
}
