// Bindings of the dense side of a block: row norm, balance loss, linear layers. Their kernels run on the current stream of the
// tensors' own device, whichever device is current.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../kernels/tile_walker.h"
#include "../kernels/token_walker.h"
#include "py_types.h"
#include "tensor_maps.h"

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

// The kernels read tensors through their pointers. A fake or wrapped tensor has none (its address reads as null, which would fault on the device); a zero
// tensor, as some backward passes hand on, has none either; a negated view's memory holds the other sign.
constexpr c10::DispatchKeySet kNotItsMemory({c10::DispatchKey::Python, c10::DispatchKey::ZeroTensor, c10::DispatchKey::Negative, c10::DispatchKey::Conjugate});
bool is_its_memory(const torch::Tensor& t) { return t.defined() && t.layout() == torch::kStrided && t.has_storage() && !t.key_set().has_any(kNotItsMemory); }
void want_memory(const char* op, const torch::Tensor& t) {
  TORCH_CHECK(is_its_memory(t), op, ": every tensor must be one of plain memory (no fake, wrapped, sparse, zero or negated tensor)");
}
void want_memory(const char* op, const OptTensor& t) { if (t.has_value()) want_memory(op, *t); }
template <class... T> void all_in_memory(const char* op, const T&... t) { (want_memory(op, t), ...); }
// An incoming gradient, made real where it is a zero tensor or a negated view.
torch::Tensor real(const char* op, const torch::Tensor& grad) {
  if (is_its_memory(grad)) return grad;
  const torch::Tensor g = grad._is_zerotensor() ? at::zeros(grad.sizes(), grad.options()) : grad.resolve_neg();
  want_memory(op, g);
  return g;
}

// What a backward pass kept, as it was: hooks of saved tensors may have brought it back otherwise. last: its last size, or -1 for any; made: by the forward pass itself, contiguous.
void want_kept(const char* op, const torch::Tensor& t, const torch::Tensor& grad, c10::ScalarType type, int64_t numel, int64_t last, bool made) {
  TORCH_CHECK(is_its_memory(t) && t.device() == grad.device() && t.scalar_type() == type && t.numel() == numel && (last < 0 || (t.dim() >= 1 && t.size(-1) == last)) && (!made || t.is_contiguous()),
              op, ": a saved tensor came back on another device, of another type, size or layout");
}

// No operator here has a forward-mode derivative: an input's tangent would be lost without a word.
void no_tangent(const char* op, const torch::Tensor& t) {
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), op, ": there is no forward-mode derivative, and an input has a tangent");
}
void no_tangent(const char* op, const OptTensor& t) { if (t.has_value()) no_tangent(op, *t); }
template <class... T> void no_tangents(const char* op, const T&... t) { (no_tangent(op, t), ...); }

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

// A new contiguous tensor on the device of `like`, without the dispatcher's way there (half of what a call of a few rows costs the host is allocation).
torch::Tensor fresh(at::IntArrayRef shape, const torch::Tensor& like, c10::ScalarType type) { return at::detail::empty_cuda(shape, type, like.device(), c10::nullopt); }
torch::Tensor fresh(at::IntArrayRef shape, const torch::Tensor& like) { return fresh(shape, like, like.scalar_type()); }

// Rows of t as a matrix whose rows are contiguous; only what cannot be seen as one is copied.
torch::Tensor as_rows(const torch::Tensor& t, int64_t cols) {
  torch::Tensor m = t.dim() == 2 ? t : t.reshape({-1, cols});
  return m.stride(1) == 1 || cols == 1 ? m : m.contiguous();
}
// Rows of t, so few that a kernel counts past the last one in 32 bits. Asked for before anything is copied or allocated.
int rows_of(const torch::Tensor& t, int64_t cols, const char* what) {
  const int64_t rows = t.numel() / cols;
  TORCH_CHECK(rows <= 1 << 30, what, ": more than 2^30 rows");
  return static_cast<int>(rows);
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
  RowNormArgs a{};
  a.T = rows_of(x, H, "add_rms_norm"); a.H = static_cast<int>(H);
  c10::cuda::CUDAGuard guard(x.device());
  const torch::Tensor xm = as_rows(x, H);
  a.x = xm.data_ptr(); a.x_stride = xm.stride(0);
  a.weight = weight.data_ptr();
  a.rows_bf16 = x.scalar_type() == torch::kBFloat16; a.weight_bf16 = weight.scalar_type() == torch::kBFloat16;
  a.eps = static_cast<float>(eps);
  torch::Tensor y = fresh(x.sizes(), x), rm;
  torch::Tensor h, q, scales, rstd;
  a.y = y.data_ptr();
  if (residual.has_value()) {
    rm = as_rows(*residual, H);
    a.residual = rm.data_ptr(); a.residual_stride = rm.stride(0);
    h = fresh(x.sizes(), x);
    a.h = h.data_ptr();
  }
  if (quantise) {
    q = fresh(x.sizes(), x, torch::kUInt8);
    auto shape = x.sizes().vec();
    shape.back() = H / 128;
    scales = fresh(shape, x, torch::kFloat32);
    a.q = q.data_ptr<uint8_t>(); a.scales = scales.data_ptr<float>();
  }
  if (keep) {
    rstd = fresh({xm.size(0)}, x, torch::kFloat32);
    a.rstd = rstd.data_ptr<float>();
  }
  cuda_check(launch_row_norm(a, sm_count(x), cur_stream()), "add_rms_norm");
  return {y, h, q, scales, rstd};
}

// (dx, dweight) from what the forward pass normalised, its rstd, dy and optionally dh.
std::tuple<torch::Tensor, torch::Tensor> row_norm_bwd(const torch::Tensor& h, const torch::Tensor& weight, const torch::Tensor& rstd, const torch::Tensor& dy, const OptTensor& dh) {
  TORCH_CHECK(h.is_cuda() && row_type(h) && row_type(weight) && dy.sizes() == h.sizes() && dy.scalar_type() == h.scalar_type() && dy.device() == h.device(), "add_rms_norm backward: gradient of y");
  TORCH_CHECK(!dh.has_value() || (dh->sizes() == h.sizes() && dh->scalar_type() == h.scalar_type() && dh->device() == h.device()), "add_rms_norm backward: gradient of the sum");
  const int64_t H = h.size(-1);
  want_kept("add_rms_norm backward", h, dy, h.scalar_type(), dy.numel(), H, false);
  want_kept("add_rms_norm backward", weight, dy, weight.scalar_type(), H, H, true);
  want_kept("add_rms_norm backward", rstd, dy, torch::kFloat32, dy.numel() / H, dy.numel() / H, true);
  c10::cuda::CUDAGuard guard(h.device());
  const torch::Tensor hm = as_rows(h, H), ym = dy.contiguous(), dm = dh.has_value() ? dh->contiguous() : torch::Tensor();
  RowNormBwdArgs a{};
  a.h = hm.data_ptr(); a.h_stride = hm.stride(0);
  a.weight = weight.data_ptr(); a.rstd = rstd.data_ptr<float>();
  a.dy = ym.data_ptr(); a.dh = dm.defined() ? dm.data_ptr() : nullptr;
  a.T = rows_of(h, H, "add_rms_norm"); a.H = static_cast<int>(H);
  a.rows_bf16 = h.scalar_type() == torch::kBFloat16; a.weight_bf16 = weight.scalar_type() == torch::kBFloat16;
  auto dx = fresh(h.sizes(), h);
  if (a.T == 0) return {dx, torch::zeros({H}, weight.options())};
  auto dweight = fresh({H}, weight);
  const int blocks = row_norm_bwd_blocks(a, sm_count(h));
  auto partials = fresh({blocks, H}, h, torch::kFloat32);
  a.dx = dx.data_ptr(); a.dweight = dweight.data_ptr(); a.partials = partials.data_ptr<float>();
  cuda_check(launch_row_norm_bwd(a, blocks, cur_stream()), "add_rms_norm backward");
  return {dx, dweight};
}

torch::Tensor dequantise_rows(const torch::Tensor& q, const torch::Tensor& scales) {
  all_in_memory("dequantise_rows", q, scales);
  no_tangents("dequantise_rows", scales);
  TORCH_CHECK(!recorded(scales), "dequantise_rows: there is no gradient of the scales, and they require one");
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kUInt8 && q.dim() >= 1 && q.is_contiguous() && q.size(-1) % 128 == 0 && q.size(-1) > 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 8 == 0,
              "dequantise_rows: q must be contiguous e4m3 bytes [..., hidden], hidden a multiple of 128");
  TORCH_CHECK(scales.device() == q.device() && scales.scalar_type() == torch::kFloat32 && scales.is_contiguous() && scales.dim() == q.dim() && scales.numel() * 128 == q.numel() &&
              scales.size(-1) * 128 == q.size(-1), "dequantise_rows: scales must be contiguous fp32 [..., hidden / 128] on q's device");
  c10::cuda::CUDAGuard guard(q.device());
  auto out = fresh(q.sizes(), q, torch::kBFloat16);
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
    torch::Tensor dx, dw, dh;
    {
      torch::NoGradGuard no_grad;
      if (residual && grads[1].defined()) dh = real("add_rms_norm backward", grads[1]);
      if (grads[0].defined()) {
        std::tie(dx, dw) = row_norm_bwd(saved[0], saved[1], saved[2], real("add_rms_norm backward", grads[0]), dh.defined() ? OptTensor(dh) : OptTensor());
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
  all_in_memory("add_rms_norm", x, weight, residual);
  no_tangents("add_rms_norm", x, weight, residual);
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
struct Balance { torch::Tensor loss, counts, kept; };
torch::Tensor mask_bytes(const OptTensor& mask) { return mask.has_value() ? mask->contiguous() : torch::Tensor(); }

Balance balance(const torch::Tensor& logits, const torch::Tensor& topk_idx, const OptTensor& mask, bool sigmoid) {
  TORCH_CHECK(logits.is_cuda() && row_type(logits) && logits.dim() >= 1, "balance_loss: logits must be a bf16 or fp32 CUDA tensor [..., experts]");
  const int64_t E = logits.size(-1);
  TORCH_CHECK(E >= 1 && E <= kBalanceMaxExperts, "balance_loss: 1 to ", kBalanceMaxExperts, " experts, got ", E);
  TORCH_CHECK(topk_idx.device() == logits.device() && topk_idx.scalar_type() == torch::kInt32 && topk_idx.dim() == logits.dim() && topk_idx.sizes().slice(0, topk_idx.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1) &&
              topk_idx.size(-1) >= 1 && topk_idx.size(-1) <= 0x7fffffff, "balance_loss: topk_idx must be int32 [..., k] on the device of logits, a row per token");
  TORCH_CHECK(!mask.has_value() || (mask->device() == logits.device() && mask->scalar_type() == torch::kBool && mask->sizes() == logits.sizes().slice(0, logits.dim() - 1)),
              "balance_loss: mask must be bool [...] on the device of logits, one value per token");
  BalanceArgs a{};
  a.T = rows_of(logits, E, "balance_loss"); a.E = static_cast<int>(E); a.K = static_cast<int>(topk_idx.size(-1)); a.sigmoid = sigmoid;
  TORCH_CHECK(static_cast<int64_t>(a.T) * a.K <= 0x7fffffff, "balance_loss: more than 2^31 - 1 choices");
  c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor lm = as_rows(logits, E), im = topk_idx.contiguous(), mm = mask_bytes(mask);
  a.logits = lm.data_ptr(); a.stride = lm.stride(0); a.logits_bf16 = logits.scalar_type() == torch::kBFloat16;
  a.topk_idx = im.data_ptr<int>();
  a.mask = mm.defined() ? reinterpret_cast<const unsigned char*>(mm.data_ptr()) : nullptr;
  Balance b{fresh(at::IntArrayRef{}, logits, torch::kFloat32), fresh({E}, logits, torch::kInt32), fresh({E + 1}, logits, torch::kInt32)};
  a.loss = b.loss.data_ptr<float>(); a.counts = b.counts.data_ptr<int>(); a.kept = b.kept.data_ptr<int>();
  const int blocks = balance_blocks(a, sm_count(logits));
  torch::Tensor scratch;
  if (blocks > 1) {
    scratch = fresh({blocks, 2 * E + 1}, logits, torch::kInt32);
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
    ctx->saved_data["kept"] = std::vector<int64_t>{topk_idx.size(-1), sigmoid, logits.size(-1), static_cast<int64_t>(logits.scalar_type()), logits.numel() / logits.size(-1)};
    ctx->save_for_backward({logits, mask_bytes(mask), b.kept});
    ctx->mark_non_differentiable({b.counts});
    return {b.loss, b.counts};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> kept = ctx->saved_data["kept"].toIntVector();
    const torch::Tensor& logits = saved[0];
    const int64_t E = kept[2];
    want_kept("balance_loss backward", logits, grads[0], static_cast<c10::ScalarType>(kept[3]), kept[4] * E, E, false);
    if (saved[1].defined()) want_kept("balance_loss backward", saved[1], grads[0], torch::kBool, kept[4], -1, true);
    want_kept("balance_loss backward", saved[2], grads[0], torch::kInt32, E + 1, E + 1, true);
    torch::Tensor dlogits;
    {
      torch::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(logits.device());
      const torch::Tensor lm = as_rows(logits, logits.size(-1)), dloss = real("balance_loss backward", grads[0]).to(torch::kFloat32);
      dlogits = fresh(logits.sizes(), logits);
      BalanceBwdArgs a{};
      a.logits = lm.data_ptr(); a.stride = lm.stride(0); a.logits_bf16 = logits.scalar_type() == torch::kBFloat16;
      a.mask = saved[1].defined() ? reinterpret_cast<const unsigned char*>(saved[1].data_ptr()) : nullptr;
      a.T = rows_of(logits, logits.size(-1), "balance_loss"); a.E = static_cast<int>(logits.size(-1)); a.K = static_cast<int>(kept[0]); a.sigmoid = static_cast<int>(kept[1]);
      a.kept = saved[2].data_ptr<int>(); a.dloss = dloss.data_ptr<float>(); a.dlogits = dlogits.data_ptr();
      cuda_check(launch_balance_bwd(a, sm_count(logits), cur_stream()), "balance_loss backward");
    }
    variable_list in = grads;
    in.push_back(logits);
    return once("balance_loss", in, {dlogits, torch::Tensor(), torch::Tensor(), torch::Tensor()});
  }
};
std::tuple<torch::Tensor, torch::Tensor> balance_loss(const torch::Tensor& logits, const torch::Tensor& topk_idx, const OptTensor& mask, bool sigmoid) {
  all_in_memory("balance_loss", logits, topk_idx, mask);
  no_tangents("balance_loss", logits);
  if (!recorded(logits)) {
    Balance b = balance(logits, topk_idx, mask, sigmoid);
    return {b.loss, b.counts};
  }
  variable_list out = BalanceLoss::apply(logits, topk_idx, mask, sigmoid);
  return {out[0], out[1]};
}

// ---- linear layers ----------------------------------------------------------------------------------------
enum class LinearKind : int { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kSwiGLU = 4 };   // the first four are Activation's

// Rows [n, cols] that TMA can read: contiguous rows, 16-byte aligned, a multiple of 16 bytes apart. What is not is copied.
torch::Tensor tma_rows(const torch::Tensor& t, int64_t cols) {
  torch::Tensor m = as_rows(t, cols);
  const bool ok = reinterpret_cast<uintptr_t>(m.data_ptr()) % 16 == 0 && m.stride(1) == 1 && (m.size(0) <= 1 || (m.stride(0) % 8 == 0 && m.stride(0) >= cols));
  return ok ? m : m.clone(at::MemoryFormat::Contiguous);
}
CUtensorMap rows_map(const torch::Tensor& m, int box_rows, int box_cols = 64) {
  const cuuint64_t rows = static_cast<cuuint64_t>(m.size(0)), cols = static_cast<cuuint64_t>(m.size(1)), dims[2] = {cols, rows}, strides[1] = {2 * (rows > 1 ? static_cast<cuuint64_t>(m.stride(0)) : cols)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  return bf16_map(2, reinterpret_cast<int64_t>(m.data_ptr()), dims, strides, box, box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

struct DenseEpilogue {
  GemmEpilogue kind = GemmEpilogue::kLinear;
  const torch::Tensor *bias = nullptr, *residual = nullptr, *pre = nullptr;   // pre: pre-activation, or gate|up of kSwiGLU and what their rounding took off
  Activation act = Activation::kNone;
};

// How the kernel with tiles of 256 features goes about `rows` tokens (more than 64: fewer are always few, see few_pays). plain: nothing but the product.
TokDenseArgs dense_args(int rows, int64_t features, int64_t reduction, bool plain, int ctas) {
  TokDenseArgs a{};
  a.num_groups = 1;
  a.dense_rows = rows; a.features = static_cast<int>(features);
  a.m_tiles = static_cast<int>((features + 255) / 256); a.red_blocks = static_cast<int>((reduction + 63) / 64);
  a.granule = 32;
  // Where all tokens fit a narrow tile, narrow tiles leave shared memory to the weights in flight.
  a.tile_n = rows <= 128 ? 128 : gemm::tok_dense_tile(rows, a.m_tiles, a.red_blocks, ctas / 2);
  // SwiGLU, whose kept gate and up would leave three stages, takes no wide tiles: us on them, without: 300 x 4096 -> 104448 233 to 273, 246; kept 312 to 331, 282 to 294;
  // 280 x 4096 -> 163840 382 to 387, 358 to 362; kept 439 to 448, 422 to 426.
  if (plain && a.tile_n == 256 && gemm::tok_wide(false, static_cast<int>(reduction), rows, (rows + 511) / 512 * (features / 256.0) / (ctas / 2))) a.tile_n = 512;
  a.band_tiles = gemm::tok_band(0, 64 * a.red_blocks, a.m_tiles, a.tile_n);
  a.back_tiles = gemm::tok_back_tiles(64 * a.red_blocks, a.band_tiles, std::max(a.tile_n, gemm::kTokAccN));
  return a;
}

// forward: out [T, N] = epilogue(x [T, K] . weight [N, K]^T); dgrad: out [T, K] = x [T, N] . weight [N, K]. All bf16 rows as tma_rows makes them.
void dense_gemm(GemmMode mode, const torch::Tensor& weight, const torch::Tensor& x, const torch::Tensor& out, const DenseEpilogue& ep, uint64_t timeout_ns) {
  const bool fwd = mode == GemmMode::kForward;
  const int64_t N = weight.size(0), K = weight.size(1), features = fwd ? N : K, reduction = fwd ? K : N;
  const int ctas = sm_count(x) & ~1;
  const bool plain = ep.kind == GemmEpilogue::kLinear && ep.act == Activation::kNone && !ep.bias && !ep.residual && !ep.pre;
  TokDenseArgs a = dense_args(static_cast<int>(x.size(0)), features, reduction, plain, ctas);
  const GemmEpilogue kind = a.tile_n == 512 ? GemmEpilogue::kStore : ep.kind;
  a.status = dense_status();
  TORCH_CHECK(a.status != nullptr, "linear: no status block on this device");
  a.timeout_ns = timeout_ns;
  const int cols = kind == GemmEpilogue::kLinear ? 32 : 64;   // of the epilogue's boxes
  CUtensorMap w, c = rows_map(out, 32, cols), c2, c3;
  TokMapsX xm;
  if (ep.kind == GemmEpilogue::kSwiGLU) {
    // [N / 256 tiles][8 groups of 16 features][gate, up][16][K], fetched as four groups with both halves
    const cuuint64_t k = static_cast<cuuint64_t>(K), dims[5] = {k, 16, 2, 8, static_cast<cuuint64_t>(N / 256)}, strides[4] = {2 * k, 256 * k, 32 * k, 512 * k};
    const cuuint32_t box[5] = {64, 16, 2, 4, 1};
    w = bf16_map(5, reinterpret_cast<int64_t>(weight.data_ptr()), dims, strides, box);
  } else {
    w = rows_map(weight, fwd ? 128 : 64);
  }
  for (int j = 0; j < kTokBoxes; ++j) xm.box[j] = rows_map(x, 16 << j);
  TokDenseMaps maps{};
  maps.w = &w; maps.x = &xm; maps.c = &c;
  if (kind == GemmEpilogue::kSwiGLU) {
    if (ep.pre) { c2 = rows_map(*ep.pre, 32); maps.c2 = &c2; a.keep_gate_up = 1; }
  } else if (kind == GemmEpilogue::kLinear) {
    a.act = ep.act;
    if (ep.bias) a.bias = reinterpret_cast<const __nv_bfloat16*>(ep.bias->data_ptr());
    if (ep.residual) { c2 = rows_map(*ep.residual, 32, cols); maps.c2 = &c2; a.has_residual = 1; }
    if (ep.pre) { c3 = rows_map(*ep.pre, 32, cols); maps.c3 = &c3; a.keep_pre = 1; }
  }
  torch::Tensor partials, counters;
  if (dense_split(a, ctas).cut_tiles > 0) {
    partials = fresh({tok_partial_floats(ctas, a.tile_n)}, x, torch::kFloat32);
    counters = torch::zeros({tok_counters(ctas)}, x.options().dtype(torch::kInt32));
    a.partials = partials.data_ptr<float>();
    a.counters = reinterpret_cast<unsigned int*>(counters.data_ptr<int>());
  }
  cuda_check(launch_dense_gemm(mode, kind, maps, a, ctas, cur_stream()), "linear");
}

// out [N, K] = dz [T, N]^T . x [T, K]. Few tiles of many rows: the rows are shared out, and the slices' fp32 sums added up by a second launch.
// us: 8000 rows, 1024 x 1024 (16 tiles, 4 slices) 45 -> 23; 4280 rows, 3376 x 136 (14 tiles, 5 slices) 28 -> 18.
void dense_wgrad(const torch::Tensor& dz, const torch::Tensor& x, const torch::Tensor& out, uint64_t timeout_ns) {
  const int64_t N = out.size(0), K = out.size(1);
  const int ctas = sm_count(x) & ~1, rows = static_cast<int>(x.size(0));
  GemmArgs g{};
  g.dense_rows = rows;
  g.fixed_m_tiles = static_cast<int>((N + 255) / 256);
  g.tiles_n = static_cast<int>((K + 255) / 256);
  const int64_t tiles = static_cast<int64_t>(g.fixed_m_tiles) * g.tiles_n;
  const int slices = static_cast<int>(std::min<int64_t>({8, ctas / 2 / tiles, (rows + 63) / 64 / 8}));
  g.status = dense_status();
  TORCH_CHECK(g.status != nullptr, "linear: no status block on this device");
  g.timeout_ns = timeout_ns;
  if (slices > 1) {
    const torch::Tensor sums = fresh({slices, tiles, 256, 256}, x, torch::kFloat32);
    g.num_groups = slices;
    g.sums = sums.data_ptr<float>();
    g.direct_epilogue = 1;
    cuda_check(launch_grouped_gemm_pair(GemmMode::kWgrad, GemmEpilogue::kStore, rows_map(dz, 64), rows_map(x, 64), rows_map(out, 128), nullptr, g, ctas, cur_stream()), "linear weight gradient");
    cuda_check(launch_fold_slices(g.sums, slices, g.fixed_m_tiles, g.tiles_n, reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), static_cast<int>(N), static_cast<int>(K), cur_stream()), "linear weight gradient");
    return;
  }
  g.num_groups = 1;
  g.wide = gemm::wgrad_wide(g.fixed_m_tiles, static_cast<int>(K), ctas / 2, rows);
  if (g.wide) g.tiles_n /= 2;
  g.c_rows_per_group = static_cast<int>(N);
  g.c = reinterpret_cast<__nv_bfloat16*>(out.data_ptr()); g.ldc = K;
  cuda_check(launch_grouped_gemm_pair(GemmMode::kWgrad, GemmEpilogue::kStore, rows_map(dz, 64), rows_map(x, 64), rows_map(out, g.wide ? 32 : 128), nullptr, g, ctas, cur_stream()), "linear weight gradient");
}

// The same on few rows, where that pays; false: nothing was done.
bool dense_few(GemmMode mode, const torch::Tensor& weight, const torch::Tensor& x, const torch::Tensor& out, const DenseEpilogue& ep, uint64_t timeout_ns) {
  const bool swiglu = ep.kind == GemmEpilogue::kSwiGLU, fwd = mode == GemmMode::kForward;
  const int64_t red_blocks = (weight.size(fwd ? 1 : 0) + 63) / 64;
  const auto sectors = [](const torch::Tensor& t) { return t.stride(0) % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 32 == 0; };
  if (!few_pays(static_cast<int>(x.size(0)), static_cast<int>(out.size(1)), static_cast<int>(red_blocks), swiglu, sectors(weight) && sectors(x), sm_count(x))) return false;
  FewArgs a{};
  a.T = static_cast<int>(x.size(0)); a.columns = static_cast<int>(out.size(1));
  a.red_blocks = static_cast<int>(red_blocks);
  const auto ptr = [](const torch::Tensor* t) { return t ? reinterpret_cast<__nv_bfloat16*>(t->data_ptr()) : nullptr; };
  a.bias = ptr(ep.bias); a.residual = ptr(ep.residual); a.out = ptr(&out); a.pre = ptr(ep.pre);
  a.residual_stride = ep.residual ? ep.residual->stride(0) : 0;
  a.status = dense_status();
  TORCH_CHECK(a.status != nullptr, "linear: no status block on this device");
  a.timeout_ns = timeout_ns;
  cuda_check(launch_linear_few(mode, ep.act, swiglu, rows_map(weight, swiglu || !fwd ? 64 : 128), rows_map(x, few_plan(a.T, a.columns, a.red_blocks, swiglu, sm_count(x)).n), a, sm_count(x), cur_stream()), "linear");
  return true;
}

struct LinearOut { torch::Tensor y, pre; };
LinearOut linear_forward(const torch::Tensor& x, const torch::Tensor& weight, const OptTensor& bias, LinearKind kind, const OptTensor& residual, bool keep, uint64_t timeout_ns) {
  const auto bf = torch::kBFloat16;
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == bf && x.dim() >= 1, "linear: x must be a bf16 CUDA tensor [..., inputs]");
  TORCH_CHECK(weight.device() == x.device() && weight.scalar_type() == bf && weight.dim() == 2 && weight.size(1) == x.size(-1), "linear: weight must be bf16 [outputs, inputs] on x's device");
  const int64_t N = weight.size(0), K = weight.size(1), cols = kind == LinearKind::kSwiGLU ? N / 2 : N;
  TORCH_CHECK(K >= 8 && K % 8 == 0 && N >= 8 && N % 8 == 0, "linear: inputs and outputs must be multiples of 8 (rows of whole 16-byte words), got ", K, " and ", N);
  TORCH_CHECK(K <= 1 << 24 && N <= 1 << 24, "linear: at most 2^24 inputs and outputs");
  TORCH_CHECK(kind != LinearKind::kSwiGLU || (N % 256 == 0 && !bias.has_value() && !residual.has_value()),
              "linear: swiglu takes weights in tiles of 128 gate rows and 128 up rows (outputs a multiple of 256), no bias and no residual");
  TORCH_CHECK(!bias.has_value() || (bias->device() == x.device() && bias->scalar_type() == bf && bias->dim() == 1 && bias->size(0) == N && bias->is_contiguous()), "linear: bias must be contiguous bf16 [outputs] on x's device");
  auto shape = x.sizes().vec();
  shape.back() = cols;
  TORCH_CHECK(!residual.has_value() || (residual->device() == x.device() && residual->scalar_type() == bf && residual->sizes() == at::IntArrayRef(shape)), "linear: residual must be bf16 with the output's shape, on x's device");
  const int64_t T = rows_of(x, K, "linear");
  c10::cuda::CUDAGuard guard(x.device());
  LinearOut o{fresh(shape, x), {}};
  const bool pre = keep && kind != LinearKind::kNone;
  if (pre) o.pre = fresh({T, kind == LinearKind::kSwiGLU ? 2 * N : N}, x);   // SwiGLU: with what the rounding took off
  if (T == 0) return o;
  const torch::Tensor xm = tma_rows(x, K), wm = kind == LinearKind::kSwiGLU && !weight.is_contiguous() ? weight.contiguous() : tma_rows(weight, K), ym = o.y.view({T, cols});
  torch::Tensor rm, bm;
  DenseEpilogue ep;
  if (kind == LinearKind::kSwiGLU) {
    ep.kind = GemmEpilogue::kSwiGLU;
  } else {
    ep.act = static_cast<Activation>(kind);
    if (bias.has_value()) { bm = reinterpret_cast<uintptr_t>(bias->data_ptr()) % 8 == 0 ? *bias : bias->clone(); ep.bias = &bm; }   // read in words of 8 bytes
    if (residual.has_value()) { rm = tma_rows(*residual, cols); ep.residual = &rm; }
  }
  if (pre) ep.pre = &o.pre;
  if (!dense_few(GemmMode::kForward, wm, xm, ym, ep, timeout_ns)) dense_gemm(GemmMode::kForward, wm, xm, ym, ep, timeout_ns);
  return o;
}

struct Linear : torch::autograd::Function<Linear> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t kind, int64_t timeout_ns) {
    const bool through = x.requires_grad() || weight.requires_grad() || wants_grad(bias);   // the gradient goes past the activation
    LinearOut o = linear_forward(x, weight, bias, static_cast<LinearKind>(kind), residual, through, timeout_ns);
    ctx->set_materialize_grads(false);
    // all numbers in one entry: every entry is a hash of its name on the way in and out
    std::vector<int64_t> kept{kind, timeout_ns, bias.has_value(), residual.has_value(), weight.size(0), weight.size(1)};
    kept.insert(kept.end(), x.sizes().begin(), x.sizes().end());
    ctx->saved_data["kept"] = std::move(kept);
    ctx->save_for_backward({weight.requires_grad() ? x : torch::Tensor(), x.requires_grad() ? weight : torch::Tensor(), o.pre});
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> kept = ctx->saved_data["kept"].toIntVector();
    const auto kind = static_cast<LinearKind>(kept[0]);
    const uint64_t timeout_ns = static_cast<uint64_t>(kept[1]);
    const bool has_bias = kept[2], has_residual = kept[3];
    const int64_t N = kept[4], K = kept[5];
    const at::IntArrayRef shape(kept.data() + 6, kept.size() - 6);   // of x
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = has_bias && ctx->needs_input_grad(2), want_r = has_residual && ctx->needs_input_grad(has_bias ? 3 : 2);
    if (want_r) out[3] = grads[0];
    if (want_x || want_w || want_b) {
      torch::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(grads[0].device());
      const torch::Tensor dy = tma_rows(real("linear backward", grads[0]), kind == LinearKind::kSwiGLU ? N / 2 : N);
      const int64_t T = dy.size(0), kept_width = kind == LinearKind::kSwiGLU ? 2 * N : N;
      if (want_w) want_kept("linear backward", saved[0], dy, torch::kBFloat16, T * K, K, false);
      if (want_x) want_kept("linear backward", saved[1], dy, torch::kBFloat16, N * K, K, false);
      if (kind != LinearKind::kNone) want_kept("linear backward", saved[2], dy, torch::kBFloat16, T * kept_width, kept_width, true);
      TORCH_CHECK(dy.scalar_type() == torch::kBFloat16, "linear backward: the gradient must be bf16");
      if (T == 0) {
        if (want_x) out[0] = torch::zeros(shape, dy.options());
        if (want_w) out[1] = torch::zeros({N, K}, dy.options());
        if (want_b) out[2] = torch::zeros({N}, dy.options());
      } else {
        torch::Tensor dz = dy;
        if (kind == LinearKind::kSwiGLU) {
          const torch::Tensor d = dy.contiguous();
          dz = fresh({T, N}, dy);
          cuda_check(launch_linear_swiglu_dz(reinterpret_cast<const __nv_bfloat16*>(d.data_ptr()), reinterpret_cast<const __nv_bfloat16*>(saved[2].data_ptr()), reinterpret_cast<__nv_bfloat16*>(dz.data_ptr()),
                                             static_cast<int>(T), static_cast<int>(N / 2), cur_stream()), "linear backward: swiglu");
        } else if (kind != LinearKind::kNone || want_b) {
          const torch::Tensor d = dy.contiguous();
          torch::Tensor partials;
          const int blocks = linear_dz_blocks(static_cast<int>(T), static_cast<int>(N), sm_count(dy));
          if (kind != LinearKind::kNone) dz = fresh({T, N}, dy);
          if (want_b) {
            out[2] = fresh({N}, dy);
            partials = fresh({blocks, N}, dy, torch::kFloat32);
          }
          const auto ptr = [](const torch::Tensor& t) { return t.defined() ? reinterpret_cast<__nv_bfloat16*>(t.data_ptr()) : nullptr; };
          cuda_check(launch_linear_dz(static_cast<Activation>(kind), ptr(d), ptr(saved[2]), kind != LinearKind::kNone ? ptr(dz) : nullptr, want_b ? partials.data_ptr<float>() : nullptr, static_cast<int>(T),
                                      static_cast<int>(N), blocks, ptr(out[2]), cur_stream()), "linear backward: activation");
        }
        if (want_x) {
          out[0] = fresh(shape, dy);
          const torch::Tensor wm = tma_rows(saved[1], K), dx = out[0].view({T, K});
          if (!dense_few(GemmMode::kDgrad, wm, dz, dx, {}, timeout_ns)) dense_gemm(GemmMode::kDgrad, wm, dz, dx, {}, timeout_ns);
        }
        if (want_w) {
          out[1] = fresh({N, K}, dy);
          dense_wgrad(dz, tma_rows(saved[0], K), out[1], timeout_ns);
        }
      }
    }
    variable_list in = grads;
    in.insert(in.end(), saved.begin(), saved.end());
    return once("linear", in, out);
  }
};
torch::Tensor linear(const torch::Tensor& x, const torch::Tensor& weight, const OptTensor& bias, const OptTensor& residual, int kind, double timeout_s) {
  all_in_memory("linear", x, weight, bias, residual);
  no_tangents("linear", x, weight, bias, residual);
  TORCH_CHECK(kind >= 0 && kind <= 4 && timeout_s > 0, "linear: activation or limit");
  const int64_t timeout_ns = static_cast<int64_t>(timeout_s * 1e9);
  if (!recorded(x, weight, bias, residual)) return linear_forward(x, weight, bias, static_cast<LinearKind>(kind), residual, false, timeout_ns).y;
  return Linear::apply(x, weight, bias, residual, kind, timeout_ns)[0];
}
// Where linear layers on the current device report a wait that gave up. All of the device's users share it, so reading leaves it as it is.
std::shared_ptr<StatusPy> dense_block() {
  DeviceStatus* d = dense_status();
  TORCH_CHECK(d != nullptr, "linear: no status block on this device");
  return std::make_shared<StatusPy>(d);
}

}  // namespace

void bind_dense(py::module_& m) {
  m.def("add_rms_norm", &add_rms_norm, py::arg("x"), py::arg("weight"), py::arg("eps"), py::arg("residual"), py::arg("quantise"));
  m.def("balance_loss", &balance_loss, py::arg("logits"), py::arg("topk_idx"), py::arg("mask"), py::arg("sigmoid"));
  m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("residual"), py::arg("kind"), py::arg("timeout_s"));
  m.def("dense_status", &dense_block);
  // Which way a product of a linear layer goes: whether the kernel for few tokens has it, and otherwise the most tokens of a tile, how many tiles are cut along the reduction, into how many
  // parts or shares, and whether as a stream.
  m.def("dense_path", [](int tokens, int64_t features, int64_t reduction, bool swiglu, bool plain, bool sectors, int sms) {
    const int ctas = sms & ~1;
    const bool few = few_pays(tokens, static_cast<int>(swiglu ? features / 2 : features), static_cast<int>((reduction + 63) / 64), swiglu, sectors, sms);
    py::dict d;
    d["few"] = few;
    if (few) return d;
    const TokDenseArgs a = dense_args(tokens, features, reduction, plain && !swiglu, ctas);
    const gemm::TokSplit s = dense_split(a, ctas);
    d["tile"] = a.tile_n; d["cut_tiles"] = s.cut_tiles; d["shares"] = s.shares; d["stream"] = s.stream;
    return d;
  }, py::arg("tokens"), py::arg("features"), py::arg("reduction"), py::arg("swiglu"), py::arg("plain"), py::arg("sectors"), py::arg("sms") = 148);
  m.def("dequantise_rows", &dequantise_rows, py::arg("q"), py::arg("scales"));
}
