// Bindings of the dense side of a block: row norm, balance loss, linear layers. Their kernels run on the current stream of the
// tensors' own device, whichever device is current.
#include <c10/cuda/CUDAGuard.h>

#include "py_types.h"

namespace py = pybind11;
using namespace fastb;
using namespace fastb_py;

namespace {

using OptTensor = c10::optional<torch::Tensor>;

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

// (y, h, q, scales, rstd): h is undefined without residual, q and scales without quantise, rstd without keep.
std::tuple<torch::Tensor, OptTensor, OptTensor, OptTensor, OptTensor> row_norm(const torch::Tensor& x, const torch::Tensor& weight, double eps, const OptTensor& residual, bool quantise, bool keep) {
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
  OptTensor h, q, scales, rstd;
  a.y = y.data_ptr();
  if (residual.has_value()) {
    rm = as_rows(*residual, H);
    a.residual = rm.data_ptr(); a.residual_stride = rm.stride(0);
    h = torch::empty(x.sizes(), x.options());
    a.h = h->data_ptr();
  }
  if (quantise) {
    q = torch::empty(x.sizes(), x.options().dtype(torch::kUInt8));
    auto shape = x.sizes().vec();
    shape.back() = H / 128;
    scales = torch::empty(shape, x.options().dtype(torch::kFloat32));
    a.q = q->data_ptr<uint8_t>(); a.scales = scales->data_ptr<float>();
  }
  if (keep) {
    rstd = torch::empty({xm.size(0)}, x.options().dtype(torch::kFloat32));
    a.rstd = rstd->data_ptr<float>();
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

}  // namespace

void bind_dense(py::module_& m) {
  m.def("row_norm", &row_norm, py::arg("x"), py::arg("weight"), py::arg("eps"), py::arg("residual"), py::arg("quantise"), py::arg("keep"));
  m.def("row_norm_bwd", &row_norm_bwd, py::arg("h"), py::arg("weight"), py::arg("rstd"), py::arg("dy"), py::arg("dh"));
  m.def("dequantise_rows", &dequantise_rows, py::arg("q"), py::arg("scales"));
}
