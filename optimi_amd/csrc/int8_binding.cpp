// PyTorch-ROCm binding of the int8 activation operators of optimi_hip.h: checks that tensors are what the kernels
// assume, makes them contiguous, allocates outputs and workspaces from PyTorch's allocator on the calling thread's
// current stream, and raises RuntimeError when the library returns a non-zero status.

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>

#include "optimi_hip.h"

namespace {

using at::Tensor;

void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed: ", optimi_hip_error_string(rc), " (status ", rc, ")");
}

int dtype_code(at::ScalarType type, const char* name) {
  switch (type) {
    case at::kFloat: return OPTIMI_F32;
    case at::kBFloat16: return OPTIMI_BF16;
    case at::kHalf: return OPTIMI_F16;
    default: TORCH_CHECK(false, "optimi_amd: unsupported dtype ", type, " of ", name, " (float32, bfloat16 and float16 are implemented)");
  }
  return -1;
}

void check_device(const Tensor& first, const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "optimi_amd: ", name, " must live on a HIP device, got ", t.device());
  TORCH_CHECK(t.layout() == at::kStrided, "optimi_amd: ", name, " must be a dense tensor");
  TORCH_CHECK(t.device() == first.device(), "optimi_amd: ", name, " is on ", t.device(), ", expected ", first.device());
}

// The trailing dimension is the row, all others count rows.
struct Rows {
  int64_t rows, cols;
};
Rows rows_of(const Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() >= 1, "optimi_amd: ", name, " must have at least one dimension");
  Rows r{1, t.size(-1)};
  for (int64_t d = 0; d + 1 < t.dim(); ++d) r.rows *= t.size(d);
  return r;
}
at::DimVector leading(const Tensor& t) { return at::DimVector(t.sizes().begin(), t.sizes().end() - 1); }
at::DimVector with_cols(const Tensor& t, int64_t cols) {
  at::DimVector sizes = leading(t);
  sizes.push_back(cols);
  return sizes;
}

// The calls are short, and on small inputs the host's part of them is what counts: tensors are made by the allocator's own
// function instead of through the dispatcher, and a contiguous one is taken as it is, unless it carries the lazy negative bit: then
// what lies in memory has the opposite sign.
Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor dense(const Tensor& t) {
  if (t.is_neg()) return t.resolve_neg().contiguous();
  return t.is_contiguous() ? t : t.contiguous();
}

// values [..., cols] with one scale per row
Tensor check_pair(const Tensor& values, const Tensor& scales, const char* name) {
  TORCH_CHECK(values.scalar_type() == at::kChar, "optimi_amd: ", name, " must hold int8 values, got ", values.scalar_type());
  TORCH_CHECK(scales.scalar_type() == at::kFloat, "optimi_amd: the scales of ", name, " must be float32, got ", scales.scalar_type());
  TORCH_CHECK(values.dim() >= 1 && scales.sizes() == values.sizes().slice(0, values.dim() - 1), "optimi_amd: ", name, " of size ", values.sizes(),
              " needs scales of size ", values.sizes().slice(0, values.dim() - 1), ", got ", scales.sizes());
  return dense(scales);
}

hipStream_t current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

Tensor workspace(int64_t bytes, const Tensor& like, const char* what) {
  if (bytes < 0) check_status((int)bytes, what);
  return bytes ? make({bytes}, at::kByte, like) : Tensor();
}
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

std::tuple<Tensor, Tensor> int8_quantize(const Tensor& x_) {
  check_device(x_, x_, "the activation");
  const int dtype = dtype_code(x_.scalar_type(), "the activation");
  const Rows r = rows_of(x_, "the activation");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x_.device());
  const Tensor x = dense(x_);
  Tensor values = make(x.sizes(), at::kChar, x);
  Tensor scales = make(leading(x), at::kFloat, x);
  check_status(optimi_hip_int8_quantize(x.data_ptr(), r.rows, r.cols, dtype, (int8_t*)values.data_ptr(), (float*)scales.data_ptr(), current_stream()),
               "optimi_hip_int8_quantize");
  return {values, scales};
}

Tensor int8_dequantize(const Tensor& values_, const Tensor& scales_, at::ScalarType type) {
  check_device(values_, values_, "values");
  check_device(values_, scales_, "scales");
  const int dtype = dtype_code(type, "the result");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(values_.device());
  const Tensor scales = check_pair(values_, scales_, "values");
  const Rows r = rows_of(values_, "values");
  const Tensor values = dense(values_);
  Tensor out = make(values.sizes(), type, values);
  check_status(optimi_hip_int8_dequantize((const int8_t*)values.data_ptr(), (const float*)scales.data_ptr(), r.rows, r.cols, dtype, out.data_ptr(),
                                          current_stream()),
               "optimi_hip_int8_dequantize");
  return out;
}

Tensor int8_matmul(const Tensor& a_, const Tensor& a_scales_, const Tensor& b_, const Tensor& b_scales_, const std::optional<Tensor>& bias_,
                   at::ScalarType type) {
  check_device(a_, a_, "the activation");
  check_device(a_, a_scales_, "the activation's scales");
  check_device(a_, b_, "the weight");
  check_device(a_, b_scales_, "the weight's scales");
  const int dtype = dtype_code(type, "the result");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a_.device());
  const Tensor a_scales = check_pair(a_, a_scales_, "the activation"), b_scales = check_pair(b_, b_scales_, "the weight");
  const Rows r = rows_of(a_, "the activation");
  TORCH_CHECK(b_.dim() == 2, "optimi_amd: the weight must be a matrix [outputs, inputs], got ", b_.dim(), " dimensions");
  TORCH_CHECK(b_.size(1) == r.cols, "optimi_amd: the weight has ", b_.size(1), " inputs, the activation ", r.cols, " columns");
  const int64_t n = b_.size(0);
  Tensor bias;
  if (bias_.has_value()) {
    check_device(a_, *bias_, "the bias");
    TORCH_CHECK(bias_->scalar_type() == type, "optimi_amd: the bias has dtype ", bias_->scalar_type(), ", the result ", type);
    TORCH_CHECK(bias_->dim() == 1 && bias_->size(0) == n, "optimi_amd: the bias must have ", n, " elements, got size ", bias_->sizes());
    bias = dense(*bias_);
  }
  const Tensor a = dense(a_), b = dense(b_);
  Tensor out = make(with_cols(a, n), type, a);
  const Tensor work = workspace(optimi_hip_int8_matmul_workspace(r.rows, n, r.cols), a, "optimi_hip_int8_matmul");
  check_status(optimi_hip_int8_matmul((const int8_t*)a.data_ptr(), (const float*)a_scales.data_ptr(), (const int8_t*)b.data_ptr(),
                                      (const float*)b_scales.data_ptr(), pointer(bias), r.rows, n, r.cols, dtype, out.data_ptr(), pointer(work),
                                      current_stream()),
               "optimi_hip_int8_matmul");
  return out;
}

std::tuple<Tensor, std::optional<Tensor>> int8_weight_grad(const Tensor& grad_, const Tensor& values_, const Tensor& scales_, bool with_bias) {
  check_device(grad_, grad_, "the gradient");
  check_device(grad_, values_, "the checkpoint's values");
  check_device(grad_, scales_, "the checkpoint's scales");
  const int dtype = dtype_code(grad_.scalar_type(), "the gradient");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(grad_.device());
  const Tensor scales = check_pair(values_, scales_, "the checkpoint");
  const Rows g = rows_of(grad_, "the gradient"), v = rows_of(values_, "the checkpoint");
  TORCH_CHECK(leading(grad_) == leading(values_), "optimi_amd: the gradient of size ", grad_.sizes(), " and the checkpoint of size ", values_.sizes(),
              " have different rows");
  const Tensor grad = dense(grad_), values = dense(values_);
  Tensor dw = make({g.cols, v.cols}, grad.scalar_type(), grad);
  std::optional<Tensor> db;
  if (with_bias) db = make({g.cols}, grad.scalar_type(), grad);
  const Tensor work = workspace(optimi_hip_int8_weight_grad_workspace(g.rows, g.cols, v.cols, dtype, with_bias), grad, "optimi_hip_int8_weight_grad");
  check_status(optimi_hip_int8_weight_grad(grad.data_ptr(), (const int8_t*)values.data_ptr(), (const float*)scales.data_ptr(), g.rows, g.cols, v.cols,
                                           dtype, dw.data_ptr(), db ? db->data_ptr() : nullptr, pointer(work), current_stream()),
               "optimi_hip_int8_weight_grad");
  return {dw, db};
}

// the column sums of grad, which need no checkpoint
Tensor int8_bias_grad(const Tensor& grad_) {
  check_device(grad_, grad_, "the gradient");
  const int dtype = dtype_code(grad_.scalar_type(), "the gradient");
  const Rows g = rows_of(grad_, "the gradient");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(grad_.device());
  const Tensor grad = dense(grad_);
  Tensor db = make({g.cols}, grad.scalar_type(), grad);
  const Tensor work = workspace(optimi_hip_int8_weight_grad_workspace(g.rows, g.cols, 0, dtype, 1), grad, "optimi_hip_int8_weight_grad");
  check_status(optimi_hip_int8_weight_grad(grad.data_ptr(), nullptr, nullptr, g.rows, g.cols, 0, dtype, nullptr, db.data_ptr(), pointer(work), current_stream()),
               "optimi_hip_int8_weight_grad");
  return db;
}

int norm_weight_code(const Tensor& weight, const Tensor& x, int64_t cols) {
  check_device(x, weight, "the norm's weight");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "optimi_amd: the norm's weight has dtype ",
              weight.scalar_type(), ": expected ", x.scalar_type(), " or float32");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == cols, "optimi_amd: the norm's weight must have ", cols, " elements, got size ", weight.sizes());
  return dtype_code(weight.scalar_type(), "the norm's weight");
}

void check_twin(const Tensor& x, const Tensor& t, const char* name) {
  check_device(x, t, name);
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), "optimi_amd: ", name, " has dtype ", t.scalar_type(), ", expected ", x.scalar_type());
  TORCH_CHECK(t.sizes() == x.sizes(), "optimi_amd: ", name, " has size ", t.sizes(), ", expected ", x.sizes());
}

// values, scales, h, 1/rms; h is x itself where there is no residual
std::tuple<Tensor, Tensor, Tensor, Tensor> add_rms_norm_int8(const Tensor& x_, const Tensor& weight_, const std::optional<Tensor>& residual_, double eps) {
  check_device(x_, x_, "the activation");
  const int dtype = dtype_code(x_.scalar_type(), "the activation");
  const Rows r = rows_of(x_, "the activation");
  const int weight_dtype = norm_weight_code(weight_, x_, r.cols);
  Tensor residual;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x_.device());
  if (residual_.has_value()) {
    check_twin(x_, *residual_, "the residual");
    residual = dense(*residual_);
  }
  const Tensor x = dense(x_), weight = dense(weight_);
  Tensor values = make(x.sizes(), at::kChar, x);
  Tensor scales = make(leading(x), at::kFloat, x), rstd = make(leading(x), at::kFloat, x);
  Tensor h = residual.defined() ? make(x.sizes(), x.scalar_type(), x) : Tensor();
  check_status(optimi_hip_add_rms_norm_int8(x.data_ptr(), pointer(residual), weight.data_ptr(), r.rows, r.cols, dtype, weight_dtype, eps, pointer(h),
                                            (int8_t*)values.data_ptr(), (float*)scales.data_ptr(), (float*)rstd.data_ptr(), current_stream()),
               "optimi_hip_add_rms_norm_int8");
  return {values, scales, h.defined() ? h : x_, rstd};
}

std::tuple<Tensor, Tensor> add_rms_norm_int8_backward(const Tensor& grad_, const Tensor& h_, const Tensor& rstd_, const Tensor& weight_,
                                                      const std::optional<Tensor>& grad_h_) {
  check_device(grad_, grad_, "the gradient");
  const int dtype = dtype_code(grad_.scalar_type(), "the gradient");
  const Rows r = rows_of(grad_, "the gradient");
  check_twin(grad_, h_, "h");
  check_device(grad_, rstd_, "rstd");
  TORCH_CHECK(rstd_.scalar_type() == at::kFloat && rstd_.sizes() == grad_.sizes().slice(0, grad_.dim() - 1), "optimi_amd: rstd must be float32 of size ",
              grad_.sizes().slice(0, grad_.dim() - 1), ", got ", rstd_.scalar_type(), " of size ", rstd_.sizes());
  const int weight_dtype = norm_weight_code(weight_, grad_, r.cols);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(grad_.device());
  Tensor grad_h;
  if (grad_h_.has_value()) {
    check_twin(grad_, *grad_h_, "the gradient of h");
    grad_h = dense(*grad_h_);
  }
  const Tensor grad = dense(grad_), h = dense(h_), rstd = dense(rstd_), weight = dense(weight_);
  Tensor dx = make(grad.sizes(), grad.scalar_type(), grad), dweight = make({r.cols}, weight.scalar_type(), weight);
  const Tensor work = workspace(optimi_hip_add_rms_norm_int8_backward_workspace(r.rows, r.cols), grad, "optimi_hip_add_rms_norm_int8_backward");
  check_status(optimi_hip_add_rms_norm_int8_backward(grad.data_ptr(), pointer(grad_h), h.data_ptr(), (const float*)rstd.data_ptr(), weight.data_ptr(),
                                                     r.rows, r.cols, dtype, weight_dtype, dx.data_ptr(), dweight.data_ptr(), pointer(work),
                                                     current_stream()),
               "optimi_hip_add_rms_norm_int8_backward");
  return {dx, dweight};
}

}  // namespace

void bind_int8(py::module& mod) {
  mod.def("int8_quantize", &int8_quantize);
  mod.def("int8_dequantize", &int8_dequantize);
  mod.def("int8_matmul", &int8_matmul);
  mod.def("int8_weight_grad", &int8_weight_grad);
  mod.def("int8_bias_grad", &int8_bias_grad);
  mod.def("add_rms_norm_int8", &add_rms_norm_int8);
  mod.def("add_rms_norm_int8_backward", &add_rms_norm_int8_backward);
}
