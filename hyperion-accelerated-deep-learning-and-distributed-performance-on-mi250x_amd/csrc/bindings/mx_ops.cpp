// Torch bindings: microscaled 4-bit floating point (kernels/mxfp4.hip).
#include "bindings/common.h"
#include "bindings/registry.h"

namespace hypbind {
namespace {

// codes [R, 16 nb], scales [R, nb] of rows of `cols` elements
void check_mx(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, const char* who) {
  HYP_CHECK_CUDA_TENSOR(codes);
  const int64_t nb = (cols + 31) / 32;
  TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte && codes.dim() == 2 && scales.dim() == 2 &&
                  codes.is_contiguous() && scales.is_contiguous() && codes.size(0) == scales.size(0) &&
                  scales.size(1) == nb && codes.size(1) == 16 * nb && scales.device() == codes.device() &&
                  reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0,
              who, ": contiguous uint8 codes [R, 16 nb] (16-byte aligned) and scales [R, nb] of one device, nb = ceil(", cols, " / 32)");
}

std::vector<at::Tensor> mx_quantize(const at::Tensor& x) {
  HYP_CHECK_CUDA_TENSOR(x);
  TORCH_CHECK(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1) && x.size(1) < (int64_t)INT32_MAX - 32,
              "mx_quantize: x [R, K] with unit stride in K");
  const int64_t nb = (x.size(1) + 31) / 32;
  TORCH_CHECK(x.size(0) * nb < hyp::kMxGridMax * 64, "mx_quantize: x is too large for one launch");
  const at::DeviceGuard guard(x.device());
  auto opt = x.options().dtype(at::kByte);
  auto codes = at::empty({x.size(0), 16 * nb}, opt), scales = at::empty({x.size(0), nb}, opt);
  HYP_CHECK_HIP(hyp::mx_quantize(dtype_code(x), x.data_ptr(), x.stride(0), x.size(0), (int)x.size(1),
                                 codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), cur_stream()));
  return {codes, scales};
}

// [R, cols] values; cols may be the whole blocks' 32 nb (zeros behind the row's own length)
at::Tensor mx_dequantize(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, at::ScalarType dtype) {
  check_mx(codes, scales, cols, "mx_dequantize");
  TORCH_CHECK(codes.size(0) * scales.size(1) < hyp::kMxGridMax * 64, "mx_dequantize: too large for one launch");
  const at::DeviceGuard guard(codes.device());
  auto out = at::empty({codes.size(0), cols}, codes.options().dtype(dtype));
  HYP_CHECK_HIP(hyp::mx_dequantize(dtype_code(dtype), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                                   codes.size(0), (int)cols, out.data_ptr(), cols, cur_stream()));
  return out;
}

int pieces_of(at::ScalarType t) { return t == at::kBFloat16 ? 1 : (t == at::kHalf ? 2 : 3); }

// x [R, K] (unit stride in K) as bf16 pieces [P R, pitch], zeros behind K
at::Tensor mx_pieces(const at::Tensor& x, int64_t pitch) {
  HYP_CHECK_CUDA_TENSOR(x);
  TORCH_CHECK(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1) && pitch % 8 == 0 && pitch >= x.size(1) &&
                  pitch < (int64_t)INT32_MAX, "mx_pieces: x [R, K] with unit stride in K, pitch >= K a multiple of 8");
  const at::DeviceGuard guard(x.device());
  const int P = pieces_of(x.scalar_type());
  auto out = at::empty({P * x.size(0), pitch}, x.options().dtype(at::kBFloat16));
  HYP_CHECK_HIP(hyp::mx_pieces(dtype_code(x), x.data_ptr(), x.stride(0), x.size(0), (int)x.size(1), (int)pitch,
                               out.data_ptr(), cur_stream()));
  return out;
}

const float* bias_ptr(const c10::optional<at::Tensor>& bias, int64_t n, const at::Device& dev, const char* who) {
  if (!bias.has_value() || !bias->defined()) return nullptr;
  TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->numel() == n && bias->device() == dev,
              who, ": bias must be a contiguous fp32 [", n, "]");
  return bias->data_ptr<float>();
}

// sum over the pieces of part [P R, pitch] (fp32), columns [0, cols), + bias -> [R, cols] in dtype
at::Tensor mx_join(const at::Tensor& part, int64_t rows, int64_t cols, const c10::optional<at::Tensor>& bias,
                   at::ScalarType dtype) {
  HYP_CHECK_CUDA_TENSOR(part);
  TORCH_CHECK(part.scalar_type() == at::kFloat && part.dim() == 2 && part.is_contiguous() && part.size(1) >= cols &&
                  rows > 0 && part.size(0) % rows == 0, "mx_join: contiguous fp32 part [P * rows, >= cols]");
  const at::DeviceGuard guard(part.device());
  auto y = at::empty({rows, cols}, part.options().dtype(dtype));
  HYP_CHECK_HIP(hyp::mx_join(dtype_code(dtype), part.data_ptr<float>(), (int)(part.size(0) / rows), rows, (int)cols,
                             part.size(1), bias_ptr(bias, cols, part.device(), "mx_join"), y.data_ptr(), cur_stream()));
  return y;
}

// x [M, 32 nb] bf16 contiguous times the weight's transpose -> [M, N] (bf16 or fp32)
at::Tensor mx_rows(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                   const c10::optional<at::Tensor>& bias, at::ScalarType dtype) {
  HYP_CHECK_CUDA_TENSOR(x);
  check_mx(codes, scales, x.size(-1), "mx_rows");
  const int64_t M = x.size(0), N = codes.size(0), nb = scales.size(1);
  TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kBFloat16 && x.is_contiguous() && x.size(1) == 32 * nb &&
                  x.device() == codes.device() && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
                  M <= 65535 * 16 && N < (int64_t)INT32_MAX - 16,
              "mx_rows: contiguous, 16-byte aligned bf16 x [M, 32 nb] on the weight's device");
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kFloat, "mx_rows: bf16 or fp32 output");
  const at::DeviceGuard guard(x.device());
  auto y = at::empty({M, N}, x.options().dtype(dtype));
  HYP_CHECK_HIP(hyp::mx_rows(x.data_ptr(), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), (int)M, (int)N, (int)nb,
                             bias_ptr(bias, N, x.device(), "mx_rows"), dtype_code(dtype), y.data_ptr(), cur_stream()));
  return y;
}

}  // namespace

void register_mx_ops(pybind11::module& m) {
  m.def("mx_quantize", &mx_quantize, "rows -> microscaled 4-bit (codes, scales)", pybind11::arg("x"));
  m.def("mx_dequantize", &mx_dequantize, "microscaled 4-bit rows -> values", pybind11::arg("codes"),
        pybind11::arg("scales"), pybind11::arg("cols"), pybind11::arg("dtype"));
  m.def("mx_pieces", &mx_pieces, "activations as exact bf16 pieces [P R, pitch]", pybind11::arg("x"), pybind11::arg("pitch"));
  m.def("mx_join", &mx_join, "sum of fp32 piece products (+ bias) in the output dtype", pybind11::arg("part"),
        pybind11::arg("rows"), pybind11::arg("cols"), pybind11::arg("bias"), pybind11::arg("dtype"));
  m.def("mx_rows", &mx_rows, "few rows x 4-bit weight (one launch)", pybind11::arg("x"), pybind11::arg("codes"),
        pybind11::arg("scales"), pybind11::arg("bias"), pybind11::arg("dtype"));
}

}  // namespace hypbind
