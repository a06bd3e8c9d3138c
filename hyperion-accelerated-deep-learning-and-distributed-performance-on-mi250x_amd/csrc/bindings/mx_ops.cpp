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

const float* bias_ptr(const c10::optional<at::Tensor>& bias, int64_t n, const at::Device& dev, const char* who) {
  if (!bias.has_value() || !bias->defined()) return nullptr;
  TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->numel() == n && bias->device() == dev &&
                  reinterpret_cast<uintptr_t>(bias->data_ptr()) % 16 == 0,
              who, ": bias must be a contiguous, 16-byte aligned fp32 [", n, "]");
  return bias->data_ptr<float>();
}

// x [M, n] (unit stride in n) as bf16 pieces [P M, pitch] whose sum it is, zeros behind n; x itself where it is that
at::Tensor pieces(const at::Tensor& x, int64_t pitch) {
  if (x.scalar_type() == at::kBFloat16 && x.size(1) == pitch && x.is_contiguous() &&
      reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0)
    return x;
  auto out = at::empty({pieces_of(x.scalar_type()) * x.size(0), pitch}, x.options().dtype(at::kBFloat16));
  HYP_CHECK_HIP(hyp::mx_pieces(dtype_code(x), x.data_ptr(), x.stride(0), x.size(0), (int)x.size(1), (int)pitch,
                               out.data_ptr(), cur_stream()));
  return out;
}

// sum over the pieces of part [P M, pitch] (fp32), columns [0, cols), + bias -> [M, cols] in dtype
at::Tensor join(const at::Tensor& part, int64_t M, int64_t cols, const float* bias, at::ScalarType dtype) {
  auto y = at::empty({M, cols}, part.options().dtype(dtype));
  HYP_CHECK_HIP(hyp::mx_join(dtype_code(dtype), part.data_ptr<float>(), (int)(part.size(0) / M), M, (int)cols, part.size(1),
                             bias, y.data_ptr(), cur_stream()));
  return y;
}

// a [R, K] (bf16 rows of stride lda) times the decoded weight wd on the tiled GEMM: b_tr = false: a wdᵀ (wd [N, K]),
// n_out >= N columns (zeros behind N); b_tr = true: a wd (wd [K, N])
at::Tensor tiled(const at::Tensor& a, int64_t K, const at::Tensor& wd, bool b_tr, int64_t n_out, const float* bias,
                 at::ScalarType dtype) {
  auto y = at::empty({a.size(0), n_out}, a.options().dtype(dtype));
  hyp::GemmTiledArgs g;
  g.in_dtype = hyp::kBF16;
  g.out_dtype = dtype_code(dtype);
  g.A = a.data_ptr();
  g.B = wd.data_ptr();
  g.C = y.data_ptr();
  g.M = (int)a.size(0);
  g.N = (int)n_out;
  g.K = (int)K;
  g.lda = (int)a.size(1);
  g.ldb = (int)wd.size(1);
  g.ldc = (int)n_out;
  g.a_tr = false;
  g.b_tr = b_tr;
  g.alpha = 1.f;
  g.b_rows = b_tr ? (int)n_out : (int)wd.size(0);
  g.zero = device_zero_page(a.device());
  if (bias) {
    g.bias = bias;
    g.bias_dtype = hyp::kF32;
  }
  hyp::mx_gemm_plan(g.M, g.N, g.K, &g.tile, &g.splits);
  const int sp = hyp::gemm_tiled_splits(g);
  at::Tensor part;
  if (sp > 1) {
    part = at::empty({(int64_t)sp * g.M * g.N}, a.options().dtype(at::kFloat));
    g.part = part.data_ptr<float>();
  }
  HYP_CHECK_HIP(hyp::gemm_tiled(g, cur_stream()));
  return y;
}

void check_rows(const at::Tensor& x, const at::Tensor& codes, int64_t n, const char* who) {
  HYP_CHECK_CUDA_TENSOR(x);
  TORCH_CHECK(x.dim() == 2 && x.size(1) == n && (x.stride(1) == 1 || n == 1) && x.device() == codes.device() &&
                  x.size(0) >= 1 && x.size(0) < (1 << 24) && codes.size(0) >= 1 && codes.size(0) < (1 << 24) && n >= 1 && n < (1 << 24),
              who, ": x [M, ", n, "] with unit column stride on the weight's device, all sizes in [1, 2^24)");
}

bool lds_ok(const at::Tensor& scales) {
  return scales.size(1) % 4 == 0 && reinterpret_cast<uintptr_t>(scales.data_ptr()) % 4 == 0;
}

at::Tensor decoded(const at::Tensor& codes, const at::Tensor& scales) {
  return mx_dequantize(codes, scales, scales.size(1) * 32, at::kBFloat16);
}

// x [M, K] times the transpose of the 4-bit weight [N, K] (+ fp32 bias) -> [M, N] in x's dtype.
// tile (A/B): -1 planned, 0 the decoded GEMM, 16 mt + nt the one-launch product
at::Tensor mx_linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                     const c10::optional<at::Tensor>& bias, int64_t tile) {
  check_mx(codes, scales, x.size(-1), "mx_linear");
  check_rows(x, codes, x.size(-1), "mx_linear");
  const at::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), N = codes.size(0), nb = scales.size(1), P = pieces_of(x.scalar_type());
  const float* b = bias_ptr(bias, N, x.device(), "mx_linear");
  const at::Tensor xp = pieces(x, 32 * nb);
  const auto dt = P == 1 ? at::kBFloat16 : at::kFloat;
  int mt, nt;
  hyp::mx_nt_plan((int)M, (int)N, (int)nb, (int)P, lds_ok(scales), &mt, &nt);
  if (tile >= 0) mt = (int)tile / 16, nt = (int)tile % 16;
  at::Tensor y;
  if (mt > hyp::kMxBig) {
    y = at::empty({M, N}, x.options());
    HYP_CHECK_HIP(hyp::mx_nt(xp.data_ptr(), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), (int)M, (int)N, (int)nb, b,
                             dtype_code(y), y.data_ptr(), cur_stream(), mt, nt, (int)P));
    return y;
  }
  if (mt > 0) {
    y = at::empty({P * M, N}, xp.options().dtype(dt));
    HYP_CHECK_HIP(hyp::mx_nt(xp.data_ptr(), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), (int)(P * M), (int)N,
                             (int)nb, P == 1 ? b : nullptr, dtype_code(dt), y.data_ptr(), cur_stream(), mt, nt, 1));
  } else {
    const int64_t Np = (N + 7) / 8 * 8;
    const bool direct = P == 1 && (b == nullptr || Np == N);  // the epilogue's bias has as many elements as columns
    y = tiled(xp, 32 * nb, decoded(codes, scales), false, Np, direct ? b : nullptr, direct ? at::kBFloat16 : at::kFloat);
    if (direct) return Np == N ? y : y.narrow(1, 0, N).contiguous();
  }
  return P == 1 && mt > 0 ? y : join(y, M, N, b, x.scalar_type());
}

// dy [M, N] times the 4-bit weight [N, K] -> [M, K] in dy's dtype.  tile (A/B): -1 planned, 0 the decoded GEMM, mt
at::Tensor mx_linear_dgrad(const at::Tensor& dy, const at::Tensor& codes, const at::Tensor& scales, int64_t K,
                           int64_t tile) {
  check_mx(codes, scales, K, "mx_linear_dgrad");
  check_rows(dy, codes, codes.size(0), "mx_linear_dgrad");
  TORCH_CHECK(K >= 1 && K < (1 << 24), "mx_linear_dgrad: K in [1, 2^24)");
  const at::DeviceGuard guard(dy.device());
  const int64_t M = dy.size(0), N = codes.size(0), nb = scales.size(1), P = pieces_of(dy.scalar_type());
  const auto dt = P == 1 ? at::kBFloat16 : at::kFloat;
  int mt;
  hyp::mx_nn_plan((int)M, (int)N, (int)nb, (int)P, lds_ok(scales), &mt);
  if (tile >= 0) mt = (int)tile;
  const int64_t unit = mt > hyp::kMxLds ? 128 : 8;  // the product through LDS takes whole groups of the reduction
  const at::Tensor dp = pieces(dy, (N + unit - 1) / unit * unit);
  at::Tensor dx;
  if (mt > hyp::kMxBig) {
    dx = at::empty({M, K}, dy.options());
    HYP_CHECK_HIP(hyp::mx_nn(dp.data_ptr(), dp.size(1), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), (int)M, (int)N,
                             (int)nb, (int)K, dtype_code(dx), dx.data_ptr(), cur_stream(), mt, (int)P));
    return dx;
  }
  if (mt > 0) {
    dx = at::empty({P * M, K}, dp.options().dtype(dt));
    HYP_CHECK_HIP(hyp::mx_nn(dp.data_ptr(), dp.size(1), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), (int)(P * M),
                             (int)N, (int)nb, (int)K, dtype_code(dt), dx.data_ptr(), cur_stream(), mt, 1));
  } else {
    dx = tiled(dp, N, decoded(codes, scales), true, 32 * nb, nullptr, dt);
    if (P == 1) return 32 * nb == K ? dx : dx.narrow(1, 0, K).contiguous();
  }
  return P == 1 ? dx : join(dx, M, K, nullptr, dy.scalar_type());
}

// the variant that mx_linear (x [M, K], weight [N, K], rows of whole groups of four blocks) or mx_linear_dgrad plans, as
// their `tile`, and the tiled GEMM's (tile, splits) where it is 0
std::tuple<int64_t, int64_t, int64_t> mx_plan(int64_t M, int64_t N, int64_t K, int64_t pieces, bool dgrad) {
  TORCH_CHECK(M >= 1 && N >= 1 && K >= 1 && M < (1 << 24) && N < (1 << 24) && K < (1 << 24) && pieces >= 1 && pieces <= 3,
              "mx_plan: sizes in [1, 2^24), 1 to 3 pieces");
  const int nb = (int)((K + 31) / 32);
  int mt = 0, nt = 0, tile, splits;
  if (dgrad) hyp::mx_nn_plan((int)M, (int)N, nb, (int)pieces, nb % 4 == 0, &mt);
  else hyp::mx_nt_plan((int)M, (int)N, nb, (int)pieces, nb % 4 == 0, &mt, &nt);
  hyp::mx_gemm_plan((int)(pieces * M), dgrad ? 32 * nb : (int)N, dgrad ? (int)N : 32 * nb, &tile, &splits);
  return {dgrad ? mt : 16 * mt + nt, tile, splits};
}

}  // namespace

void register_mx_ops(pybind11::module& m) {
  m.def("mx_quantize", &mx_quantize, "rows -> microscaled 4-bit (codes, scales)", pybind11::arg("x"));
  m.def("mx_dequantize", &mx_dequantize, "microscaled 4-bit rows -> values", pybind11::arg("codes"),
        pybind11::arg("scales"), pybind11::arg("cols"), pybind11::arg("dtype"));
  m.def("mx_linear", &mx_linear, "x times the transposed 4-bit weight (+ bias)", pybind11::arg("x"), pybind11::arg("codes"),
        pybind11::arg("scales"), pybind11::arg("bias") = pybind11::none(), pybind11::arg("tile") = -1);
  m.def("mx_plan", &mx_plan, "the planned variant of a product, and the tiled GEMM's tile and splits", pybind11::arg("M"),
        pybind11::arg("N"), pybind11::arg("K"), pybind11::arg("pieces") = 1, pybind11::arg("dgrad") = false);
  m.def("mx_linear_dgrad", &mx_linear_dgrad, "dy times the 4-bit weight", pybind11::arg("dy"), pybind11::arg("codes"),
        pybind11::arg("scales"), pybind11::arg("K"), pybind11::arg("tile") = -1);
}

}  // namespace hypbind
