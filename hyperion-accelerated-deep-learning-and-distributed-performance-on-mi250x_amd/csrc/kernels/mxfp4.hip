// Microscaled 4-bit floating point: quantisation, its inverse, and the product of a few rows with a
// 4-bit weight.
//
// Format: 32 consecutive elements of a row share the scale 2^e, kept as the byte e + 127; an element is
// a sign and one of the magnitudes 0 .5 1 1.5 2 3 4 6 (e2m1) in 4 bits, two in a byte, the first in
// the low half.  e = floor(log2(max |x|)) - 2, at least -127; magnitudes are rounded to the nearest
// (ties to the even code) and saturate at 6.  Scale byte 255 is NaN: a block with a NaN or an
// infinity.  A row holds whole blocks, the last one padded with zeros.
//
// gfx950 converts both ways with the scale applied (v_cvt_scalef32_pk_*): two elements an
// instruction, rounding and saturating as above, exact for all 256 scale bytes (0 and 255 among them).
#include "hyp_common.h"
#include "hyp_kernels.h"
#include "mfma_lds.h"

namespace hyp {
namespace {

using mfl::f32x4;
using mfl::u16x8;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4a __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kMxBlock = 32;

__device__ __forceinline__ float mx_scale(unsigned byte) { return __uint_as_float(byte << 23); }

// ---- quantisation ---------------------------------------------------------------------------------
// eight consecutive elements at p, `left` of them inside the row (zeros behind it)
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
  if (left >= 8) {
    if (sizeof(T) == 4) {
      const u32x4a a = reinterpret_cast<const u32x4a*>(p)[0], b = reinterpret_cast<const u32x4a*>(p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = __uint_as_float(a[i]);
        v[4 + i] = __uint_as_float(b[i]);
      }
    } else {
      const u32x4a a = reinterpret_cast<const u32x4a*>(p)[0];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = sizeof(T) == 2 && __is_same(T, bf16_t) ? __uint_as_float(a[i] << 16) : f16_lo(a[i]);
        v[2 * i + 1] = sizeof(T) == 2 && __is_same(T, bf16_t) ? __uint_as_float(a[i] & 0xffff0000u) : f16_hi(a[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? ld1<T>(p + i) : 0.f;
  }
}

constexpr int kQThreads = 256;

// Four lanes a block, eight elements a lane: one 16-byte load, the maximum over the four by two lane
// exchanges, one 4-byte store of codes.  HBM-bound (2 or 4 bytes in, 17/32 out per element).
template <typename T>
__global__ __launch_bounds__(kQThreads) void mx_quantize_k(const T* __restrict__ x, int64_t ld, int cols, int nb,
                                                           int64_t total, uint32_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * kQThreads + threadIdx.x;  // lane group (row, block), lane quarter
  const int64_t bi = i >> 2;
  const int quarter = (int)(i & 3);
  if (bi >= total) return;  // whole groups of four lanes
  const int64_t row = bi / nb;
  const int c0 = (int)(bi - row * nb) * kMxBlock + quarter * 8;
  float v[8];
  load8<T>(x + row * ld + c0, cols - c0, v);
  unsigned top = 0;  // the largest magnitude, in the order of the bits: a NaN or an infinity is above all numbers
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  top = max(top, (unsigned)__shfl_xor((int)top, 1, 4));
  top = max(top, (unsigned)__shfl_xor((int)top, 2, 4));
  const unsigned e = top >> 23;
  const unsigned byte = e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
  const float s = mx_scale(byte);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
  codes[i] = w;
  if (quarter == 0) scales[bi] = (uint8_t)byte;
}

// ---- the values ------------------------------------------------------------------------------------
// eight elements a thread: 4 bytes of codes in, one or two 16-byte stores (out rows of `pitch` elements)
template <typename T>
__device__ __forceinline__ void mx_values(unsigned w, float s, float (&v)[8]) {
#define HYP_MX_PAIR(I)                                                          \
  {                                                                             \
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, I);          \
    v[2 * I] = p[0];                                                            \
    v[2 * I + 1] = p[1];                                                        \
  }
  HYP_MX_PAIR(0) HYP_MX_PAIR(1) HYP_MX_PAIR(2) HYP_MX_PAIR(3)
#undef HYP_MX_PAIR
}

template <typename T>
__global__ __launch_bounds__(kQThreads) void mx_dequantize_k(const uint32_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, int cols, int nb,
                                                             int64_t total, T* __restrict__ out, int64_t pitch) {
  const int64_t i = (int64_t)blockIdx.x * kQThreads + threadIdx.x;
  const int64_t bi = i >> 2;
  if (bi >= total) return;
  const int64_t row = bi / nb;
  const int c0 = (int)(bi - row * nb) * kMxBlock + (int)(i & 3) * 8;
  float v[8];
  mx_values<T>(codes[i], mx_scale(scales[bi]), v);
  T* o = out + row * pitch + c0;
  if (c0 + 8 <= cols && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
    Vec8<T>::store(o, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j < cols) st1<T>(o + j, v[j]);
  }
}

// ---- activations as bf16 pieces ---------------------------------------------------------------------
// x = the sum of P bf16 numbers exactly (P = 1 bf16, 2 fp16, 3 fp32: 8 significant bits each, cut, not
// rounded, so that none overflows): the products then run on the bf16 matrix instructions with
// nothing lost.  out [P, rows, pitch], zeros behind `cols`.
template <typename T, int P>
__global__ __launch_bounds__(kQThreads) void mx_pieces_k(const T* __restrict__ x, int64_t ld, int64_t rows, int cols,
                                                         int pitch, bf16_t* __restrict__ out) {
  const int per = pitch >> 3;
  const int64_t i = (int64_t)blockIdx.x * kQThreads + threadIdx.x;
  const int64_t row = i / per;
  if (row >= rows) return;
  const int c0 = (int)(i - row * per) * 8;
  float v[8];
  load8<T>(x + row * ld + c0, cols - c0, v);
#pragma unroll
  for (int p = 0; p < P; ++p) {
    float h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned b = __float_as_uint(v[j]);
      h[j] = v[j] != v[j] ? v[j] : __uint_as_float(P == 1 ? b : b & 0xffff0000u);
      v[j] = (b & 0x7f800000u) == 0x7f800000u ? 0.f : v[j] - h[j];
    }
    Vec8<bf16_t>::store(out + ((int64_t)p * rows + row) * pitch + c0, h);
  }
}

// y [rows, cols] = the sum of P fp32 slabs [P, rows, pitch] (+ bias), rounded once
template <typename T>
__global__ __launch_bounds__(kQThreads) void mx_join_k(const float* __restrict__ part, int P, int64_t rows, int cols,
                                                       int64_t pitch, const float* __restrict__ bias,
                                                       T* __restrict__ y) {
  const int64_t i = (int64_t)blockIdx.x * kQThreads + threadIdx.x;
  if (i >= rows * cols) return;
  const int64_t row = i / cols;
  const int c = (int)(i - row * cols);
  float s = 0.f;
  for (int p = P - 1; p >= 0; --p) s += part[((int64_t)p * rows + row) * pitch + c];  // the small pieces first
  if (bias) s += bias[c];
  st1<T>(y + i, s);
}

// ---- few rows times a 4-bit weight ---------------------------------------------------------------------
// y [M, N] = x [M, 32 nb] Wt, W [N, 32 nb] in blocks.  A workgroup owns 16 columns of y and 16 MT rows; its
// 8 waves share the reduction (wave w takes the groups of four blocks w, w + 8, ...), so that the few
// columns of a thin product still fill the chip and one launch does it: no partial sums in memory.
// v_mfma_f32_16x16x32_bf16: lane l holds 8 reduction elements of row / column l & 15.  The order of the
// reduction is free as long as both operands share it: lane group g = l >> 4 takes block 4 kk + g whole, so
// that a lane's 16-byte load of codes is one block under one scale and feeds four matrix instructions.
// The eight partial tiles meet in LDS in wave order (the result does not depend on timing).
constexpr int kRowWaves = 8;

template <int MT, typename O>
__global__ __launch_bounds__(kRowWaves * 64) void mx_rows_k(const bf16_t* __restrict__ x, const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int M, int N, int nb,
                                                            const float* __restrict__ bias, O* __restrict__ y) {
  __shared__ float part[kRowWaves][MT][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * MT);
  const int64_t K = (int64_t)nb * kMxBlock;
  const int n = n0 + l15;
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int groups = (nb + 3) >> 2;
  for (int kk = wave; kk < groups; kk += kRowWaves) {
    const int b = kk * 4 + g;
    u32x4 w = {0u, 0u, 0u, 0u};
    unsigned sb = 127;
    const bool in = b < nb;
    if (in && n < N) {
      w = *reinterpret_cast<const u32x4*>(codes + ((int64_t)n * nb + b) * 16);
      sb = scales[(int64_t)n * nb + b];
    }
    const float s = mx_scale(sb);
    u16x8 a[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + i * 16 + l15;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[i][j] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (in && m < M) a[i][j] = *reinterpret_cast<const u16x8*>(x + m * K + (int64_t)b * kMxBlock + j * 8);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      union {
        bf16x2 p[4];
        u16x8 v;
      } f;
      f.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], s, 0);
      f.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], s, 1);
      f.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], s, 2);
      f.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], s, 3);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = mfl::mma16<bf16_t>(a[i][j], f.v, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][i][(4 * g + e) * 16 + l15] = acc[i][e];
  }
  __syncthreads();
  for (int t = threadIdx.x; t < MT * 256; t += kRowWaves * 64) {
    const int i = t >> 8, r = (t >> 4) & 15, c = t & 15;
    const int m = m0 + i * 16 + r;
    if (m >= M || n0 + c >= N) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) sum += part[w][i][t & 255];
    if (bias) sum += bias[n0 + c];
    st1<O>(y + (int64_t)m * N + n0 + c, sum);
  }
}

}  // namespace

hipError_t mx_quantize(int dtype, const void* x, int64_t ld, int64_t rows, int cols, uint8_t* codes, uint8_t* scales,
                       hipStream_t stream) {
  const int nb = (cols + kMxBlock - 1) / kMxBlock;
  const int64_t total = rows * nb, grid = (total * 4 + kQThreads - 1) / kQThreads;
  if (total == 0) return hipSuccess;
  if (grid >= kMxGridMax) return hipErrorInvalidValue;
  HYP_DISPATCH_FLOAT(dtype, T, {
    hipLaunchKernelGGL((mx_quantize_k<T>), dim3(grid), dim3(kQThreads), 0, stream, static_cast<const T*>(x), ld, cols,
                       nb, total, reinterpret_cast<uint32_t*>(codes), scales);
  });
  return hipGetLastError();
}

hipError_t mx_dequantize(int dtype, const uint8_t* codes, const uint8_t* scales, int64_t rows, int cols, void* out,
                         int64_t pitch, hipStream_t stream) {
  const int nb = (cols + kMxBlock - 1) / kMxBlock;
  const int64_t total = rows * nb, grid = (total * 4 + kQThreads - 1) / kQThreads;
  if (total == 0) return hipSuccess;
  if (grid >= kMxGridMax || pitch < cols) return hipErrorInvalidValue;
  HYP_DISPATCH_FLOAT(dtype, T, {
    hipLaunchKernelGGL((mx_dequantize_k<T>), dim3(grid), dim3(kQThreads), 0, stream,
                       reinterpret_cast<const uint32_t*>(codes), scales, cols, nb, total, static_cast<T*>(out), pitch);
  });
  return hipGetLastError();
}

hipError_t mx_pieces(int dtype, const void* x, int64_t ld, int64_t rows, int cols, int pitch, void* out,
                     hipStream_t stream) {
  if (pitch % 8 != 0 || pitch < cols) return hipErrorInvalidValue;
  const int64_t grid = (rows * (pitch / 8) + kQThreads - 1) / kQThreads;
  if (grid == 0) return hipSuccess;
  if (grid >= kMxGridMax) return hipErrorInvalidValue;
  bf16_t* o = static_cast<bf16_t*>(out);
  if (dtype == kBF16)
    hipLaunchKernelGGL((mx_pieces_k<bf16_t, 1>), dim3(grid), dim3(kQThreads), 0, stream,
                       static_cast<const bf16_t*>(x), ld, rows, cols, pitch, o);
  else if (dtype == kF16)
    hipLaunchKernelGGL((mx_pieces_k<f16_t, 2>), dim3(grid), dim3(kQThreads), 0, stream, static_cast<const f16_t*>(x), ld,
                       rows, cols, pitch, o);
  else
    hipLaunchKernelGGL((mx_pieces_k<float, 3>), dim3(grid), dim3(kQThreads), 0, stream, static_cast<const float*>(x), ld,
                       rows, cols, pitch, o);
  return hipGetLastError();
}

hipError_t mx_join(int dtype, const float* part, int pieces, int64_t rows, int cols, int64_t pitch, const float* bias,
                   void* y, hipStream_t stream) {
  const int64_t grid = (rows * cols + kQThreads - 1) / kQThreads;
  if (grid == 0) return hipSuccess;
  if (grid >= kMxGridMax) return hipErrorInvalidValue;
  HYP_DISPATCH_FLOAT(dtype, T, {
    hipLaunchKernelGGL((mx_join_k<T>), dim3(grid), dim3(kQThreads), 0, stream, part, pieces, rows, cols, pitch, bias,
                       static_cast<T*>(y));
  });
  return hipGetLastError();
}

hipError_t mx_rows(const void* x, const uint8_t* codes, const uint8_t* scales, int M, int N, int nb, const float* bias,
                   int out_dtype, void* y, hipStream_t stream) {
  if (M == 0 || N == 0) return hipSuccess;
  if (out_dtype != kBF16 && out_dtype != kF32) return hipErrorInvalidValue;
  const int mt = M <= 16 ? 1 : (M <= 32 ? 2 : 4);
  const dim3 grid((N + 15) / 16, (M + 16 * mt - 1) / (16 * mt)), block(kRowWaves * 64);
  if (grid.y > 65535) return hipErrorInvalidValue;
  const bf16_t* xp = static_cast<const bf16_t*>(x);
#define HYP_MX_ROWS(MT)                                                                                       \
  if (out_dtype == kBF16)                                                                                     \
    hipLaunchKernelGGL((mx_rows_k<MT, bf16_t>), grid, block, 0, stream, xp, codes, scales, M, N, nb, bias,    \
                       static_cast<bf16_t*>(y));                                                              \
  else                                                                                                        \
    hipLaunchKernelGGL((mx_rows_k<MT, float>), grid, block, 0, stream, xp, codes, scales, M, N, nb, bias,     \
                       static_cast<float*>(y));
  if (mt == 1) { HYP_MX_ROWS(1) } else if (mt == 2) { HYP_MX_ROWS(2) } else { HYP_MX_ROWS(4) }
#undef HYP_MX_ROWS
  return hipGetLastError();
}

}  // namespace hyp
