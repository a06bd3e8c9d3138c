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

// ---- activations times a 4-bit weight, decoded on the way to the matrix instructions ---------------------
// Both products run on v_mfma_f32_16x16x32_bf16 (lane l: 8 reduction elements 8 (l >> 4) .. of row / column
// l & 15) without LDS or barriers in their loops: the waves of a workgroup share one output tile and
// split its reduction into contiguous ranges, so that thin products still fill the chip, every wave
// streams its own operands from L2, and one launch does it.  The partial tiles meet in LDS in wave order
// (the result does not depend on timing).  Workgroups of one weight tile and different rows are 8 ids
// apart, on one XCD: the weight comes from HBM once.
constexpr int kMxWaves = 8;

struct MxArgs {
  const bf16_t* x;  // NT: [M, 32 nb]; NN: [M, ld]
  const uint8_t* codes;
  const uint8_t* scales;
  const float* bias;  // NT: [N] or null
  void* y;
  int M, N, nb;  // weight [N, 32 nb]
  int cols;      // NN: columns of y (K of the weight)
  int64_t ld;    // NN: row stride of x
};

// workgroup -> (row block, weight tile)
__device__ __forceinline__ void mx_tile(int rows, int tiles, int* mb, int* tile) {
  const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
  *mb = i % rows;
  *tile = (i / rows) * 8 + xcd;
}

// Lanes 16 g + l hold words w[0..3] of block g of row l; afterwards word j is word g of block j (a 4 x 4
// transposition over the lane groups): reduction elements 8 g .. 8 g + 7 of block j, as the matrix
// instruction wants them, so that the activations are read in rows of 64 bytes.
__device__ __forceinline__ void mx_group_transpose(u32x4& w) {
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  const u32x2 b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  const u32x2 c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const u32x2 d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  w = u32x4{c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ u16x8 mx_fragment(unsigned w, float s) {
  union {
    bf16x2 p[4];
    u16x8 v;
  } f;
  f.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0);
  f.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
  f.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2);
  f.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  return f.v;
}

// the four scales of a group of blocks as bytes of a word (127, that is 1, behind the row's end)
__device__ __forceinline__ unsigned mx_group_scales(const uint8_t* row, int b, int nb) {
  if (b + 4 <= nb) {
    typedef unsigned u32a __attribute__((aligned(1)));
    return *reinterpret_cast<const u32a*>(row + b);
  }
  unsigned s = 0x7f7f7f7fu;
  for (int i = 0; i < 4 && b + i < nb; ++i) s = (s & ~(255u << (8 * i))) | ((unsigned)row[b + i] << (8 * i));
  return s;
}

// y [M, N] = x Wt (+ bias): a workgroup owns 16 MT rows and 16 NT columns.  The reduction goes in groups of
// four blocks (128 elements); a lane's 16-byte load of codes is one block of its column.  Groups are loaded
// one ahead of the matrix instructions that use them.
template <int MT, int NT, typename O>
__global__ __launch_bounds__(kMxWaves * 64) void mx_nt_k(const MxArgs a) {
  extern __shared__ float part[];  // [waves][MT][NT][256]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  int mb, tile;
  mx_tile((a.M + 16 * MT - 1) / (16 * MT), (a.N + 16 * NT - 1) / (16 * NT), &mb, &tile);
  const int n0 = tile * 16 * NT, m0 = mb * 16 * MT;
  if (n0 >= a.N) return;  // the last ids of a tile count that is no multiple of 8
  const int64_t K = (int64_t)a.nb * kMxBlock;
  const int groups = (a.nb + 3) >> 2;
  const int kb = (int)((int64_t)wave * groups / kMxWaves), ke = (int)((int64_t)(wave + 1) * groups / kMxWaves);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Stage {
    u32x4 w[NT];
    unsigned s[NT];
    u16x8 x[MT][4];
  };
  auto load = [&](Stage& t, int kk) {
    const int b = kk * 4 + g;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = n0 + 16 * j + l15;
      t.w[j] = u32x4{0u, 0u, 0u, 0u};
      t.s[j] = 0x7f7f7f7fu;
      if (n < a.N) {
        if (b < a.nb) t.w[j] = *reinterpret_cast<const u32x4*>(a.codes + ((int64_t)n * a.nb + b) * 16);
        t.s[j] = mx_group_scales(a.scales + (int64_t)n * a.nb, kk * 4, a.nb);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + 16 * i + l15;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        t.x[i][q] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (m < a.M && kk * 4 + q < a.nb)
          t.x[i][q] = *reinterpret_cast<const u16x8*>(a.x + m * K + (int64_t)(kk * 4 + q) * kMxBlock + g * 8);
      }
    }
  };
  auto use = [&](Stage& t) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      mx_group_transpose(t.w[j]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u16x8 f = mx_fragment(t.w[j][q], mx_scale((t.s[j] >> (8 * q)) & 255u));
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = mfl::mma16<bf16_t>(t.x[i][q], f, acc[i][j]);
      }
    }
  };
  if (kb < ke) {
    Stage t[2];
    load(t[0], kb);
    int kk = kb;
    for (; kk + 2 <= ke; kk += 2) {
      load(t[1], kk + 1);
      use(t[0]);
      if (kk + 2 < ke) load(t[0], kk + 2);
      use(t[1]);
    }
    if (kk < ke) use(t[0]);
  }
  constexpr int kTile = MT * NT * 256;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave * kTile + (16 * i + 4 * g + e) * (16 * NT) + 16 * j + l15] = acc[i][j][e];
  __syncthreads();
  O* y = static_cast<O*>(a.y);
  for (int t = threadIdx.x; t < kTile; t += kMxWaves * 64) {
    const int m = m0 + t / (16 * NT), n = n0 + t % (16 * NT);
    if (m >= a.M || n >= a.N) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMxWaves; ++w) sum += part[w * kTile + t];
    if (a.bias) sum += a.bias[n];
    st1<O>(y + (int64_t)m * a.N + n, sum);
  }
}

// y [M, cols] = x W, x [M, N]: the reduction runs over the weight's rows.  A workgroup owns 16 MT rows and 128
// columns, 32 weight rows a step: a lane loads 8 elements (4 bytes) of each of 8 weight rows, decodes them
// under each row's own scale and transposes the 8 x 8 in registers (v_perm), which gives the fragments of
// columns 8 (l & 15) + c, c = 0..7: no transposed copy of the weight, and 16 consecutive bytes of y a lane.
template <int MT, typename O>
__global__ __launch_bounds__(kMxWaves * 64) void mx_nn_k(const MxArgs a) {
  extern __shared__ float part[];  // [waves][16 MT][128]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  int mb, tile;
  mx_tile((a.M + 16 * MT - 1) / (16 * MT), (a.cols + 127) / 128, &mb, &tile);
  const int k0 = tile * 128, m0 = mb * 16 * MT;
  if (k0 >= a.cols) return;
  const int steps = (a.N + 31) >> 5;
  const int sb = (int)((int64_t)wave * steps / kMxWaves), se = (int)((int64_t)(wave + 1) * steps / kMxWaves);
  const int blk = (k0 >> 5) + (l15 >> 2);
  const bool in = blk < a.nb;
  const uint8_t* cp = a.codes + (int64_t)blk * 16 + (l15 & 3) * 4;
  const uint8_t* sp = a.scales + blk;
  f32x4 acc[MT][8];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Stage {
    unsigned w[8], s[8];
    u16x8 x[MT];
  };
  auto load = [&](Stage& t, int st) {
    const int n0 = st * 32 + g * 8;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      t.w[r] = 0u;
      t.s[r] = 127u;
      if (in && n0 + r < a.N) {
        t.w[r] = *reinterpret_cast<const unsigned*>(cp + (int64_t)(n0 + r) * a.nb * 16);
        t.s[r] = sp[(int64_t)(n0 + r) * a.nb];
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + 16 * i + l15;
      t.x[i] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (m < a.M && n0 < a.N) t.x[i] = *reinterpret_cast<const u16x8*>(a.x + m * a.ld + n0);
    }
  };
  auto use = [&](const Stage& t) {
    union {
      u16x8 v;
      unsigned w[4];
    } row[8], f;  // row[r].w[q]: columns 2 q, 2 q + 1 of weight row r
#pragma unroll
    for (int r = 0; r < 8; ++r) row[r].v = mx_fragment(t.w[r], mx_scale(t.s[r]));
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int h = 0; h < 4; ++h)  // rows 2 h, 2 h + 1 of column c
        f.w[h] = __builtin_amdgcn_perm(row[2 * h + 1].w[c >> 1], row[2 * h].w[c >> 1], (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][c] = mfl::mma16<bf16_t>(t.x[i], f.v, acc[i][c]);
    }
  };
  if (sb < se) {
    Stage t[2];
    load(t[0], sb);
    int st = sb;
    for (; st + 2 <= se; st += 2) {
      load(t[1], st + 1);
      use(t[0]);
      if (st + 2 < se) load(t[0], st + 2);
      use(t[1]);
    }
    if (st < se) use(t[0]);
  }
  constexpr int kTile = MT * 16 * 128;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float* p = part + wave * kTile + (16 * i + 4 * g + e) * 128 + 8 * l15;
      reinterpret_cast<float4*>(p)[0] = make_float4(acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]);
      reinterpret_cast<float4*>(p)[1] = make_float4(acc[i][4][e], acc[i][5][e], acc[i][6][e], acc[i][7][e]);
    }
  __syncthreads();
  O* y = static_cast<O*>(a.y);
  for (int t = threadIdx.x; t < kTile; t += kMxWaves * 64) {
    const int m = m0 + (t >> 7), k = k0 + (t & 127);
    if (m >= a.M || k >= a.cols) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMxWaves; ++w) sum += part[w * kTile + t];
    st1<O>(y + (int64_t)m * a.cols + k, sum);
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

namespace {

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename K>
hipError_t mx_launch(K kernel, int rows, int tiles, size_t lds, const MxArgs& a, hipStream_t stream) {
  const int64_t grid = (int64_t)rows * ((tiles + 7) / 8 * 8);
  if (grid >= kMxGridMax) return hipErrorInvalidValue;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kMxWaves * 64), lds, stream, a);
  return hipGetLastError();
}

}  // namespace

// Measured (MI355X, bf16): the one-launch product against decoding the weight (8 us for 4096 x 4096, 18 for 11008 x
// 4096) plus the tiled GEMM (17 us at least): the larger tiles while they give every CU a workgroup.
void mx_nt_plan(int M, int N, int nb, int* mt, int* nt) {
  struct T {
    int mt, nt;
  };
  static const T kOrder[] = {{4, 4}, {2, 4}, {2, 2}, {1, 2}, {1, 1}};
  const int64_t work = (int64_t)M * N * nb;
  *mt = *nt = 0;
  if (M > 128 && work > (int64_t)256 * 4096 * 128) return;
  for (const T& t : kOrder) {
    *mt = t.mt;
    *nt = t.nt;
    if (16 * t.mt <= M && (int64_t)ceil_div(M, 16 * t.mt) * ceil_div(N, 16 * t.nt) >= 256) return;
  }
}

void mx_nn_plan(int M, int N, int nb, int* mt) {
  const int64_t work = (int64_t)M * N * nb;
  *mt = M > 128 && work > (int64_t)256 * 4096 * 128 ? 0 : (ceil_div(M, 32) * ceil_div(nb, 4) >= 256 ? 2 : 1);
}

// The tiled GEMM's 256x256 ping-pong tile (one workgroup a CU) or its 128x128 tile (two a CU), by the rounds that
// their workgroups need: a 32-deep step of a round takes 1.0 us / 0.62 us (measured at 2032 .. 4064 rows), a split
// another pass over fp32 partial sums.
void mx_gemm_plan(int M, int N, int K, int* tile, int* splits) {
  double best = 1e30;
  *tile = 3;
  *splits = 1;
  for (int t : {8, 3}) {
    const int b = t == 8 ? 256 : 128;
    if (t == 8 && (M < 256 || N < 256)) continue;
    const int64_t tiles = (int64_t)ceil_div(M, b) * ceil_div(N, b);
    for (int s : {1, 2, 4, 8}) {
      if (s > 1 && K / s < 512) break;
      const int slots = t == 8 ? 256 : 512;
      double us = (double)((tiles * s + slots - 1) / slots) * ceil_div(ceil_div(K, 32), s) * (t == 8 ? 1.0 : 0.62);
      if (s > 1) us += 4.0 + (double)M * N * 4.0 * (s + 1) / 4e6;
      if (us < best) {
        best = us;
        *tile = t;
        *splits = s;
      }
    }
  }
}

hipError_t mx_nt(const void* x, const uint8_t* codes, const uint8_t* scales, int M, int N, int nb, const float* bias,
                 int out_dtype, void* y, hipStream_t stream, int mt, int nt) {
  if (M == 0 || N == 0) return hipSuccess;
  if (out_dtype != kBF16 && out_dtype != kF32) return hipErrorInvalidValue;
  MxArgs a{static_cast<const bf16_t*>(x), codes, scales, bias, y, M, N, nb, 0, 0};
#define HYP_MX_NT(MT, NT)                                                                                      \
  if (mt == MT && nt == NT) {                                                                                  \
    const size_t lds = sizeof(float) * kMxWaves * MT * NT * 256;                                               \
    const int rows = ceil_div(M, 16 * MT), tiles = ceil_div(N, 16 * NT);                                       \
    return out_dtype == kBF16 ? mx_launch(mx_nt_k<MT, NT, bf16_t>, rows, tiles, lds, a, stream)                \
                              : mx_launch(mx_nt_k<MT, NT, float>, rows, tiles, lds, a, stream);                \
  }
  HYP_MX_NT(1, 1) HYP_MX_NT(1, 2) HYP_MX_NT(2, 2) HYP_MX_NT(2, 4) HYP_MX_NT(4, 4)
#undef HYP_MX_NT
  return hipErrorInvalidValue;
}

hipError_t mx_nn(const void* x, int64_t ld, const uint8_t* codes, const uint8_t* scales, int M, int N, int nb, int cols,
                 int out_dtype, void* y, hipStream_t stream, int mt) {
  if (M == 0 || cols == 0) return hipSuccess;
  if ((out_dtype != kBF16 && out_dtype != kF32) || ld % 8 != 0) return hipErrorInvalidValue;
  MxArgs a{static_cast<const bf16_t*>(x), codes, scales, nullptr, y, M, N, nb, cols, ld};
#define HYP_MX_NN(MT)                                                                                          \
  if (mt == MT) {                                                                                              \
    const size_t lds = sizeof(float) * kMxWaves * MT * 2048;                                                   \
    const int rows = ceil_div(M, 16 * MT), tiles = ceil_div(cols, 128);                                        \
    return out_dtype == kBF16 ? mx_launch(mx_nn_k<MT, bf16_t>, rows, tiles, lds, a, stream)                    \
                              : mx_launch(mx_nn_k<MT, float>, rows, tiles, lds, a, stream);                    \
  }
  HYP_MX_NN(1) HYP_MX_NN(2)
#undef HYP_MX_NN
  return hipErrorInvalidValue;
}

}  // namespace hyp
