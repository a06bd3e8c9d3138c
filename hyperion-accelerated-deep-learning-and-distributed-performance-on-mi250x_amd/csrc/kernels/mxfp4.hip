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
#include <algorithm>
#include <cmath>

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
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
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
  for (int64_t i = (int64_t)blockIdx.x * kQThreads + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * kQThreads) {
    const int64_t row = i / cols;
    const int c = (int)(i - row * cols);
    float s = 0.f;
    for (int p = P - 1; p >= 0; --p) s += part[((int64_t)p * rows + row) * pitch + c];  // the small pieces first
    if (bias) s += bias[c];
    st1<T>(y + i, s);
  }
}

// ---- activations times a 4-bit weight, decoded on the way to the matrix instructions ---------------------
// Both products run on v_mfma_f32_16x16x32_bf16 (lane l: 8 reduction elements 8 (l >> 4) .. of row / column
// l & 15) without LDS or barriers in their loops: the waves of a workgroup share one output tile and
// split its reduction into contiguous ranges, so that thin products still fill the chip, every wave
// streams its own operands from L2, and one launch does it.  The partial tiles meet in LDS in wave order
// (the result does not depend on timing).
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
  int group;     // row blocks of a group (mx_tile)
  int pieces;    // 128-column tiles: x is [pieces, M, 32 nb], their sum the activations
};

// workgroup -> (row block, weight tile): every XCD takes a contiguous piece of the order row group, weight tile, row
// block of the group.  A group's activations (at most 2 MB) and the piece's weight tiles stay in the XCD's L2.
__device__ __forceinline__ void mx_tile(const MxArgs& a, int rows, int tiles, int* mb, int* tile) {
  const int id = mfl::xcd_remap(blockIdx.x, gridDim.x);
  const int group = id / (a.group * tiles), r = id - group * a.group * tiles;
  const int size = min(a.group, rows - group * a.group);
  *tile = r / size;
  *mb = group * a.group + r % size;
}

// Lanes 16 g + l hold words w[0..3] of block g of row l; afterwards word j is word g of block j (a 4 x 4
// transposition over the lane groups): reduction elements 8 g .. 8 g + 7 of block j, as the matrix
// instruction wants them, so that the activations are read in rows of 64 bytes.
__device__ __forceinline__ void mx_group_transpose(u32x4& w) {
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
  mx_tile(a, (a.M + 16 * MT - 1) / (16 * MT), (a.N + 16 * NT - 1) / (16 * NT), &mb, &tile);
  const int n0 = tile * 16 * NT, m0 = mb * 16 * MT;
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

// ---- the same product through LDS --------------------------------------------------------------------------
// Lanes 16 apart hold one row's neighbours in a fragment, so a fragment loaded from memory asks for 64 single 16-byte
// pieces (64 clocks a KiB of a CU's 16).  Where rows are whole groups of four blocks, each wave therefore moves its
// own operands with LDS-DMA, 256 contiguous bytes of an activation row and 64 of a weight row at a time, into a ring
// of its own (no barrier in the loop), and reads the fragments from there.  Lane group g takes block g of the group:
// one scale a lane and no exchange; the activation's fragment of step q is chunk 4 g + q of its row.
// Images: activations [16 MT rows][16 chunks], chunk c of row r at slot c ^ h(r), h = the low four bits of r with
// their halves swapped; weight [16 NT rows][4 chunks], chunk c of row r at c ^ f(r >> 2 & 3), f = 0 2 3 1; scales
// [64 rows] of 4 bytes.  Both make every group of lanes that LDS serves at once touch 64 different banks.
constexpr int kLdsWaves = 4;

template <int N>
__device__ __forceinline__ void mx_wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

__device__ __forceinline__ void lds_dma16(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
__device__ __forceinline__ void lds_dma4(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}

// Fragment reads as asm, each block with its own wait (the compiler would wait for the whole ring before an LDS read).
// four chunks of one 16-row image; the image begins OFF bytes behind the lane addresses
template <int OFF>
__device__ __forceinline__ void mx_read_x1(const unsigned (&ad)[4], u32x4 (&x)[4]) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%8\n\tds_read_b128 %1, %5 offset:%8\n\tds_read_b128 %2, %6 offset:%8\n\t"
      "ds_read_b128 %3, %7 offset:%8\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
      : "v"(ad[0]), "v"(ad[1]), "v"(ad[2]), "v"(ad[3]), "i"(OFF)
      : "memory");
}
__device__ __forceinline__ void mx_read_x2(const unsigned (&ad)[4], u32x4 (&x)[2][4]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\tds_read_b128 %6, %10 offset:4096\n\t"
      "ds_read_b128 %7, %11 offset:4096\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[0][2]), "=&v"(x[0][3]), "=&v"(x[1][0]), "=&v"(x[1][1]),
        "=&v"(x[1][2]), "=&v"(x[1][3])
      : "v"(ad[0]), "v"(ad[1]), "v"(ad[2]), "v"(ad[3])
      : "memory");
}
__device__ __forceinline__ void mx_read_w(unsigned wa, unsigned sa, u32x4 (&w)[1], unsigned (&s)[1]) {
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b32 %1, %3\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(w[0]), "=&v"(s[0])
               : "v"(wa), "v"(sa)
               : "memory");
}
__device__ __forceinline__ void mx_read_w(unsigned wa, unsigned sa, u32x4 (&w)[2], unsigned (&s)[2]) {
  asm volatile(
      "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\tds_read_b32 %2, %5\n\tds_read_b32 %3, %5 offset:64\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(s[0]), "=&v"(s[1])
      : "v"(wa), "v"(sa)
      : "memory");
}
__device__ __forceinline__ void mx_read_w(unsigned wa, unsigned sa, u32x4 (&w)[4], unsigned (&s)[4]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:1024\n\tds_read_b128 %2, %8 offset:2048\n\t"
      "ds_read_b128 %3, %8 offset:%10\n\tds_read_b32 %4, %9\n\tds_read_b32 %5, %9 offset:64\n\t"
      "ds_read_b32 %6, %9 offset:128\n\tds_read_b32 %7, %9 offset:192\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
      : "v"(wa), "v"(sa), "i"(3 * 1024)
      : "memory");
}

template <int MT, int NT>
constexpr int mx_nt_lds_bytes(int stages) {
  return kLdsWaves * stages * (MT * 4096 + NT * 1024 + 256);
}

template <int MT, int NT, int S, typename O>
__global__ __launch_bounds__(kLdsWaves * 64) void mx_nt_lds_k(const MxArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int kX = MT * 4096, kW = NT * 1024, kStage = kX + kW + 256;
  constexpr int L = MT * 4 + NT + 1;  // DMA instructions of a stage
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  int mb, tile;
  mx_tile(a, (a.M + 16 * MT - 1) / (16 * MT), (a.N + 16 * NT - 1) / (16 * NT), &mb, &tile);
  const int n0 = tile * 16 * NT, m0 = mb * 16 * MT;
  const int64_t K = (int64_t)a.nb * kMxBlock;
  const int groups = a.nb >> 2;
  const int kb = (int)((int64_t)wave * groups / kLdsWaves), n = (int)((int64_t)(wave + 1) * groups / kLdsWaves) - kb;
  uint8_t* ring = lds + wave * (S * kStage);
  // rows behind the ends read the last row: their outputs are not stored
  const uint8_t* xs[MT * 4];
  const uint8_t* ws[NT];
#pragma unroll
  for (int i = 0; i < MT * 4; ++i) {
    const int r = 4 * i + (lane >> 4), m = min(m0 + r, a.M - 1);
    const int h = ((r & 3) << 2) | ((r >> 2) & 3);
    xs[i] = reinterpret_cast<const uint8_t*>(a.x + m * K) + kb * 256 + ((l15 ^ h) << 4);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = lane >> 2, nn = min(n0 + 16 * j + r, a.N - 1);
    ws[j] = a.codes + ((int64_t)nn * a.nb + kb * 4 + ((lane & 3) ^ ((0x78 >> (2 * (r >> 2))) & 3))) * 16;
  }
  const uint8_t* ss = a.scales + (int64_t)min(n0 + min(lane, 16 * NT - 1), a.N - 1) * a.nb + kb * 4;
  auto issue = [&](int t) {
    uint8_t* st = ring + (t % S) * kStage;
#pragma unroll
    for (int i = 0; i < MT * 4; ++i) lds_dma16(xs[i] + t * 256, st + i * 1024);
#pragma unroll
    for (int j = 0; j < NT; ++j) lds_dma16(ws[j] + t * 64, st + kX + j * 1024);
    lds_dma4(ss + t * 4, st + kX + kW);
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int h = ((l15 & 3) << 2) | (l15 >> 2);
  const unsigned base = mfl::lds_addr(ring);
  for (int t = 0; t < S - 1 && t < n; ++t) issue(t);
  for (int t = 0; t < n; ++t) {
    if (t + S - 1 < n) issue(t + S - 1);
    const int ahead = n - 1 - t;
    if (ahead >= S - 1) mx_wait_vm<(S - 1) * L>();
    else if (S > 2 && ahead == 1) mx_wait_vm<L>();
    else mx_wait_vm<0>();
    const unsigned sb = base + (t % S) * kStage;
    unsigned xa[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) xa[q] = sb + l15 * 256 + (((4 * g + q) ^ h) << 4);
    u32x4 w[NT], x[MT][4];
    unsigned sc[NT];
    mx_read_w(sb + kX + l15 * 64 + ((g ^ ((0x78 >> (2 * (l15 >> 2))) & 3)) << 4), sb + kX + kW + l15 * 4, w, sc);
    if constexpr (MT == 2) mx_read_x2(xa, x);
    else mx_read_x1<0>(xa, x[0]);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float s = mx_scale((sc[j] >> (8 * g)) & 255u);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u16x8 f = mx_fragment(w[j][q], s);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = mfl::mma16<bf16_t>(__builtin_bit_cast(u16x8, x[i][q]), f, acc[i][j]);
      }
    }
  }
  __syncthreads();  // the rings become the partial tiles
  constexpr int kTile = MT * NT * 256;
  float* part = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave * kTile + (16 * i + 4 * g + e) * (16 * NT) + 16 * j + l15] = acc[i][j][e];
  __syncthreads();
  O* y = static_cast<O*>(a.y);
  for (int t = threadIdx.x; t < kTile; t += kLdsWaves * 64) {
    const int m = m0 + t / (16 * NT), c = n0 + t % (16 * NT);
    if (m >= a.M || c >= a.N) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kLdsWaves; ++w) sum += part[w * kTile + t];
    if (a.bias) sum += a.bias[c];
    st1<O>(y + (int64_t)m * a.N + c, sum);
  }
}

// ---- the same product in 128-column tiles -----------------------------------------------------------------
// For more rows: 8 waves share a ring of stages (one barrier a stage) over 32 MI rows and 128 columns, so that a
// decoded fragment meets MI fragments of activations.  Waves 4 h + 2 i + j own the i-th half of the rows and the j-th of
// the columns for half h of every block's elements: two waves a SIMD (one alone issues at half rate), whose
// sums meet in LDS.  2048 x 11008 x 4096 in 185 us in 64-row tiles, 197 in 128-row ones (1.0 PFLOP/s; decoded
// weight and tiled GEMM 248), 450 x 4096 x 4096 in 23 us against 34 in 32-row tiles.  At 1024 x 4096 x 4096 the matrix pipe works
// 43 % of the time, LDS 25 %, and waves wait 36 %.  Halves a barrier apart (one multiplies while the other
// reads) were slower, 37.6 against 34.6 us for one round of 128-row tiles, and so was every wave bringing its own scales
// (42 against 36 us at 700 rows in 64-row tiles).  The images are those above.  x holds P pieces [M, 32 nb] whose sum the activations are: the
// reduction runs over the weight once for each, the smallest first, into the same fp32 sums.
constexpr int kBigStages = 3, kBigCols = 128;

__device__ __forceinline__ void st4(float* y, const float (&v)[4]) { *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void st4(bf16_t* y, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ void st4(f16_t* y, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(y) = make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
}

// LDS-DMA as asm (it has no result): with the builtin in flight the compiler waits for the whole ring before an LDS read,
// and here it is to schedule the fragment reads among the matrix instructions.
__device__ __forceinline__ void big_dma16(const void* src, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void big_dma4(const void* src, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(src) : "memory", "m0");
}
template <typename V>
__device__ __forceinline__ V lds_at(unsigned addr) {
  return *(const __attribute__((address_space(3))) V*)addr;
}

template <int MI>
constexpr int mx_big_bytes() {
  return kBigStages * (MI * 8192 + 8192 + 512);
}

template <int MI, typename O>
__global__ __launch_bounds__(512) void mx_nt_big_k(const MxArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int kX = MI * 8192, kW = 8192, kStage = kX + kW + 512, S = kBigStages;
  constexpr int L = MI + 1;  // DMA instructions of a wave and stage; waves 0 and 1 also bring the scales
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  const int half = wave >> 2, wm = (wave >> 1) & 1, wn = wave & 1;
  int mb, tile;
  mx_tile(a, (a.M + 32 * MI - 1) / (32 * MI), (a.N + kBigCols - 1) / kBigCols, &mb, &tile);
  const int n0 = tile * kBigCols, m0 = mb * 32 * MI;
  const int64_t K = (int64_t)a.nb * kMxBlock, piece = (int64_t)a.M * K;
  const int groups = a.nb >> 2, n = a.pieces * groups;
  // rows behind the ends read the last row: their outputs are not stored
  const uint8_t* xs[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int r = 4 * (wave * MI + i) + g, m = min(m0 + r, a.M - 1);
    const int h = ((r & 3) << 2) | ((r >> 2) & 3);
    xs[i] = reinterpret_cast<const uint8_t*>(a.x + (a.pieces - 1) * piece + m * K) + ((l15 ^ h) << 4);
  }
  const int wr = lane >> 2;
  const uint8_t* ws = a.codes + ((int64_t)min(n0 + 16 * wave + wr, a.N - 1) * a.nb + ((lane & 3) ^ ((0x78 >> (2 * (wr >> 2))) & 3))) * 16;
  const uint8_t* ss = a.scales + (int64_t)min(n0 + 64 * wn + lane, a.N - 1) * a.nb;  // (waves 0 and 1)
  const unsigned base = mfl::lds_addr(lds);
  int at = 0, slot = 0;  // the next stage's group of its piece, and its place
  auto issue = [&]() {
    const unsigned st = __builtin_amdgcn_readfirstlane(base + slot * kStage);
#pragma unroll
    for (int i = 0; i < MI; ++i) big_dma16(xs[i] + at * 256, st + (wave * MI + i) * 1024);
    big_dma16(ws + at * 64, st + kX + wave * 1024);
    if (wave < 2) big_dma4(ss + at * 4, st + kX + kW + wave * 256);
    slot = slot + 1 == S ? 0 : slot + 1;
    if (++at == groups) {
      at = 0;
#pragma unroll
      for (int i = 0; i < MI; ++i) xs[i] -= piece * 2;
    }
  };
  f32x4 acc[MI][4];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int h = ((l15 & 3) << 2) | (l15 >> 2);
  const unsigned xr = (16 * MI * wm + l15) * 256, q0 = ((4 * g + 2 * half) ^ h) << 4, q1 = ((4 * g + 2 * half + 1) ^ h) << 4;
  const unsigned wo = kX + (64 * wn + l15) * 64 + ((g ^ ((0x78 >> (2 * (l15 >> 2))) & 3)) << 4) + 8 * half;
  const unsigned so = kX + kW + wn * 256 + l15 * 4;
  for (int t = 0; t < S - 1 && t < n; ++t) issue();
  int use = 0;
  for (int t = 0; t < n; ++t) {
    if (t + 1 == n) mx_wait_vm<0>();
    else if (wave < 2) mx_wait_vm<L + 1>();
    else mx_wait_vm<L>();
    mfl::barrier_keep_vm();  // every wave's part of stage t is there, and stage t - 1 has been read
    asm volatile("" ::: "memory");  // no read moves up
    if (t + S - 1 < n) issue();
    const unsigned sb = base + use * kStage;
    use = use + 1 == S ? 0 : use + 1;
    u32x4 x[MI][2];
    u32x2 w[4];
    unsigned sc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = lds_at<u32x2>(sb + wo + j * 1024);
      sc[j] = lds_at<unsigned>(sb + so + j * 64);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      x[i][0] = lds_at<u32x4>(sb + xr + q0 + i * 4096);
      x[i][1] = lds_at<u32x4>(sb + xr + q1 + i * 4096);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float s = mx_scale((sc[j] >> (8 * g)) & 255u);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const u16x8 f = mx_fragment(w[j][q], s);
#pragma unroll
        for (int i = 0; i < MI; ++i) acc[i][j] = mfl::mma16<bf16_t>(f, __builtin_bit_cast(u16x8, x[i][q]), acc[i][j]);
      }
    }
  }
  // each half keeps MI / 2 of the row fragments and takes the other half's sums for them
  __syncthreads();
  constexpr int H = MI / 2;
  f32x4* part = reinterpret_cast<f32x4*>(lds) + lane;
#pragma unroll
  for (int i = 0; i < H; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 lo = acc[i][j], hi = acc[i + H][j];
      part[((wave * H + i) * 4 + j) * 64] = half ? lo : hi;
    }
  __syncthreads();
  O* y = static_cast<O*>(a.y);
  const bool vec = a.N % 4 == 0;
#pragma unroll
  for (int i = 0; i < H; ++i) {
    const int m = m0 + 16 * (MI * wm + i + (half ? H : 0)) + l15;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 o = part[(((wave ^ 4) * H + i) * 4 + j) * 64], lo = acc[i][j], hi = acc[i + H][j];
      float sum[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = o[e] + (half ? hi : lo)[e];
      const int c = n0 + 64 * wn + 16 * j + 4 * g;
      O* to = y + (int64_t)m * a.N + c;
      if (vec && c < a.N) {
        if (a.bias) {
          const float4 b = *reinterpret_cast<const float4*>(a.bias + c);
          sum[0] += b.x, sum[1] += b.y, sum[2] += b.z, sum[3] += b.w;
        }
        st4(to, sum);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < a.N) st1<O>(to + e, sum[e] + (a.bias ? a.bias[c + e] : 0.f));
      }
    }
  }
}

// y [M, cols] = x W, x [M, N]: the reduction runs over the weight's rows.  A workgroup owns 16 rows and 128
// columns, 32 weight rows a step: a lane loads 8 elements (4 bytes) of each of 8 weight rows, decodes them
// under each row's own scale and transposes the 8 x 8 in registers (v_perm), which gives the fragments of
// columns 8 (l & 15) + c, c = 0..7: no transposed copy of the weight, and 16 consecutive bytes of y a lane.
template <typename O>
__global__ __launch_bounds__(kMxWaves * 64) void mx_nn_k(const MxArgs a) {
  constexpr int MT = 1;
  extern __shared__ float part[];  // [waves][16][128]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  int mb, tile;
  mx_tile(a, (a.M + 16 * MT - 1) / (16 * MT), (a.cols + 127) / 128, &mb, &tile);
  const int k0 = tile * 128, m0 = mb * 16 * MT;
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

// ---- the data gradient through LDS ------------------------------------------------------------------------
// y [M, cols] = x W, x [M, ld] with zeros from N to ld, a multiple of 128: the reduction runs over the weight's rows, 128 a
// stage.  A workgroup owns 16 MT rows and 128 columns; the waves split the reduction and each fills a ring of its own as
// above.  A lane reads 8 elements (4 bytes) of each of 8 weight rows, decodes them under each row's own scale
// and transposes the 8 x 8 in registers (v_perm), which gives the fragments of columns 8 (l & 15) + c, c = 0..7:
// no transposed copy of the weight, and 32 consecutive bytes of the partial tile a lane.  Every workgroup
// walks all of the weight's rows, 0.33 us for 128 of them: up to 16 rows of x over 4096 columns are 32 workgroups on 256 CUs and
// take one walk's time (14 us for 4096 weight rows), and 128 rows of x (17 us) decode each strip eight times.
// Images: activations as above with h(r) = r; weight rows 8 g + r of every 32 at place 4 r + g, 64 bytes each, so
// that the four lane groups read 256 consecutive bytes; scales [128 rows] of 4 bytes.
template <int S0>
__device__ __forceinline__ void mx_read_nn(unsigned wa, unsigned sa, unsigned xa0, unsigned xa1, u32x2 (&w)[8], u32x4 (&s)[4],
                                           u32x4 (&x)[1][2]) {
  asm volatile(
      "ds_read2st64_b32 %0, %14 offset0:%18 offset1:%19\n\t"
      "ds_read2st64_b32 %1, %14 offset0:%20 offset1:%21\n\t"
      "ds_read2st64_b32 %2, %14 offset0:%22 offset1:%23\n\t"
      "ds_read2st64_b32 %3, %14 offset0:%24 offset1:%25\n\t"
      "ds_read2st64_b32 %4, %14 offset0:%26 offset1:%27\n\t"
      "ds_read2st64_b32 %5, %14 offset0:%28 offset1:%29\n\t"
      "ds_read2st64_b32 %6, %14 offset0:%30 offset1:%31\n\t"
      "ds_read2st64_b32 %7, %14 offset0:%32 offset1:%33\n\t"
      "ds_read_b128 %8, %15 offset:%34\n\t"
      "ds_read_b128 %9, %15 offset:%35\n\t"
      "ds_read_b128 %10, %15 offset:%36\n\t"
      "ds_read_b128 %11, %15 offset:%37\n\t"
      "ds_read_b128 %12, %16\n\t"
      "ds_read_b128 %13, %17\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7]),
        "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3]), "=&v"(x[0][0]), "=&v"(x[0][1])
      : "v"(wa), "v"(sa), "v"(xa0), "v"(xa1), "i"(8 * (S0 + 0) + 0), "i"(8 * (S0 + 0) + 1), "i"(8 * (S0 + 0) + 2),
        "i"(8 * (S0 + 0) + 3), "i"(8 * (S0 + 0) + 4), "i"(8 * (S0 + 0) + 5), "i"(8 * (S0 + 0) + 6),
        "i"(8 * (S0 + 0) + 7), "i"(8 * (S0 + 1) + 0), "i"(8 * (S0 + 1) + 1), "i"(8 * (S0 + 1) + 2),
        "i"(8 * (S0 + 1) + 3), "i"(8 * (S0 + 1) + 4), "i"(8 * (S0 + 1) + 5), "i"(8 * (S0 + 1) + 6),
        "i"(8 * (S0 + 1) + 7), "i"(128 * (S0 + 0) + 0), "i"(128 * (S0 + 0) + 16), "i"(128 * (S0 + 1) + 0),
        "i"(128 * (S0 + 1) + 16)
      : "memory");
}
template <int S0>
__device__ __forceinline__ void mx_read_nn(unsigned wa, unsigned sa, unsigned xa0, unsigned xa1, u32x2 (&w)[8], u32x4 (&s)[4],
                                           u32x4 (&x)[2][2]) {
  asm volatile(
      "ds_read2st64_b32 %0, %16 offset0:%20 offset1:%21\n\t"
      "ds_read2st64_b32 %1, %16 offset0:%22 offset1:%23\n\t"
      "ds_read2st64_b32 %2, %16 offset0:%24 offset1:%25\n\t"
      "ds_read2st64_b32 %3, %16 offset0:%26 offset1:%27\n\t"
      "ds_read2st64_b32 %4, %16 offset0:%28 offset1:%29\n\t"
      "ds_read2st64_b32 %5, %16 offset0:%30 offset1:%31\n\t"
      "ds_read2st64_b32 %6, %16 offset0:%32 offset1:%33\n\t"
      "ds_read2st64_b32 %7, %16 offset0:%34 offset1:%35\n\t"
      "ds_read_b128 %8, %17 offset:%36\n\t"
      "ds_read_b128 %9, %17 offset:%37\n\t"
      "ds_read_b128 %10, %17 offset:%38\n\t"
      "ds_read_b128 %11, %17 offset:%39\n\t"
      "ds_read_b128 %12, %18\n\t"
      "ds_read_b128 %13, %19\n\t"
      "ds_read_b128 %14, %18 offset:4096\n\t"
      "ds_read_b128 %15, %19 offset:4096\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7]),
        "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3]), "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]),
        "=&v"(x[1][1])
      : "v"(wa), "v"(sa), "v"(xa0), "v"(xa1), "i"(8 * (S0 + 0) + 0), "i"(8 * (S0 + 0) + 1), "i"(8 * (S0 + 0) + 2),
        "i"(8 * (S0 + 0) + 3), "i"(8 * (S0 + 0) + 4), "i"(8 * (S0 + 0) + 5), "i"(8 * (S0 + 0) + 6),
        "i"(8 * (S0 + 0) + 7), "i"(8 * (S0 + 1) + 0), "i"(8 * (S0 + 1) + 1), "i"(8 * (S0 + 1) + 2),
        "i"(8 * (S0 + 1) + 3), "i"(8 * (S0 + 1) + 4), "i"(8 * (S0 + 1) + 5), "i"(8 * (S0 + 1) + 6),
        "i"(8 * (S0 + 1) + 7), "i"(128 * (S0 + 0) + 0), "i"(128 * (S0 + 0) + 16), "i"(128 * (S0 + 1) + 0),
        "i"(128 * (S0 + 1) + 16)
      : "memory");
}

template <int MT>
constexpr int mx_nn_lds_bytes(int stages) {
  return kLdsWaves * (stages * (MT * 4096 + 8192 + 512) > MT * 8192 ? stages * (MT * 4096 + 8192 + 512) : MT * 8192);
}

template <int MT, int S, typename O>
__global__ __launch_bounds__(kLdsWaves * 64) void mx_nn_lds_k(const MxArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int kX = MT * 4096, kW = 8192, kStage = kX + kW + 512;
  constexpr int L = MT * 4 + 8 + 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  int mb, tile;
  mx_tile(a, (a.M + 16 * MT - 1) / (16 * MT), (a.cols + 127) >> 7, &mb, &tile);
  const int k0 = tile * 128, m0 = mb * 16 * MT;
  const int stages = (a.N + 127) >> 7;
  const int sb = (int)((int64_t)wave * stages / kLdsWaves), n = (int)((int64_t)(wave + 1) * stages / kLdsWaves) - sb;
  uint8_t* ring = lds + wave * (S * kStage);
  const uint8_t* xs[MT * 4];
#pragma unroll
  for (int i = 0; i < MT * 4; ++i) {
    const int r = 4 * i + (lane >> 4), m = min(m0 + r, a.M - 1);
    xs[i] = reinterpret_cast<const uint8_t*>(a.x + m * a.ld) + sb * 256 + ((l15 ^ (r & 15)) << 4);
  }
  const int wrow = ((lane >> 2) & 3) * 8 + (lane >> 4);
  const uint8_t* wcol = a.codes + (int64_t)tile * 64 + (lane & 3) * 16;
  const uint8_t* scol = a.scales + tile * 4;
  const int64_t wld = (int64_t)a.nb * 16;
  // weight rows behind the end read the last row: the activations there are zeros
  auto issue = [&](int t) {
    uint8_t* st = ring + (t % S) * kStage;
    const int nn = (sb + t) * 128;
#pragma unroll
    for (int i = 0; i < MT * 4; ++i) lds_dma16(xs[i] + t * 256, st + i * 1024);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      lds_dma16(wcol + min(nn + wrow + 4 * (j & 1) + 32 * (j >> 1), a.N - 1) * wld, st + kX + j * 1024);
#pragma unroll
    for (int j = 0; j < 2; ++j) lds_dma4(scol + (int64_t)min(nn + 64 * j + lane, a.N - 1) * a.nb, st + kX + kW + j * 256);
  };
  f32x4 acc[MT][8];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const unsigned turn = 8 * (l15 >> 2) + 9;  // rotates the scale byte of this lane's block to a float's exponent
  auto use = [&](const u32x2 (&w)[8], const u32x4 (&s)[4], const u32x4 (&x)[MT][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      union {
        u16x8 v;
        unsigned w[4];
      } row[8], f;  // row[r].w[q]: columns 2 q, 2 q + 1 of weight row r
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const unsigned b = s[2 * h + (r >> 2)][r & 3];
        row[r].v = mx_fragment(w[4 * h + (r >> 1)][r & 1], __uint_as_float(__builtin_amdgcn_alignbit(b, b, turn) & 0x7f800000u));
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
#pragma unroll
        for (int q = 0; q < 4; ++q)  // rows 2 q, 2 q + 1 of column c
          f.w[q] = __builtin_amdgcn_perm(row[2 * q + 1].w[c >> 1], row[2 * q].w[c >> 1], (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][c] = mfl::mma16<bf16_t>(__builtin_bit_cast(u16x8, x[i][h]), f.v, acc[i][c]);
      }
    }
  };
  const unsigned base = mfl::lds_addr(ring);
  for (int t = 0; t < S - 1 && t < n; ++t) issue(t);
  for (int t = 0; t < n; ++t) {
    if (t + S - 1 < n) issue(t + S - 1);
    const int ahead = n - 1 - t;
    if (ahead >= S - 1) mx_wait_vm<(S - 1) * L>();
    else if (S > 2 && ahead == 1) mx_wait_vm<L>();
    else mx_wait_vm<0>();
    const unsigned at = base + (t % S) * kStage;
    const unsigned wa = at + kX + g * 64 + l15 * 4, sa = at + kX + kW + g * 32, xr = at + l15 * 256;
    u32x2 w[8];
    u32x4 s[4], x[MT][2];
    mx_read_nn<0>(wa, sa, xr + ((g ^ l15) << 4), xr + (((4 + g) ^ l15) << 4), w, s, x);
    use(w, s, x);
    mx_read_nn<2>(wa, sa, xr + (((8 + g) ^ l15) << 4), xr + (((12 + g) ^ l15) << 4), w, s, x);
    use(w, s, x);
  }
  __syncthreads();  // the rings become the partial tiles
  constexpr int kTile = MT * 16 * 128;
  float* part = reinterpret_cast<float*>(lds);
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
  for (int t = threadIdx.x; t < kTile; t += kLdsWaves * 64) {
    const int m = m0 + (t >> 7), k = k0 + (t & 127);
    if (m >= a.M || k >= a.cols) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kLdsWaves; ++w) sum += part[w * kTile + t];
    st1<O>(y + (int64_t)m * a.cols + k, sum);
  }
}

// ---- the data gradient in tiles of 32 MI rows -------------------------------------------------------------
// As the forward's 128-column tiles: 8 waves share the ring, waves 4 i + q own the i-th half of the rows and the q-th 32
// weight rows of a stage, all 128 columns; the decoding and the transposition of a fragment are paid once for MI of them.
// The four partial sums meet in LDS: wave q keeps the rows 4 g + q of every 16, 8 consecutive columns a lane.
template <int MI, typename O>
__global__ __launch_bounds__(512) void mx_nn_big_k(const MxArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int kX = MI * 8192, kW = 8192, kStage = kX + kW + 512, S = kBigStages;
  constexpr int L = MI + 1;  // DMA instructions of a wave and stage; waves 0 and 1 also bring the scales
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  const int wm = wave >> 2, q = wave & 3;
  int mb, tile;
  mx_tile(a, (a.M + 32 * MI - 1) / (32 * MI), (a.cols + kBigCols - 1) / kBigCols, &mb, &tile);
  const int k0 = tile * kBigCols, m0 = mb * 32 * MI;
  const int64_t piece = (int64_t)a.M * a.ld;
  const int groups = (a.N + 127) >> 7, n = a.pieces * groups;
  // rows behind the ends repeat the last one: outputs that are not stored, weight rows that meet zeros of x
  const uint8_t* xs[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int r = 4 * (wave * MI + i) + g, m = min(m0 + r, a.M - 1);
    xs[i] = reinterpret_cast<const uint8_t*>(a.x + (a.pieces - 1) * piece + m * a.ld) + ((l15 ^ (r & 15)) << 4);
  }
  const int wrow = 32 * (wave >> 1) + 8 * ((lane >> 2) & 3) + 4 * (wave & 1) + (lane >> 4), srow = 64 * wave + lane;
  const uint8_t* ws = a.codes + (int64_t)tile * 64 + (lane & 3) * 16;
  const uint8_t* ss = a.scales + tile * 4;
  const unsigned base = mfl::lds_addr(lds);
  int at = 0, slot = 0;  // the next stage's group of its piece, and its place
  auto issue = [&]() {
    const unsigned st = __builtin_amdgcn_readfirstlane(base + slot * kStage);
#pragma unroll
    for (int i = 0; i < MI; ++i) big_dma16(xs[i] + at * 256, st + (wave * MI + i) * 1024);
    big_dma16(ws + (int64_t)min(at * 128 + wrow, a.N - 1) * a.nb * 16, st + kX + wave * 1024);
    if (wave < 2) big_dma4(ss + (int64_t)min(at * 128 + srow, a.N - 1) * a.nb, st + kX + kW + wave * 256);
    slot = slot + 1 == S ? 0 : slot + 1;
    if (++at == groups) {
      at = 0;
#pragma unroll
      for (int i = 0; i < MI; ++i) xs[i] -= piece * 2;
    }
  };
  f32x4 acc[MI][8];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const unsigned turn = 8 * (l15 >> 2) + 9;  // rotates the scale byte of this lane's block to a float's exponent
  const unsigned xo = (16 * MI * wm + l15) * 256 + (((4 * q + g) ^ l15) << 4);
  const unsigned wo = kX + q * 2048 + g * 64 + l15 * 4, so = kX + kW + q * 128 + g * 32;
  for (int t = 0; t < S - 1 && t < n; ++t) issue();
  int use = 0;
  for (int t = 0; t < n; ++t) {
    if (t + 1 == n) mx_wait_vm<0>();
    else if (wave < 2) mx_wait_vm<L + 1>();
    else mx_wait_vm<L>();
    mfl::barrier_keep_vm();  // every wave's part of stage t is there, and stage t - 1 has been read
    asm volatile("" ::: "memory");  // no read moves up
    if (t + S - 1 < n) issue();
    const unsigned sb = base + use * kStage;
    use = use + 1 == S ? 0 : use + 1;
    u32x4 x[MI], s[2];
    union {
      u16x8 v;
      unsigned w[4];
    } row[8], f;  // row[r].w[p]: columns 2 p, 2 p + 1 of weight row r
    unsigned w[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) w[r] = lds_at<unsigned>(sb + wo + r * 256);
#pragma unroll
    for (int r = 0; r < 2; ++r) s[r] = lds_at<u32x4>(sb + so + r * 16);
#pragma unroll
    for (int i = 0; i < MI; ++i) x[i] = lds_at<u32x4>(sb + xo + i * 4096);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const unsigned b = s[r >> 2][r & 3];
      row[r].v = mx_fragment(w[r], __uint_as_float(__builtin_amdgcn_alignbit(b, b, turn) & 0x7f800000u));
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int p = 0; p < 4; ++p)  // rows 2 p, 2 p + 1 of column c
        f.w[p] = __builtin_amdgcn_perm(row[2 * p + 1].w[c >> 1], row[2 * p].w[c >> 1], (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int i = 0; i < MI; ++i) acc[i][c] = mfl::mma16<bf16_t>(__builtin_bit_cast(u16x8, x[i]), f.v, acc[i][c]);
    }
  }
  constexpr int H = MI / 2;  // 16-row fragments a round of the exchange
  f32x4* part = reinterpret_cast<f32x4*>(lds) + lane;
  O* y = static_cast<O*>(a.y);
  const int k = k0 + 8 * l15;
#pragma unroll
  for (int round = 0; round < 2; ++round) {
    __syncthreads();  // the ring, or the last round's sums, have been read
#pragma unroll
    for (int p = 0; p < 4; ++p) {  // wave q's sums for wave p, in the place that leaves q's own out
      if (p == q) continue;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const auto& v = acc[round * H + i];
        f32x4* to = part + ((wave * 3 + p - (p > q)) * H + i) * 128;
        to[0] = f32x4{v[0][p], v[1][p], v[2][p], v[3][p]};
        to[64] = f32x4{v[4][p], v[5][p], v[6][p], v[7][p]};
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const auto& v = acc[round * H + i];
      float sum[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) sum[c] = q == 0 ? v[c][0] : q == 1 ? v[c][1] : q == 2 ? v[c][2] : v[c][3];
      for (int p = 0; p < 4; ++p) {
        if (p == q) continue;
        const f32x4* from = part + (((4 * wm + p) * 3 + q - (q > p)) * H + i) * 128;
        const f32x4 lo = from[0], hi = from[64];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += lo[e], sum[4 + e] += hi[e];
      }
      const int m = m0 + 16 * (MI * wm + round * H + i) + 4 * g + q;
      if (m >= a.M) continue;
      O* to = y + (int64_t)m * a.cols + k;
      if (a.cols % 8 == 0) {
        if (k < a.cols) Vec8<O>::store(to, sum);
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (k + c < a.cols) st1<O>(to + c, sum[c]);
      }
    }
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
  const int64_t grid = std::min(kMxGridMax - 1, (rows * cols + kQThreads - 1) / kQThreads);
  if (grid == 0) return hipSuccess;
  HYP_DISPATCH_FLOAT(dtype, T, {
    hipLaunchKernelGGL((mx_join_k<T>), dim3(grid), dim3(kQThreads), 0, stream, part, pieces, rows, cols, pitch, bias,
                       static_cast<T*>(y));
  });
  return hipGetLastError();
}

namespace {

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename K>
hipError_t mx_launch(K kernel, int rows, int tiles, int waves, size_t lds, const MxArgs& a, hipStream_t stream) {
  const int64_t grid = (int64_t)rows * tiles;
  if (grid >= kMxGridMax) return hipErrorInvalidValue;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(waves * 64), lds, stream, a);
  return hipGetLastError();
}

// rows of a workgroup's tile
int mx_rows(int mt) { return mt > kMxBig ? 32 * (mt - kMxBig) : 16 * (mt % kMxLds); }

// row blocks (of M rows) whose activations, rows of `bytes`, take at most 2 MB
int mx_group(int M, int mt, int64_t bytes) {
  const int rows = mx_rows(mt);
  return rows == 0 ? 1 : (int)std::min<int64_t>(ceil_div(M, rows), std::max<int64_t>(1, (2 << 20) / (rows * bytes)));
}

bool mx_lds_ok(const uint8_t* scales, int nb) { return nb % 4 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0; }

}  // namespace

// Planning.  A variant is a tile, + kMxLds in its rows where the operands go through LDS (rows of whole groups of four
// blocks); 0 is decoding the weight and the tiled GEMM.  Every variant is priced by its workgroups' rounds over 256 CUs:
// a start, and for each round a part for its ends and a part for each stage of its reduction.  The prices (us) are fitted
// to every variant's time over 28 weights (N 768 .. 11008, K 768 .. 11008) and 16 numbers of rows (1 .. 4064), bf16; within
// 10 % for 8 shapes in 10.  Choosing by them costs 0.3 % (forward) and 0.1 % (gradient) more than the best
// variant of each shape, on average over the 448; 0.8 % and 1 % where rows are no whole groups, over 250 more (K 96 .. 4064).
// Measured, us, with what was chosen:
//   forward      rows   1     16    32    64    128   300   700   1500  4064    decoded: 128   700   1500  4064
//   4096 x 4096       4.6   4.8   5.6   7.3   10.0  22    34    55    128          29    55    78    128
//   11008 x 4096      6.8   7.1   9.4   17    23    35    69    150   366          50    133   231   368
//   768 x 2048        4.0   4.0   4.0   4.0   4.2   5.2   10    13    20           17    21    25    33
//   11008 x 2048      4.8   5.1   6.6   12    13    20    38    80    194          33    80    138   208
//   gradient (N -> K)
//   4096 -> 4096      13    14    14    15    17    26    36    63    134          29    57    84    134
//   11008 -> 4096     32    34    34    35    39    63    87    160   330          50    112   214   330
//   4096 -> 11008     15    16    16    18    27    42    80    175   378          50    139   241   378
//   768 -> 768        5.4   5.8   5.8   5.8   5.9   6.0   7.5   8.7   12           19    19    19    20
// (in tiles of at most 32 rows, 1500 rows take 99 us forward at 4096 x 4096 and 96 at 4096 -> 4096; without LDS the gradient
// takes 19 .. 21 there up to 100 rows).

// the tiled GEMM's 256 x 256 ping-pong tile (one workgroup a CU) or its 128 x 128 tile (one or two a CU), chosen by the
// rounds that their workgroups need: a 32-deep step of a round takes 0.92 / 0.62 us, a split another pass over fp32 partial
// sums.  Returns the choice's time, with the ends of a round apart from its steps.
double mx_gemm_plan(int M, int N, int K, int* tile, int* splits) {
  double best = 1e30;
  *tile = 3;
  *splits = 1;
  int64_t groups = 0;
  for (int t : {8, 3}) {
    const int b = t == 8 ? 256 : 128;
    if (t == 8 && (M < 256 || N < 256)) continue;
    const int64_t tiles = (int64_t)ceil_div(M, b) * ceil_div(N, b);
    for (int s : {1, 2, 4, 8}) {
      if (s > 1 && K / s < 512) break;
      const int slots = t == 8 ? 256 : 512;
      double us = (double)((tiles * s + slots - 1) / slots) * ceil_div(ceil_div(K, 32), s) * (t == 8 ? 0.92 : 0.62);
      if (s > 1) us += 4.0 + (double)M * N * 4.0 * (s + 1) / 4e6;
      if (us < best) {
        best = us;
        groups = tiles * s;
        *tile = t;
        *splits = s;
      }
    }
  }
  const int steps = ceil_div(ceil_div(K, 32), *splits);
  const double two = 5.9 + 0.52 * steps, one = 2.0 + 0.47 * steps;
  const double last = groups % 512 > 256 ? two : groups % 512 > 0 ? one : 0.0;
  return (*tile == 8 ? (double)((groups + 255) / 256) * (12.8 + 0.82 * steps) : (double)(groups / 512) * two + last) +
         (*splits > 1 ? 3.3 + (double)M * N * 4.0 * (*splits + 1) / 10e6 : 0.0);
}

namespace {

// decoding (2.5 bytes an element), and the GEMM of an [M, n] result over k
double decoded_us(int M, int n, int k, int64_t weight) {
  int tile, splits;
  return 5.7 + (double)weight * 0.375e-6 + mx_gemm_plan(M, n, k, &tile, &splits);
}

struct Price {
  double start, round, stage;
  double rounds(double n, int stages) const { return n * (round + stage * stages); }
};

// 128-column tiles of 128 rows (*mi 4), one workgroup a CU, or of 64 rows (*mi 2), one (`one`) or two (`two`)
double big_us(int M, int cols, int stages, const Price& p128, double lone, const Price& one, const Price& two, int* mi) {
  const double w4 = (double)ceil_div(M, 128) * ceil_div(cols, 128) / 256.0, w2 = (double)ceil_div(M, 64) * ceil_div(cols, 128) / 256.0;
  const double full = std::floor(w2 / 2), last = w2 - 2 * full;
  const double r4 = p128.start + p128.rounds(w4 <= 1 ? lone : std::ceil(w4), stages);  // (a lone round runs a little faster)
  const double o = one.rounds(1, stages), t = two.rounds(1, stages);
  const double r2 = one.start + full * t + (last > 1 ? o + 0.8 * (t - o) : last > 0 ? o : 0.0);
  *mi = r2 < r4 ? 2 : 4;
  return std::min(r2, r4);
}

// joining the pieces' products, which the 128-column tiles need not do
double join_us(int M, int cols, int pieces) { return pieces > 1 ? 2.5 + (double)M * cols * (4 * pieces + 4) / 3.5e6 : 0.0; }

int64_t rounds_of(int rows, int row_tile, int cols, int col_tile) {
  return ((int64_t)ceil_div(rows, row_tile) * ceil_div(cols, col_tile) + 255) / 256;
}

}  // namespace

void mx_nt_plan(int M, int N, int nb, int pieces, bool lds, int* mt, int* nt) {
  static const struct {
    int mt, nt;
    Price p;  // a stage: a group of four blocks, over the waves that share it
  } kTiles[] = {{2 + kMxLds, 4, {1.1, 2.4, 0.185}},    {2 + kMxLds, 2, {1.5, 1.75, 0.12}}, {1 + kMxLds, 4, {1.5, 1.65, 0.131}},
                {1 + kMxLds, 2, {2.8, 0.43, 0.0736}}, {1 + kMxLds, 1, {2.7, 0.43, 0.051}}, {2, 4, {0.95, 3.35, 0.271}},
                {1, 1, {3.45, 0.256, 0.0755}}};
  const int K = 32 * nb, rows = pieces * M;
  const double join = join_us(M, N, pieces);
  double best = 1e30;
  for (const auto& t : kTiles) {
    if (lds != (t.mt > kMxLds)) continue;  // (where both exist, through LDS is faster)
    const int tile = mx_rows(t.mt);
    const double us = join + t.p.start + t.p.rounds((double)rounds_of(rows, tile, N, 16 * t.nt), ceil_div(nb, 4));
    if (us < best) {
      best = us;
      *mt = t.mt;
      *nt = t.nt;
    }
  }
  if (lds) {
    int mi;
    const double us = big_us(M, N, nb / 4 * pieces, {0.6, 4.0, 0.91}, 0.94, {3.4, 0.25, 0.56}, {0.0, 2.5, 0.98}, &mi);
    if (us < best) {
      best = us;
      *mt = kMxBig + mi;
      *nt = kBigCols / 16;
    }
  }
  if (join + decoded_us(rows, N, K, (int64_t)N * K) < best) *mt = *nt = 0;
}

void mx_nn_plan(int M, int N, int nb, int pieces, bool lds, int* mt) {
  const int K = 32 * nb, all = pieces * M, stages = ceil_div(N, 128);
  const double join = join_us(M, K, pieces);
  // what goes through LDS takes whole stages; pieces are written padded, other activations have to be copied for it
  const double padding = pieces == 1 && N % 128 != 0 ? 2.5 + (double)M * N * 4 / 4.5e6 : 0.0;
  double best = join + 2.8 + (double)rounds_of(all, 16, K, 128) * std::max(1.2, 0.5 * N / 128);
  *mt = 1;
  auto take = [&](double us, int variant) {
    if (us < best) {
      best = us;
      *mt = variant;
    }
  };
  if (lds) {
    take(join + padding + 0.8 + Price{0.0, 3.15, 0.332}.rounds((double)rounds_of(all, 16, K, 128), stages), 1 + kMxLds);
    take(join + padding + 0.8 + Price{0.0, 4.1, 0.369}.rounds((double)rounds_of(all, 32, K, 128), stages), 2 + kMxLds);
    int mi;
    const double us = big_us(M, K, stages * pieces, {1.0, 5.0, 0.944}, 0.965, {4.2, 0.0, 0.675}, {0.0, 2.7, 1.13}, &mi);
    take(padding + us, kMxBig + mi);
  }
  take(join + decoded_us(all, K, N, (int64_t)N * K), 0);
}

hipError_t mx_nt(const void* x, const uint8_t* codes, const uint8_t* scales, int M, int N, int nb, const float* bias,
                 int out_dtype, void* y, hipStream_t stream, int mt, int nt, int pieces) {
  if (M == 0 || N == 0) return hipSuccess;
  if (mx_rows(mt) == 0 || nt <= 0 || (mt > kMxLds && !mx_lds_ok(scales, nb))) return hipErrorInvalidValue;
  MxArgs a{static_cast<const bf16_t*>(x), codes, scales, bias, y, M, N, nb, 0, 0, mx_group(M, mt, (int64_t)64 * nb), pieces};
  const int rows = ceil_div(M, mx_rows(mt)), tiles = ceil_div(N, 16 * nt);
#define HYP_MX_NT_BIG(MI)                                                                                      \
  if (mt == kMxBig + MI && nt == kBigCols / 16)                                                                \
    return out_dtype == kBF16  ? mx_launch(mx_nt_big_k<MI, bf16_t>, rows, tiles, 8, mx_big_bytes<MI>(), a, stream) \
           : out_dtype == kF16 ? mx_launch(mx_nt_big_k<MI, f16_t>, rows, tiles, 8, mx_big_bytes<MI>(), a, stream) \
                               : mx_launch(mx_nt_big_k<MI, float>, rows, tiles, 8, mx_big_bytes<MI>(), a, stream);
  HYP_MX_NT_BIG(2) HYP_MX_NT_BIG(4)
#undef HYP_MX_NT_BIG
  if (pieces != 1 || (out_dtype != kBF16 && out_dtype != kF32)) return hipErrorInvalidValue;
#define HYP_MX_NT(MT, NT)                                                                                      \
  if (mt == MT && nt == NT) {                                                                                  \
    const size_t lds = sizeof(float) * kMxWaves * MT * NT * 256;                                               \
    return out_dtype == kBF16 ? mx_launch(mx_nt_k<MT, NT, bf16_t>, rows, tiles, kMxWaves, lds, a, stream)      \
                              : mx_launch(mx_nt_k<MT, NT, float>, rows, tiles, kMxWaves, lds, a, stream);      \
  }
#define HYP_MX_NT_LDS(MT, NT)                                                                                  \
  if (mt == MT + kMxLds && nt == NT) {                                                                         \
    const size_t lds = mx_nt_lds_bytes<MT, NT>(3);                                                             \
    return out_dtype == kBF16 ? mx_launch(mx_nt_lds_k<MT, NT, 3, bf16_t>, rows, tiles, kLdsWaves, lds, a, stream) \
                              : mx_launch(mx_nt_lds_k<MT, NT, 3, float>, rows, tiles, kLdsWaves, lds, a, stream); \
  }
  HYP_MX_NT(1, 1) HYP_MX_NT(2, 4)
  HYP_MX_NT_LDS(1, 1) HYP_MX_NT_LDS(1, 2) HYP_MX_NT_LDS(1, 4) HYP_MX_NT_LDS(2, 2) HYP_MX_NT_LDS(2, 4)
#undef HYP_MX_NT
#undef HYP_MX_NT_LDS
  return hipErrorInvalidValue;
}

hipError_t mx_nn(const void* x, int64_t ld, const uint8_t* codes, const uint8_t* scales, int M, int N, int nb, int cols,
                 int out_dtype, void* y, hipStream_t stream, int mt, int pieces) {
  if (M == 0 || cols == 0) return hipSuccess;
  if (ld % 8 != 0 || mx_rows(mt) == 0) return hipErrorInvalidValue;
  MxArgs a{static_cast<const bf16_t*>(x), codes, scales, nullptr, y, M, N, nb, cols, ld, mx_group(M, mt, 2 * ld), pieces};
  const int rows = ceil_div(M, mx_rows(mt)), tiles = ceil_div(cols, 128);
  if (mt > kMxLds && (!mx_lds_ok(scales, nb) || ld % 128 != 0)) return hipErrorInvalidValue;
#define HYP_MX_NN_BIG(MI)                                                                                      \
  if (mt == kMxBig + MI)                                                                                       \
    return out_dtype == kBF16  ? mx_launch(mx_nn_big_k<MI, bf16_t>, rows, tiles, 8, mx_big_bytes<MI>(), a, stream) \
           : out_dtype == kF16 ? mx_launch(mx_nn_big_k<MI, f16_t>, rows, tiles, 8, mx_big_bytes<MI>(), a, stream) \
                               : mx_launch(mx_nn_big_k<MI, float>, rows, tiles, 8, mx_big_bytes<MI>(), a, stream);
  HYP_MX_NN_BIG(2) HYP_MX_NN_BIG(4)
#undef HYP_MX_NN_BIG
  if (pieces != 1 || (out_dtype != kBF16 && out_dtype != kF32)) return hipErrorInvalidValue;
  if (mt == 1) {
    const size_t lds = sizeof(float) * kMxWaves * 2048;
    return out_dtype == kBF16 ? mx_launch(mx_nn_k<bf16_t>, rows, tiles, kMxWaves, lds, a, stream)
                              : mx_launch(mx_nn_k<float>, rows, tiles, kMxWaves, lds, a, stream);
  }
#define HYP_MX_NN_LDS(MT, S)                                                                                   \
  if (mt == MT + kMxLds) {                                                                                     \
    const size_t lds = mx_nn_lds_bytes<MT>(S);                                                                 \
    return out_dtype == kBF16 ? mx_launch(mx_nn_lds_k<MT, S, bf16_t>, rows, tiles, kLdsWaves, lds, a, stream) \
                              : mx_launch(mx_nn_lds_k<MT, S, float>, rows, tiles, kLdsWaves, lds, a, stream); \
  }
  HYP_MX_NN_LDS(1, 3) HYP_MX_NN_LDS(2, 2)
#undef HYP_MX_NN_LDS
  return hipErrorInvalidValue;
}

}  // namespace hyp
