// Multi-tensor Adam / AdamW whose two moments are held in 8 bits: one launch for every parameter, and
// one more that decodes them.
//
// Blocks of 256 elements in memory order (a tensor's last block may be shorter) share one fp32 scale S for
// each moment, the block's largest magnitude.  The codes are companded, so that small elements of a
// block keep relative precision:
//   m:  int8 q in [-127, 127],  m = q |q| S / 127^2,   q = sign(m) round(127 (|m| / S)^(1/2))
//   v: uint8 q in [0, 255],     v = q^4 S / 255^4,     q = round(255 (v / S)^(1/4)), at least 1 where v > 0
// where a half goes to the lower code (levels 127^2 and 255^4 apart in a block; v > 0 never becomes 0, which would
// divide by eps alone).
// A scale below the smallest normal number is kept as 0 and its block as zeros; a scale that is not
// finite is kept as NaN: its block is NaN.
//
// The new moments m' = b1 m + (1 - b1) g and v' = b2 v + (1 - b2) g^2 are fp64, and so is the decision
// between two codes: the fp32 square roots only find k = floor(r), and |m'| becomes k + 1 where it is above the
// border S ((k + 1/2) / 127)^2 (v' above S ((k + 1/2) / 255)^4).  The codes are thus those of the exact
// formula, whatever the instructions' rounding.  The fp64 operations are those of the PyTorch path, one by
// one and uncontracted, so that scales and codes are the same bits on CPU and GPU (0.9 S + 0.1 g is
// often exactly halfway between two fp32 numbers, where a fused product would round the other way).
// The parameter's update uses the uncoded moments, in fp32 and with the reciprocal and square root instructions (1 ulp
// each); the PyTorch path computes it in fp64, so that parameters agree to a few roundings, not bit for bit.
//
// A half wave holds one block, 8 elements a lane; the block's maxima meet over the 32 lanes by lane
// exchanges in registers.  Per element: gradient 2 or 4 bytes, fp32 parameter 4 + 4 (+ 2 its bf16 / fp16
// copy), codes 2 + 2, scales 16 / 256.  Measured (MI355X): 180M bf16 parameters with masters 588 us (4.9 TB/s; a large copy
// reaches 5.1), 16.8M in 256 tensors 64 us, 6.8M fp32 in 52 tensors 28 us.  About 80 VALU slots an element keep the
// lanes nearly as busy as HBM; accesses of the masters past the caches gained 2% of the first, lost 7% of the second.
#include "hyp_common.h"
#include "hyp_kernels.h"

namespace hyp {
namespace {

constexpr int kThreads = 256;
constexpr int kLane = 8;  // elements a lane; 32 lanes hold a block
// 1 / 127^2 and 1 / 255^4: products with them, not quotients (PyTorch divides by a number with a product on the GPU and a
// quotient on the CPU, which differ in the last bit and, at those halves, in the scale)
constexpr double kUnitM = 1.0 / 16129.0, kUnitV = 1.0 / 4228250625.0;

struct Adam8Args {
  float lr, eps, wd, ln_b1, ln_b2;
  double b1, b2, l2;
  int adamw, zero_grad;
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// a tensor's address out of a table: global memory (the compiler would have to use flat accesses, which also
// occupy the LDS counter)
template <typename T>
__device__ __forceinline__ T* table_ptr(int64_t a) {
  typedef __attribute__((address_space(1))) T G;
  return (T*)reinterpret_cast<G*>(a);
}

template <typename T>
__device__ __forceinline__ void load_lane(const T* p, int left, float (&v)[8]) {
  if (left >= 8) {
    Vec8<T>::load(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? ld1<T>(p + i) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_lane(T* p, int left, const float (&v)[8]) {
  if (left >= 8) {
    Vec8<T>::store(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) st1<T>(p + i, v[i]);
  }
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int left) {
  if (left >= 8) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* p, int left, const uint32_t (&w)[2]) {
  if (left >= 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}
__device__ __forceinline__ int code_m(const uint2& w, int i) {  // sign-extended byte i
  return (int)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
}
__device__ __forceinline__ unsigned code_v(const uint2& w, int i) { return ((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 255u; }

// maximum over the 32 lanes of a half wave (non-negative floats order like their bits, NaN above all)
__device__ __forceinline__ unsigned half_max(unsigned v) {
#define HYP_DPP_MAX(CTRL) v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true));
  HYP_DPP_MAX(0xb1)   // lane ^ 1
  HYP_DPP_MAX(0x4e)   // lane ^ 2
  HYP_DPP_MAX(0x141)  // mirrored within 8
  HYP_DPP_MAX(0x140)  // mirrored within 16
#undef HYP_DPP_MAX
  return max(v, (unsigned)__builtin_amdgcn_ds_swizzle((int)v, 0x401f));  // lane ^ 16
}

__device__ __forceinline__ float kept_scale(unsigned bits) {
  if (bits < 0x00800000u) return 0.f;
  return __uint_as_float(bits >= 0x7f800000u ? 0x7fc00000u : bits);
}

// ptrs [6 + MASTER][T]: parameter PL, gradient G, m codes, v codes, m scales, v scales (, fp32 master)
template <typename G, typename PL, bool MASTER>
__global__ __launch_bounds__(kThreads) void adam8_mt_k(const int64_t* __restrict__ ptrs, const int64_t* __restrict__ sizes,
                                                       const int* __restrict__ blocks, int T, int chunk, Adam8Args a,
                                                       const float* __restrict__ lr_t, const float* __restrict__ step_t,
                                                       const float* __restrict__ inv_scale,
                                                       const float* __restrict__ found_inf) {
#pragma clang fp contract(off)
  const int t = blocks[2 * blockIdx.x], ck = blocks[2 * blockIdx.x + 1];
  const int64_t n = sizes[t];
  const int64_t start = (int64_t)ck * chunk, end = min(n, start + chunk);
  G* g = table_ptr<G>(ptrs[T + t]);
  if (found_inf != nullptr && *found_inf != 0.f) {  // an overflowed step is skipped
    if (a.zero_grad)
      for (int64_t i = start + threadIdx.x; i < end; i += kThreads) st1<G>(g + i, 0.f);
    return;
  }
  PL* pl = table_ptr<PL>(ptrs[t]);
  float* p = table_ptr<float>(MASTER ? ptrs[6 * T + t] : ptrs[t]);
  uint8_t* mq = table_ptr<uint8_t>(ptrs[2 * T + t]);
  uint8_t* vq = table_ptr<uint8_t>(ptrs[3 * T + t]);
  float* ms = table_ptr<float>(ptrs[4 * T + t]);
  float* vs = table_ptr<float>(ptrs[5 * T + t]);
  const float step = *step_t;
  const float lr = lr_t ? *lr_t : a.lr, gs = inv_scale ? *inv_scale : 1.f;
  const float lr1 = lr / -expm1f(step * a.ln_b1), rb2 = rsqrtf(-expm1f(step * a.ln_b2));
  const float decay = lr * a.wd;
  const double omb1 = 1.0 - a.b1, omb2 = 1.0 - a.b2;
  // the whole half wave follows the loop while its block begins before the end: lanes behind it hold zeros
  for (int64_t b0 = start + (threadIdx.x >> 5) * 256; b0 < end; b0 += kThreads * kLane) {
    const int64_t i0 = b0 + (threadIdx.x & 31) * kLane, blk = b0 >> 8;
    const int left = (int)min((int64_t)8, end - i0);  // <= 0 behind the end
    float pv[8], gv[8];
    uint2 mw = make_uint2(0u, 0u), vw = make_uint2(0u, 0u);
    load_lane<float>(p + i0, left, pv);
    load_lane<G>(g + i0, left, gv);
    mw = load_codes(mq + i0, left);
    vw = load_codes(vq + i0, left);
    const double m_step = (double)ms[blk] * kUnitM, v_step = (double)vs[blk] * kUnitV;
    double md[8], vd[8];
    unsigned m_top = 0, v_top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double gd = (double)(gv[i] * gs);
      if (!a.adamw) gd = gd + (double)pv[i] * a.l2;  // fp64: gradient and decay may cancel
      const int q = code_m(mw, i);
      const unsigned q2 = code_v(vw, i) * code_v(vw, i);
      md[i] = (double)(q * abs(q)) * m_step * a.b1 + gd * omb1;
      vd[i] = (double)(q2 * q2) * v_step * a.b2 + gd * gd * omb2;
      const float mf = (float)md[i], vf = (float)vd[i];
      m_top = max(m_top, __float_as_uint(mf) & 0x7fffffffu);
      v_top = max(v_top, __float_as_uint(vf) & 0x7fffffffu);
      if (a.adamw) pv[i] = fmaf(-decay, pv[i], pv[i]);
      pv[i] = fmaf(-lr1 * mf, __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(vf), rb2, a.eps)), pv[i]);
    }
    const float m_s = kept_scale(half_max(m_top)), v_s = kept_scale(half_max(v_top));
    const bool m_live = m_s > 0.f, v_live = v_s > 0.f;  // neither 0 nor NaN
    const float m_inv = m_live ? __builtin_amdgcn_rcpf(m_s) : 0.f, v_inv = v_live ? __builtin_amdgcn_rcpf(v_s) : 0.f;
    const double m_unit = (double)m_s * kUnitM, v_unit = (double)v_s * kUnitV;
    uint32_t mo[2] = {0u, 0u}, vo[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double x = fabs(md[i]), y = vd[i];
      const float km = fminf(floorf(__builtin_amdgcn_sqrtf((float)x * m_inv) * 127.f), 127.f);
      const int qm = (int)km + (x > m_unit * (double)(fmaf(km, km, km) + 0.25f));
      mo[i >> 2] |= ((unsigned)(md[i] < 0.0 ? -qm : qm) & 255u) << (8 * (i & 3));
      const float r = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)y * v_inv));
      const float kv = fminf(floorf(r * 255.f), 255.f), h = kv + 0.5f;
      const double h2 = (double)(h * h);
      const unsigned qv = (unsigned)kv + (y > v_unit * (h2 * h2));
      vo[i >> 2] |= (qv == 0u && y > 0.0 ? 1u : qv) << (8 * (i & 3));
    }
    if (!m_live) mo[0] = mo[1] = 0u;
    if (!v_live) vo[0] = vo[1] = 0u;
    if (left > 0) {
      store_lane<float>(p + i0, left, pv);
      if (MASTER) store_lane<PL>(pl + i0, left, pv);
      if (a.zero_grad) {
        const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        store_lane<G>(g + i0, left, zero);
      }
      store_codes(mq + i0, left, mo);
      store_codes(vq + i0, left, vo);
    }
    if ((threadIdx.x & 31) == 0) {
      ms[blk] = m_s;
      vs[blk] = v_s;
    }
  }
}

// ptrs [4][T]: m codes, v codes, m scales, v scales -> fp32 values at offs[t] of two dense vectors
__global__ __launch_bounds__(kThreads) void adam8_values_k(const int64_t* __restrict__ ptrs, const int64_t* __restrict__ sizes,
                                                           const int* __restrict__ blocks, const int64_t* __restrict__ offs,
                                                           int T, int chunk, float* __restrict__ mo, float* __restrict__ vo) {
  const int t = blocks[2 * blockIdx.x], ck = blocks[2 * blockIdx.x + 1];
  const int64_t n = sizes[t];
  const int64_t start = (int64_t)ck * chunk, end = min(n, start + chunk), at = offs[t];
  const uint8_t* mq = table_ptr<const uint8_t>(ptrs[t]);
  const uint8_t* vq = table_ptr<const uint8_t>(ptrs[T + t]);
  const float* ms = table_ptr<const float>(ptrs[2 * T + t]);
  const float* vs = table_ptr<const float>(ptrs[3 * T + t]);
  for (int64_t i0 = start + threadIdx.x * 4; i0 < end; i0 += kThreads * 4) {
    const int left = (int)min((int64_t)4, end - i0);
    uint32_t mw = 0, vw = 0;
    if (left >= 4) {
      mw = *reinterpret_cast<const uint32_t*>(mq + i0);
      vw = *reinterpret_cast<const uint32_t*>(vq + i0);
    } else {
      for (int i = 0; i < left; ++i) {
        mw |= (uint32_t)mq[i0 + i] << (8 * i);
        vw |= (uint32_t)vq[i0 + i] << (8 * i);
      }
    }
    const double m_step = (double)ms[i0 >> 8] * kUnitM, v_step = (double)vs[i0 >> 8] * kUnitV;
    float m[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = (int)(int8_t)(mw >> (8 * i));
      const unsigned w = (vw >> (8 * i)) & 255u, w2 = w * w;
      m[i] = (float)((double)(q * abs(q)) * m_step);
      v[i] = (float)((double)(w2 * w2) * v_step);
    }
    if (left >= 4) {
      *reinterpret_cast<f32x4u*>(mo + at + i0) = f32x4u{m[0], m[1], m[2], m[3]};
      *reinterpret_cast<f32x4u*>(vo + at + i0) = f32x4u{v[0], v[1], v[2], v[3]};
    } else {
      for (int i = 0; i < left; ++i) {
        mo[at + i0 + i] = m[i];
        vo[at + i0 + i] = v[i];
      }
    }
  }
}

}  // namespace

hipError_t adam8_multi_tensor(int grad_dtype, int param_dtype, const int64_t* ptrs, const int64_t* sizes,
                              const int* blocks, int nblocks, int T, int chunk, float lr, double b1, double b2, float eps,
                              double wd, int adamw, const float* lr_t, const float* step_t, const float* inv_scale,
                              const float* found_inf, hipStream_t stream, int zero_grad) {
  if (nblocks == 0) return hipSuccess;
  if (chunk % (kThreads * kLane) != 0) return hipErrorInvalidValue;  // whole blocks, 16-byte lanes
  Adam8Args a{lr, eps, (float)wd, (float)log(b1), (float)log(b2), b1, b2, wd, adamw, zero_grad};
  HYP_DISPATCH_FLOAT(grad_dtype, G, {
    if (param_dtype == kF32)
      hipLaunchKernelGGL((adam8_mt_k<G, float, false>), dim3(nblocks), dim3(kThreads), 0, stream, ptrs, sizes, blocks, T,
                         chunk, a, lr_t, step_t, inv_scale, found_inf);
    else if (param_dtype == kBF16)
      hipLaunchKernelGGL((adam8_mt_k<G, bf16_t, true>), dim3(nblocks), dim3(kThreads), 0, stream, ptrs, sizes, blocks, T,
                         chunk, a, lr_t, step_t, inv_scale, found_inf);
    else
      hipLaunchKernelGGL((adam8_mt_k<G, f16_t, true>), dim3(nblocks), dim3(kThreads), 0, stream, ptrs, sizes, blocks, T,
                         chunk, a, lr_t, step_t, inv_scale, found_inf);
  });
  return hipGetLastError();
}

hipError_t adam8_values(const int64_t* ptrs, const int64_t* sizes, const int* blocks, const int64_t* offs, int nblocks,
                        int T, int chunk, float* m, float* v, hipStream_t stream) {
  if (nblocks == 0) return hipSuccess;
  if (chunk % (kThreads * kLane) != 0) return hipErrorInvalidValue;
  hipLaunchKernelGGL(adam8_values_k, dim3(nblocks), dim3(kThreads), 0, stream, ptrs, sizes, blocks, offs, T, chunk, m, v);
  return hipGetLastError();
}

}  // namespace hyp
