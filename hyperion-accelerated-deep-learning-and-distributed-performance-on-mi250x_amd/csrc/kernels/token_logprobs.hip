// Log probabilities of given tokens, the entropy of each row and its most likely tokens, and the
// gradient of the first two into the logits.
//
// Per row of logits z with y = z / T, in base 2 (c = log2(e) / T, t_j = (z_j - m) c, m the row's
// largest logit; the difference first, so that a row of the type's lowest value stays finite), one
// pass with a running maximum:
//   s = sum 2^t_j,  u = sum 2^t_j t_j
//   logprob = (z_target - m) / T - log2 s ln 2,   H = (log2 s - u / s) ln 2
// and from the saved (m, log2 s, H), with q_j = t_j - log2 s, p_j = 2^q_j:
//   dz_j = [ dlogp (delta_j - p_j) - dH p_j (q_j ln 2 + H) ] / T
// Sums are fp32.  The forward reads every logit once, the backward reads it once and writes its
// gradient once: HBM bounds both, with about 11 VALU slots per logit (exp2 takes 4 of them) close behind.
// Measured, bf16: 2032 x 50257 forward 38 us (5.4 TB/s); 4064 x 50257 forward 112 us and backward 139 us under a profiler,
// 240 together in a loop (5.1 TB/s, a large copy's rate; reading the first rows past the last-level cache, or the rows backwards in the
// backward, changed nothing); one row with 20 alternatives 12 us, of which the launch is 3.
//
// Rows start at any element (V = 50257 rows of 2-byte logits are 2-byte aligned).  The forward reads the
// 16-byte aligned part of a row in 16-byte pieces; the backward, whose logits and gradient rows need not
// have the same alignment, loads and stores 16 bytes at the row's own.
//
// An empty row (every logit -inf) has logprob -inf, entropy 0 and no gradient; a NaN or +inf logit
// makes its row's results and gradient NaN; a target outside [0, V) is never read and makes the
// row's logprob and gradient NaN; a row whose target is ignore_index is not read: 0 everywhere, ids -1.
#include <type_traits>

#include "hyp_common.h"
#include "hyp_kernels.h"

namespace hyp {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -200.f;  // 2^-200 is 0 in fp32: a finite stand-in for -inf in products with p = 0
constexpr int kTopCap = 1024;     // candidates of the top alternatives kept in LDS, and batches that hold them
constexpr int kTopStep = 128;     // ids looked at together for logits equal to the bound
constexpr int kTopPrefix = 7 * kTopStep;  // .. and at most: they fit beside fewer than k above it
static_assert(kTopPrefix + kTokenTopMax <= kTopCap, "candidates");

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4a __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at a row's own alignment

template <typename T>
struct Row16 {  // 16 bytes of a row
  static constexpr int N = 16 / (int)sizeof(T);
  static __device__ __forceinline__ u32x4 raw(const T* p) { return *reinterpret_cast<const u32x4a*>(p); }
  static __device__ __forceinline__ void open(const u32x4& r, float (&v)[N]);
};
template <>
__device__ __forceinline__ void Row16<float>::open(const u32x4& r, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
template <>
__device__ __forceinline__ void Row16<bf16_t>::open(const u32x4& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(r[i] << 16);
    v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void Row16<f16_t>::open(const u32x4& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = f16_lo(r[i]);
    v[2 * i + 1] = f16_hi(r[i]);
  }
}

__device__ __forceinline__ u32x4a close16(const float (&v)[4], const float*) {
  return u32x4a{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ u32x4a close16(const float (&v)[8], const bf16_t*) {
  return u32x4a{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ u32x4a close16(const float (&v)[8], const f16_t*) {
  return u32x4a{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7])};
}

// running (m, s, u) of a set of logits: m the largest logit, s = sum 2^((z - m) c), u = sum of the
// same weighted by its exponent.  NaN stays in s; m = -inf with s = 0 is the empty set.
struct Run {
  float m, s, u;
};

__device__ __forceinline__ Run run_join(const Run& a, const Run& b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = a.m == m ? 0.f : (a.m - m) * c, db = b.m == m ? 0.f : (b.m - m) * c;
  const float fa = exp2f(da), fb = exp2f(db);
  return {m, a.s * fa + b.s * fb, fa * (a.u + fmaxf(da, kFloor) * a.s) + fb * (b.u + fmaxf(db, kFloor) * b.s)};
}

// takes `mx`, the largest of the logits to be added next, into the running maximum
__device__ __forceinline__ void run_raise(Run& r, float mx, float c) {
  if (mx > r.m) {  // also the first values: from m = -inf the old sums are 0
    const float d = (r.m - mx) * c, f = exp2f(d);
    r.u = f * (r.u + fmaxf(d, kFloor) * r.s);
    r.s *= f;
    r.m = mx;
  }
}
// adds N logits that are not above the running maximum
template <int N>
__device__ __forceinline__ void run_add(Run& r, const float (&v)[N], float c) {
  const float at = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = (v[i] - at) * c, e = __builtin_amdgcn_exp2f(t);
    r.s += e;
    r.u = fmaf(e, fmaxf(t, kFloor), r.u);
  }
}
template <int N>
__device__ __forceinline__ float largest(const float (&v)[N]) {
  float mx = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = fmaxf(mx, v[i]);
  return mx;
}

// order of the alternatives: larger logit first (NaN above everything, -0 = +0), then the lower id.  Every key is below
// ~0, the sweeps' start, and above 0: the row's k <= V keys are distinct, so each of k sweeps finds one.
__device__ __forceinline__ uint64_t top_key(float z, int id) {
  const uint32_t b = __float_as_uint(z + 0.f);
  uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (z != z) k = 0xfffffffeu;
  return ((uint64_t)k << 32) | (0xffffffffu - (uint32_t)id);
}
__device__ __forceinline__ uint64_t shfl_max64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}

struct LpArgs {
  const void* z;
  int64_t s0, s1;  // element strides of row r: (r / inner) * s0 + (r % inner) * s1
  int inner, V;
  const int64_t* target;
  int64_t ignore;
  float c, inv_t;
  float *logp, *ent, *stats;  // stats [rows, 3]: m, log2 s, H; null without a backward to come
  int k;
  float* top_lp;
  int64_t* top_id;
};

template <typename T>
__device__ __forceinline__ const T* row_ptr(const LpArgs& a, int64_t r) {
  return static_cast<const T*>(a.z) + (r / a.inner) * a.s0 + (r % a.inner) * a.s1;
}

// the r-th largest of the 64 lanes' values (with repetitions), in every lane
__device__ __forceinline__ float wave_rth(float v, int r) {
  const int lane = threadIdx.x & 63;
  bool in = true;
  float top = 0.f;
  for (int i = 0; i < r; ++i) {
    top = wave_max(in ? v : -INFINITY);
    const uint64_t who = __ballot(in && v == top);
    if (who != 0 && lane == __ffsll((unsigned long long)who) - 1) in = false;
  }
  return top;
}

// One workgroup per row: up to 15 elements before the first and behind the last 16-byte boundary, one to a
// thread, and the aligned body in batches of U loads a thread (a long read reaches 6.2 TB/s aligned, 5.2
// at odd elements).
// TOP: also the k most likely tokens.
//   1. during the pass every batch's largest logit goes to LDS; with r = floor(k / full waves) + 1, T is the
//      smallest of the full waves' r-th largest thread maxima: at least k + 1 logits are >= T, so that k are above it where
//      no two are equal;
//   2. the batches that hold more than T (their maxima say which, nothing is read again for it) are read
//      again, a few dozen, and their logits above T become candidates;
//   3. if these are fewer than k, logits equal to T follow in the order of their ids: those of the first 896 ids, which
//      hold a mask's value often enough, else all of them, where the batches that hold T are few;
//   4. every candidate writes itself to the place given by how many are larger.
//   Where that does not serve (a NaN or +inf in the row, more candidates than fit, ties elsewhere), k sweeps
//   over the row pick one maximum each.
template <typename T, int THREADS, int U, bool TOP>
__global__ __launch_bounds__(THREADS) void token_lp_fwd_k(const LpArgs a) {
  constexpr int N = Row16<T>::N, W = THREADS / 64;
  extern __shared__ float batch_max[];  // TOP: [iterations][THREADS]
  __shared__ Run wr[W];
  __shared__ uint64_t cand[TOP ? kTopCap : 1];
  __shared__ int batches[TOP ? kTopCap : 1];
  __shared__ uint64_t wkey[TOP ? W : 1];
  __shared__ float wtop[TOP ? W : 1];
  __shared__ int nbatch, ncand;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t tgt = a.target[row];
  if (tgt == a.ignore) {
    if (tid == 0) {
      a.logp[row] = 0.f;
      a.ent[row] = 0.f;
      if (a.stats) a.stats[3 * row] = a.stats[3 * row + 1] = a.stats[3 * row + 2] = 0.f;
    }
    if (TOP && tid < a.k) {
      a.top_lp[row * a.k + tid] = 0.f;
      a.top_id[row * a.k + tid] = -1;
    }
    return;
  }
  const T* z = row_ptr<T>(a, row);
  const int head = min(a.V, (int)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int)sizeof(T));
  const int nv = (a.V - head) / N, tail = head + nv * N;  // 16-byte pieces; elements [0, head) and [tail, V) are single
  const u32x4* body = reinterpret_cast<const u32x4*>(z + head);
  const bool has_one = tid < a.V - tail + head;           // (differences first: V may be close to 2^31)
  const int one = tid < head ? tid : has_one ? tail + (tid - head) : 0;  // this thread's single element, if any
  const float lone = has_one ? ld1<T>(z + one) : -INFINITY;
  Run run{-INFINITY, 0.f, 0.f};
  float best = -INFINITY;
  int it = 0;
  auto batch = [&](int v0, auto whole) {  // pieces v0, v0 + THREADS, ...; whole: all U of them exist
    u32x4 r[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      r[i] = u32x4{0u, 0u, 0u, 0u};
      if (whole || v0 + i * THREADS < nv)
        r[i] = body[v0 + i * THREADS];
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (!whole && v0 + i * THREADS >= nv) break;
      float x[N];
      Row16<T>::open(r[i], x);
      top = fmaxf(top, largest<N>(x));
    }
    run_raise(run, top, a.c);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (!whole && v0 + i * THREADS >= nv) break;
      float x[N];
      Row16<T>::open(r[i], x);
      run_add<N>(run, x, a.c);
    }
    if (TOP) {
      batch_max[it * THREADS + tid] = top;
      best = fmaxf(best, top);
    }
    ++it;
  };
  const int whole_end = nv / (U * THREADS) * (U * THREADS);
  for (int v0 = tid; v0 < whole_end; v0 += U * THREADS) batch(v0, std::true_type{});
  if (whole_end + tid < nv) batch(whole_end + tid, std::false_type{});
  if (has_one) {
    const float x[1] = {lone};
    run_raise(run, lone, a.c);
    run_add<1>(run, x, a.c);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    run = run_join(run, Run{__shfl_xor(run.m, o, 64), __shfl_xor(run.s, o, 64), __shfl_xor(run.u, o, 64)}, a.c);
  if (lane == 0) wr[wv] = run;
  int full = 0;
  if (TOP) {
    full = min(W, nv / 64);  // waves whose every thread holds a piece
    if (wv < full) {
      const float t = wave_rth(best, a.k / full + 1);
      if (lane == 0) wtop[wv] = t;
    }
    if (tid == 0) nbatch = ncand = 0;
  }
  __syncthreads();
  run = lane < W ? wr[lane] : Run{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
    run = run_join(run, Run{__shfl_xor(run.m, o, 64), __shfl_xor(run.s, o, 64), __shfl_xor(run.u, o, 64)}, a.c);
  run = {__shfl(run.m, 0, 64), __shfl(run.s, 0, 64), __shfl(run.u, 0, 64)};
  const bool empty = run.s == 0.f;  // NaN is not
  const float m = empty ? 0.f : run.m, ls = empty ? INFINITY : __log2f(run.s);
  if (tid == 0) {
    float lp = __uint_as_float(0x7fc00000u);
    if (tgt >= 0 && tgt < a.V) lp = empty ? -INFINITY : fmaf(ld1<T>(z + tgt) - m, a.inv_t, -ls * kLn2);
    float h = empty ? 0.f : (ls - run.u / run.s) * kLn2;
    if (h < 0.f) h = 0.f;  // rounding, in a row of one token
    a.logp[row] = lp;
    a.ent[row] = h;
    if (a.stats) {
      a.stats[3 * row] = m;
      a.stats[3 * row + 1] = ls;
      a.stats[3 * row + 2] = h;
    }
  }
  if (!TOP) return;
  auto write = [&](int at, uint64_t key) {
    const int id = (int)(0xffffffffu - (uint32_t)key);
    a.top_id[row * a.k + at] = id;
    a.top_lp[row * a.k + at] = empty ? -INFINITY : fmaf(ld1<T>(z + id) - m, a.inv_t, -ls * kLn2);
  };
  auto put = [&](float x, int id) {
    const int at = atomicAdd(&ncand, 1);
    if (at < kTopCap) cand[at] = top_key(x, id);
  };
  // the logits of batches [b0, b1) of the list that `keep` takes become candidates
  auto take = [&](int b0, int b1, auto keep) {
    for (int i = tid; i < (b1 - b0) * U; i += THREADS) {
      const int b = batches[b0 + i / U], v = (b / THREADS) * (U * THREADS) + (i % U) * THREADS + b % THREADS;
      if (v >= nv) continue;
      float x[N];
      Row16<T>::open(body[v], x);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (keep(x[j])) put(x[j], head + v * N + j);
    }
  };
  bool served = run.s == run.s;  // uniform, like every decision below
  if (served && full == 0) {  // a short row: every logit is a candidate
    for (int i = tid; i < a.V; i += THREADS) put(ld1<T>(z + i), i);
  } else if (served) {
    float bound = wtop[0];
    for (int i = 1; i < full; ++i) bound = fminf(bound, wtop[i]);
    for (int i = 0; i < it; ++i)
      if (batch_max[i * THREADS + tid] > bound) {
        const int at = atomicAdd(&nbatch, 1);
        if (at < kTopCap) batches[at] = i * THREADS + tid;
      }
    if (has_one && lone > bound) put(lone, one);
    __syncthreads();
    const int nb = nbatch;
    served = nb <= kTopCap;
    if (served) {
      take(0, nb, [&](float x) { return x > bound; });
      __syncthreads();
      const int above = ncand;
      __syncthreads();
      if (above < a.k) {
        bool few = true;
        for (int p0 = 0; few && p0 < min(a.V, kTopPrefix); p0 += kTopStep) {  // in order, and no more than it takes
          const int i = p0 + tid;
          if (tid < kTopStep && i < a.V) {
            const float x = ld1<T>(z + i);
            if (x == bound) put(x, i);
          }
          __syncthreads();
          few = ncand < a.k;
          __syncthreads();
        }
        if (few) {  // the places behind the first `above` are written anew
          if (tid == 0) ncand = above;
          for (int i = 0; i < it; ++i)
            if (batch_max[i * THREADS + tid] == bound) {
              const int at = atomicAdd(&nbatch, 1);
              if (at < kTopCap) batches[at] = i * THREADS + tid;
            }
          __syncthreads();
          if (has_one && lone == bound) put(lone, one);
          served = nbatch <= kTopCap;
          if (served) take(0, nbatch, [&](float x) { return x == bound; });
        }
      }
    }
  }
  __syncthreads();
  const int n = ncand;
  if (served && n >= a.k && n <= kTopCap) {
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t key = cand[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += cand[j] > key;
      if (rank < a.k) write(rank, key);
    }
    return;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < a.k; ++i) {
    uint64_t top = 0;
    for (int e = tid; e < a.V; e += THREADS) {
      const uint64_t k = top_key(ld1<T>(z + e), e);
      if (k < last && k > top) top = k;
    }
    top = shfl_max64(top);
    __syncthreads();
    if (lane == 0) wkey[wv] = top;
    __syncthreads();
    last = wkey[0];
    for (int j = 1; j < W; ++j) last = wkey[j] > last ? wkey[j] : last;
    if (tid == 0) write(i, last);
  }
}

constexpr int kBwdThreads = 256, kBwdU = 4;

// A workgroup writes kBwdThreads * kBwdU 16-byte pieces of one row's gradient.
template <typename T>
__global__ __launch_bounds__(kBwdThreads) void token_lp_bwd_k(const LpArgs a, const float* __restrict__ dlogp,
                                                              const float* __restrict__ dent, T* __restrict__ dz,
                                                              int chunks) {
  constexpr int N = Row16<T>::N;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const int64_t tgt = a.target[row];
  const bool ignored = tgt == a.ignore;
  T* g = dz + row * a.V;
  const int nv = a.V / N, tail = nv * N;
  const bool lone = (int)threadIdx.x < a.V - tail;  // one of the last elements is this thread's (V may be close to 2^31)
  const int v0 = chunk * (kBwdThreads * kBwdU) + threadIdx.x;
  const float m = a.stats[3 * row], ls = a.stats[3 * row + 1], h = a.stats[3 * row + 2];
  float wl = 0.f, wh = 0.f;  // both 0 in an ignored or empty row
  if (!ignored && ls != INFINITY) {
    wl = dlogp ? dlogp[row] : 0.f;
    wh = dent ? dent[row] : 0.f;
    if (tgt < 0 || tgt >= a.V) wl = __uint_as_float(0x7fc00000u);
  }
  const float hot = wl * a.inv_t;
  // dz = -p (A + B q),  A = (wl + wh H) / T,  B = wh ln2 / T
  const float A = (wl + wh * h) * a.inv_t, B = wh * kLn2 * a.inv_t;
  auto grad = [&](float x, int id) {
    const float q = (x - m) * a.c - ls;
    const float d = -__builtin_amdgcn_exp2f(q) * fmaf(B, fmaxf(q, kFloor), A);
    return id == tgt ? d + hot : d;
  };
  if (ignored) {
    const u32x4a zero{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kBwdU; ++i) {
      const int v = v0 + i * kBwdThreads;
      if (v < nv) *reinterpret_cast<u32x4a*>(g + (int64_t)v * N) = zero;
    }
    if (chunk == 0 && lone) st1<T>(g + tail + threadIdx.x, 0.f);
    return;
  }
  const T* z = row_ptr<T>(a, row);
  u32x4 r[kBwdU];
#pragma unroll
  for (int i = 0; i < kBwdU; ++i) {
    const int v = v0 + i * kBwdThreads;
    if (v < nv) r[i] = Row16<T>::raw(z + (int64_t)v * N);
  }
#pragma unroll
  for (int i = 0; i < kBwdU; ++i) {
    const int v = v0 + i * kBwdThreads;
    if (v < nv) {
      float x[N];
      Row16<T>::open(r[i], x);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = grad(x[j], v * N + j);
      *reinterpret_cast<u32x4a*>(g + (int64_t)v * N) = close16(x, (const T*)nullptr);
    }
  }
  if (chunk == 0 && lone)
    st1<T>(g + tail + threadIdx.x, grad(ld1<T>(z + tail + threadIdx.x), tail + threadIdx.x));
}

LpArgs lp_args(const void* z, int64_t s0, int64_t s1, int inner, int V, const int64_t* target, int64_t ignore,
               float inv_t) {
  LpArgs a{};
  a.z = z;
  a.s0 = s0;
  a.s1 = s1;
  a.inner = inner;
  a.V = V;
  a.target = target;
  a.ignore = ignore;
  a.inv_t = inv_t;
  a.c = inv_t * 1.4426950408889634f;
  return a;
}

}  // namespace

hipError_t token_logprobs_fwd(int dtype, const void* z, int64_t s0, int64_t s1, int inner, int64_t rows, int V,
                              const int64_t* target, int64_t ignore, float inv_t, float* logp, float* ent, float* stats,
                              int k, float* top_lp, int64_t* top_id, hipStream_t stream) {
  if (rows == 0) return hipSuccess;
  if (V < 1 || inner < 1 || k < 0 || k > kTokenTopMax || k > V || rows >= kTokenRowsMax || (k > 0 && V > kTokenTopVocab)) return hipErrorInvalidValue;
  LpArgs a = lp_args(z, s0, s1, inner, V, target, ignore, inv_t);
  a.logp = logp;
  a.ent = ent;
  a.stats = stats;
  a.k = k;
  a.top_lp = top_lp;
  a.top_id = top_id;
  // 1024 threads have a long row's loads in flight at once; 256 leave room for other rows' workgroups, and their reductions
  // and lists are shorter.  Wide where at most one row comes to a CU (256) and it is long, or, without alternatives, two.
  // Us with 256 / 1024 threads.  None: 64 x 32000 bf16 7.2 / 6.6, 64 x 20000 bf16 5.2 / 5.7, 256 x 50257 fp32 21 / 13; 400 x 32000
  // fp32 15.7 / 14.5, 264 x 50257 bf16 11.9 / 13.8, 700 x 50257 fp32 28.0 / 28.9.  Five alternatives: 200 x 80000 bf16 18.2 / 17.2,
  // 256 x 32000 fp32 13.0 / 14.4, 64 x 50257 fp32 15.3 / 13.4, 264 x 50257 fp32 21.7 / 23.2, 400 x 32000 bf16 13.0 / 20.6;
  // one x 50257 bf16 11.0 / 11.4, with 20 alternatives, of which a wave finds k / waves + 1 in turn, 12.6 / 12.3.
  const int64_t bytes = (int64_t)V * (dtype == kF32 ? 4 : 2);
  const bool wide = rows <= 256 ? bytes >= (k > 8 ? 100000 : k > 0 ? 150000 : 64000) : k == 0 && rows <= 512 && bytes >= 128000;
#define HYP_LP(TH, U, TOP)                                                                                             \
  do {                                                                                                                 \
    const int its = V / (Row16<T>::N * TH * U) + 1;                                                                    \
    hipLaunchKernelGGL((token_lp_fwd_k<T, TH, U, TOP>), dim3(rows), dim3(TH), TOP ? its * TH * sizeof(float) : 0, stream, a); \
  } while (0)
  HYP_DISPATCH_FLOAT(dtype, T, {
    if (k > 0) {
      if (wide) HYP_LP(1024, 8, true);
      else HYP_LP(256, (sizeof(T) == 4 ? 8 : 4), true);
    } else {
      if (wide) HYP_LP(1024, 4, false);
      else HYP_LP(256, 4, false);
    }
  });
#undef HYP_LP
  return hipGetLastError();
}

hipError_t token_logprobs_bwd(int dtype, const void* z, int64_t s0, int64_t s1, int inner, int64_t rows, int V,
                              const int64_t* target, int64_t ignore, float inv_t, const float* stats,
                              const float* dlogp, const float* dent, void* dz, hipStream_t stream) {
  if (rows == 0) return hipSuccess;
  if (V < 1 || inner < 1) return hipErrorInvalidValue;
  LpArgs a = lp_args(z, s0, s1, inner, V, target, ignore, inv_t);
  a.stats = const_cast<float*>(stats);
  HYP_DISPATCH_FLOAT(dtype, T, {
    const int per = kBwdThreads * kBwdU * Row16<T>::N;
    const int64_t chunks = ((int64_t)V + per - 1) / per;
    if (rows * chunks >= kTokenRowsMax) return hipErrorInvalidValue;
    hipLaunchKernelGGL((token_lp_bwd_k<T>), dim3(rows * chunks), dim3(kBwdThreads), 0, stream, a, dlogp, dent,
                       static_cast<T*>(dz), (int)chunks);
  });
  return hipGetLastError();
}

}  // namespace hyp
