// One AdamW step over many tensors, with states in 32 or in 8 bits.
//
// For every element of every tensor (torch.optim.AdamW's decoupled form):
//   g  = grad * min(1, max_norm / (|grad|_2 over all tensors + 1e-6))    (optional)
//   m += (1 - b1) (g - m);   v = b2 v + (1 - b2) g^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// HBM-bound: p and g are read and p written once in their own type, the states are
// read and written once: 28 bytes an element with 32-bit states, 16 with 8-bit ones
// (fp32 tensors; 22 and 10 for bf16). The norm reads g once more.
//
// 8-bit states: blocks of 256 consecutive elements of a tensor share one fp32 scale,
// absmax / 448, for m and one for sqrt(v); each element is an e4m3 number. The root
// halves v's span of magnitudes, so that the 18 octaves of e4m3 below a block's
// largest value cover 36 octaves of v; a root that is not 0 is never rounded to 0,
// since m / (0 + eps) would be a huge step. The block's largest value is held to 32
// bits (it is 448 times the scale), the others to half a step of 2^-4; the update
// itself uses m and v before they are rounded. Rounding is to nearest: the blocks'
// common growth and decay goes into the scales, so values do not stall where a single
// step's change is below half a step of the format.
//
// A warp takes blocks of 256: 8 elements a lane in two 16-byte loads (one for 16-bit
// tensors), the maxima by one integer reduction each, the arithmetic on packed pairs. The
// tensors' table (pointers and sizes) comes as a kernel argument, so that a launch needs
// no copy and can be captured.
#include <cuda_fp8.h>
#include <stdio.h>

#include <mutex>
#include <type_traits>

#include "soup_common.cuh"

namespace soup {
namespace {

constexpr int kBlock = 256;              // elements that share a scale
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kE4m3Max = 448.f;
constexpr float kMostV = 3.3e38f;        // second moments past 32 bits stay at their end,
constexpr float kMostRoot = 1.8e19f;     // with roots from here on

struct Tensor {
  void* p;
  const void* g;
  int64_t n;
  int block0;   // first state block
  int first;    // blocks of the tensors before it in this launch
};

template <int N>
struct Table {
  int count, blocks;
  Tensor t[N];
};

// CTAs of the step's kernel on an SM (40 to 48 registers a thread). Each warp takes one
// block and is done: CTAs then come in the order of memory. A grid of resident CTAs that
// stride over the tensors, or walk a run of them each, drifts apart, and DRAM serves many
// pages at a time: 8-bit states of 233 M bf16 elements took 407 us this way, 464 to 619
// us with resident CTAs of every depth tried, with or without a ring of cp.async copies.
// With exactly rounded codes (root_pair, to_codes) it is 417 to 425 us, 5.6 TB/s (8 warps a
// CTA 430, 16 453, 2 473); 100 M fp32 elements with 32-bit states 405 us, 6.9 TB/s.
__host__ __device__ constexpr int step_ctas(int es) { return es == 4 ? 10 : 12; }

struct Hyper {
  float one_minus_beta1, beta2, one_minus_beta2, eps, decay;  // decay: 1 - lr wd
  float one;  // an argument, so that a * b + c written as (a * b) * one + c keeps its two roundings
};

// What a step's elements share, left by adamw_coef_kernel.
struct Coefs {
  float step_size, root_scale, clip, pad;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

struct States {
  void* m;          // fp32, or e4m3
  void* v;          // fp32 v, or e4m3 sqrt(v)
  float* m_scale;   // [blocks]
  float* v_scale;
};

// The tensor that holds block c of the launch.
template <int N>
__device__ __forceinline__ int find_tensor(const Table<N>& tab, int c) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Pairs of elements in packed 32-bit arithmetic: one instruction for two.
__device__ __forceinline__ uint64_t f2_same(float x) { return f2_pack(x, x); }

// Eight consecutive elements as they lie in memory.
template <typename T>
struct Raw8 {
  static constexpr int kWords = 2 * (int)sizeof(T);
  uint32_t u[kWords];
  __device__ __forceinline__ void load(const T* p, int left, bool vec) {
    if (left >= 8 && vec) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p) + i / 4);
        u[i] = q.x;
        u[i + 1] = q.y;
        u[i + 2] = q.z;
        u[i + 3] = q.w;
      }
    } else {
      union {
        T t[8];
        uint32_t w[kWords];
      } r;
#pragma unroll
      for (int i = 0; i < 8; ++i) r.t[i] = i < left ? p[i] : Cvt<T>::from_f(0.f);
#pragma unroll
      for (int i = 0; i < kWords; ++i) u[i] = r.w[i];
    }
  }
  __device__ __forceinline__ uint64_t pair(int i) const {
    if constexpr (sizeof(T) == 4) {
      return f2_pack(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return f2_pack(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      return f2_pack(f.x, f.y);
    }
  }
  __device__ __forceinline__ void set(int i, uint64_t v) {
    float x, y;
    f2_unpack(v, x, y);
    if constexpr (sizeof(T) == 4) {
      u[2 * i] = __float_as_uint(x);
      u[2 * i + 1] = __float_as_uint(y);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
      u[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 h = __floats2half2_rn(x, y);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  __device__ __forceinline__ void store(T* p, int left, bool vec) const {
    if (left >= 8 && vec) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4)
        __stcs(reinterpret_cast<uint4*>(p) + i / 4, make_uint4(u[i], u[i + 1], u[i + 2], u[i + 3]));
    } else {
      union {
        T t[8];
        uint32_t w[kWords];
      } r;
#pragma unroll
      for (int i = 0; i < kWords; ++i) r.w[i] = u[i];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = r.t[i];
    }
  }
};

__device__ __forceinline__ uint64_t pair_of_codes(uint2 c, int i) {
  const uint32_t w = i < 2 ? c.x : c.y;
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * (i & 1))), __NV_E4M3);
  const float2 v = __half22float2(__half2(h));
  return f2_pack(v.x, v.y);
}

// Reciprocal and reciprocal root to 2^-22, subnormals as 0: the IEEE forms cost more
// instructions than all the rest.
__device__ __forceinline__ float recip_root_approx(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float recip_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Square roots of a pair of finite numbers, rounded as exact ones are but for rare last bits:
// one step of Newton's method, s + (x - s^2) / (2 sqrt(x)), from x times the approximate
// reciprocal root (of x + 2^-126, which leaves 0 its root and numbers above 2^-102 as they
// are; roots of smaller ones come out low, by kRootError at most).
constexpr double kRootError = 2.1e-20;
__device__ __forceinline__ uint64_t root_pair(uint64_t x) {
  float lo, hi;
  f2_unpack(f2_add(x, f2_same(1.17549435e-38f)), lo, hi);
  const uint64_t h = f2_pack(recip_root_approx(lo), recip_root_approx(hi));
  const uint64_t s = f2_mul(x, h);
  return f2_fma(f2_fma(s, s, f2_mul(x, f2_same(-1.f))), f2_mul(h, f2_same(-0.5f)), s);
}

// The same of every number: those below 2^-100 are scaled up by 2^64 first.
__device__ __forceinline__ uint64_t root_pair_tiny(uint64_t x) {
  constexpr float kLeast = 7.8886091e-31f;
  float lo, hi, r0, r1, s0, s1;
  f2_unpack(x, lo, hi);
  f2_unpack(root_pair(x), r0, r1);
  f2_unpack(f2_mul(root_pair(f2_mul(x, f2_same(1.8446744e19f))), f2_same(2.3283064e-10f)), s0, s1);
  return f2_pack(lo < kLeast ? s0 : r0, hi < kLeast ? s1 : r1);
}

// Scale of the warp's block and its codes. Values that are not finite are left out of
// the maximum (they must not wipe out the other 255): fmaxf passes NaN over, and a
// maximum that is infinite, which no sound step has, is taken again without them. Roots
// are of moments that were held below kMostV, NaN too: beside a root that large, which no
// sound step has either, those whose first moment is not finite become NaN and are left
// out. (As a number it would be the block's largest, and the other 255 its smallest code,
// beside which their steps are nothing.) The bits of numbers of 0 or more order as the
// numbers do, so one integer reduction of the warp gives the maximum.
template <bool ROOT>
__device__ __forceinline__ uint2 to_codes(uint64_t (&f)[4], const uint64_t (&first)[4], float& scale) {
  float v[8], top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f2_unpack(f[i], v[2 * i], v[2 * i + 1]);
    top = fmaxf(top, fmaxf(fabsf(v[2 * i]), fabsf(v[2 * i + 1])));
  }
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
  if (top >= (ROOT ? kMostRoot : __int_as_float(0x7f800000))) {  // warp-uniform
    if constexpr (ROOT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float lo, hi;
        f2_unpack(first[i], lo, hi);
        if (!(fabsf(lo) <= 3.4028235e38f)) v[2 * i] = __int_as_float(0x7fffffff);
        if (!(fabsf(hi) <= 3.4028235e38f)) v[2 * i + 1] = __int_as_float(0x7fffffff);
        f[i] = f2_pack(v[2 * i], v[2 * i + 1]);
      }
    }
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]) <= 3.4028235e38f ? fabsf(v[i]) : 0.f);
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
  }
  scale = top / kE4m3Max;
  uint64_t y[4];
  if (scale >= 1.17549435e-38f) {  // warp-uniform
    // quotients corrected by their remainder, as an exact division rounds them but for rare
    // last bits: which of two codes a value between them takes is then that of the formula
    const uint64_t inv = f2_same(recip_approx(scale)), minus = f2_same(-scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t q = f2_mul(f[i], inv);
      y[i] = f2_fma(f2_fma(q, minus, f[i]), inv, q);
    }
  } else {
    // no finite reciprocal: scaled up by 2^64 first (a block of zeros stays 0)
    const float inv = scale > 0.f ? 1.f / (scale * 1.8446744e19f) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = f2_pack(v[2 * i] * 1.8446744e19f * inv, v[2 * i + 1] * 1.8446744e19f * inv);
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2_unpack(y[i], lo, hi);
    w[i >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3) << (16 * (i & 1));
  }
  if constexpr (ROOT) {
    // roots that are not 0 and were rounded to it (rare: a code of 0 is looked for first)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if ((w[j] - 0x01010101u) & ~w[j] & 0x80808080u) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (((w[j] >> (8 * i)) & 0xffu) == 0 && v[4 * j + i] > 0.f) w[j] |= 1u << (8 * i);
      }
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ double block_sum(double v, double* share) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) share[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += share[i];
  return s;
}

// Sum of squares of the gradients: eight squares in 32 bits, then one partial a CTA in
// 64 bits (the clip coefficient scales every element, so its error is in all of them).
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) grad_square_kernel(const __grid_constant__ Table<N> tab,
                                                               double* __restrict__ partial) {
  __shared__ double share[kWarps];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0.0;
  constexpr int U = 4;  // blocks of a warp in flight
  for (int c = blockIdx.x * U * kWarps + warp; c < tab.blocks; c += gridDim.x * U * kWarps) {
    int ti = find_tensor(tab, c);  // (a turn may pass over hundreds of small tensors)
    Raw8<T> g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int blk = c + u * kWarps;
      int left = 0;
      const T* at = nullptr;
      bool vec = false;
      if (blk < tab.blocks) {
        while (ti + 1 < tab.count && tab.t[ti + 1].first <= blk) ++ti;
        const Tensor& t = tab.t[ti];
        const int64_t e = (int64_t)(blk - t.first) * kBlock + lane * 8;
        const int64_t rest = t.n - e;
        left = rest >= 8 ? 8 : rest < 0 ? 0 : (int)rest;
        at = static_cast<const T*>(t.g) + e;
        vec = (reinterpret_cast<uintptr_t>(t.g) & 15) == 0;
      }
      g[u].load(at, left, vec);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t sq = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sq = f2_fma(g[u].pair(i), g[u].pair(i), sq);
      float lo, hi;
      f2_unpack(sq, lo, hi);
      lo += hi;
      if (lo > 3.4028235e38f) {  // squares past 32 bits
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f2_unpack(g[u].pair(i), lo, hi);
          sum += (double)lo * lo + (double)hi * hi;
        }
      } else {
        sum += lo;
      }
    }
  }
  sum = block_sum(sum, share);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The coefficients of step t = *step + 1 and, from the sums of squares, the clip
// coefficient and the norm. `raise`: the step's last call, after which the count is t.
__global__ void __launch_bounds__(kThreads) adamw_coef_kernel(double lr, double log_beta1, double log_beta2,
                                                              double max_norm, const double* __restrict__ partial,
                                                              int partials, float* __restrict__ norm_out,
                                                              float* __restrict__ step, int raise,
                                                              Coefs* __restrict__ out) {
  __shared__ double share[kWarps];
  pdl_wait();
  pdl_trigger();
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += kThreads) sum += partial[i];
  sum = block_sum(sum, share);
  if (threadIdx.x != 0) return;
  const double t = (double)*step + 1.0;
  Coefs c;
  // 1 - b^t = -expm1(t log b): exact also in the first steps
  c.step_size = (float)(lr / -expm1(t * log_beta1));
  c.root_scale = (float)(1.0 / sqrt(-expm1(t * log_beta2)));
  c.clip = 1.f;
  c.pad = 0.f;
  if (partials > 0) {
    const double norm = sqrt(sum), k = max_norm / (norm + 1e-6);
    c.clip = k > 1.0 ? 1.f : (float)k;  // a norm that is not a number stays visible in every element
    if (norm_out) *norm_out = (float)norm;
  }
  *out = c;
  if (raise) *step = (float)t;
}

// The step: a warp a block. TINY: eps is so small that roots of second moments below
// 2^-102 count beside it (see step_run). As a branch for each pair of elements it took the
// other steps 24 of 418 us.
template <typename T, bool EIGHT, bool TINY, int N>
__global__ void __launch_bounds__(kThreads, step_ctas(sizeof(T))) adamw_multi_kernel(const __grid_constant__ Table<N> tab,
                                                                                 States st, Hyper h,
                                                                                 const Coefs* __restrict__ coefs) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * kWarps + warp;
  const int ti = find_tensor(tab, min(c, tab.blocks - 1));
  pdl_wait();
  pdl_trigger();
  if (c >= tab.blocks) return;  // warp-uniform; no barrier follows
  const float4 co = *reinterpret_cast<const float4*>(coefs);
  const uint64_t step_size = f2_same(-co.x), root_scale = f2_same(co.y), clip = f2_same(co.z);
  const uint64_t c1 = f2_same(h.one_minus_beta1), c2 = f2_same(h.one_minus_beta2), b2 = f2_same(h.beta2);
  const uint64_t eps = f2_same(h.eps), decay = f2_same(h.decay), one = f2_same(h.one), minus = f2_same(-h.one);
  const Tensor& t = tab.t[ti];
  const int64_t e = (int64_t)(c - t.first) * kBlock + lane * 8;
  const int64_t rest = t.n - e;
  const int left = rest >= 8 ? 8 : rest < 0 ? 0 : (int)rest;
  const int64_t blk = t.block0 + (c - t.first), at = blk * kBlock + lane * 8;
  const bool vg = (reinterpret_cast<uintptr_t>(t.g) & 15) == 0, vp = (reinterpret_cast<uintptr_t>(t.p) & 15) == 0;
  Raw8<T> p, g;
  Raw8<float> m32, v32;
  uint2 mc, vc;
  float ms = 0.f, vs = 0.f;
  g.load(static_cast<const T*>(t.g) + e, left, vg);
  p.load(static_cast<const T*>(t.p) + e, left, vp);
  if constexpr (EIGHT) {
    mc = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(st.m) + at));
    vc = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(st.v) + at));
    ms = st.m_scale[blk];
    vs = st.v_scale[blk];
  } else {
    m32.load(static_cast<const float*>(st.m) + at, 8, true);
    v32.load(static_cast<const float*>(st.v) + at, 8, true);
  }
  uint64_t m[4], v[4], root[4];
  const uint64_t msc = f2_same(ms), vsc = f2_same(vs);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (EIGHT) {
      m[i] = f2_mul(pair_of_codes(mc, i), msc);
      v[i] = f2_mul(pair_of_codes(vc, i), vsc);
      v[i] = f2_mul(v[i], v[i]);
    } else {
      m[i] = m32.pair(i);
      v[i] = v32.pair(i);
    }
    const uint64_t gi = f2_mul(g.pair(i), clip);
    // each operation of the moments rounds by itself, as elementwise tensor operations do:
    // what lies between two codes then goes the same way as there (one code off is a
    // sixteenth of a moment, or twice a small root)
    m[i] = f2_fma(f2_mul(c1, f2_fma(m[i], minus, gi)), one, m[i]);
    float lo, hi;
    f2_unpack(f2_fma(f2_mul(v[i], b2), one, f2_mul(c2, f2_mul(gi, gi))), lo, hi);
    v[i] = f2_pack(fminf(lo, kMostV), fminf(hi, kMostV));
    root[i] = TINY ? root_pair_tiny(v[i]) : root_pair(v[i]);
    f2_unpack(f2_fma(root[i], root_scale, eps), lo, hi);
    const uint64_t inv = f2_pack(recip_approx(lo), recip_approx(hi));
    p.set(i, f2_fma(f2_mul(m[i], step_size), inv, f2_mul(p.pair(i), decay)));
  }
  p.store(static_cast<T*>(t.p) + e, left, vp);
  if (left < 8) {
    // what lies behind a tensor's end stays 0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool a = 2 * i < left, b = 2 * i + 1 < left;
      float x, y;
      f2_unpack(m[i], x, y);
      m[i] = f2_pack(a ? x : 0.f, b ? y : 0.f);
      f2_unpack(v[i], x, y);
      v[i] = f2_pack(a ? x : 0.f, b ? y : 0.f);
      f2_unpack(root[i], x, y);
      root[i] = f2_pack(a ? x : 0.f, b ? y : 0.f);
    }
  }
  if constexpr (EIGHT) {
    float sm, sv;
    const uint2 cv = to_codes<true>(root, m, sv);
    const uint2 cm = to_codes<false>(m, m, sm);
    __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(st.m) + at), cm);
    __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(st.v) + at), cv);
    if (lane == 0) {
      st.m_scale[blk] = sm;
      st.v_scale[blk] = sv;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m32.set(i, m[i]);
      v32.set(i, v[i]);
    }
    m32.store(static_cast<float*>(st.m) + at, 8, true);
    v32.store(static_cast<float*>(st.v) + at, 8, true);
  }
}

// What a DLPack exchange interface fills in for a tensor (DLTensor of DLPack 1).
struct DlTensor {
  void* data;
  int32_t device_type, device;
  int32_t ndim;
  uint8_t type_code, type_bits;
  uint16_t lanes;
  const int64_t* shape;
  const int64_t* strides;
  uint64_t byte_offset;
};
constexpr int kDlFloat = 2, kDlBfloat = 4;

// t is dense in the order of its axes and has n elements of that type on that device.
bool dense_tensor(const DlTensor& t, int64_t n, int dtype, int device_type, int device) {
  if (t.device_type != device_type || t.device != device || t.lanes != 1 ||
      t.type_code != (dtype == SOUP_BF16 ? kDlBfloat : kDlFloat) || t.type_bits != (dtype == SOUP_F32 ? 32 : 16))
    return false;
  int64_t e = 1;
  bool dense = true;
  for (int d = t.ndim - 1; d >= 0; --d) {
    if (t.shape[d] != 1 && t.strides && t.strides[d] != e) dense = false;
    e *= t.shape[d];
  }
  return dense && e == n && t.data;
}

constexpr int kSquareCtas = 12;             // of grad_square_kernel on an SM, each with a partial sum
constexpr int kSmall = 64, kLarge = 960;  // tensors of a launch: arguments of 2 and 30 KB

inline int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

// CTAs of a launch: a block for every warp, as far as they are resident together
inline int grid_of(int blocks, int per_sm) {
  const int cap = num_sms() * per_sm, want = (blocks + kWarps - 1) / kWarps;
  return want < cap ? want : cap;
}

struct Args {
  void* const* params;
  const void* const* grads;
  const int64_t* sizes;
  const int32_t* blocks;
  int count;
};

// Tensors [i0, i1) into a table.
template <int N>
void fill_table(Table<N>& tab, const Args& a, int i0, int i1) {
  int blocks = 0;
  for (int i = i0; i < i1; ++i) {
    tab.t[i - i0] = Tensor{a.params ? a.params[i] : nullptr, a.grads[i], a.sizes[i], a.blocks ? a.blocks[i] : 0, blocks};
    blocks += (int)blocks_of(a.sizes[i]);
  }
  tab.count = i1 - i0;
  tab.blocks = blocks;
}

// The end of the launch that starts with tensor i0: at most `most` tensors and 2^30 blocks
// (a tensor has at most as many).
int launch_end(const Args& a, int i0, int most) {
  int64_t blocks = 0;
  int i = i0;
  while (i < a.count && i - i0 < most) {
    blocks += blocks_of(a.sizes[i]);
    if (i > i0 && blocks > (1 << 30)) break;
    ++i;
  }
  return i;
}

// A launch that takes the table by reference (launch_pdl would copy its 30 KB twice).
template <typename... KArgs, typename... PArgs>
int launch_table(void (*kernel)(KArgs...), int grid, cudaStream_t st, const PArgs&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* ptrs[] = {const_cast<void*>(static_cast<const void*>(&args))...};
  return cuda_status(cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), ptrs));
}

template <typename T, int N>
int square_launch(const Args& a, int i0, int i1, double* partial, int* used, cudaStream_t st) {
  Table<N> tab;
  fill_table(tab, a, i0, i1);
  const int grid = grid_of(tab.blocks, kSquareCtas);
  *used += grid;
  return launch_table(grad_square_kernel<T, N>, grid, st, tab, partial);
}

template <typename T, bool EIGHT, bool TINY, int N>
int step_launch(const Args& a, int i0, int i1, const States& s, const Hyper& h, const Coefs* coefs, cudaStream_t st) {
  Table<N> tab;
  fill_table(tab, a, i0, i1);
  const int grid = (tab.blocks + kWarps - 1) / kWarps;
  return launch_table(adamw_multi_kernel<T, EIGHT, TINY, N>, grid, st, tab, s, h, coefs);
}

int check_tensors(const char* fn, const Args& a, bool step) {
  bool ok = a.grads && a.sizes && a.count > 0 && (!step || (a.params && a.blocks));
  for (int i = 0; ok && i < a.count; ++i)
    ok = a.grads[i] && a.sizes[i] > 0 && a.sizes[i] <= (int64_t(1) << 38) &&
         (!step || (a.params[i] && a.blocks[i] >= 0));
  if (ok) return SOUP_OK;
  char msg[96];
  snprintf(msg, sizeof(msg), "%s: bad tensor table", fn);
  set_last_error(msg);
  return SOUP_ERR_INVALID;
}

template <typename T>
int square_run(const Args& a, double* partial, int cap, int* used, cudaStream_t st) {
  const int most = a.count <= kSmall ? kSmall : kLarge;
  for (int i0 = 0; i0 < a.count;) {
    const int i1 = launch_end(a, i0, most);
    if (*used + num_sms() * kSquareCtas > cap) {
      set_last_error("soup_grad_square: workspace too small");
      return SOUP_ERR_WORKSPACE;
    }
    double* at = partial + *used;
    const int rc = most == kSmall ? square_launch<T, kSmall>(a, i0, i1, at, used, st)
                                  : square_launch<T, kLarge>(a, i0, i1, at, used, st);
    if (rc) return rc;
    i0 = i1;
  }
  return SOUP_OK;
}

template <typename T, bool EIGHT, bool TINY>
int step_run(const Args& a, const States& s, const Hyper& h, const Coefs* coefs, cudaStream_t st) {
  const int most = a.count <= kSmall ? kSmall : kLarge;
  for (int i0 = 0; i0 < a.count;) {
    const int i1 = launch_end(a, i0, most);
    const int rc = most == kSmall ? step_launch<T, EIGHT, TINY, kSmall>(a, i0, i1, s, h, coefs, st)
                                  : step_launch<T, EIGHT, TINY, kLarge>(a, i0, i1, s, h, coefs, st);
    if (rc) return rc;
    i0 = i1;
  }
  return SOUP_OK;
}

// Below 2^-102 root_pair's roots are low by kRootError at most, times 1 / sqrt(1 - b2) in the
// denominator: less than a rounding of eps where eps is larger than this (1e-11 for b2 of
// 0.999). Steps with a smaller eps take the roots of every number (442 us for 233 M bf16
// elements, 418 without).
template <typename T, bool EIGHT>
int step_run(const Args& a, const States& s, const Hyper& h, double beta2, const Coefs* coefs, cudaStream_t st) {
  const bool tiny = h.eps * 5.9604645e-8 < kRootError / sqrt(1.0 - beta2);
  return tiny ? step_run<T, EIGHT, true>(a, s, h, coefs, st) : step_run<T, EIGHT, false>(a, s, h, coefs, st);
}

}  // namespace
}  // namespace soup

using namespace soup;

extern "C" {

int soup_tensor_addresses(void* const* reader, void* list, const int64_t* sizes, int count, int dtype, int device_type,
                          int device, uint64_t* addresses) {
  if (!reader || !reader[0] || !reader[1] || !list || !sizes || count <= 0 || !addresses ||
      (dtype != SOUP_F32 && dtype != SOUP_BF16 && dtype != SOUP_F16)) {
    set_last_error("soup_tensor_addresses: bad arguments");
    return SOUP_ERR_INVALID;
  }
  const auto fill = reinterpret_cast<int (*)(void*, DlTensor*)>(reader[0]);
  const auto item = reinterpret_cast<void* (*)(void*, intptr_t)>(reader[1]);
  for (int i = 0; i < count; ++i) {
    void* object = item(list, i);
    DlTensor t{};
    if (!object || object == reader[2] || fill(object, &t) != 0 ||
        !dense_tensor(t, sizes[i], dtype, device_type, device))
      return -1 - i;
    addresses[i] = reinterpret_cast<uint64_t>(t.data) + t.byte_offset;
  }
  return SOUP_OK;
}

size_t soup_grad_square_workspace_bytes(int64_t tensors) {
  if (tensors <= 0) return 0;
  return sizeof(double) * kSquareCtas * (size_t)num_sms() * (size_t)((tensors + kLarge - 1) / kLarge);
}

int soup_grad_square(const void* const* grads, const int64_t* sizes, int count, int dtype, void* workspace,
                     size_t workspace_bytes, int* partials, void* stream) {
  const Args a{nullptr, grads, sizes, nullptr, count};
  if (int rc = check_tensors("soup_grad_square", a, false)) return rc;
  if (!workspace || !aligned16(workspace) || !partials || *partials < 0) {
    set_last_error("soup_grad_square: bad arguments");
    return SOUP_ERR_INVALID;
  }
  double* ws = static_cast<double*>(workspace);
  const int cap = (int)(workspace_bytes / sizeof(double) > (1u << 30) ? (1u << 30) : workspace_bytes / sizeof(double));
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_F32) return square_run<float>(a, ws, cap, partials, st);
  if (dtype == SOUP_BF16) return square_run<__nv_bfloat16>(a, ws, cap, partials, st);
  if (dtype == SOUP_F16) return square_run<__half>(a, ws, cap, partials, st);
  set_last_error("soup_grad_square: unsupported dtype");
  return SOUP_ERR_INVALID;
}

int soup_adamw_multi(void* const* params, const void* const* grads, const int64_t* sizes, const int32_t* blocks,
                     int count, int dtype, int state_bits, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                     float* exp_avg_sq_scale, double lr, double beta1, double beta2, double eps, double weight_decay,
                     double max_norm, const void* grad_squares, int partials, float* norm_out, float* step, int last,
                     float* coefs, void* stream) {
  const Args a{params, grads, sizes, blocks, count};
  if (int rc = check_tensors("soup_adamw_multi", a, true)) return rc;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 1e-30) || !exp_avg || !exp_avg_sq ||
      !step || !coefs || (state_bits != 8 && state_bits != 32) ||
      (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) || partials < 0 || (partials > 0 && !grad_squares) ||
      !aligned16(exp_avg) || !aligned16(exp_avg_sq) || !aligned16(coefs) ||
      (dtype != SOUP_F32 && dtype != SOUP_BF16 && dtype != SOUP_F16)) {
    set_last_error("soup_adamw_multi: bad arguments");
    return SOUP_ERR_INVALID;
  }
  const States s{exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale};
  const Hyper h{(float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, (float)(1.0 - lr * weight_decay),
                1.f};
  cudaStream_t st = as_stream(stream);
  Coefs* co = reinterpret_cast<Coefs*>(coefs);
  if (int rc = cuda_status(launch_pdl(adamw_coef_kernel, dim3(1), dim3(kThreads), 0, st, lr, log(beta1), log(beta2),
                                      max_norm, static_cast<const double*>(grad_squares), partials, norm_out, step,
                                      last, co)))
    return rc;
#define RUN(T) \
  return state_bits == 8 ? step_run<T, true>(a, s, h, beta2, co, st) : step_run<T, false>(a, s, h, beta2, co, st)
  if (dtype == SOUP_F32) RUN(float);
  if (dtype == SOUP_BF16) RUN(__nv_bfloat16);
  RUN(__half);
#undef RUN
}

}  // extern "C"
