// SwiGLU with its inputs kept in 8 bits between the forward and the backward.
//
// Format of a kept [rows, cols] tensor: one signed byte per element and one
// fp32 scale per block of 64 consecutive columns of a row (the last block of a
// row may be shorter),
//   scale = absmax / 127,  code = rint(x * (127 / absmax)),  value = code * scale,
// each fp32 operation rounded to nearest (the divisions too), so the codes are the
// same on every path. A block whose absmax is below 2^-100 is all zeros (there
// 127 / absmax would overflow); one that holds an infinity or a NaN stands for
// NaN throughout, so a diverged forward stays visible in the gradient.
// 64 columns match the base weights' NF4 block; rounding a value is off by at
// most absmax / 254 (half a code).
//
// The forward computes h = silu(g) u from the exact g and u and stores the
// codes; the backward is SwiGLU's derivative at the values the codes stand for.
#include "soup_common.cuh"

namespace soup {
namespace {

constexpr int kBlk = 64;

template <typename T>
__device__ __forceinline__ float q8_sigmoid(float g) {
  return swiglu_sigmoid(g);
}
// fp32 tensors: the fast exponential's error would show in the result
template <>
__device__ __forceinline__ float q8_sigmoid<float>(float g) {
  return 1.f / (1.f + expf(-g));
}

// silu(g) u of two elements; 16-bit types on packed pairs, with the hardware exponential
// and reciprocal (2^-22 each, far below the types' rounding). For g -> -inf the divisor
// overflows and the result is the limit 0.
template <typename T>
__device__ __forceinline__ void q8_swiglu2(float g0, float g1, float u0, float u1, float& o0, float& o1) {
  const uint64_t g = f2_pack(g0, g1);
  float e0, e1;
  f2_unpack(f2_mul(g, f2_pack(-kLog2e, -kLog2e)), e0, e1);
  f2_unpack(f2_add(f2_pack(fast_exp2(e0), fast_exp2(e1)), f2_pack(1.f, 1.f)), e0, e1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e1));
  f2_unpack(f2_mul(f2_mul(g, f2_pack(e0, e1)), f2_pack(u0, u1)), o0, o1);
}
template <>
__device__ __forceinline__ void q8_swiglu2<float>(float g0, float g1, float u0, float u1, float& o0,
                                                  float& o1) {
  o0 = (g0 * q8_sigmoid<float>(g0)) * u0;
  o1 = (g1 * q8_sigmoid<float>(g1)) * u1;
}

// |x| as ordered bits: NaN above infinity above every number, so an integer
// maximum over a block also finds a NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// inv = 127 / absmax and scale = absmax / 127, both correctly rounded. The second
// divides by a constant: a product with the rounded reciprocal and one residual step
// (Markstein's theorem) instead of a division.
__device__ __forceinline__ void q8_scale(float top, float& inv, float& scale) {
  constexpr float kR = 1.f / 127.f;
  const bool tiny = top < 7.8886090522101181e-31f;  // 2^-100: the block stands for zeros
  inv = tiny ? 0.f : __fdiv_rn(127.f, top);
  const float q = __fmul_rn(top, kR);
  scale = tiny ? 0.f : __fmaf_rn(__fmaf_rn(-127.f, q, top), kR, q);
}
// rint(x * inv) for |x * inv| <= 127 as the low byte of the result: adding 1.5 * 2^23
// rounds to an integer, to even on ties, without the conversion unit, whose rate (that of
// the exponential) would bound the kernel. The product is rounded by itself: a fused
// multiply-add, or packed pairs, which the compiler fuses, give other codes on ties.
constexpr float kMagic = 12582912.f;
__device__ __forceinline__ uint32_t q8_code(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), kMagic));
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Byte j of a word of codes as a float (exact): the code + 128 as the low bits of 2^23.
__device__ __forceinline__ float code_float(uint32_t biased, int j) {
  return __uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7550 | j)) - 8388736.f;
}

// i / d for 0 <= i < 2^31 by a product (Granlund and Montgomery): d >= 1.
struct FastDiv {
  uint32_t d, mul, shift;
  explicit FastDiv(uint32_t div) : d(div) {
    shift = 0;
    while ((1ull << shift) < div) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - div)) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t i) const {
    return (uint32_t)(((uint64_t)__umulhi(i, mul) + i) >> shift);
  }
};

// Maxima of |g| and |u| over groups of L neighbouring lanes (a block of 64 columns), from
// this lane's vectors. 16-bit types: as pairs of 16-bit integers, both tensors in one word
// for the exchange between lanes.
template <typename T, int L>
__device__ __forceinline__ void block_tops(const Vec16<T>& g, const Vec16<T>& u, float& gt, float& ut) {
  if (sizeof(T) == 2) {
    const uint4 a = g.u, b = u.u;
    constexpr uint32_t kAbs = 0x7fff7fffu;
    const uint32_t x = __vmaxu2(__vmaxu2(a.x & kAbs, a.y & kAbs), __vmaxu2(a.z & kAbs, a.w & kAbs));
    const uint32_t y = __vmaxu2(__vmaxu2(b.x & kAbs, b.y & kAbs), __vmaxu2(b.z & kAbs, b.w & kAbs));
    // low halves of x and y in one word, high halves in another
    uint32_t m = __vmaxu2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    union {
      uint16_t s;
      T t;
    } c;
    c.s = (uint16_t)(m & 0xffffu);
    gt = Cvt<T>::to_f(c.t);
    c.s = (uint16_t)(m >> 16);
    ut = Cvt<T>::to_f(c.t);
  } else {
    uint32_t x = 0, y = 0;
#pragma unroll
    for (int j = 0; j < Vec16<T>::N; ++j) {
      x = max(x, abs_bits(Cvt<T>::to_f(g.v[j])));
      y = max(y, abs_bits(Cvt<T>::to_f(u.v[j])));
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
      y = max(y, __shfl_xor_sync(0xffffffffu, y, o));
    }
    gt = __uint_as_float(x);
    ut = __uint_as_float(y);
  }
}

struct FwdArgs {
  const void* gate;
  const void* up;
  void* out;
  int64_t gate_ld, up_ld, out_ld;
  int8_t* gq;
  int8_t* uq;
  float* gs;
  float* us;
  int64_t q_ld, s_ld;
  int64_t rows, cols;
};

struct BwdArgs {
  const void* dy;
  int64_t dy_ld;
  const int8_t* gq;
  const int8_t* uq;
  const float* gs;
  const float* us;
  int64_t q_ld, s_ld;
  void* dg;
  void* du;
  void* h;  // optional: silu(g) u of the kept values
  int64_t dg_ld, du_ld, h_ld;
  int64_t rows, cols;
};

// The codes of one vector of NE floats in one store.
template <int NE>
__device__ __forceinline__ void store_codes(int8_t* p, const float (&v)[NE], float inv) {
  uint32_t w[NE / 4];
#pragma unroll
  for (int j = 0; j < NE; j += 4)
    w[j / 4] = low_bytes(q8_code(v[j], inv), q8_code(v[j + 1], inv), q8_code(v[j + 2], inv),
                         q8_code(v[j + 3], inv));
  if (NE == 8)
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[NE / 4 - 1]));
  else
    __stcs(reinterpret_cast<uint32_t*>(p), w[0]);
}
template <int NE>
__device__ __forceinline__ void load_codes(const int8_t* p, uint32_t (&w)[NE / 4]) {
  if (NE == 8) {
    const uint2 t = __ldcs(reinterpret_cast<const uint2*>(p));
    w[0] = t.x;
    w[NE / 4 - 1] = t.y;
  } else {
    w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
  }
}

// Vector path: every row start 16-byte aligned (codes: 8 or 4 bytes), cols a
// multiple of the vector. 64 / NE neighbouring lanes share a block.
// kHasAct: SwiGLU forward (gate and up); otherwise quantise `gate` alone.
// Bound by HBM: 8192 x 8960 bf16 (596 MB) in 105 us, 5.7 TB/s, with two vectors a thread in
// flight (118 us with one). Before the conversions left the special-function unit and the row
// index its 64-bit division, issue slots bounded it (150 us).
template <typename T, bool kHasAct>
__global__ void __launch_bounds__(256) q8_fwd_vec_kernel(FwdArgs a, FastDiv vpr, uint32_t total) {
  constexpr int NE = Vec16<T>::N;
  constexpr int L = kBlk / NE;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const T* gate = static_cast<const T*>(a.gate);
  const T* up = static_cast<const T*>(a.up);
  T* out = static_cast<T*>(a.out);
  // total: vectors, rows padded to whole blocks (vpr vectors a row); below 2^31
  struct Item {
    Vec16<T> g, u;
    uint32_t r, c;
    bool in, blk;  // the vector / its block exists
  };
  auto load = [&](uint32_t i, Item& t) {
    t.r = vpr.div(i);
    t.c = (i - t.r * vpr.d) * NE;
    t.in = i < total && t.c < a.cols;
    t.blk = i < total && t.c - (lane & (L - 1)) * NE < a.cols;
    t.g.u = t.u.u = make_uint4(0, 0, 0, 0);
    if (t.in) {
      t.g = ld16_stream(gate + t.r * a.gate_ld + t.c);
      if (kHasAct) t.u = ld16_stream(up + t.r * a.up_ld + t.c);
    }
  };
  auto process = [&](const Item& t) {
    float gt, ut;
    block_tops<T, L>(t.g, t.u, gt, ut);
    // half of a block's lanes divide for gate, the other half for up
    const bool second = kHasAct && (lane & (L / 2));
    float inv, sc;
    q8_scale(second ? ut : gt, inv, sc);
    const float inv_x = kHasAct ? __shfl_xor_sync(0xffffffffu, inv, L / 2) : 0.f;
    if ((lane & (L / 2 - 1)) == 0 && t.blk) {
      if (second)
        a.us[t.r * a.s_ld + t.c / kBlk] = sc;
      else if (kHasAct || (lane & (L - 1)) == 0)
        a.gs[t.r * a.s_ld + t.c / kBlk] = sc;
    }
    if (!t.in) return;
    float gf[NE], uf[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      gf[j] = Cvt<T>::to_f(t.g.v[j]);
      uf[j] = Cvt<T>::to_f(t.u.v[j]);
    }
    store_codes<NE>(a.gq + t.r * a.q_ld + t.c, gf, second ? inv_x : inv);
    if (kHasAct) {
      store_codes<NE>(a.uq + t.r * a.q_ld + t.c, uf, second ? inv : inv_x);
      Vec16<T> o;
#pragma unroll
      for (int j = 0; j < NE; j += 2) {
        float x0, x1;
        q8_swiglu2<T>(gf[j], gf[j + 1], uf[j], uf[j + 1], x0, x1);
        o.v[j] = Cvt<T>::from_f(x0);
        o.v[j + 1] = Cvt<T>::from_f(x1);
      }
      st16_stream(out + t.r * a.out_ld + t.c, o);
    }
  };
  const uint32_t step = gridDim.x * blockDim.x;
  for (uint32_t base = blockIdx.x * blockDim.x + (threadIdx.x & ~31u); base < total; base += 2 * step) {
    Item t0, t1;
    load(base + lane, t0);
    load(base + step + lane, t1);
    process(t0);
    if (base + step < total) process(t1);  // warp-uniform
  }
}

// Any alignment: one warp per block of 64 columns, two columns per lane.
template <typename T, bool kHasAct>
__global__ void __launch_bounds__(256) q8_fwd_scalar_kernel(FwdArgs a, int64_t bpr) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const T* gate = static_cast<const T*>(a.gate);
  const T* up = static_cast<const T*>(a.up);
  T* out = static_cast<T*>(a.out);
  const int64_t total = a.rows * bpr;
  for (int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; w < total;
       w += ((int64_t)gridDim.x * blockDim.x) >> 5) {
    const int64_t r = w / bpr, b = w - r * bpr;
    float g[2], u[2];
    uint32_t gm = 0, um = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t c = b * kBlk + lane + 32 * e;
      const bool in = c < a.cols;
      g[e] = in ? Cvt<T>::to_f(gate[r * a.gate_ld + c]) : 0.f;
      u[e] = kHasAct && in ? Cvt<T>::to_f(up[r * a.up_ld + c]) : 0.f;
      gm = max(gm, abs_bits(g[e]));
      um = max(um, abs_bits(u[e]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, o));
      um = max(um, __shfl_xor_sync(0xffffffffu, um, o));
    }
    float ginv, gsc, uinv = 0.f, usc = 0.f;
    q8_scale(__uint_as_float(gm), ginv, gsc);
    if (kHasAct) q8_scale(__uint_as_float(um), uinv, usc);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t c = b * kBlk + lane + 32 * e;
      if (c >= a.cols) continue;
      a.gq[r * a.q_ld + c] = (int8_t)q8_code(g[e], ginv);
      if (kHasAct) {
        a.uq[r * a.q_ld + c] = (int8_t)q8_code(u[e], uinv);
        out[r * a.out_ld + c] = Cvt<T>::from_f((g[e] * q8_sigmoid<T>(g[e])) * u[e]);
      }
    }
    if (lane == 0) {
      a.gs[r * a.s_ld + b] = gsc;
      if (kHasAct) a.us[r * a.s_ld + b] = usc;
    }
  }
}

template <typename T>
__device__ __forceinline__ void q8_bwd_f(float d, float g, float u, float& dg, float& du, float& h) {
  const float sg = q8_sigmoid<T>(g);
  const float si = g * sg;
  du = d * si;
  dg = d * u * sg * (1.f + g * (1.f - sg));
  h = si * u;
}

// Bound by HBM: 8192 x 8960 bf16 (596 MB) in 102 us, 5.8 TB/s (108 with conversion instructions
// and 64-bit divisions; a second vector in flight gains nothing here).
template <typename T, bool kHasH>
__global__ void __launch_bounds__(256) q8_bwd_vec_kernel(BwdArgs a, FastDiv vpr, uint32_t total) {
  constexpr int NE = Vec16<T>::N;
  pdl_wait();
  pdl_trigger();
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) {
    const uint32_t r = vpr.div(i);
    const uint32_t c = (i - r * vpr.d) * NE;
    const Vec16<T> d = ld16_stream(static_cast<const T*>(a.dy) + r * a.dy_ld + c);
    uint32_t gw[NE / 4], uw[NE / 4];
    load_codes<NE>(a.gq + r * a.q_ld + c, gw);
    load_codes<NE>(a.uq + r * a.q_ld + c, uw);
    const float gs = a.gs[r * a.s_ld + c / kBlk], us = a.us[r * a.s_ld + c / kBlk];
    Vec16<T> dg, du, h;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      float x, y, z;
      q8_bwd_f<T>(Cvt<T>::to_f(d.v[j]), code_float(gw[j / 4] ^ 0x80808080u, j & 3) * gs,
                  code_float(uw[j / 4] ^ 0x80808080u, j & 3) * us, x, y, z);
      dg.v[j] = Cvt<T>::from_f(x);
      du.v[j] = Cvt<T>::from_f(y);
      if (kHasH) h.v[j] = Cvt<T>::from_f(z);
    }
    st16_stream(static_cast<T*>(a.dg) + r * a.dg_ld + c, dg);
    st16_stream(static_cast<T*>(a.du) + r * a.du_ld + c, du);
    if (kHasH) st16_stream(static_cast<T*>(a.h) + r * a.h_ld + c, h);
  }
}

template <typename T, bool kHasH>
__global__ void __launch_bounds__(256) q8_bwd_scalar_kernel(BwdArgs a) {
  pdl_wait();
  pdl_trigger();
  const int64_t total = a.rows * a.cols;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / a.cols, c = i - r * a.cols;
    const float g = (float)a.gq[r * a.q_ld + c] * a.gs[r * a.s_ld + c / kBlk];
    const float u = (float)a.uq[r * a.q_ld + c] * a.us[r * a.s_ld + c / kBlk];
    float x, y, z;
    q8_bwd_f<T>(Cvt<T>::to_f(static_cast<const T*>(a.dy)[r * a.dy_ld + c]), g, u, x, y, z);
    static_cast<T*>(a.dg)[r * a.dg_ld + c] = Cvt<T>::from_f(x);
    static_cast<T*>(a.du)[r * a.du_ld + c] = Cvt<T>::from_f(y);
    if (kHasH) static_cast<T*>(a.h)[r * a.h_ld + c] = Cvt<T>::from_f(z);
  }
}

int grid_for(int64_t threads) {
  int64_t blocks = (threads + 255) / 256;
  const int64_t cap = (int64_t)num_sms() * 8;
  if (blocks > cap) blocks = cap;
  return blocks < 1 ? 1 : (int)blocks;
}

// The vector kernels index vectors in 31 bits and step past the end by up to two grids
// (2 x 8 x 256 threads on each SM), and columns in 32; larger tensors take the scalar kernels'
// 64-bit indices.
constexpr int64_t kMaxCols = int64_t(1) << 31;
constexpr int64_t kMaxVecs = (int64_t(1) << 31) - (int64_t(1) << 20);

template <typename T>
bool vec_ok(const void* p, int64_t ld) {
  return aligned16(p) && (ld * (int64_t)sizeof(T)) % 16 == 0;
}
template <int NE>
bool codes_ok(const int8_t* p, int64_t ld) {
  return reinterpret_cast<uintptr_t>(p) % NE == 0 && ld % NE == 0;
}

template <typename T, bool kHasAct>
int run_fwd(const FwdArgs& a, cudaStream_t st) {
  constexpr int NE = Vec16<T>::N;
  const int64_t bpr = (a.cols + kBlk - 1) / kBlk;
  const bool vec = a.cols % NE == 0 && vec_ok<T>(a.gate, a.gate_ld) && codes_ok<NE>(a.gq, a.q_ld) &&
                   (!kHasAct || (vec_ok<T>(a.up, a.up_ld) && vec_ok<T>(a.out, a.out_ld) &&
                                 codes_ok<NE>(a.uq, a.q_ld)));
  const int64_t vpr = bpr * (kBlk / NE), total = a.rows * vpr;
  if (vec && total < kMaxVecs && a.cols < kMaxCols)
    return cuda_status(launch_pdl(q8_fwd_vec_kernel<T, kHasAct>, dim3(grid_for(total)), dim3(256), 0,
                                  st, a, FastDiv((uint32_t)vpr), (uint32_t)total));
  return cuda_status(launch_pdl(q8_fwd_scalar_kernel<T, kHasAct>, dim3(grid_for(a.rows * bpr * 32)),
                                dim3(256), 0, st, a, bpr));
}

template <typename T, bool kHasH>
int run_bwd_h(const BwdArgs& a, cudaStream_t st) {
  constexpr int NE = Vec16<T>::N;
  const bool vec = a.cols % NE == 0 && vec_ok<T>(a.dy, a.dy_ld) && vec_ok<T>(a.dg, a.dg_ld) &&
                   vec_ok<T>(a.du, a.du_ld) && codes_ok<NE>(a.gq, a.q_ld) &&
                   codes_ok<NE>(a.uq, a.q_ld) && (!kHasH || vec_ok<T>(a.h, a.h_ld));
  const int64_t vpr = a.cols / NE, total = a.rows * vpr;
  if (vec && total < kMaxVecs && a.cols < kMaxCols)
    return cuda_status(launch_pdl(q8_bwd_vec_kernel<T, kHasH>, dim3(grid_for(total)), dim3(256), 0,
                                  st, a, FastDiv((uint32_t)vpr), (uint32_t)total));
  return cuda_status(launch_pdl(q8_bwd_scalar_kernel<T, kHasH>, dim3(grid_for(a.rows * a.cols)),
                                dim3(256), 0, st, a));
}
template <typename T>
int run_bwd(const BwdArgs& a, cudaStream_t st) {
  return a.h ? run_bwd_h<T, true>(a, st) : run_bwd_h<T, false>(a, st);
}

}  // namespace
}  // namespace soup

using namespace soup;

extern "C" {

int soup_swiglu_q8_fwd(const void* gate, int64_t gate_row_stride, const void* up,
                       int64_t up_row_stride, void* out, int64_t out_row_stride, int8_t* gate_codes,
                       int8_t* up_codes, int64_t codes_row_stride, float* gate_scales,
                       float* up_scales, int64_t scales_row_stride, int64_t rows, int64_t cols,
                       int dtype, void* stream) {
  if (!gate || !up || !out || !gate_codes || !up_codes || !gate_scales || !up_scales || rows < 0 ||
      cols <= 0 || gate_row_stride < cols || up_row_stride < cols || out_row_stride < cols ||
      codes_row_stride < cols || scales_row_stride < (cols + kBlk - 1) / kBlk) {
    set_last_error("soup_swiglu_q8_fwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (rows == 0) return SOUP_OK;
  FwdArgs a{gate, up, out, gate_row_stride, up_row_stride, out_row_stride, gate_codes, up_codes,
            gate_scales, up_scales, codes_row_stride, scales_row_stride, rows, cols};
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_BF16) return run_fwd<__nv_bfloat16, true>(a, st);
  if (dtype == SOUP_F16) return run_fwd<__half, true>(a, st);
  if (dtype == SOUP_F32) return run_fwd<float, true>(a, st);
  set_last_error("soup_swiglu_q8_fwd: unsupported dtype");
  return SOUP_ERR_INVALID;
}

int soup_q8_quantize(const void* x, int64_t x_row_stride, int8_t* codes, int64_t codes_row_stride,
                     float* scales, int64_t scales_row_stride, int64_t rows, int64_t cols, int dtype,
                     void* stream) {
  if (!x || !codes || !scales || rows < 0 || cols <= 0 || x_row_stride < cols ||
      codes_row_stride < cols || scales_row_stride < (cols + kBlk - 1) / kBlk) {
    set_last_error("soup_q8_quantize: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (rows == 0) return SOUP_OK;
  FwdArgs a{x, nullptr, nullptr, x_row_stride, 0, 0, codes, nullptr, scales, nullptr,
            codes_row_stride, scales_row_stride, rows, cols};
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_BF16) return run_fwd<__nv_bfloat16, false>(a, st);
  if (dtype == SOUP_F16) return run_fwd<__half, false>(a, st);
  if (dtype == SOUP_F32) return run_fwd<float, false>(a, st);
  set_last_error("soup_q8_quantize: unsupported dtype");
  return SOUP_ERR_INVALID;
}

int soup_swiglu_q8_bwd(const void* dy, int64_t dy_row_stride, const int8_t* gate_codes,
                       const int8_t* up_codes, int64_t codes_row_stride, const float* gate_scales,
                       const float* up_scales, int64_t scales_row_stride, void* dgate,
                       int64_t dgate_row_stride, void* dup, int64_t dup_row_stride, void* h,
                       int64_t h_row_stride, int64_t rows, int64_t cols, int dtype, void* stream) {
  if (!dy || !gate_codes || !up_codes || !gate_scales || !up_scales || !dgate || !dup || rows < 0 ||
      cols <= 0 || dy_row_stride < cols || codes_row_stride < cols ||
      scales_row_stride < (cols + kBlk - 1) / kBlk || dgate_row_stride < cols ||
      dup_row_stride < cols || (h && h_row_stride < cols)) {
    set_last_error("soup_swiglu_q8_bwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (rows == 0) return SOUP_OK;
  BwdArgs a{dy, dy_row_stride, gate_codes, up_codes, gate_scales, up_scales, codes_row_stride,
            scales_row_stride, dgate, dup, h, dgate_row_stride, dup_row_stride, h_row_stride, rows,
            cols};
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_BF16) return run_bwd<__nv_bfloat16>(a, st);
  if (dtype == SOUP_F16) return run_bwd<__half>(a, st);
  if (dtype == SOUP_F32) return run_bwd<float>(a, st);
  set_last_error("soup_swiglu_q8_bwd: unsupported dtype");
  return SOUP_ERR_INVALID;
}

}  // extern "C"
