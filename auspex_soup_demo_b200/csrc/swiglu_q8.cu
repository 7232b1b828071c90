// SwiGLU with its inputs kept in 8 bits between the forward and the backward.
//
// Format of a kept [rows, cols] tensor: one signed byte per element and one
// fp32 scale per block of 64 consecutive columns of a row (the last block of a
// row may be shorter),
//   scale = absmax / 127,  code = rint(x * (127 / absmax)),  value = code * scale,
// each fp32 operation rounded to nearest (IEEE divisions), so the codes are the
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

// |x| as ordered bits: NaN above infinity above every number, so an integer
// maximum over a block also finds a NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ void q8_scale(uint32_t top_bits, float& inv, float& scale) {
  const float top = __uint_as_float(top_bits);
  inv = top < 7.8886090522101181e-31f ? 0.f : __fdiv_rn(127.f, top);  // 2^-100
  scale = __fdiv_rn(top, 127.f);
}
__device__ __forceinline__ int q8_code(float x, float inv) { return __float2int_rn(__fmul_rn(x, inv)); }

template <int L>  // maximum over groups of L neighbouring lanes
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    const uint32_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = v > w ? v : w;
  }
  return v;
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

// 8 / NE x 16-byte codes pieces: NE codes as one store.
template <int NE>
__device__ __forceinline__ void st_codes(int8_t* p, const int (&q)[NE]) {
  if (NE == 8) {
    uint2 w;
    w.x = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | (uint32_t)q[3] << 24;
    w.y = (q[4] & 255) | (q[5] & 255) << 8 | (q[6] & 255) << 16 | (uint32_t)q[7] << 24;
    *reinterpret_cast<uint2*>(p) = w;
  } else {
    *reinterpret_cast<uint32_t*>(p) =
        (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | (uint32_t)q[3] << 24;
  }
}
template <int NE>
__device__ __forceinline__ void ld_codes(const int8_t* p, float (&v)[NE], float scale) {
  uint32_t w[2];
  if (NE == 8) {
    const uint2 t = __ldcs(reinterpret_cast<const uint2*>(p));
    w[0] = t.x;
    w[1] = t.y;
  } else {
    w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
    w[1] = 0;
  }
#pragma unroll
  for (int j = 0; j < NE; ++j)
    v[j] = (float)(int)(int8_t)(w[j >> 2] >> (8 * (j & 3))) * scale;
}

// Vector path: every row start 16-byte aligned (codes: 8 or 4 bytes), cols a
// multiple of the vector. 64 / NE neighbouring lanes share a block.
// kHasAct: SwiGLU forward (gate and up); otherwise quantise `gate` alone.
template <typename T, bool kHasAct>
__global__ void __launch_bounds__(256) q8_fwd_vec_kernel(FwdArgs a, int64_t vpr) {
  constexpr int NE = Vec16<T>::N;
  constexpr int L = kBlk / NE;
  pdl_wait();
  pdl_trigger();
  const int64_t total = a.rows * vpr;  // vpr: vectors per row, padded to whole blocks
  const int lane = threadIdx.x & 31;
  const T* gate = static_cast<const T*>(a.gate);
  const T* up = static_cast<const T*>(a.up);
  T* out = static_cast<T*>(a.out);
  for (int64_t base = blockIdx.x * (int64_t)blockDim.x + (threadIdx.x & ~31); base < total;
       base += (int64_t)gridDim.x * blockDim.x) {
    const int64_t i = base + lane;
    const int64_t r = i / vpr;
    const int64_t c = (i - r * vpr) * NE;
    const bool in = i < total && c < a.cols;
    Vec16<T> g, u;
    g.u = u.u = make_uint4(0, 0, 0, 0);
    if (in) {
      g = ld16_stream(gate + r * a.gate_ld + c);
      if (kHasAct) u = ld16_stream(up + r * a.up_ld + c);
    }
    float gf[NE], uf[NE];
    uint32_t gm = 0, um = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      gf[j] = Cvt<T>::to_f(g.v[j]);
      gm = max(gm, abs_bits(gf[j]));
      if (kHasAct) {
        uf[j] = Cvt<T>::to_f(u.v[j]);
        um = max(um, abs_bits(uf[j]));
      }
    }
    gm = group_max<L>(gm);
    if (kHasAct) um = group_max<L>(um);
    if (!in) continue;
    float inv, sc;
    int q[NE];
    q8_scale(gm, inv, sc);
#pragma unroll
    for (int j = 0; j < NE; ++j) q[j] = q8_code(gf[j], inv);
    st_codes<NE>(a.gq + r * a.q_ld + c, q);
    if ((lane & (L - 1)) == 0) a.gs[r * a.s_ld + c / kBlk] = sc;
    if (kHasAct) {
      q8_scale(um, inv, sc);
#pragma unroll
      for (int j = 0; j < NE; ++j) q[j] = q8_code(uf[j], inv);
      st_codes<NE>(a.uq + r * a.q_ld + c, q);
      if ((lane & (L - 1)) == 0) a.us[r * a.s_ld + c / kBlk] = sc;
      Vec16<T> o;
#pragma unroll
      for (int j = 0; j < NE; ++j)
        o.v[j] = Cvt<T>::from_f((gf[j] * q8_sigmoid<T>(gf[j])) * uf[j]);
      st16_stream(out + r * a.out_ld + c, o);
    }
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
    gm = group_max<32>(gm);
    um = group_max<32>(um);
    float ginv, gsc, uinv = 0.f, usc = 0.f;
    q8_scale(gm, ginv, gsc);
    if (kHasAct) q8_scale(um, uinv, usc);
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

template <typename T, bool kHasH>
__global__ void __launch_bounds__(256) q8_bwd_vec_kernel(BwdArgs a, int64_t vpr) {
  constexpr int NE = Vec16<T>::N;
  pdl_wait();
  pdl_trigger();
  const int64_t total = a.rows * vpr;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / vpr;
    const int64_t c = (i - r * vpr) * NE;
    const Vec16<T> d = ld16_stream(static_cast<const T*>(a.dy) + r * a.dy_ld + c);
    float g[NE], u[NE];
    ld_codes<NE>(a.gq + r * a.q_ld + c, g, a.gs[r * a.s_ld + c / kBlk]);
    ld_codes<NE>(a.uq + r * a.q_ld + c, u, a.us[r * a.s_ld + c / kBlk]);
    Vec16<T> dg, du, h;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      float x, y, z;
      q8_bwd_f<T>(Cvt<T>::to_f(d.v[j]), g[j], u[j], x, y, z);
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
  if (vec) {
    const int64_t vpr = bpr * (kBlk / NE);
    return cuda_status(launch_pdl(q8_fwd_vec_kernel<T, kHasAct>, dim3(grid_for(a.rows * vpr)),
                                  dim3(256), 0, st, a, vpr));
  }
  return cuda_status(launch_pdl(q8_fwd_scalar_kernel<T, kHasAct>, dim3(grid_for(a.rows * bpr * 32)),
                                dim3(256), 0, st, a, bpr));
}

template <typename T, bool kHasH>
int run_bwd_h(const BwdArgs& a, cudaStream_t st) {
  constexpr int NE = Vec16<T>::N;
  const bool vec = a.cols % NE == 0 && vec_ok<T>(a.dy, a.dy_ld) && vec_ok<T>(a.dg, a.dg_ld) &&
                   vec_ok<T>(a.du, a.du_ld) && codes_ok<NE>(a.gq, a.q_ld) &&
                   codes_ok<NE>(a.uq, a.q_ld) && (!kHasH || vec_ok<T>(a.h, a.h_ld));
  if (vec) {
    const int64_t vpr = a.cols / NE;
    return cuda_status(launch_pdl(q8_bwd_vec_kernel<T, kHasH>, dim3(grid_for(a.rows * vpr)),
                                  dim3(256), 0, st, a, vpr));
  }
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
