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
// A warp takes a block: 8 elements a lane in two 16-byte loads (one for 16-bit
// tensors), the maxima by shuffles. A CTA takes 2048 elements at a time and a
// contiguous run of such chunks over all tensors, whose table (pointers and sizes)
// comes as a kernel argument, so that a launch needs no copy and can be captured.
#include <cuda_fp8.h>
#include <stdio.h>

#include "soup_common.cuh"

namespace soup {
namespace {

constexpr int kBlock = 256;              // elements that share a scale
constexpr int kWarps = 8;
constexpr int kChunk = kBlock * kWarps;  // elements of a CTA's turn
constexpr int kThreads = 32 * kWarps;
constexpr float kE4m3Max = 448.f;
constexpr float kE4m3Least = 0.001953125f;  // 2^-9

struct Tensor {
  void* p;
  const void* g;
  int64_t n;
  int block0;   // first state block
  int chunk0;   // chunks of the tensors before it in this launch
};

template <int N>
struct Table {
  int count, chunks;
  Tensor t[N];
};

struct Hyper {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, lr, decay;  // decay: 1 - lr wd
  double log_beta1, log_beta2;
  float max_norm;
};

struct States {
  void* m;          // fp32, or e4m3
  void* v;          // fp32 v, or e4m3 sqrt(v)
  float* m_scale;   // [blocks]
  float* v_scale;
};

// The tensor that holds chunk c.
template <int N>
__device__ __forceinline__ int find_tensor(const Table<N>& tab, int c) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].chunk0 <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void chunk_run(int chunks, int& c0, int& c1) {
  c0 = (int)((int64_t)chunks * blockIdx.x / gridDim.x);
  c1 = (int)((int64_t)chunks * (blockIdx.x + 1) / gridDim.x);
}

// 8 consecutive elements as floats; `left` of them exist, the others read 0.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, bool vec, float (&f)[8]) {
  constexpr int NE = Vec16<T>::N;
  if (left >= 8 && vec) {
#pragma unroll
    for (int i = 0; i < 8; i += NE) {
      const Vec16<T> q = ld16_stream(p + i);
#pragma unroll
      for (int e = 0; e < NE; ++e) f[i + e] = Cvt<T>::to_f(q.v[e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < left ? Cvt<T>::to_f(p[i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int left, bool vec, const float (&f)[8]) {
  constexpr int NE = Vec16<T>::N;
  if (left >= 8 && vec) {
#pragma unroll
    for (int i = 0; i < 8; i += NE) {
      Vec16<T> q;
#pragma unroll
      for (int e = 0; e < NE; ++e) q.v[e] = Cvt<T>::from_f(f[i + e]);
      st16_stream(p + i, q);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = Cvt<T>::from_f(f[i]);
  }
}

__device__ __forceinline__ void from_codes(uint2 c, float scale, float (&f)[8]) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
    const float2 v = __half22float2(__half2(h));
    f[2 * i] = v.x * scale;
    f[2 * i + 1] = v.y * scale;
  }
}

// Scale of the warp's block and its codes. Values that are not finite are left out of
// the maximum: they must not wipe out the other 255.
template <bool ROOT>
__device__ __forceinline__ uint2 to_codes(const float (&f)[8], float& scale) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(f[i]);
    top = a <= 3.4028235e38f ? fmaxf(top, a) : top;
  }
  top = warp_max(top);
  scale = top / kE4m3Max;
  // a subnormal scale has no finite reciprocal: such a block is divided
  const float inv = scale >= 1.17549435e-38f ? 1.f / scale : 0.f;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 y = make_float2(f[2 * i] * inv, f[2 * i + 1] * inv);
    if (inv == 0.f && scale > 0.f) y = make_float2(f[2 * i] / scale, f[2 * i + 1] / scale);
    if constexpr (ROOT) {
      if (f[2 * i] > 0.f) y.x = fmaxf(y.x, kE4m3Least);
      if (f[2 * i + 1] > 0.f) y.y = fmaxf(y.y, kE4m3Least);
    }
    w[i >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3) << (16 * (i & 1));
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

// Sum of squares of the gradients: one partial a CTA, in 64 bits (the clip coefficient
// scales every element, so its error would be in all of them).
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) grad_square_kernel(const __grid_constant__ Table<N> tab,
                                                               double* __restrict__ partial) {
  __shared__ double share[kWarps];
  pdl_wait();
  pdl_trigger();
  int c0, c1;
  chunk_run(tab.chunks, c0, c1);
  double sum = 0.0;
  int ti = c0 < c1 ? find_tensor(tab, c0) : 0;
  for (int c = c0; c < c1; ++c) {
    while (ti + 1 < tab.count && tab.t[ti + 1].chunk0 <= c) ++ti;
    const Tensor& t = tab.t[ti];
    const int64_t e = (int64_t)(c - t.chunk0) * kChunk + threadIdx.x * 8;
    if (e >= t.n) continue;
    const int64_t rest = t.n - e;
    float g[8];
    load8(static_cast<const T*>(t.g) + e, rest < 8 ? (int)rest : 8, (reinterpret_cast<uintptr_t>(t.g) & 15) == 0, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fma((double)g[i], (double)g[i], sum);
  }
  sum = block_sum(sum, share);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The step. `partial`: the sums of squares of all of the step's tensors, or null.
// `step` counts the steps done; `ticket` is 0 between launches. The last CTA of the
// step's last launch (bump) raises the count after every CTA has read it.
template <typename T, bool EIGHT, int N>
__global__ void __launch_bounds__(kThreads) adamw_multi_kernel(const __grid_constant__ Table<N> tab, States st,
                                                               Hyper h, const double* __restrict__ partial,
                                                               int partials, float* __restrict__ norm_out,
                                                               float* __restrict__ step, int* __restrict__ ticket,
                                                               int bump) {
  __shared__ double share[kWarps];
  __shared__ float coefs[3];
  pdl_wait();
  pdl_trigger();
  double sum = 0.0;
  if (partial) {
    for (int i = threadIdx.x; i < partials; i += kThreads) sum += partial[i];
    sum = block_sum(sum, share);
  }
  if (threadIdx.x == 0) {
    const double t = (double)*step + 1.0;
    // 1 - b^t = -expm1(t log b): exact also in the first steps
    coefs[0] = (float)((double)h.lr / -expm1(t * h.log_beta1));
    coefs[1] = (float)(1.0 / sqrt(-expm1(t * h.log_beta2)));
    float clip = 1.f;
    if (partial) {
      const double norm = sqrt(sum);
      const double c = (double)h.max_norm / (norm + 1e-6);
      clip = c > 1.0 ? 1.f : (float)c;  // a norm that is not a number stays visible in every element
      if (blockIdx.x == 0 && norm_out) *norm_out = (float)norm;
    }
    coefs[2] = clip;
  }
  __syncthreads();
  const float step_size = coefs[0], root_scale = coefs[1], clip = coefs[2];
  int c0, c1;
  chunk_run(tab.chunks, c0, c1);
  const int lane8 = threadIdx.x * 8;
  int ti = c0 < c1 ? find_tensor(tab, c0) : 0;
  for (int c = c0; c < c1; ++c) {
    while (ti + 1 < tab.count && tab.t[ti + 1].chunk0 <= c) ++ti;
    const Tensor& t = tab.t[ti];
    const int64_t e = (int64_t)(c - t.chunk0) * kChunk + lane8;
    const int64_t rest = t.n - e;
    // a warp's block is there as a whole or in part, or not at all
    if (t.n <= e - (threadIdx.x & 31) * 8) continue;
    const int left = rest >= 8 ? 8 : rest < 0 ? 0 : (int)rest;
    const bool vp = (reinterpret_cast<uintptr_t>(t.p) & 15) == 0, vg = (reinterpret_cast<uintptr_t>(t.g) & 15) == 0;
    const int64_t blk = t.block0 + (e >> 8);
    const int64_t at = blk * kBlock + (threadIdx.x & 31) * 8;
    float p[8], g[8], m[8], v[8];
    load8(static_cast<const T*>(t.g) + e, left, vg, g);
    load8(static_cast<const T*>(t.p) + e, left, vp, p);
    if constexpr (EIGHT) {
      const uint2 mc = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(st.m) + at));
      const uint2 vc = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(st.v) + at));
      from_codes(mc, st.m_scale[blk], m);
      from_codes(vc, st.v_scale[blk], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= v[i];
    } else {
      load8(static_cast<const float*>(st.m) + at, 8, true, m);
      load8(static_cast<const float*>(st.v) + at, 8, true, v);
    }
    float root[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float gi = g[i] * clip;
      m[i] = fmaf(h.one_minus_beta1, gi - m[i], m[i]);
      v[i] = fmaf(h.one_minus_beta2 * gi, gi, v[i] * h.beta2);
      root[i] = sqrtf(v[i]);
      p[i] = fmaf(p[i], h.decay, -(step_size * m[i] / fmaf(root[i], root_scale, h.eps)));
    }
    store8(static_cast<T*>(t.p) + e, left, vp, p);
    if constexpr (EIGHT) {
      // what lies behind a tensor's end stays 0
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= left) m[i] = root[i] = 0.f;
      float ms, vs;
      const uint2 mc = to_codes<false>(m, ms);
      const uint2 vc = to_codes<true>(root, vs);
      __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(st.m) + at), mc);
      __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(st.v) + at), vc);
      if ((threadIdx.x & 31) == 0) {
        st.m_scale[blk] = ms;
        st.v_scale[blk] = vs;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= left) m[i] = v[i] = 0.f;
      store8(static_cast<float*>(st.m) + at, 8, true, m);
      store8(static_cast<float*>(st.v) + at, 8, true, v);
    }
  }
  if (bump && threadIdx.x == 0) {
    // every CTA has read the count before its ticket
    __threadfence();
    if (atomicAdd(ticket, 1) == (int)gridDim.x - 1) {
      *ticket = 0;
      *step += 1.f;
    }
  }
}

constexpr int kSmall = 64, kLarge = 960;  // tensors of a launch: arguments of 2 and 30 KB

inline int chunks_of(int64_t n) { return (int)((n + kChunk - 1) / kChunk); }

inline int grid_of(int chunks) {
  const int cap = num_sms() * 4;
  return chunks < cap ? (chunks < 1 ? 1 : chunks) : cap;
}

struct Args {
  void* const* params;
  const void* const* grads;
  const int64_t* sizes;
  const int32_t* blocks;
  int count;
};

// Tensors [i0, i1) into a table; returns the chunks.
template <int N>
void fill_table(Table<N>& tab, const Args& a, int i0, int i1) {
  int chunks = 0;
  for (int i = i0; i < i1; ++i) {
    tab.t[i - i0] = Tensor{a.params ? a.params[i] : nullptr, a.grads[i], a.sizes[i], a.blocks ? a.blocks[i] : 0, chunks};
    chunks += chunks_of(a.sizes[i]);
  }
  tab.count = i1 - i0;
  tab.chunks = chunks;
}

// The end of the launch that starts with tensor i0: at most `most` tensors and 2^30 chunks.
int launch_end(const Args& a, int i0, int most) {
  int64_t chunks = 0;
  int i = i0;
  while (i < a.count && i - i0 < most) {
    const int64_t c = chunks_of(a.sizes[i]);
    if (i > i0 && chunks + c > (1 << 30)) break;
    chunks += c;
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
  const int grid = grid_of(tab.chunks) < num_sms() * 2 ? grid_of(tab.chunks) : num_sms() * 2;
  *used += grid;
  return launch_table(grad_square_kernel<T, N>, grid, st, tab, partial);
}

template <typename T, bool EIGHT, int N>
int step_launch(const Args& a, int i0, int i1, const States& s, const Hyper& h, const double* partial, int partials,
                float* norm_out, float* step, int* ticket, int bump, cudaStream_t st) {
  Table<N> tab;
  fill_table(tab, a, i0, i1);
  return launch_table(adamw_multi_kernel<T, EIGHT, N>, grid_of(tab.chunks), st, tab, s, h, partial, partials, norm_out,
                      step, ticket, bump);
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
    if (*used + num_sms() * 2 > cap) {
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

template <typename T, bool EIGHT>
int step_run(const Args& a, const States& s, const Hyper& h, const double* partial, int partials, float* norm_out,
             float* step, int* ticket, int bump, cudaStream_t st) {
  const int most = a.count <= kSmall ? kSmall : kLarge;
  for (int i0 = 0; i0 < a.count;) {
    const int i1 = launch_end(a, i0, most);
    const int b = bump && i1 == a.count ? 1 : 0;
    const int rc = most == kSmall
                       ? step_launch<T, EIGHT, kSmall>(a, i0, i1, s, h, partial, partials, norm_out, step, ticket, b, st)
                       : step_launch<T, EIGHT, kLarge>(a, i0, i1, s, h, partial, partials, norm_out, step, ticket, b, st);
    if (rc) return rc;
    i0 = i1;
  }
  return SOUP_OK;
}

}  // namespace
}  // namespace soup

using namespace soup;

extern "C" {

size_t soup_grad_square_workspace_bytes(int64_t tensors) {
  if (tensors <= 0) return 0;
  // two partials an SM for each launch
  return sizeof(double) * 2 * (size_t)num_sms() * (size_t)((tensors + kLarge - 1) / kLarge);
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
                     double max_norm, const void* grad_squares, int partials, float* norm_out, float* step,
                     int* ticket, int last, void* stream) {
  const Args a{params, grads, sizes, blocks, count};
  if (int rc = check_tensors("soup_adamw_multi", a, true)) return rc;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps > 0.0) || !exp_avg || !exp_avg_sq ||
      !step || !ticket || (state_bits != 8 && state_bits != 32) ||
      (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) || partials < 0 || (partials > 0 && !grad_squares) ||
      !aligned16(exp_avg) || !aligned16(exp_avg_sq)) {
    set_last_error("soup_adamw_multi: bad arguments");
    return SOUP_ERR_INVALID;
  }
  const States s{exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale};
  const Hyper h{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, (float)lr,
                (float)(1.0 - lr * weight_decay), log(beta1), log(beta2), (float)max_norm};
  const double* sq = partials > 0 ? static_cast<const double*>(grad_squares) : nullptr;
  cudaStream_t st = as_stream(stream);
#define RUN(T)                                                                                                  \
  return state_bits == 8 ? step_run<T, true>(a, s, h, sq, partials, norm_out, step, ticket, last, st)           \
                         : step_run<T, false>(a, s, h, sq, partials, norm_out, step, ticket, last, st)
  if (dtype == SOUP_F32) RUN(float);
  if (dtype == SOUP_BF16) RUN(__nv_bfloat16);
  if (dtype == SOUP_F16) RUN(__half);
#undef RUN
  set_last_error("soup_adamw_multi: unsupported dtype");
  return SOUP_ERR_INVALID;
}

}  // extern "C"
