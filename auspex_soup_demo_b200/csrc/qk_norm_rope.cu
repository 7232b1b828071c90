// Norms of queries and keys for each head and their rotation, in one pass.
//
//   n = x * rstd * w,  rstd = 1 / sqrt(mean(x^2) + eps)      (w may be absent: n = x)
//   y1 = n1 c - n2 s,  y2 = n1 s + n2 c                      (halves of the head dim)
// backward:
//   dn1 = g1 c + g2 s, dn2 = g2 c - g1 s
//   dx  = rstd (dn w - x rstd^2 mean(dn w x)),  dw = sum over tokens and heads of dn x rstd
// c and s of frequency i come from cos / sin tables, or from the token's position
// on that frequency's axis: theta = pos[axis(i)] * inv_freq[i], reduced to a
// fraction of a turn in 64 bits (a position of 100000 leaves 3e-3 of an angle in
// 32 bits), then one sincospi in 32 bits.
//
// HBM-bound: q and k are read once and written once (backward: x and dy read, dx
// written; rstd is formed again from x, which is read anyway). Everything between
// is in 32 bits; the one rounding is the output's.
//
// A row (token, head) is `lanes` threads of one warp, each with a 16-byte vector
// of the first half and the matching vector of the second, so a rotation needs no
// exchange and a norm needs log2(lanes) shuffles. A CTA takes P tokens at a time:
// their rows' loads are in flight while the CTA forms the P tables in shared
// memory, which all heads then read. Head dims whose half is not a multiple of a
// vector, or rows that are not 16-byte aligned, take a warp per row instead.
#include "soup_common.cuh"

namespace soup {
namespace {

constexpr int kMaxDim = 512;        // head dim
constexpr int kMaxHalf = kMaxDim / 2;
constexpr int kMaxThreads = 512;

struct HeadRows {
  const void* x;       // q or k
  const void* g;       // backward: gradient of the rotated rows
  void* out;           // rotated rows, or dx
  int64_t xb, xh, xs;  // strides in elements (the head dim is contiguous)
  int64_t gb, gh, gs;
  int64_t ob, oh, os;
  const void* w;       // norm weight [D], or null
  int heads;
};

struct Angles {
  const void* cos;     // tables, or null
  const void* sin;
  int64_t tb, ts;      // strides of both
  int dtype;
  const void* pos;     // positions, axis pa apart
  int64_t pa, pb, ps;
  int pos64;
  const float* inv_freq;
  uint8_t axis[kMaxHalf];
};

struct Shape {
  int64_t tokens;      // batch * seq
  int64_t seq;
  int half;
  int lanes;           // threads of a row (a power of two)
  float eps;
  int w_dtype;
  float sign;          // -1: the inverse rotation
};

__device__ __forceinline__ float load_as_f(const void* p, int64_t i, int dtype) {
  if (dtype == SOUP_F32) return static_cast<const float*>(p)[i];
  if (dtype == SOUP_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// cos and sin of frequency i for the token at (b, s)
__device__ __forceinline__ void angle_of(const Angles& a, int64_t b, int64_t s, int i, float& c, float& sn) {
  if (a.cos) {
    const int64_t at = b * a.tb + s * a.ts + i;
    c = load_as_f(a.cos, at, a.dtype);
    sn = load_as_f(a.sin, at, a.dtype);
  } else {
    const int64_t at = a.axis[i] * a.pa + b * a.pb + s * a.ps;
    const double pos = a.pos64 ? (double)static_cast<const long long*>(a.pos)[at]
                               : (double)static_cast<const int*>(a.pos)[at];
    const double turns = pos * ((double)a.inv_freq[i] * 0.15915494309189533577);  // 1 / (2 pi)
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &c);
  }
}

// The tables of tokens [n0, n0 + P) into shared memory (cos, then sin, half each).
template <int P>
__device__ __forceinline__ void fill_tables(const Angles& a, const Shape& sh, int64_t n0, float* tab) {
  for (int e = threadIdx.x; e < P * sh.half; e += blockDim.x) {
    const int p = e / sh.half, i = e - p * sh.half;
    const int64_t n = n0 + p;
    if (n >= sh.tokens) break;
    const int64_t b = n / sh.seq;
    float c, s;
    angle_of(a, b, n - b * sh.seq, i, c, s);
    tab[p * 2 * sh.half + i] = c;
    tab[(p * 2 + 1) * sh.half + i] = sh.sign * s;
  }
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int NE>
__device__ __forceinline__ void load_table(const float* t, float (&v)[NE]) {
#pragma unroll
  for (int e = 0; e < NE; e += 4) {
    const float4 q = *reinterpret_cast<const float4*>(t + e);
    v[e] = q.x;
    v[e + 1] = q.y;
    v[e + 2] = q.z;
    v[e + 3] = q.w;
  }
}

// Forward (and, without weights and with sign -1, the backward of a rotation alone).
template <typename T, int P, bool NORM>
__global__ void __launch_bounds__(kMaxThreads) qk_rope_fwd_kernel(HeadRows q, HeadRows k,
                                                                  const __grid_constant__ Angles ang,
                                                                  Shape sh) {
  constexpr int NE = Vec16<T>::N;
  __shared__ __align__(16) float tab[P * 2 * kMaxHalf];
  pdl_wait();
  pdl_trigger();
  const int half = sh.half, chunks = half / NE;
  const int shift = __ffs(sh.lanes) - 1;
  const int slots = (q.heads + k.heads) << shift;
  const int64_t n0 = (int64_t)blockIdx.x * P;
  bool ready = false;
  for (int base = 0; base < slots; base += blockDim.x) {
    const int i = base + threadIdx.x;
    const int h = i >> shift, d = (i & (sh.lanes - 1)) * NE;
    const bool on = i < slots && d < chunks * NE;
    const bool isq = h < q.heads;
    const HeadRows& t = isq ? q : k;
    const int64_t hh = isq ? h : h - q.heads;
    Vec16<T> x1[P], x2[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      x1[p].u = make_uint4(0, 0, 0, 0);
      x2[p].u = make_uint4(0, 0, 0, 0);
      const int64_t n = n0 + p;
      if (on && n < sh.tokens) {
        const int64_t b = n / sh.seq, s = n - b * sh.seq;
        const T* xp = static_cast<const T*>(t.x) + b * t.xb + hh * t.xh + s * t.xs + d;
        x1[p] = ld16_stream(xp);
        x2[p] = ld16_stream(xp + half);
      }
    }
    float w1[NE], w2[NE];
    if constexpr (NORM) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        w1[e] = on ? load_as_f(t.w, d + e, sh.w_dtype) : 0.f;
        w2[e] = on ? load_as_f(t.w, half + d + e, sh.w_dtype) : 0.f;
      }
    }
    if (!ready) {  // block-uniform
      fill_tables<P>(ang, sh, n0, tab);
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int64_t n = n0 + p;
      if (n >= sh.tokens) break;  // block-uniform
      float a[NE], bb[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        a[e] = Cvt<T>::to_f(x1[p].v[e]);
        bb[e] = Cvt<T>::to_f(x2[p].v[e]);
      }
      if constexpr (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) ss = fmaf(a[e], a[e], fmaf(bb[e], bb[e], ss));
        ss = lanes_sum(ss, sh.lanes);
        const float rstd = 1.f / sqrtf(ss / (float)(2 * half) + sh.eps);
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          a[e] = a[e] * rstd * w1[e];
          bb[e] = bb[e] * rstd * w2[e];
        }
      }
      if (on) {
        float c[NE], s[NE];
        load_table<NE>(tab + p * 2 * half + d, c);
        load_table<NE>(tab + (p * 2 + 1) * half + d, s);
        const int64_t b = n / sh.seq, sp = n - b * sh.seq;
        T* op = static_cast<T*>(t.out) + b * t.ob + hh * t.oh + sp * t.os + d;
        Vec16<T> y1, y2;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          y1.v[e] = Cvt<T>::from_f(a[e] * c[e] - bb[e] * s[e]);
          y2.v[e] = Cvt<T>::from_f(a[e] * s[e] + bb[e] * c[e]);
        }
        st16_stream(op, y1);
        st16_stream(op + half, y2);
      }
    }
  }
}

// Backward with norms. One (head, vector) slot a thread for all of the CTA's
// tokens, so a thread's share of dw stays in its registers; blockIdx.y takes the
// next blockDim.x slots. The CTA joins its rows of dw in the order of the heads and
// leaves one partial row [2][D] (q, k), which dw_join_kernel sums in block order.
template <typename T, int P>
__global__ void __launch_bounds__(kMaxThreads) qk_norm_rope_bwd_kernel(HeadRows q, HeadRows k,
                                                                       const __grid_constant__ Angles ang,
                                                                       Shape sh, float* __restrict__ dw_part) {
  constexpr int NE = Vec16<T>::N;
  extern __shared__ __align__(16) float smem[];  // tables [P][2][half], later dw [blockDim][2 NE]
  pdl_wait();
  pdl_trigger();
  const int half = sh.half, chunks = half / NE;
  const int shift = __ffs(sh.lanes) - 1;
  const int slots = (q.heads + k.heads) << shift;
  const int i = blockIdx.y * blockDim.x + threadIdx.x;
  const int h = i >> shift, d = (i & (sh.lanes - 1)) * NE;
  const bool on = i < slots && d < chunks * NE;
  const bool isq = h < q.heads;
  const HeadRows& t = isq ? q : k;
  const int64_t hh = isq ? h : h - q.heads;
  float w1[NE], w2[NE], dw1[NE], dw2[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    w1[e] = on ? load_as_f(t.w, d + e, sh.w_dtype) : 0.f;
    w2[e] = on ? load_as_f(t.w, half + d + e, sh.w_dtype) : 0.f;
    dw1[e] = dw2[e] = 0.f;
  }
  const int64_t tiles = (sh.tokens + P - 1) / P;
  const float inv_d = 1.f / (float)(2 * half);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t n0 = tile * P;
    Vec16<T> x1[P], x2[P], g1[P], g2[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      x1[p].u = x2[p].u = g1[p].u = g2[p].u = make_uint4(0, 0, 0, 0);
      const int64_t n = n0 + p;
      if (on && n < sh.tokens) {
        const int64_t b = n / sh.seq, s = n - b * sh.seq;
        const T* xp = static_cast<const T*>(t.x) + b * t.xb + hh * t.xh + s * t.xs + d;
        const T* gp = static_cast<const T*>(t.g) + b * t.gb + hh * t.gh + s * t.gs + d;
        x1[p] = ld16_stream(xp);
        x2[p] = ld16_stream(xp + half);
        g1[p] = ld16_stream(gp);
        g2[p] = ld16_stream(gp + half);
      }
    }
    __syncthreads();  // the tables of the tile before are read
    fill_tables<P>(ang, sh, n0, smem);
    __syncthreads();
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int64_t n = n0 + p;
      if (n >= sh.tokens) break;  // block-uniform
      float c[NE], s[NE], dn1[NE], dn2[NE];
      const int dt = on ? d : 0;
      load_table<NE>(smem + p * 2 * half + dt, c);
      load_table<NE>(smem + (p * 2 + 1) * half + dt, s);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const float a = Cvt<T>::to_f(x1[p].v[e]), bb = Cvt<T>::to_f(x2[p].v[e]);
        const float ga = Cvt<T>::to_f(g1[p].v[e]), gb = Cvt<T>::to_f(g2[p].v[e]);
        dn1[e] = ga * c[e] + gb * s[e];
        dn2[e] = gb * c[e] - ga * s[e];
        ss = fmaf(a, a, fmaf(bb, bb, ss));
        dot = fmaf(dn1[e] * w1[e], a, fmaf(dn2[e] * w2[e], bb, dot));
      }
      for (int o = sh.lanes >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
      const float rstd = 1.f / sqrtf(ss * inv_d + sh.eps);
      const float back = dot * inv_d * rstd * rstd;
      Vec16<T> y1, y2;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const float a = Cvt<T>::to_f(x1[p].v[e]), bb = Cvt<T>::to_f(x2[p].v[e]);
        dw1[e] = fmaf(dn1[e], a * rstd, dw1[e]);
        dw2[e] = fmaf(dn2[e], bb * rstd, dw2[e]);
        y1.v[e] = Cvt<T>::from_f(rstd * (dn1[e] * w1[e] - a * back));
        y2.v[e] = Cvt<T>::from_f(rstd * (dn2[e] * w2[e] - bb * back));
      }
      if (on) {
        const int64_t b = n / sh.seq, sp = n - b * sh.seq;
        T* op = static_cast<T*>(t.out) + b * t.ob + hh * t.oh + sp * t.os + d;
        st16_stream(op, y1);
        st16_stream(op + half, y2);
      }
    }
  }
  if (!dw_part) return;
  __syncthreads();
  float* mine = smem + threadIdx.x * 2 * NE;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    mine[e] = dw1[e];
    mine[NE + e] = dw2[e];
  }
  __syncthreads();
  // this block's heads, in order; a block's slots start at a head's first
  const int dim = 2 * half;
  const int h0 = (blockIdx.y * blockDim.x) >> shift;
  const int h1 = min((int)((blockIdx.y + 1) * blockDim.x) >> shift, q.heads + k.heads);
  float* row = dw_part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * dim;
  for (int e = threadIdx.x; e < 2 * dim; e += blockDim.x) {
    const int which = e / dim, col = e - which * dim;
    const int second = col >= half ? 1 : 0, c = col - second * half;
    const int lo = which ? max(h0, q.heads) : h0, hi = which ? h1 : min(h1, q.heads);
    float sum = 0.f;
    for (int hd = lo; hd < hi; ++hd) {
      const int th = (hd << shift) + c / NE - blockIdx.y * blockDim.x;
      sum += smem[th * 2 * NE + second * NE + c % NE];
    }
    row[e] = sum;
  }
}

// dw [2][D] = sum of the partial rows in block order: a warp-wide group of 32
// threads a column group, 32 rows apart, joined in shared memory.
__global__ void __launch_bounds__(1024) dw_join_kernel(const float* __restrict__ part, int rows, int dim,
                                                       void* __restrict__ dwq, void* __restrict__ dwk,
                                                       int w_dtype) {
  __shared__ float acc[32][33];
  pdl_wait();
  pdl_trigger();
  const int col = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (col < 2 * dim)
    for (int r = threadIdx.y; r < rows; r += 32) s += part[(int64_t)r * 2 * dim + col];
  acc[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < 2 * dim) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += acc[r][threadIdx.x];
    void* dst = col < dim ? dwq : dwk;
    const int c = col < dim ? col : col - dim;
    if (!dst) return;
    if (w_dtype == SOUP_F32) static_cast<float*>(dst)[c] = t;
    else if (w_dtype == SOUP_BF16) static_cast<__nv_bfloat16*>(dst)[c] = __float2bfloat16_rn(t);
    else static_cast<__half*>(dst)[c] = __float2half_rn(t);
  }
}

// Any alignment and any even head dim: a warp a row, lane l on the pairs l, l + 32, ...
// Forward and backward; dw shares stay in registers while the warp walks rows of
// one tensor, and are joined per block as above (a block is rows of q or of k).
constexpr int kAnyWarps = 8;
constexpr int kAnyPairs = kMaxHalf / 32;

template <typename T, bool NORM, bool BWD>
__global__ void __launch_bounds__(32 * kAnyWarps) qk_rope_any_kernel(HeadRows q, HeadRows k,
                                                                     const __grid_constant__ Angles ang,
                                                                     Shape sh, float* __restrict__ dw_part) {
  __shared__ float share[BWD && NORM ? kAnyWarps * kMaxDim : 1];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const HeadRows& t = blockIdx.y ? k : q;
  const int half = sh.half;
  const int64_t rows = sh.tokens * t.heads;
  float dw1[kAnyPairs], dw2[kAnyPairs];
#pragma unroll
  for (int j = 0; j < kAnyPairs; ++j) dw1[j] = dw2[j] = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * kAnyWarps + warp; r < rows; r += (int64_t)gridDim.x * kAnyWarps) {
    const int64_t n = r / t.heads, hh = r - n * t.heads;
    const int64_t b = n / sh.seq, s = n - b * sh.seq;
    const T* xp = static_cast<const T*>(t.x) + b * t.xb + hh * t.xh + s * t.xs;
    const T* gp = BWD && NORM ? static_cast<const T*>(t.g) + b * t.gb + hh * t.gh + s * t.gs : nullptr;
    T* op = static_cast<T*>(t.out) + b * t.ob + hh * t.oh + s * t.os;
    float a[kAnyPairs], bb[kAnyPairs], c[kAnyPairs], sn[kAnyPairs], d1[kAnyPairs], d2[kAnyPairs];
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < kAnyPairs; ++j) {
      const int i = lane + 32 * j;
      a[j] = bb[j] = d1[j] = d2[j] = 0.f;
      c[j] = sn[j] = 0.f;
      if (i >= half) continue;
      a[j] = Cvt<T>::to_f(xp[i]);
      bb[j] = Cvt<T>::to_f(xp[half + i]);
      angle_of(ang, b, s, i, c[j], sn[j]);
      sn[j] *= sh.sign;
      if constexpr (NORM) ss = fmaf(a[j], a[j], fmaf(bb[j], bb[j], ss));
      if constexpr (BWD && NORM) {
        const float g1 = Cvt<T>::to_f(gp[i]), g2 = Cvt<T>::to_f(gp[half + i]);
        d1[j] = g1 * c[j] + g2 * sn[j];
        d2[j] = g2 * c[j] - g1 * sn[j];
        dot += d1[j] * load_as_f(t.w, i, sh.w_dtype) * a[j] + d2[j] * load_as_f(t.w, half + i, sh.w_dtype) * bb[j];
      }
    }
    float rstd = 1.f;
    if constexpr (NORM) rstd = 1.f / sqrtf(warp_sum(ss) / (float)(2 * half) + sh.eps);
    float back = 0.f;
    if constexpr (BWD && NORM) back = warp_sum(dot) / (float)(2 * half) * rstd * rstd;
#pragma unroll
    for (int j = 0; j < kAnyPairs; ++j) {
      const int i = lane + 32 * j;
      if (i >= half) continue;
      const float u = NORM ? load_as_f(t.w, i, sh.w_dtype) : 1.f;
      const float v = NORM ? load_as_f(t.w, half + i, sh.w_dtype) : 1.f;
      if constexpr (BWD && NORM) {
        dw1[j] = fmaf(d1[j], a[j] * rstd, dw1[j]);
        dw2[j] = fmaf(d2[j], bb[j] * rstd, dw2[j]);
        op[i] = Cvt<T>::from_f(rstd * (d1[j] * u - a[j] * back));
        op[half + i] = Cvt<T>::from_f(rstd * (d2[j] * v - bb[j] * back));
      } else {
        const float y1 = a[j] * rstd * u, y2 = bb[j] * rstd * v;
        op[i] = Cvt<T>::from_f(y1 * c[j] - y2 * sn[j]);
        op[half + i] = Cvt<T>::from_f(y1 * sn[j] + y2 * c[j]);
      }
    }
  }
  if constexpr (BWD && NORM) {
    if (!dw_part) return;
#pragma unroll
    for (int j = 0; j < kAnyPairs; ++j) {
      const int i = lane + 32 * j;
      if (i >= half) continue;
      share[warp * kMaxDim + i] = dw1[j];
      share[warp * kMaxDim + half + i] = dw2[j];
    }
    __syncthreads();
    float* row = dw_part + (int64_t)blockIdx.x * 4 * half + blockIdx.y * 2 * half;
    for (int e = threadIdx.x; e < 2 * half; e += blockDim.x) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kAnyWarps; ++w) sum += share[w * kMaxDim + e];
      row[e] = sum;
    }
  }
}

// Threads of a CTA and rows of dw partials of the backward, from sizes alone (the
// caller's workspace is sized by them).
struct BwdPlan {
  int threads, groups, blocks;  // groups: CTAs that share a token tile
};

constexpr int kBwdTokens = 2;

inline int row_lanes(int chunks) {
  int l = 1;
  while (l < chunks) l <<= 1;
  return l;
}

BwdPlan bwd_plan(int64_t tokens, int64_t heads, int lanes) {
  BwdPlan p;
  const int64_t slots = heads * lanes;
  p.threads = slots >= kMaxThreads ? kMaxThreads : (int)((slots + 31) / 32 * 32);
  // whole heads in a block: lanes divides 32, so also the thread count
  p.groups = (int)((slots + p.threads - 1) / p.threads);
  int64_t cap = (int64_t)num_sms() * (p.threads <= 128 ? 6 : p.threads <= 256 ? 4 : 2) / p.groups;
  if (cap < 1) cap = 1;
  const int64_t tiles = (tokens + kBwdTokens - 1) / kBwdTokens;
  p.blocks = (int)(tiles < cap ? tiles : cap);
  return p;
}

constexpr int kAnyBlocks = 592;  // of each tensor, at most

int any_blocks(int64_t tokens, int64_t heads) {
  const int64_t b = (tokens * heads + kAnyWarps - 1) / kAnyWarps;
  return (int)(b < kAnyBlocks ? (b < 1 ? 1 : b) : kAnyBlocks);
}

bool rows_ok(const HeadRows& t, bool grads, int64_t es) {
  if (t.heads == 0) return true;
  auto ok = [&](const void* p, int64_t b, int64_t h, int64_t s) {
    return aligned16(p) && (b * es) % 16 == 0 && (h * es) % 16 == 0 && (s * es) % 16 == 0;
  };
  return ok(t.x, t.xb, t.xh, t.xs) && ok(t.out, t.ob, t.oh, t.os) && (!grads || ok(t.g, t.gb, t.gh, t.gs));
}

template <typename T>
bool vector_path(const HeadRows& q, const HeadRows& k, int half, bool grads) {
  constexpr int NE = Vec16<T>::N;
  return half % NE == 0 && half / NE <= 32 && rows_ok(q, grads, sizeof(T)) && rows_ok(k, grads, sizeof(T));
}

template <typename T>
int run_fwd(const HeadRows& q, const HeadRows& k, const Angles& a, Shape sh, bool norm, cudaStream_t st) {
  constexpr int NE = Vec16<T>::N;
  const int heads = q.heads + k.heads;
  cudaError_t e;
  if (vector_path<T>(q, k, sh.half, false)) {
    sh.lanes = row_lanes(sh.half / NE);
    const int64_t slots = (int64_t)heads * sh.lanes;
    int threads = slots >= 256 ? 256 : (int)((slots + 31) / 32 * 32);
    // four tokens a CTA keep 128 bytes a thread in flight; with few tokens one a
    // CTA, so that more SMs share them
    if (sh.tokens >= 4 * (int64_t)num_sms()) {
      const dim3 grid((unsigned)((sh.tokens + 3) / 4));
      e = norm ? launch_pdl(qk_rope_fwd_kernel<T, 4, true>, grid, dim3(threads), 0, st, q, k, a, sh)
               : launch_pdl(qk_rope_fwd_kernel<T, 4, false>, grid, dim3(threads), 0, st, q, k, a, sh);
    } else {
      const dim3 grid((unsigned)sh.tokens);
      e = norm ? launch_pdl(qk_rope_fwd_kernel<T, 1, true>, grid, dim3(threads), 0, st, q, k, a, sh)
               : launch_pdl(qk_rope_fwd_kernel<T, 1, false>, grid, dim3(threads), 0, st, q, k, a, sh);
    }
  } else {
    const int most = q.heads > k.heads ? q.heads : k.heads;
    const dim3 grid(any_blocks(sh.tokens, most), k.heads ? 2 : 1);
    float* none = nullptr;
    e = norm ? launch_pdl(qk_rope_any_kernel<T, true, false>, grid, dim3(32 * kAnyWarps), 0, st, q, k, a, sh, none)
             : launch_pdl(qk_rope_any_kernel<T, false, false>, grid, dim3(32 * kAnyWarps), 0, st, q, k, a, sh, none);
  }
  return cuda_status(e);
}

template <typename T>
int run_bwd(const HeadRows& q, const HeadRows& k, const Angles& a, Shape sh, void* dwq, void* dwk, float* part,
            cudaStream_t st) {
  constexpr int NE = Vec16<T>::N;
  const int heads = q.heads + k.heads, dim = 2 * sh.half;
  const bool dw = dwq || dwk;
  int rows;
  cudaError_t e;
  if (vector_path<T>(q, k, sh.half, true)) {
    sh.lanes = row_lanes(sh.half / NE);
    const BwdPlan p = bwd_plan(sh.tokens, heads, sh.lanes);
    size_t smem = sizeof(float) * (size_t)kBwdTokens * dim;
    const size_t join = sizeof(float) * (size_t)p.threads * 2 * NE;
    if (dw && join > smem) smem = join;
    rows = p.blocks * p.groups;
    e = launch_pdl(qk_norm_rope_bwd_kernel<T, kBwdTokens>, dim3(p.blocks, p.groups), dim3(p.threads), smem, st, q,
                   k, a, sh, dw ? part : nullptr);
  } else {
    const int most = q.heads > k.heads ? q.heads : k.heads;
    rows = any_blocks(sh.tokens, most);
    e = launch_pdl(qk_rope_any_kernel<T, true, true>, dim3(rows, 2), dim3(32 * kAnyWarps), 0, st, q, k, a, sh,
                   dw ? part : nullptr);
  }
  if (e != cudaSuccess || !dw) return cuda_status(e);
  return cuda_status(launch_pdl(dw_join_kernel, dim3((2 * dim + 31) / 32), dim3(32, 32), 0, st,
                                static_cast<const float*>(part), rows, dim, dwq, dwk, sh.w_dtype));
}

bool fill_angles(Angles& a, const void* cos, const void* sin, int64_t tb, int64_t ts, int dtype, const void* pos,
                 int pos64, int64_t pa, int64_t pb, int64_t ps, const float* inv_freq, const uint8_t* axis,
                 int64_t half) {
  a = Angles{};
  if (cos && sin) {
    a.cos = cos;
    a.sin = sin;
    a.tb = tb;
    a.ts = ts;
    a.dtype = dtype;
    return dtype == SOUP_F32 || dtype == SOUP_BF16 || dtype == SOUP_F16;
  }
  if (cos || sin || !pos || !inv_freq || !axis) return false;
  a.pos = pos;
  a.pos64 = pos64;
  a.pa = pa;
  a.pb = pb;
  a.ps = ps;
  a.inv_freq = inv_freq;
  for (int64_t i = 0; i < half; ++i) a.axis[i] = axis[i];
  return true;
}

}  // namespace
}  // namespace soup

using namespace soup;

extern "C" {

size_t soup_qk_norm_rope_bwd_workspace_bytes(int64_t batch, int64_t seq, int64_t hq, int64_t hk,
                                             int64_t head_dim) {
  if (batch <= 0 || seq <= 0 || hq <= 0 || hk <= 0 || head_dim <= 0) return 0;
  // the most partial rows any dtype and alignment gives
  const int64_t tokens = batch * seq;
  int64_t rows = any_blocks(tokens, hq > hk ? hq : hk);
  for (int ne = 4; ne <= 8; ne += 4) {
    if ((head_dim / 2) % ne || head_dim / 2 / ne > 32) continue;
    const BwdPlan p = bwd_plan(tokens, hq + hk, row_lanes((int)(head_dim / 2 / ne)));
    if ((int64_t)p.blocks * p.groups > rows) rows = (int64_t)p.blocks * p.groups;
  }
  return sizeof(float) * (size_t)(rows * 2 * head_dim);
}

int soup_qk_norm_rope(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int64_t hq,
                      const void* k, const int64_t* k_strides, void* k_out, const int64_t* k_out_strides,
                      int64_t hk, const void* q_weight, const void* k_weight, float eps, const void* cos,
                      const void* sin, int64_t table_sb, int64_t table_ss, int table_dtype, const void* positions,
                      int positions_64, int64_t pos_sa, int64_t pos_sb, int64_t pos_ss, const float* inv_freq,
                      const uint8_t* axes, int64_t batch, int64_t seq, int64_t head_dim, int dtype, int w_dtype,
                      int inverse, void* stream) {
  const bool norm = q_weight || k_weight;
  if (!q || !q_strides || !q_out || !q_out_strides || hq <= 0 || !k || !k_strides || !k_out || !k_out_strides ||
      hk <= 0 || batch <= 0 || seq <= 0 || head_dim <= 0 || head_dim % 2 || head_dim > kMaxDim || hq > 4096 ||
      hk > 4096 || batch > (int64_t(1) << 31) / seq || (norm && (!q_weight || !k_weight || inverse))) {
    set_last_error("soup_qk_norm_rope: bad arguments");
    return SOUP_ERR_INVALID;
  }
  Angles a;
  if (!fill_angles(a, cos, sin, table_sb, table_ss, table_dtype, positions, positions_64, pos_sa, pos_sb, pos_ss,
                   inv_freq, axes, head_dim / 2)) {
    set_last_error("soup_qk_norm_rope: cos and sin tables, or positions with inv_freq and axes");
    return SOUP_ERR_INVALID;
  }
  HeadRows tq{q, nullptr, q_out, q_strides[0], q_strides[1], q_strides[2], 0, 0, 0,
              q_out_strides[0], q_out_strides[1], q_out_strides[2], q_weight, (int)hq};
  HeadRows tk{k, nullptr, k_out, k_strides[0], k_strides[1], k_strides[2], 0, 0, 0,
              k_out_strides[0], k_out_strides[1], k_out_strides[2], k_weight, (int)hk};
  Shape sh{batch * seq, seq, (int)(head_dim / 2), 32, eps, w_dtype, inverse ? -1.f : 1.f};
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_BF16) return run_fwd<__nv_bfloat16>(tq, tk, a, sh, norm, st);
  if (dtype == SOUP_F16) return run_fwd<__half>(tq, tk, a, sh, norm, st);
  if (dtype == SOUP_F32) return run_fwd<float>(tq, tk, a, sh, norm, st);
  set_last_error("soup_qk_norm_rope: unsupported dtype");
  return SOUP_ERR_INVALID;
}

int soup_qk_norm_rope_bwd(const void* dq_out, const int64_t* dq_out_strides, const void* q, const int64_t* q_strides,
                          void* dq, const int64_t* dq_strides, int64_t hq, const void* dk_out,
                          const int64_t* dk_out_strides, const void* k, const int64_t* k_strides, void* dk,
                          const int64_t* dk_strides, int64_t hk, const void* q_weight, const void* k_weight,
                          float eps, void* dq_weight, void* dk_weight, const void* cos, const void* sin,
                          int64_t table_sb, int64_t table_ss, int table_dtype, const void* positions,
                          int positions_64, int64_t pos_sa, int64_t pos_sb, int64_t pos_ss, const float* inv_freq,
                          const uint8_t* axes, int64_t batch, int64_t seq, int64_t head_dim, int dtype, int w_dtype,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!dq_out || !dq_out_strides || !q || !q_strides || !dq || !dq_strides || hq <= 0 || !dk_out ||
      !dk_out_strides || !k || !k_strides || !dk || !dk_strides || hk <= 0 || !q_weight || !k_weight || batch <= 0 ||
      seq <= 0 || head_dim <= 0 || head_dim % 2 || head_dim > kMaxDim || hq > 4096 || hk > 4096 ||
      batch > (int64_t(1) << 31) / seq) {
    set_last_error("soup_qk_norm_rope_bwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  Angles a;
  if (!fill_angles(a, cos, sin, table_sb, table_ss, table_dtype, positions, positions_64, pos_sa, pos_sb, pos_ss,
                   inv_freq, axes, head_dim / 2)) {
    set_last_error("soup_qk_norm_rope_bwd: cos and sin tables, or positions with inv_freq and axes");
    return SOUP_ERR_INVALID;
  }
  if ((dq_weight || dk_weight) &&
      (!workspace || !aligned16(workspace) ||
       workspace_bytes < soup_qk_norm_rope_bwd_workspace_bytes(batch, seq, hq, hk, head_dim))) {
    set_last_error("soup_qk_norm_rope_bwd: workspace missing, unaligned or too small");
    return SOUP_ERR_WORKSPACE;
  }
  HeadRows tq{q, dq_out, dq, q_strides[0], q_strides[1], q_strides[2],
              dq_out_strides[0], dq_out_strides[1], dq_out_strides[2],
              dq_strides[0], dq_strides[1], dq_strides[2], q_weight, (int)hq};
  HeadRows tk{k, dk_out, dk, k_strides[0], k_strides[1], k_strides[2],
              dk_out_strides[0], dk_out_strides[1], dk_out_strides[2],
              dk_strides[0], dk_strides[1], dk_strides[2], k_weight, (int)hk};
  Shape sh{batch * seq, seq, (int)(head_dim / 2), 32, eps, w_dtype, 1.f};
  float* part = static_cast<float*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_BF16) return run_bwd<__nv_bfloat16>(tq, tk, a, sh, dq_weight, dk_weight, part, st);
  if (dtype == SOUP_F16) return run_bwd<__half>(tq, tk, a, sh, dq_weight, dk_weight, part, st);
  if (dtype == SOUP_F32) return run_bwd<float>(tq, tk, a, sh, dq_weight, dk_weight, part, st);
  set_last_error("soup_qk_norm_rope_bwd: unsupported dtype");
  return SOUP_ERR_INVALID;
}

}  // extern "C"
