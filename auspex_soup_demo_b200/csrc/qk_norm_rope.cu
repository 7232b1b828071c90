// Norms of queries and keys for each head and their rotation, in one pass.
//
//   n = x * rstd * w,  rstd = 1 / sqrt(mean(x^2) + eps)      (w may be absent: n = x)
//   y1 = n1 c - n2 s,  y2 = n1 s + n2 c                      (halves of the head dim)
// backward:
//   dn1 = g1 c + g2 s, dn2 = g2 c - g1 s
//   dx  = rstd (dn w - x rstd * rstd mean(dn w x)),  dw = sum over tokens and heads of dn x rstd
// c and s of frequency i come from cos / sin tables, or from the token's position
// on that frequency's axis: theta = pos[axis(i)] * inv_freq[i], reduced to a
// fraction of a turn in 64 bits (a position of 100000 leaves 3e-3 of an angle in
// 32 bits), then one sincospi in 32 bits.
//
// HBM-bound: q and k are read once and written once (backward: x and dy read, dx
// written; rstd is formed again from x, which is read anyway). Everything between
// is in 32 bits; the one rounding is the output's.
//
// A row (token, head) is `lanes` threads of one warp, each with NE elements of the
// first half and the matching NE of the second, so a rotation needs no exchange and a
// norm needs log2(lanes) shuffles. Forward: a thread takes the rows of two tokens and is
// done. Backward: a CTA walks a run of tokens and a thread keeps its (head, elements) slot
// for all of them, so that its share of dw stays in registers; its rows arrive by cp.async
// in a ring of shared memory of its own (nobody else reads them, so no barrier), several
// tokens ahead, which keeps enough bytes in flight without the registers for them. Head
// dims whose half is not a multiple of a vector, or rows that are not 16-byte aligned,
// take a warp per row instead.
#include <stdio.h>

#include <mutex>
#include <type_traits>

#include "soup_common.cuh"

namespace soup {
namespace {

constexpr int kMaxDim = 512;        // head dim
constexpr int kMaxHalf = kMaxDim / 2;
constexpr int kMaxThreads = 256;
// Stages of a thread's ring, and resident CTAs of 256 threads on an SM by the bytes of a
// half that a thread holds: the rings take 128 to 196 KB of an SM's shared memory.
constexpr int kBwdStages = 4;
constexpr int kFwdTokens = 2;
__host__ __device__ constexpr int fwd_ctas(int bytes) { return bytes == 16 ? 4 : 2; }
__host__ __device__ constexpr int bwd_ctas(int bytes) { return bytes == 16 ? 2 : 1; }

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

// Division of an index below 2^31 by d as a product: with l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d), n m >> (31 + l) is n / d (Granlund and Montgomery's division
// by an invariant).
struct Div {
  uint32_t m;
  int shift;
  uint32_t d;
  __device__ __forceinline__ void split(uint32_t n, int64_t& q, int64_t& r) const {
    const uint32_t t = (uint32_t)(((uint64_t)n * m) >> shift);
    q = t;
    r = n - t * d;
  }
};

inline Div make_div(int64_t d) {
  int l = 0;
  while ((int64_t(1) << l) < d) ++l;
  return Div{(uint32_t)((((uint64_t)1 << (31 + l)) + (uint64_t)d - 1) / (uint64_t)d), 31 + l, (uint32_t)d};
}

struct Shape {
  int batch, seq;
  Div tokens;          // of a sequence
  int half;
  int lanes;           // threads of a row (a power of two)
  int group_heads;     // heads of a CTA
  int side;            // tokens that it takes side by side
  float eps, inv_d;    // inv_d: 1 / D
  int w_dtype;
  float sign;          // -1: the inverse rotation
};

__device__ __forceinline__ float load_as_f(const void* p, int64_t i, int dtype) {
  if (dtype == SOUP_F32) return static_cast<const float*>(p)[i];
  if (dtype == SOUP_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// cos and sin of a position on frequency i
__device__ __forceinline__ void turn(const Angles& a, int64_t b, int64_t s, int i, float& c, float& sn) {
  const int64_t at = a.axis[i] * a.pa + b * a.pb + s * a.ps;
  const double pos = a.pos64 ? (double)static_cast<const long long*>(a.pos)[at]
                             : (double)static_cast<const int*>(a.pos)[at];
  const double turns = pos * ((double)a.inv_freq[i] * 0.15915494309189533577);  // 1 / (2 pi)
  sincospif((float)(2.0 * (turns - rint(turns))), &sn, &c);
}
__device__ __forceinline__ void angle_of(const Angles& a, int64_t b, int64_t s, int i, float& c, float& sn) {
  if (a.cos) {
    const int64_t at = b * a.tb + s * a.ts + i;
    c = load_as_f(a.cos, at, a.dtype);
    sn = load_as_f(a.sin, at, a.dtype);
  } else {
    turn(a, b, s, i, c, sn);
  }
}

// NE consecutive elements of type T in loads of up to 16 bytes, read and written as
// packed pairs of 32-bit numbers.
template <typename T, int NE>
struct Pack {
  static constexpr int kBytes = NE * (int)sizeof(T);
  static constexpr int kWords = kBytes / 4;
  uint32_t u[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) u[i] = 0;
  }
  template <bool STREAM>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4* q = reinterpret_cast<const uint4*>(p) + i / 4;
        const uint4 r = STREAM ? __ldcs(q) : *q;
        u[i] = r.x;
        u[i + 1] = r.y;
        u[i + 2] = r.z;
        u[i + 3] = r.w;
      }
    } else {
      static_assert(kBytes == 8, "8 or a multiple of 16 bytes");
      const uint2* q = reinterpret_cast<const uint2*>(p);
      const uint2 r = STREAM ? __ldcs(q) : *q;
      u[0] = r.x;
      u[1] = r.y;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4)
        __stcs(reinterpret_cast<uint4*>(p) + i / 4, make_uint4(u[i], u[i + 1], u[i + 2], u[i + 3]));
    } else {
      __stcs(reinterpret_cast<uint2*>(p), make_uint2(u[0], u[1]));
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
};

__device__ __forceinline__ uint64_t f2_same(float x) { return f2_pack(x, x); }
__device__ __forceinline__ float f2_sum(uint64_t p) {
  float x, y;
  f2_unpack(p, x, y);
  return x + y;
}
// a c - b s
__device__ __forceinline__ uint64_t f2_cross(uint64_t a, uint64_t c, uint64_t b, uint64_t s) {
  return f2_fma(f2_mul(b, s), f2_same(-1.f), f2_mul(a, c));
}

// Where cos and sin come from.
constexpr int kTableT = 0;    // tables of the rows' type
constexpr int kTableF = 1;    // fp32 tables
constexpr int kPositions = 2;

template <typename T, int SRC>
struct TableType {
  using type = typename std::conditional<SRC == kTableT, T, float>::type;
};

template <typename T, int NE>
__device__ __forceinline__ void load_weights(const void* w, int at, int dtype, uint64_t (&f)[NE / 2]) {
  if (dtype == SOUP_F32) {
    Pack<float, NE> p;
    p.template load<false>(static_cast<const float*>(w) + at);
#pragma unroll
    for (int e = 0; e < NE / 2; ++e) f[e] = p.pair(e);
  } else {
    Pack<T, NE> p;
    p.template load<false>(static_cast<const T*>(w) + at);
#pragma unroll
    for (int e = 0; e < NE / 2; ++e) f[e] = p.pair(e);
  }
}

// A thread's slot: its rows and its place in them.
struct Slot {
  bool on, isq;
  int64_t hh;
  int d, token;  // token: among those that the CTA takes side by side
  __device__ __forceinline__ Slot(const HeadRows& q, const HeadRows& k, const Shape& sh, int ne) {
    const int shift = __ffs(sh.lanes) - 1;
    const int row = threadIdx.x >> shift;
    token = threadIdx.y;
    const int h = blockIdx.y * sh.group_heads + row;
    d = (threadIdx.x & (sh.lanes - 1)) * ne;
    on = row < sh.group_heads && h < q.heads + k.heads && d < sh.half;
    isq = h < q.heads;
    hh = isq ? h : h - q.heads;
    if (!on) d = 0;
  }
};

// cos and sin of a thread's elements for a token.
template <typename T, int NE, int SRC>
struct Turn {
  using TT = typename TableType<T, SRC>::type;
  Pack<TT, NE> c, s;
  __device__ __forceinline__ void load(const TT* cos, const TT* sin) {
    c.template load<false>(cos);
    s.template load<false>(sin);
  }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A place in a run of tokens: their sequence and position, and the offset of the
// thread's elements in one strided tensor (or of the tables' row).
struct Cursor {
  int64_t at, step, wrap;  // wrap: from the last token of a sequence to the next one's first
  int s;
  __device__ __forceinline__ Cursor(int64_t b, int64_t s0, int64_t sb, int64_t ss, int seq)
      : at(b * sb + s0 * ss), step(ss), wrap(sb - (int64_t)(seq - 1) * ss), s((int)s0) {}
  __device__ __forceinline__ void next(int seq) {
    const bool last = ++s == seq;
    at += last ? wrap : step;
    if (last) s = 0;
  }
};

constexpr int kGroup = 4;  // tokens whose tables a CTA forms together (kPositions)

// The tables of `count` tokens from n0 on, as far as n1, into shared memory.
__device__ __forceinline__ void fill_tables(const Angles& a, const Shape& sh, int n0, int n1, int count, float* tab) {
  const int threads = blockDim.x * blockDim.y;
  for (int e = threadIdx.y * blockDim.x + threadIdx.x; e < count * sh.half; e += threads) {
    const int p = e / sh.half, i = e - p * sh.half;
    if (n0 + p >= n1) break;
    int64_t b, s;
    sh.tokens.split(n0 + p, b, s);
    float c, sn;
    turn(a, b, s, i, c, sn);
    tab[p * 2 * sh.half + i] = c;
    tab[(p * 2 + 1) * sh.half + i] = sn;
  }
}

// The CTA's run of tokens.
__device__ __forceinline__ void token_run(const Shape& sh, int& n0, int& n1) {
  const int64_t total = (int64_t)sh.batch * sh.seq;
  n0 = (int)(total * blockIdx.x / gridDim.x);
  n1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
}

// Walks the run: ring of S stages of PIECES 16-byte pieces a thread, filled by
// issue(token's stage address), tables from `src`, then work(stage address, tables).
template <int S, int SRC, class Issue, class Work>
__device__ __forceinline__ void walk_tokens(const Angles& ang, const Shape& sh, float* tab, uint32_t ring,
                                            uint32_t stage_bytes, Issue&& issue, Work&& work) {
  int n0, n1;
  token_run(sh, n0, n1);
  int put = 0;
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (n0 + i < n1) issue(ring + put * stage_bytes);
    copy_commit();
    put = put + 1 == S ? 0 : put + 1;
  }
  int get = 0;
  for (int n = n0; n < n1; ++n) {
    if (n + S - 1 < n1) issue(ring + put * stage_bytes);
    copy_commit();
    put = put + 1 == S ? 0 : put + 1;
    const float* table = tab;
    if constexpr (SRC == kPositions) {
      // two groups' tables in turn: what a group overwrites was read before the last barrier
      const int g = n - n0;
      float* mine = tab + (g / kGroup & 1) * kGroup * 2 * sh.half;
      if (g % kGroup == 0) {
        fill_tables(ang, sh, n, n1, kGroup, mine);
        __syncthreads();
      }
      table = mine + g % kGroup * 2 * sh.half;
    }
    copy_wait<S - 1>();
    work(ring + get * stage_bytes, table);
    get = get + 1 == S ? 0 : get + 1;
  }
}

// A piece is NE elements of every thread: 16-byte parts, `pitch` (16 x threads) apart.
template <typename T, int NE>
__device__ __forceinline__ void take(Pack<T, NE>& p, uint32_t at, uint32_t pitch) {
#pragma unroll
  for (int i = 0; i < Pack<T, NE>::kWords; i += 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(p.u[i]), "=r"(p.u[i + 1]), "=r"(p.u[i + 2]), "=r"(p.u[i + 3])
                 : "r"(at + i / 4 * pitch)
                 : "memory");
}
template <typename T, int NE>
__device__ __forceinline__ void give(uint32_t at, const T* src, uint32_t pitch) {
#pragma unroll
  for (int i = 0; i < Pack<T, NE>::kWords; i += 4) copy16(at + i / 4 * pitch, src + i * 4 / sizeof(T));
}

// Forward (and, without weights and with sign -1, the backward of a rotation alone). A
// thread takes one row's elements of P tokens; CTA (x, y) the tokens [x C P, ...) of all
// its heads, C of them side by side. CTAs come in the order of memory: DRAM then serves
// few pages at a time. 2 x 16001 tokens of 32/8 heads of 128 in bf16: 117 us, 5.6 TB/s;
// 130 us with resident CTAs that walk runs of tokens behind rings of cp.async.
template <typename T, int NE, int P, bool NORM, int SRC>
__global__ void __launch_bounds__(kMaxThreads, fwd_ctas(NE * (int)sizeof(T))) qk_rope_fwd_kernel(
    HeadRows q, HeadRows k, const __grid_constant__ Angles ang, Shape sh) {
  using Tr = Turn<T, NE, SRC>;
  using TT = typename Tr::TT;
  extern __shared__ __align__(16) float tab[];  // (kPositions) tables of the CTA's tokens
  pdl_wait();
  pdl_trigger();
  const int half = sh.half, total = sh.batch * sh.seq;
  const int base = blockIdx.x * sh.side * P;
  const Slot slot(q, k, sh, NE);
  const HeadRows& t = slot.isq ? q : k;
  const T* x = static_cast<const T*>(t.x) + slot.hh * t.xh + slot.d;
  T* out = static_cast<T*>(t.out) + slot.hh * t.oh + slot.d;
  Pack<T, NE> x1[P], x2[P];
  Tr tr[P];
  int64_t to[P];
  bool on[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int n = base + p * sh.side + slot.token;
    on[p] = slot.on && n < total;
    x1[p].zero();
    x2[p].zero();
    if (on[p]) {
      int64_t b, s;
      sh.tokens.split(n, b, s);
      const T* r = x + b * t.xb + s * t.xs;
      to[p] = b * t.ob + s * t.os;
      x1[p].template load<true>(r);
      x2[p].template load<true>(r + half);
      if constexpr (SRC != kPositions) {
        const int64_t at = b * ang.tb + s * ang.ts + slot.d;
        tr[p].load(static_cast<const TT*>(ang.cos) + at, static_cast<const TT*>(ang.sin) + at);
      }
    }
  }
  uint64_t w1[NE / 2], w2[NE / 2];
  if constexpr (NORM) {
    load_weights<T, NE>(t.w, slot.d, sh.w_dtype, w1);
    load_weights<T, NE>(t.w, half + slot.d, sh.w_dtype, w2);
  }
  if constexpr (SRC == kPositions) {
    fill_tables(ang, sh, base, min(base + P * sh.side, total), P * sh.side, tab);
    __syncthreads();
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    uint64_t r = 0;
    if constexpr (NORM) {
      uint64_t ss = 0;
#pragma unroll
      for (int e = 0; e < NE / 2; ++e) {
        const uint64_t u = x1[p].pair(e), v = x2[p].pair(e);
        ss = f2_fma(u, u, f2_fma(v, v, ss));
      }
      float sum = f2_sum(ss);
      for (int o = sh.lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      r = f2_same(rsqrtf(fmaf(sum, sh.inv_d, sh.eps)));
    }
    if (!on[p]) continue;
    if constexpr (SRC == kPositions) {
      const float* mine = tab + (p * sh.side + slot.token) * 2 * half + slot.d;
      tr[p].load(mine, mine + half);
    }
    const uint64_t sign = f2_same(sh.sign);
    Pack<T, NE> y1, y2;
#pragma unroll
    for (int e = 0; e < NE / 2; ++e) {
      uint64_t u = x1[p].pair(e), v = x2[p].pair(e);
      uint64_t cs = tr[p].c.pair(e), sn = tr[p].s.pair(e);
      if constexpr (NORM) {
        u = f2_mul(f2_mul(u, r), w1[e]);
        v = f2_mul(f2_mul(v, r), w2[e]);
      } else {
        sn = f2_mul(sn, sign);
      }
      y1.set(e, f2_cross(u, cs, v, sn));
      y2.set(e, f2_fma(u, sn, f2_mul(v, cs)));
    }
    y1.store(out + to[p]);
    y2.store(out + to[p] + half);
  }
}

// Backward with norms. The thread's share of dw stays in its registers. The CTA joins
// its rows of dw in the order of the heads and leaves one partial row [2][D] (q, k),
// which dw_join_kernel sums in block order. 2 x 16001 tokens of 32/8 heads of 128 in
// bf16: 193 us, 5.1 TB/s.
template <typename T, int NE, int SRC>
__global__ void __launch_bounds__(kMaxThreads, bwd_ctas(NE * (int)sizeof(T))) qk_norm_rope_bwd_kernel(
    HeadRows q, HeadRows k, const __grid_constant__ Angles ang, Shape sh, float* __restrict__ dw_part) {
  using Tr = Turn<T, NE, SRC>;
  using TT = typename Tr::TT;
  extern __shared__ __align__(16) uint8_t smem[];  // ring, tables; later dw [blockDim][2 NE]
  pdl_wait();
  const int half = sh.half;
  const Slot slot(q, k, sh, NE);
  const HeadRows& t = slot.isq ? q : k;
  const T* x = static_cast<const T*>(t.x) + slot.hh * t.xh + slot.d;
  const T* g = static_cast<const T*>(t.g) + slot.hh * t.gh + slot.d;
  T* out = static_cast<T*>(t.out) + slot.hh * t.oh + slot.d;
  uint64_t w1[NE / 2], w2[NE / 2], dw1[NE / 2], dw2[NE / 2];
  load_weights<T, NE>(t.w, slot.d, sh.w_dtype, w1);
  load_weights<T, NE>(t.w, half + slot.d, sh.w_dtype, w2);
#pragma unroll
  for (int e = 0; e < NE / 2; ++e) dw1[e] = dw2[e] = 0;
  const uint32_t pitch = 16 * blockDim.x, piece = NE * sizeof(T) / 16 * pitch;
  constexpr int S = kBwdStages;
  float* tab = reinterpret_cast<float*>(smem + S * 4 * piece);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16;
  int n0, n1;
  token_run(sh, n0, n1);
  int64_t b, s0;
  sh.tokens.split(n0, b, s0);
  Cursor in(b, s0, t.xb, t.xs, sh.seq), gin(b, s0, t.gb, t.gs, sh.seq), to(b, s0, t.ob, t.os, sh.seq),
      row(b, s0, ang.tb, ang.ts, sh.seq);
  // The tables' rows come a token ahead: loaded where they are used they cost each token an
  // L2 round trip (212 us, so 193).
  Tr ahead;
  int left = n1 - n0;
  if constexpr (SRC != kPositions) {
    ahead.load(static_cast<const TT*>(ang.cos) + row.at + slot.d, static_cast<const TT*>(ang.sin) + row.at + slot.d);
    row.next(sh.seq);
  }
  walk_tokens<S, SRC>(
      ang, sh, tab, ring, 4 * piece,
      [&](uint32_t at) {
        if (slot.on) {
          give<T, NE>(at, x + in.at, pitch);
          give<T, NE>(at + piece, x + in.at + half, pitch);
          give<T, NE>(at + 2 * piece, g + gin.at, pitch);
          give<T, NE>(at + 3 * piece, g + gin.at + half, pitch);
        }
        in.next(sh.seq);
        gin.next(sh.seq);
      },
      [&](uint32_t at, const float* table) {
        Tr tr;
        if constexpr (SRC == kPositions) {
          tr.load(table + slot.d, table + half + slot.d);
        } else {
          tr = ahead;
          if (--left > 0) {
            ahead.load(static_cast<const TT*>(ang.cos) + row.at + slot.d,
                       static_cast<const TT*>(ang.sin) + row.at + slot.d);
            row.next(sh.seq);
          }
        }
        Pack<T, NE> x1, x2, g1, g2;
        if (slot.on) {
          take(x1, at, pitch);
          take(x2, at + piece, pitch);
          take(g1, at + 2 * piece, pitch);
          take(g2, at + 3 * piece, pitch);
        } else {
          x1.zero();
          x2.zero();
          g1.zero();
          g2.zero();
        }
        uint64_t sq = 0, dt = 0;
#pragma unroll
        for (int e = 0; e < NE / 2; ++e) {
          const uint64_t u = x1.pair(e), v = x2.pair(e), cs = tr.c.pair(e), sn = tr.s.pair(e);
          const uint64_t ga = g1.pair(e), gb = g2.pair(e);
          sq = f2_fma(u, u, f2_fma(v, v, sq));
          dt = f2_fma(f2_mul(f2_fma(ga, cs, f2_mul(gb, sn)), w1[e]), u, dt);
          dt = f2_fma(f2_mul(f2_cross(gb, cs, ga, sn), w2[e]), v, dt);
        }
        float ss = f2_sum(sq), dot = f2_sum(dt);
        for (int o = sh.lanes >> 1; o > 0; o >>= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, o);
          dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        const float rstd = rsqrtf(fmaf(ss, sh.inv_d, sh.eps));
        const uint64_t r = f2_same(rstd);
        const uint64_t mean = f2_same(-dot * sh.inv_d * rstd);
        Pack<T, NE> y1, y2;
#pragma unroll
        for (int e = 0; e < NE / 2; ++e) {
          const uint64_t cs = tr.c.pair(e), sn = tr.s.pair(e);
          const uint64_t ga = g1.pair(e), gb = g2.pair(e);
          const uint64_t d1 = f2_fma(ga, cs, f2_mul(gb, sn)), d2 = f2_cross(gb, cs, ga, sn);
          const uint64_t h1 = f2_mul(x1.pair(e), r), h2 = f2_mul(x2.pair(e), r);
          dw1[e] = f2_fma(d1, h1, dw1[e]);
          dw2[e] = f2_fma(d2, h2, dw2[e]);
          y1.set(e, f2_mul(r, f2_fma(h1, mean, f2_mul(d1, w1[e]))));
          y2.set(e, f2_mul(r, f2_fma(h2, mean, f2_mul(d2, w2[e]))));
        }
        if (slot.on) {
          y1.store(out + to.at);
          y2.store(out + to.at + half);
        }
        to.next(sh.seq);
      });
  pdl_trigger();
  if (!dw_part) return;
  __syncthreads();
  float* join = reinterpret_cast<float*>(smem);
  float* mine = join + threadIdx.x * 2 * NE;
#pragma unroll
  for (int e = 0; e < NE / 2; ++e) {
    f2_unpack(dw1[e], mine[2 * e], mine[2 * e + 1]);
    f2_unpack(dw2[e], mine[NE + 2 * e], mine[NE + 2 * e + 1]);
  }
  __syncthreads();
  // this block's heads, in order
  const int dim = 2 * half;
  const int h0 = blockIdx.y * sh.group_heads;
  const int h1 = min(h0 + sh.group_heads, q.heads + k.heads);
  float* part = dw_part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * dim;
  for (int e = threadIdx.x; e < 2 * dim; e += blockDim.x) {
    const int which = e / dim, col = e - which * dim;
    const int second = col >= half ? 1 : 0, c = col - second * half;
    const int lo = which ? max(h0, q.heads) : h0, hi = which ? h1 : min(h1, q.heads);
    float sum = 0.f;
    for (int hd = lo; hd < hi; ++hd)
      sum += join[((hd - h0) * sh.lanes + c / NE) * 2 * NE + second * NE + c % NE];
    part[e] = sum;
  }
}

// dw [2][D] = sum of the partial rows in block order: eight columns a CTA, 64 threads a
// column, 64 rows apart, joined in shared memory.
constexpr int kJoinCols = 8, kJoinRows = 64;
__global__ void __launch_bounds__(kJoinCols * kJoinRows) dw_join_kernel(const float* __restrict__ part, int rows,
                                                                        int dim, void* __restrict__ dwq,
                                                                        void* __restrict__ dwk, int w_dtype) {
  __shared__ float acc[kJoinRows][kJoinCols + 1];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % kJoinCols, r0 = threadIdx.x / kJoinCols;
  const int col = blockIdx.x * kJoinCols + lane;
  float s = 0.f;
  if (col < 2 * dim) {
#pragma unroll 8
    for (int r = r0; r < rows; r += kJoinRows) s += part[(int64_t)r * 2 * dim + col];
  }
  acc[r0][lane] = s;
  __syncthreads();
  if (threadIdx.x < kJoinCols && col < 2 * dim) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r) t += acc[r][lane];
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
  const int64_t rows = (int64_t)sh.batch * sh.seq * t.heads;
  float dw1[kAnyPairs], dw2[kAnyPairs];
#pragma unroll
  for (int j = 0; j < kAnyPairs; ++j) dw1[j] = dw2[j] = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * kAnyWarps + warp; r < rows; r += (int64_t)gridDim.x * kAnyWarps) {
    const int64_t n = r / t.heads, hh = r - n * t.heads;
    int64_t b, s;
    sh.tokens.split((uint32_t)n, b, s);
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

// Threads, groups of heads and blocks of a launch, from sizes alone (the caller's
// workspace is sized by them). many: tokens side by side fill the CTA's threads.
struct Plan {
  int lanes, group_heads, groups, threads, side;
};

Plan plan_of(int heads, int half, int ne, bool many) {
  Plan p;
  p.lanes = 1;
  while (p.lanes < half / ne) p.lanes <<= 1;
  const int64_t slots = (int64_t)heads * p.lanes;
  p.groups = (int)((slots + kMaxThreads - 1) / kMaxThreads);
  p.group_heads = (heads + p.groups - 1) / p.groups;
  p.groups = (heads + p.group_heads - 1) / p.group_heads;
  p.threads = p.group_heads * p.lanes;
  p.side = many ? kMaxThreads / p.threads : 1;
  if (p.side == 1) p.threads = (p.threads + 31) / 32 * 32;
  return p;
}

// CTAs along the tokens: as many as are resident together.
int blocks_of(int64_t tokens, int ctas, const Plan& p) {
  int64_t cap = (int64_t)num_sms() * (ctas * kMaxThreads / p.threads) / p.groups;
  if (cap < 1) cap = 1;
  return (int)(tokens < cap ? tokens : cap);
}

// Elements of a half that a thread holds: 16 bytes, or 32 where 32 threads would not
// hold the half (fp32 beyond a head dim of 256); 0: no vector form.
int row_ne(int half, int es) {
  const int ne = 16 / es;
  return half % ne == 0 && half / ne <= 32 ? ne : half % (2 * ne) == 0 && half / (2 * ne) <= 32 ? 2 * ne : 0;
}

constexpr int kAnyBlocks = 592;  // of each tensor, at most

int any_blocks(int64_t tokens, int64_t heads) {
  const int64_t b = (tokens * heads + kAnyWarps - 1) / kAnyWarps;
  return (int)(b < kAnyBlocks ? (b < 1 ? 1 : b) : kAnyBlocks);
}

// 16-byte aligned rows, tables and weights.
bool rows_ok(const HeadRows& t, bool grads, int64_t es) {
  auto ok = [&](const void* p, int64_t b, int64_t h, int64_t s) {
    return aligned16(p) && (b * es) % 16 == 0 && (h * es) % 16 == 0 && (s * es) % 16 == 0;
  };
  return ok(t.x, t.xb, t.xh, t.xs) && ok(t.out, t.ob, t.oh, t.os) && (!grads || ok(t.g, t.gb, t.gh, t.gs)) &&
         (!t.w || aligned16(t.w));
}

template <typename T>
bool vectors_ok(const HeadRows& q, const HeadRows& k, const Angles& a, int dtype, int ne, bool grads) {
  if (ne == 0 || !rows_ok(q, grads, sizeof(T)) || !rows_ok(k, grads, sizeof(T))) return false;
  if (!a.cos) return true;
  const int64_t es = a.dtype == SOUP_F32 ? 4 : 2;
  return (a.dtype == dtype || a.dtype == SOUP_F32) && aligned16(a.cos) && aligned16(a.sin) && (a.tb * es) % 16 == 0 &&
         (a.ts * es) % 16 == 0;
}

// Shared memory of a launch: the rings, and with positions two groups' tables.
inline size_t ring_bytes(int stages, int pieces, int bytes, int threads, int src, int half) {
  return (size_t)stages * pieces * bytes * threads +
         (src == kPositions ? sizeof(float) * 2 * kGroup * 2 * half : 0);
}

// A launch of a kernel with more than 48 KB of shared memory, allowed once a device.
template <typename... KArgs, typename... Args>
cudaError_t launch_ring(void (*kernel)(KArgs...), bool (&ready)[64], dim3 grid, int threads, size_t smem,
                        cudaStream_t st, Args... args) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lock(cache_mutex());
    if (!ready[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
      if (e != cudaSuccess) return e;
      ready[dev] = true;
    }
  }
  return launch_pdl(kernel, grid, dim3(threads), smem, st, args...);
}

template <typename T, int NE, bool NORM, int SRC>
cudaError_t fwd_launch(const HeadRows& q, const HeadRows& k, const Angles& a, Shape sh, cudaStream_t st) {
  const int64_t tokens = (int64_t)sh.batch * sh.seq;
  // few tokens: one a CTA, so that more SMs share them
  const Plan p = plan_of(q.heads + k.heads, sh.half, NE, tokens >= 4 * num_sms());
  sh.lanes = p.lanes;
  sh.group_heads = p.group_heads;
  sh.side = p.side;
  constexpr int P = kFwdTokens;
  const size_t smem = SRC == kPositions ? sizeof(float) * P * p.side * 2 * sh.half : 0;
  const dim3 grid((unsigned)((tokens + P * p.side - 1) / (P * p.side)), p.groups);
  return launch_pdl(qk_rope_fwd_kernel<T, NE, P, NORM, SRC>, grid, dim3(p.threads, p.side), smem, st, q, k, a, sh);
}

template <typename T, int NE>
cudaError_t fwd_launch(const HeadRows& q, const HeadRows& k, const Angles& a, const Shape& sh, bool norm, int src,
                       cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {  // fp32 tables of fp32 rows are kTableF
    if (norm && src == kTableT) return fwd_launch<T, NE, true, kTableT>(q, k, a, sh, st);
    if (src == kTableT) return fwd_launch<T, NE, false, kTableT>(q, k, a, sh, st);
  }
  if (norm && src == kTableF) return fwd_launch<T, NE, true, kTableF>(q, k, a, sh, st);
  if (norm) return fwd_launch<T, NE, true, kPositions>(q, k, a, sh, st);
  if (src == kTableF) return fwd_launch<T, NE, false, kTableF>(q, k, a, sh, st);
  return fwd_launch<T, NE, false, kPositions>(q, k, a, sh, st);
}

template <typename T, int NE, int SRC>
cudaError_t bwd_launch(const HeadRows& q, const HeadRows& k, const Angles& a, Shape sh, float* part, int* rows,
                       cudaStream_t st) {
  static bool ready[64] = {false};
  const Plan p = plan_of(q.heads + k.heads, sh.half, NE, false);
  sh.lanes = p.lanes;
  sh.group_heads = p.group_heads;
  sh.side = 1;
  const dim3 grid(blocks_of((int64_t)sh.batch * sh.seq, bwd_ctas(NE * sizeof(T)), p), p.groups);
  *rows = (int)(grid.x * grid.y);
  return launch_ring(qk_norm_rope_bwd_kernel<T, NE, SRC>, ready, grid, p.threads,
                     ring_bytes(kBwdStages, 4, NE * sizeof(T), p.threads, SRC, sh.half), st, q, k, a, sh, part);
}

template <typename T, int NE>
cudaError_t bwd_launch(const HeadRows& q, const HeadRows& k, const Angles& a, const Shape& sh, int src, float* part,
                       int* rows, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (src == kTableT) return bwd_launch<T, NE, kTableT>(q, k, a, sh, part, rows, st);
  if (src == kTableF) return bwd_launch<T, NE, kTableF>(q, k, a, sh, part, rows, st);
  return bwd_launch<T, NE, kPositions>(q, k, a, sh, part, rows, st);
}

int source_of(const Angles& a, int dtype) {
  return !a.cos ? kPositions : a.dtype == dtype && dtype != SOUP_F32 ? kTableT : kTableF;
}

template <typename T>
int run_fwd(const HeadRows& q, const HeadRows& k, const Angles& a, const Shape& sh, bool norm, int dtype,
            cudaStream_t st) {
  constexpr int NE = 16 / (int)sizeof(T);
  const int ne = row_ne(sh.half, sizeof(T));
  if (vectors_ok<T>(q, k, a, dtype, ne, false)) {
    const int src = source_of(a, dtype);
    if constexpr (sizeof(T) == 4)  // (eight 16-bit elements reach every half of up to 256)
      if (ne == 2 * NE) return cuda_status(fwd_launch<T, 2 * NE>(q, k, a, sh, norm, src, st));
    return cuda_status(fwd_launch<T, NE>(q, k, a, sh, norm, src, st));
  }
  const int most = q.heads > k.heads ? q.heads : k.heads;
  const dim3 grid(any_blocks((int64_t)sh.batch * sh.seq, most), 2), block(32 * kAnyWarps);
  float* none = nullptr;
  return cuda_status(norm ? launch_pdl(qk_rope_any_kernel<T, true, false>, grid, block, 0, st, q, k, a, sh, none)
                          : launch_pdl(qk_rope_any_kernel<T, false, false>, grid, block, 0, st, q, k, a, sh, none));
}

template <typename T>
int run_bwd(const HeadRows& q, const HeadRows& k, const Angles& a, const Shape& sh, void* dwq, void* dwk, float* part,
            int dtype, cudaStream_t st) {
  constexpr int NE = 16 / (int)sizeof(T);
  const int dim = 2 * sh.half;
  const bool dw = dwq || dwk;
  if (!dw) part = nullptr;
  int rows;
  cudaError_t e;
  const int ne = row_ne(sh.half, sizeof(T));
  if (vectors_ok<T>(q, k, a, dtype, ne, true)) {
    const int src = source_of(a, dtype);
    if constexpr (sizeof(T) == 4)
      e = ne == NE ? bwd_launch<T, NE>(q, k, a, sh, src, part, &rows, st)
                   : bwd_launch<T, 2 * NE>(q, k, a, sh, src, part, &rows, st);
    else
      e = bwd_launch<T, NE>(q, k, a, sh, src, part, &rows, st);
  } else {
    const int most = q.heads > k.heads ? q.heads : k.heads;
    rows = any_blocks((int64_t)sh.batch * sh.seq, most);
    e = launch_pdl(qk_rope_any_kernel<T, true, true>, dim3(rows, 2), dim3(32 * kAnyWarps), 0, st, q, k, a, sh, part);
  }
  if (e != cudaSuccess || !dw) return cuda_status(e);
  return cuda_status(launch_pdl(dw_join_kernel, dim3((2 * dim + kJoinCols - 1) / kJoinCols),
                                dim3(kJoinCols * kJoinRows), 0, st, static_cast<const float*>(part), rows, dim, dwq,
                                dwk, sh.w_dtype));
}

bool fill_angles(Angles& a, const soup_qk_rope& d, const void* table, const void* second, const uint8_t* axes) {
  a = Angles{};
  if (!table || !second) return false;
  if (d.source == SOUP_ROPE_TABLES) {
    a.cos = table;
    a.sin = second;
    a.tb = d.table[1];
    a.ts = d.table[2];
    a.dtype = (int)d.table_dtype;
    return a.dtype == SOUP_F32 || a.dtype == SOUP_BF16 || a.dtype == SOUP_F16;
  }
  if (!axes || (d.source != SOUP_ROPE_INT32 && d.source != SOUP_ROPE_INT64)) return false;
  a.pos = table;
  a.pos64 = d.source == SOUP_ROPE_INT64;
  a.pa = d.table[0];
  a.pb = d.table[1];
  a.ps = d.table[2];
  a.inv_freq = static_cast<const float*>(second);
  for (int64_t i = 0; i < d.head_dim / 2; ++i) a.axis[i] = axes[i];
  return true;
}

int check_desc(const char* fn, const soup_qk_rope* d) {
  if (d && d->batch > 0 && d->seq > 0 && d->head_dim > 0 && d->head_dim % 2 == 0 && d->head_dim <= kMaxDim &&
      d->hq > 0 && d->hk > 0 && d->hq <= 4096 && d->hk <= 4096 && d->batch < (int64_t(1) << 31) / d->seq &&
      d->q[3] == 1 && d->q_out[3] == 1 && d->k[3] == 1 && d->k_out[3] == 1 && d->eps >= 0.0 &&
      (d->w_dtype == d->dtype || d->w_dtype == SOUP_F32))
    return SOUP_OK;
  char msg[96];
  snprintf(msg, sizeof(msg), "%s: bad sizes, strides or types", fn);
  set_last_error(msg);
  return SOUP_ERR_INVALID;
}

HeadRows rows_of(const void* x, const void* g, void* out, const int64_t* xs, const int64_t* gs, const int64_t* os,
                 const void* w, int64_t heads) {
  return HeadRows{x, g, out, xs[0], xs[1], xs[2], gs[0], gs[1], gs[2], os[0], os[1], os[2], w, (int)heads};
}

Shape shape_of(const soup_qk_rope& d) {
  return Shape{(int)d.batch, (int)d.seq, make_div(d.seq), (int)(d.head_dim / 2), 32, 0, 1, (float)d.eps,
               1.f / (float)d.head_dim, (int)d.w_dtype, d.inverse ? -1.f : 1.f};
}

}  // namespace
}  // namespace soup

using namespace soup;

extern "C" {

size_t soup_qk_norm_rope_bwd_workspace_bytes(int64_t batch, int64_t seq, int64_t hq, int64_t hk,
                                             int64_t head_dim) {
  if (batch <= 0 || seq <= 0 || hq <= 0 || hk <= 0 || head_dim <= 0) return 0;
  // the most partial rows of the forms
  const int64_t tokens = batch * seq;
  int64_t rows = any_blocks(tokens, hq > hk ? hq : hk);
  for (int es = 2; es <= 4; es += 2) {
    const int ne = row_ne((int)(head_dim / 2), es);
    if (!ne) continue;
    const Plan p = plan_of((int)(hq + hk), (int)(head_dim / 2), ne, false);
    const int64_t r = (int64_t)blocks_of(tokens, bwd_ctas(ne * es), p) * p.groups;
    if (r > rows) rows = r;
  }
  return sizeof(float) * (size_t)(rows * 2 * head_dim);
}

int soup_qk_norm_rope(const void* q, void* q_out, const void* k, void* k_out, const void* q_weight,
                      const void* k_weight, const void* table, const void* second, const uint8_t* axes,
                      const soup_qk_rope* desc, void* stream) {
  if (int rc = check_desc("soup_qk_norm_rope", desc)) return rc;
  const bool norm = q_weight || k_weight;
  Angles a;
  if (!q || !q_out || !k || !k_out || (norm && (!q_weight || !k_weight || desc->inverse)) ||
      !fill_angles(a, *desc, table, second, axes)) {
    set_last_error("soup_qk_norm_rope: bad arguments");
    return SOUP_ERR_INVALID;
  }
  const soup_qk_rope& d = *desc;
  const HeadRows tq = rows_of(q, nullptr, q_out, d.q, d.q, d.q_out, q_weight, d.hq);
  const HeadRows tk = rows_of(k, nullptr, k_out, d.k, d.k, d.k_out, k_weight, d.hk);
  const Shape sh = shape_of(d);
  const int dtype = (int)d.dtype;
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_BF16) return run_fwd<__nv_bfloat16>(tq, tk, a, sh, norm, dtype, st);
  if (dtype == SOUP_F16) return run_fwd<__half>(tq, tk, a, sh, norm, dtype, st);
  if (dtype == SOUP_F32) return run_fwd<float>(tq, tk, a, sh, norm, dtype, st);
  set_last_error("soup_qk_norm_rope: unsupported dtype");
  return SOUP_ERR_INVALID;
}

int soup_qk_norm_rope_bwd(const void* dq_out, const void* q, void* dq, const void* dk_out, const void* k, void* dk,
                          const void* q_weight, const void* k_weight, void* dq_weight, void* dk_weight,
                          const void* table, const void* second, const uint8_t* axes, const soup_qk_rope* desc,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_desc("soup_qk_norm_rope_bwd", desc)) return rc;
  const soup_qk_rope& d = *desc;
  Angles a;
  if (!dq_out || !q || !dq || !dk_out || !k || !dk || !q_weight || !k_weight || d.inverse || d.q_grad[3] != 1 ||
      d.k_grad[3] != 1 || !fill_angles(a, d, table, second, axes)) {
    set_last_error("soup_qk_norm_rope_bwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if ((dq_weight || dk_weight) &&
      (!workspace || !aligned16(workspace) ||
       workspace_bytes < soup_qk_norm_rope_bwd_workspace_bytes(d.batch, d.seq, d.hq, d.hk, d.head_dim))) {
    set_last_error("soup_qk_norm_rope_bwd: workspace missing, unaligned or too small");
    return SOUP_ERR_WORKSPACE;
  }
  const HeadRows tq = rows_of(q, dq_out, dq, d.q, d.q_grad, d.q_out, q_weight, d.hq);
  const HeadRows tk = rows_of(k, dk_out, dk, d.k, d.k_grad, d.k_out, k_weight, d.hk);
  const Shape sh = shape_of(d);
  const int dtype = (int)d.dtype;
  float* part = static_cast<float*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (dtype == SOUP_BF16) return run_bwd<__nv_bfloat16>(tq, tk, a, sh, dq_weight, dk_weight, part, dtype, st);
  if (dtype == SOUP_F16) return run_bwd<__half>(tq, tk, a, sh, dq_weight, dk_weight, part, dtype, st);
  if (dtype == SOUP_F32) return run_bwd<float>(tq, tk, a, sh, dq_weight, dk_weight, part, dtype, st);
  set_last_error("soup_qk_norm_rope_bwd: unsupported dtype");
  return SOUP_ERR_INVALID;
}

}  // extern "C"
