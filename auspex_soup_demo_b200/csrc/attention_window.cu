// Causal grouped-query attention with a sliding window and sinks for sm_100a
// (tcgen05.mma, accumulators in TMEM, operands staged by TMA), head dim 128,
// bf16 in / fp32 accumulate: query q sees key k iff k <= q and (q - k < window or
// k < sinks). No kernel in the reference; transformers masks SDPA for its
// sliding-window layers.
//
// Key tiles without a visible pair are never loaded, so the products cover about
// window + sinks keys a query.
// Forward: one CTA per (batch, query head, 128-query tile), keys in blocks of 64, one
// thread per query row.
// Backward: dK / dV per (batch, KV head, key tile): the CTA runs through the query
// heads of its group and their queries in 128-query steps and keeps dK, dV in TMEM, so
// no per-head partials reach memory; the far queries of the sink tiles, which every
// later query sees, are cut into segments with fp32 partials summed in a fixed order.
// dQ per (batch, query head, query tile). Both recompute P from the log-sum-exp; no
// atomics, results are bitwise reproducible.
// Maxima, sums, log-sum-exps, D and all accumulators are fp32. P and dS are rounded to bf16,
// as operands of products that run at the bf16 rate: at most 2^-8 of each entry, of either
// sign, so it averages out in a sum over many keys and adds about the result's own bf16
// rounding where a few keys dominate. D takes the bf16 output, the one that the caller holds.
// Hidden keys of a block that is read have weight 0 by selection, but 0 x NaN in a product is
// NaN: V must be finite there, as for any masked softmax attention.
//
// A product that overwrites TMEM columns which an earlier product reads waits for that one's
// commit: PTX keeps only products of one accumulator and shape in issue order. The waits cost
// about 1 % (forward and backward of 16001 tokens 532 us against 526, of 4 x 2048 186 in both).
// A CTA leaves only after every asynchronous arrival on its barriers has landed: the
// producer waits for its copies, the MMA warp for its commits.
// Every mbarrier wait is bounded as in attention.cu: on expiry the role records a
// code in the device error word, raises the CTA's abort flag, the producer waits
// (bounded) for its copies, the MMA warp drains its MMAs, and the CTA frees TMEM and
// returns. Launches are plain ones: for kernels of 15 us and more an early start gains nothing.
#include "attention_common.cuh"

namespace soup {
namespace attn {
namespace {

constexpr int kWarps = 16;  // compute warps
constexpr int kThreads = 64 + 32 * kWarps;

constexpr int kErrWinProducer = 0x131;
constexpr int kErrWinMma = 0x132;
constexpr int kErrWinSoftmax = 0x133;
constexpr int kErrWinSmem = 0x134;

constexpr int kBlk = 64;  // keys per block of the forward and of dQ
// The key blocks that query tile qt needs, in the order the kernels take them: the sinks'
// before the window, then from the first block that the tile's first row sees to the diagonal.
struct KeyBlocks {
  int n_sink, lo, n;  // leading sink blocks; first block of the window; blocks
  __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : lo + (i - n_sink); }
};
__device__ __forceinline__ KeyBlocks key_blocks(int qt, int S, int window, int sinks) {
  KeyBlocks k;
  const int first = qt * kTile - window + 1;
  k.lo = first > 0 ? first / kBlk : 0;
  const int ns = (sinks + kBlk - 1) / kBlk;
  k.n_sink = ns < k.lo ? ns : k.lo;
  const int nb = (S + kBlk - 1) / kBlk;
  k.n = k.n_sink + (2 * qt + 2 < nb ? 2 * qt + 2 : nb) - k.lo;
  return k;
}
// Some pair of the block of keys from k0 and the query tile from q0 is hidden.
__device__ __forceinline__ bool block_edge(int k0, int q0, int S, int window, int sinks) {
  return k0 + kBlk > S || k0 + kBlk > q0 + 1 || (q0 + kTile - 1 - k0 >= window && k0 + kBlk > sinks);
}
// Some pair of the tile of keys [k0, k0 + 128) and the queries up to q_max is
// hidden by the window.
__device__ __forceinline__ bool win_edge(int q_max, int k0, int window, int sinks) {
  return q_max - k0 >= window && k0 + kTile > sinks;
}
// Which of 32 keys from key0 on query q sees, as bits; and which of 32 queries
// from q0 on see key. A tile that some border crosses is masked by these words:
// three clamped shifts a row instead of four comparisons an element (half of the
// forward's instructions before: 101 against 85 us at 4 x 2048 tokens, 12 heads, window
// 512), and a warp whose words are all empty skips the exponentials.
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}
__device__ __forceinline__ uint32_t keys_seen(int q, int key0, int S, int window, int sinks) {
  const int end = (q + 1 < S ? q + 1 : S) - key0;
  return low_bits(end) & (~low_bits(q - window + 1 - key0) | low_bits(sinks - key0));
}
__device__ __forceinline__ uint32_t queries_seeing(int key, int q0, int S, int window, int sinks) {
  const uint32_t in = key < sinks ? 0xffffffffu : low_bits(key + window - q0);
  return low_bits(S - q0) & ~low_bits(key - q0) & in;
}
// Warp-uniform: 0 no lane's word has a bit of `all`, 1 every one, 2 otherwise.
__device__ __forceinline__ int mask_kind(uint32_t m, uint32_t all) {
  if (__all_sync(0xffffffffu, (m & all) == 0u)) return 0;
  return __all_sync(0xffffffffu, (m & all) == all) ? 1 : 2;
}

// 2^x of a pair on the FMA pipe, for x <= 127: x = n + f with n whole and |f| <= 1/2, a cubic
// for 2^f (relative error 7.5e-5, a fiftieth of P's rounding to bf16) and n into the exponent.
// NaN stays NaN; below -126 the result is 2^-126.
__device__ __forceinline__ void exp2_fma(float& x0, float& x1) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x0));  // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x1));
  constexpr float kMagic = 12582912.f + 127.f;  // 1.5 * 2^23: the sum's low bits are n + 127
  const uint64_t x = f2_pack(x0, x1);
  const uint64_t t = f2_add(x, f2_pack(kMagic, kMagic));
  const uint64_t f = f2_fma(f2_add(t, f2_pack(-kMagic, -kMagic)), f2_pack(-1.f, -1.f), x);
  uint64_t y = f2_fma(f, f2_pack(0.0551716648f, 0.0551716648f), f2_pack(0.242611125f, 0.242611125f));
  y = f2_fma(f, y, f2_pack(0.693260968f, 0.693260968f));
  y = f2_fma(f, y, f2_pack(0.999928057f, 0.999928057f));
  float t0, t1;
  f2_unpack(t, t0, t1);
  const float s0 = __uint_as_float(__float_as_uint(t0) << 23);
  const float s1 = __uint_as_float(__float_as_uint(t1) << 23);
  f2_unpack(f2_mul(y, f2_pack(s0, s1)), x0, x1);
}

// ---- the MMA warp ----
// The whole warp walks the schedule converged, so that waits are one instruction and
// descriptors and addresses are uniform; each group of products and its commits runs in the
// branch of an elected thread. From a lane == 0 branch around the whole schedule each product
// took about 110 cycles, more than a 128 x 64 x 16 product does (75), and the issuing thread
// bounded all three kernels. Do not issue them from the converged warp under a predicate
// that only one thread has set instead of a branch: that is 2 % faster, but commits then
// go astray now and then (a wait that expires, or an illegal address).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(v));
  return v;
}
// Bounded wait of a converged warp; the result is warp-uniform.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          int* err, int code, uint64_t wait_ns) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = bounded_wait(bar, parity, abort_flag, err, code, wait_ns);
  return warp_ok(ok);
}
// An operand descriptor (128-byte swizzle) of which steps only change the address.
struct Desc {
  uint32_t lo, hi;
  __device__ __forceinline__ Desc(uint64_t d)
      : lo(static_cast<uint32_t>(d)), hi(static_cast<uint32_t>(d >> 32)) {}
  __device__ __forceinline__ uint32_t at(uint32_t bytes) const { return lo + (bytes >> 4); }
};
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                       uint32_t b_hi, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
      : "memory");
}
// Offsets in bytes of k-step kk (16 wide): of a K-major 128-column tile whose two
// 64-column boxes are `box` bytes apart, and of an MN-major tile (16 rows of 128 B).
__device__ __forceinline__ uint32_t kmajor_step(int kk, uint32_t box) {
  return (kk >> 2) * box + (kk & 3) * 32;
}
__device__ __forceinline__ uint32_t mnmajor_step(int kk) { return kk * 2048; }

__device__ __forceinline__ float max32(const float (&v)[32]) {
  float mx[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) mx[u] = v[u];
#pragma unroll
  for (int i = 4; i < 32; i += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) mx[u] = fmaxf(mx[u], v[i + u]);
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// This thread's O row (128 fp32 TMEM columns) times alpha (rare: kept out of line so
// that its registers stay out of the softmax loop). Warp-collective.
__device__ __noinline__ void rescale_o_row(uint32_t o_t, float alpha) {
  const uint64_t al2 = f2_pack(alpha, alpha);
#pragma unroll 1
  for (int c = 0; c < kHeadDim / 16; ++c) {
    uint32_t o[16];
    tmem_ld16u(o_t + c * 16, o);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float o0, o1;
      f2_unpack(f2_mul(f2_pack(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), al2), o0, o1);
      o[i] = __float_as_uint(o0);
      o[i + 1] = __float_as_uint(o1);
    }
    tmem_st16u(o_t + c * 16, o);
    tmem_st_wait();
  }
}

struct FwdArgs {
  int B, H, Hk, S;
  float scale_log2;  // softmax scale * log2(e)
  int window, sinks;
  bf16* out;   // [B, S, H, D] contiguous
  float* lse;  // [B, H, S_pad]
  uint64_t wait_ns;
};

// ------------------------------------------------------------- forward ----
// One CTA per (batch, query head, 128-query tile), keys in blocks of 64, two CTAs an SM.
// TMEM (256 columns): two S buffers of 64 columns, O at 128; P of a block overwrites the
// first 32 columns of its own S buffer as bf16 pairs and is the A operand of O += P V
// read from TMEM. With S double buffered the products run a block ahead: the softmax
// finds its next S ready and its chain holds no product; the other CTA's products fill the
// time in which this one starts and ends. Shared memory: Q (32 KB), one
// ring of 5 x 16 KB through which K and V blocks pass (K0 V0 K1 V1 ...), barriers.
// At 1 x 16001 tokens, 12 heads over 2, window 1000, 16 sinks: 134 us, 722 TFLOP/s of the
// visible pairs' products; 168 us with one CTA an SM for a pair of query tiles that shares
// the K and V blocks. A block takes a CTA 2080 cycles, of which the products of both CTAs
// on the SM are 1800 (N = 64 ones take as long as N = 128 ones). Two threads a row (154 us)
// or maxima only where a block's sum grows (137 us) are no faster.
constexpr int kFwdWarps = 4;  // softmax warps, one row per thread
constexpr int kFwdThreads = 64 + 32 * kFwdWarps;
constexpr int kRing = 5;
struct WinFwdSmem {
  static constexpr int kQ = 0;
  static constexpr int kKV = kQ + kTileBytes;
  static constexpr int kBar = kKV + kRing * kStepTile;
  // q_full, full[5], empty[5], then per S buffer: s_full, p_full, pv_done; drain
  static constexpr int kNumBars = 1 + 2 * kRing + 6 + 1;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kUsed = kMisc + 16;
  static constexpr int kBytes = 115712;  // half of an SM's 228 KB less 1 KB a CTA
};
static_assert(WinFwdSmem::kUsed + 512 <= WinFwdSmem::kBytes, "window attention forward shared memory");

__global__ void __launch_bounds__(kFwdThreads, 2)
    win_fwd_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_k,
                   const __grid_constant__ CUtensorMap tma_v, FwdArgs a, int* err) {
  using L = WinFwdSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  if ((uint32_t)(smem - smem_raw) + L::kUsed > dynamic_smem_bytes()) {  // grid-uniform
    if (threadIdx.x == 0) atomicCAS(err, 0, kErrWinSmem);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::kBar;
  const uint32_t q_full = bar0;
  auto full = [&](int s) { return bar0 + 8u * (1 + s); };
  auto empty = [&](int s) { return bar0 + 8u * (1 + kRing + s); };
  constexpr int kB = 1 + 2 * kRing;
  // of block i: its S buffer is i & 1, the phase (i >> 1) & 1
  auto s_full = [&](int i) { return bar0 + 8u * (kB + (i & 1)); };
  auto p_full = [&](int i) { return bar0 + 8u * (kB + 2 + (i & 1)); };
  auto pv_done = [&](int i) { return bar0 + 8u * (kB + 4 + (i & 1)); };
  const uint32_t drain_bar = bar0 + 8u * (kB + 6);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nq = (a.S + kTile - 1) / kTile;
  const int bh = blockIdx.x % (a.B * a.H);
  const int qt = nq - 1 - blockIdx.x / (a.B * a.H);  // late tiles first: early ones are short
  const int b = bh / a.H, h = bh % a.H;
  const int hk = h / (a.H / a.Hk);
  const KeyBlocks kb = key_blocks(qt, a.S, a.window, a.sinks);
  const int n = kb.n;
  const uint64_t wait_ns = a.wait_ns;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kNumBars; ++i) {
      const uint32_t bar = bar0 + 8u * i;
      mbar_init(bar, bar == p_full(0) || bar == p_full(1) ? kFwdWarps : 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc::tma_prefetch_desc(&tma_q);
    tc::tma_prefetch_desc(&tma_k);
    tc::tma_prefetch_desc(&tma_v);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_holder)),
                 "r"(256)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer ----
      mbar_arrive_expect_tx(q_full, kTileBytes);
      tma_load_4d(sbase + L::kQ, &tma_q, q_full, 0, qt * kTile, h, b);
      tma_load_4d(sbase + L::kQ + kBox, &tma_q, q_full, 64, qt * kTile, h, b);
      int issued = 0;
      for (int i = 0; i < 2 * n; ++i) {  // K of block j is load 2 j, V load 2 j + 1
        const int st = i % kRing;
        if (!bounded_wait(empty(st), ((i / kRing) & 1) ^ 1, abort_flag, err, kErrWinProducer, wait_ns))
          break;
        const int key0 = kb.at(i >> 1) * kBlk;
        const CUtensorMap* map = (i & 1) ? &tma_v : &tma_k;
        const uint32_t d = sbase + L::kKV + st * kStepTile;
        mbar_arrive_expect_tx(full(st), kStepTile);
        tma_load_4d(d, map, full(st), 0, key0, hk, b);
        tma_load_4d(d + kStepBox, map, full(st), 64, key0, hk, b);
        ++issued;
      }
      // let every issued copy land before the CTA may leave (bounded)
      uint64_t t0 = tc::globaltimer();
      while (!mbar_try_wait(q_full, 0) && tc::globaltimer() - t0 < wait_ns) {
      }
      for (int i = issued > kRing ? issued - kRing : 0; i < issued; ++i) {
        t0 = tc::globaltimer();
        while (!mbar_try_wait(full(i % kRing), (i / kRing) & 1) && tc::globaltimer() - t0 < wait_ns) {
        }
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------- MMA issuer ----
    // S of blocks 0 and 1, then per block i: P V (i) and, once it is done, S(i + 2) into the
    // buffer that it has read P from.
    auto wait = [&](uint32_t bar, int parity) {
      return warp_wait(bar, parity, abort_flag, err, kErrWinMma, wait_ns);
    };
    bool ok = wait(q_full, 0);
    bool issued = false;
    const Desc q_desc(smem_desc_sw128(sbase + L::kQ, 16, 1024));
    const Desc k_desc(smem_desc_sw128(sbase + L::kKV, 16, 1024));
    const Desc v_desc(smem_desc_sw128(sbase + L::kKV, kStepBox, 1024));
    auto issue_s = [&](int i) -> bool {
      const int st = (2 * i) % kRing;
      if (!wait(full(st), (2 * i / kRing) & 1)) return false;
      tc_fence_after();
      const uint32_t d = tmem + (i & 1) * 64;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kHeadDim / 16; ++kk)
          mma_ss(d, q_desc.at(kmajor_step(kk, kBox)), q_desc.hi,
                 k_desc.at(st * kStepTile + kmajor_step(kk, kStepBox)), k_desc.hi, kIdescKK64,
                 kk > 0 ? 1u : 0u);
        tc_commit(s_full(i));
        tc_commit(empty(st));
      }
      __syncwarp();
      issued = true;
      return true;
    };
    auto issue_pv = [&](int i) -> bool {
      const int st = (2 * i + 1) % kRing;
      if (!wait(full(st), ((2 * i + 1) / kRing) & 1)) return false;
      if (!wait(p_full(i), (i >> 1) & 1)) return false;
      tc_fence_after();
      const uint32_t p = tmem + (i & 1) * 64;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kBlk / 16; ++kk)
          mma_ts(tmem + 128, p + kk * 8, v_desc.at(st * kStepTile + mnmajor_step(kk)), v_desc.hi,
                 kIdescKM, (i > 0 || kk > 0) ? 1u : 0u);
        tc_commit(pv_done(i));
        tc_commit(empty(st));
      }
      __syncwarp();
      return true;
    };
    if (ok) ok = issue_s(0);
    if (ok && n > 1) ok = issue_s(1);
    for (int i = 0; i < n && ok; ++i) {
      ok = issue_pv(i);
      if (ok && i + 2 < n) ok = wait(pv_done(i), (i >> 1) & 1) && issue_s(i + 2);
    }
    // the ring's last arrivals (nothing else waits for them)
    for (int i = 2 * n > kRing ? 2 * n - kRing : 0; i < 2 * n && ok; ++i)
      ok = wait(empty(i % kRing), (i / kRing) & 1);
    if (!ok && issued) {
      if (elect_one()) tc_commit(drain_bar);
      __syncwarp();
      uint64_t t0 = tc::globaltimer();
      while (!mbar_try_wait(drain_bar, 0) && tc::globaltimer() - t0 < wait_ns) {
      }
    }
  } else {
    // ------------------------------------------------------- softmax ----
    const int quarter = warp & 3;                    // TMEM lanes this warp may access
    const int q = qt * kTile + quarter * 32 + lane;  // query row of this thread
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_base = tmem + lane_off;
    const uint32_t o_t = tmem + 128 + lane_off;
    const uint64_t sl2 = f2_pack(a.scale_log2, a.scale_log2);
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      if (!(ok = warp_wait(s_full(i), (i >> 1) & 1, abort_flag, err, kErrWinSoftmax, wait_ns))) break;
      tc_fence_after();
      const uint32_t s_t = s_base + (i & 1) * 64;
      float s0[32], s1[32];
      tmem_ld32_async(s_t, s0);
      tmem_ld32_async(s_t + 32, s1);
      const int k0 = kb.at(i) * kBlk;
      int kind0 = 1, kind1 = 1;
      uint32_t mk0 = 0xffffffffu, mk1 = 0xffffffffu;
      if (block_edge(k0, qt * kTile, a.S, a.window, a.sinks)) {
        mk0 = keys_seen(q, k0, a.S, a.window, a.sinks);
        mk1 = keys_seen(q, k0 + 32, a.S, a.window, a.sinks);
        kind0 = mask_kind(mk0, 0xffffffffu);
        kind1 = mask_kind(mk1, 0xffffffffu);
      }
      tmem_ld_wait();
      if (kind0 == 2) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(mk0 & (1u << e))) s0[e] = -INFINITY;
      }
      if (kind1 == 2) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(mk1 & (1u << e))) s1[e] = -INFINITY;
      }
      const float mt = fmaxf(kind0 ? max32(s0) : -INFINITY, kind1 ? max32(s1) : -INFINITY) *
                       a.scale_log2;
      bool rescale = false;
      float alpha = 1.f;
      if (mt > m_used + 8.f) {  // also when m_used is still -inf
        alpha = fast_exp2(m_used - mt);
        m_used = mt;
        rescale = true;
      }
      if (i > 0 && __any_sync(0xffffffffu, rescale)) {
        // O is stable once P V (i - 1) is done (S(i) came before it; P V (i - 2) before S(i))
        if (!(ok = warp_wait(pv_done(i - 1), ((i - 1) >> 1) & 1, abort_flag, err, kErrWinSoftmax, wait_ns))) break;
        tc_fence_after();
        rescale_o_row(o_t, alpha);
      }
      // a row whose keys are all hidden so far: exp2(-inf - 0) = 0 instead of NaN
      const float nm = m_used == -INFINITY ? 0.f : -m_used;
      const uint64_t nm2 = f2_pack(nm, nm);
      uint64_t sm2[4] = {0, 0, 0, 0};
      uint32_t pw[32];
      auto exps = [&](const float (&v)[32], int kind, int w0) {
        if (kind == 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) pw[w0 + e] = 0u;
          return;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(v[e], v[e + 1]), sl2, nm2), x0, x1);
          x0 = fast_exp2(x0);
          x1 = fast_exp2(x1);
          sm2[(e >> 1) & 3] = f2_add(sm2[(e >> 1) & 3], f2_pack(x0, x1));
          pw[w0 + (e >> 1)] = pack_bf16(x0, x1);
        }
      };
      exps(s0, kind0, 0);
      exps(s1, kind1, 16);
      tmem_st32u(s_t, pw);
      float t0, t1, t2, t3;
      f2_unpack(f2_add(sm2[0], sm2[1]), t0, t1);
      f2_unpack(f2_add(sm2[2], sm2[3]), t2, t3);
      const float sum = (t0 + t1) + (t2 + t3);
      l = rescale ? l * alpha + sum : l + sum;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(i));
    }
    if (ok) {
      bool w = true;
      if (lane == 0)
        w = bounded_wait(pv_done(n - 1), ((n - 1) >> 1) & 1, abort_flag, err, kErrWinSoftmax, wait_ns);
      ok = warp_ok(w);
    }
    if (ok) {
      tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : 0.f;
      bf16* orow = a.out + ((int64_t)b * a.S + q) * (int64_t)(a.H * kHeadDim) + h * kHeadDim;
#pragma unroll
      for (int c = 0; c < kHeadDim / 32; ++c) {
        float o[32];
        tmem_ld32(o_t + c * 32, o);
        if (q < a.S) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint4*>(orow + c * 32 + 8 * g) =
                make_uint4(pack_bf16(o[8 * g] * inv, o[8 * g + 1] * inv),
                           pack_bf16(o[8 * g + 2] * inv, o[8 * g + 3] * inv),
                           pack_bf16(o[8 * g + 4] * inv, o[8 * g + 5] * inv),
                           pack_bf16(o[8 * g + 6] * inv, o[8 * g + 7] * inv));
        }
      }
      if (q < a.S)
        a.lse[((int64_t)b * a.H + h) * ((int64_t)nq * kTile) + q] = (m_used + __log2f(l)) * kLn2;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256)
                 : "memory");
  }
}

// ------------------------------------------------------------ backward ----
struct BwdArgs {
  int B, H, Hk, S;
  float scale;       // softmax scale (applied to dK, dQ in fp32)
  float scale_log2;  // scale * log2(e)
  int window, sinks;
  float* Dv;         // [B, H, S_pad] dO . O: written by the dQ kernel, read by dK / dV's
  float* nl2;        // [B, H, S_pad] -lse * log2(e), the same
  const bf16* out;   // [B, S, H, D]
  const bf16* dout;
  const float* lse;  // [B, H, S_pad]
  bf16* dq;          // [B, S, H, D]
  bf16* dk;          // [B, S, Hk, D]
  bf16* dv;
  float* part;       // fp32 partials, one slot of dK, dV [2][128][D] per entry
  int groups;        // parts that a KV head's query heads are split into
  int heads_per;     // query heads per part
  int n_sink;        // sink tiles
  int segs, seg_steps;  // most segments of a sink tile's 128-query steps, and their length
  int sink_slots;       // segments that the sink tiles of one KV head have, together
  uint64_t wait_ns;
};

// One unit of dK / dV work: a key tile, a range of 128-query steps, query heads
// [h0, h0 + nh), and the slot its sums go to (-1: straight to dk, dv).
struct DkvUnit {
  int b, hk, kt, h0, nh, step0, n, slot;
};
__host__ __device__ __forceinline__ int dkv_sink_units(const BwdArgs& a) {
  return a.B * a.Hk * a.n_sink * a.groups * a.segs;
}
// Sink tile kt has ceil((nq - kt) / seg_steps) segments; those of the tiles before it:
__host__ __device__ __forceinline__ int64_t segments_of_last(int64_t tiles, int64_t seg_steps) {
  const int64_t n = tiles / seg_steps, r = tiles % seg_steps;  // sum of ceil(m / seg_steps), m = 1..tiles
  return seg_steps * (n * (n + 1) / 2) + r * (n + 1);
}
__host__ __device__ __forceinline__ int segments_before(int kt, int nq, int seg_steps) {
  return static_cast<int>(segments_of_last(nq, seg_steps) - segments_of_last(nq - kt, seg_steps));
}
__host__ __device__ __forceinline__ int segments_of(int kt, int nq, int seg_steps) {
  return (nq - kt + seg_steps - 1) / seg_steps;
}
__device__ __forceinline__ DkvUnit dkv_unit(const BwdArgs& a, int i) {
  DkvUnit u;
  const int nq = (a.S + kTile - 1) / kTile;
  const int n_sink_units = dkv_sink_units(a);
  const int rep = a.H / a.Hk;
  int g, bhk;
  if (i < n_sink_units) {
    const int seg = i % a.segs;
    i /= a.segs;
    g = i % a.groups;
    i /= a.groups;
    u.kt = i % a.n_sink;
    bhk = i / a.n_sink;
    u.slot = (bhk * a.sink_slots + segments_before(u.kt, nq, a.seg_steps)) * a.groups +
             g * segments_of(u.kt, nq, a.seg_steps) + seg;
    u.step0 = u.kt + seg * a.seg_steps;
    const int end = u.step0 + a.seg_steps < nq ? u.step0 + a.seg_steps : nq;
    u.n = end > u.step0 ? end - u.step0 : 0;
  } else {
    i -= n_sink_units;
    u.slot = a.groups > 1 ? a.B * a.Hk * a.sink_slots * a.groups + i : -1;
    g = i % a.groups;
    i /= a.groups;
    bhk = i % (a.B * a.Hk);
    u.kt = a.n_sink + i / (a.B * a.Hk);
    u.step0 = u.kt;
    // the last query that sees a key of this tile
    const int last = (u.kt * kTile + kTile - 1 + a.window - 1) / kTile;
    u.n = (last < nq - 1 ? last : nq - 1) - u.step0 + 1;
  }
  u.b = bhk / a.Hk;
  u.hk = bhk % a.Hk;
  u.h0 = u.hk * rep + g * a.heads_per;
  const int h1 = (u.hk + 1) * rep;
  u.nh = u.h0 + a.heads_per < h1 ? a.heads_per : h1 - u.h0;
  if (u.nh < 0) u.nh = 0;
  return u;
}

// dK / dV of one unit, keys on the rows: per step of 128 queries S^T = K Q^T, dP^T = V dO^T,
// dV += P^T dO, dK += dS^T Q. TMEM: S^T at column 0, dP^T 128, dV 256, dK 384. P^T and
// dS^T overwrite the columns that they were computed from (bf16 pairs, the 32 queries of
// a compute warp in the first 16 of its own 32 columns, so no warp writes what another
// still reads) and are A operands from TMEM. The issue order
//   dV(i), S^T(i + 1), dK(i), dP^T(i + 1), dV(i + 1), ...
// leaves the softmax the time of two products between S^T and dV, and dS the same between
// dP^T and dK, so the tensor pipe need not wait; products of N = 128 run at twice the rate
// of N = 64 ones (75 cycles of issue either way). Shared memory: K, V (32 KB each, loaded
// once for all query heads), two stages of (Q, dO) tiles with their nl2 / D vectors. A
// compute thread owns 32 queries of one key row.
// Bound by the loop dV(i), S^T(i + 1), P(i + 1): about 3400 cycles a step, of which the two
// products take 1200, the TMEM read up to 800 (beside products), the exponentials 800-1000
// (at the special-function rate 1024 for 128 x 128) and handoffs the rest; dP and dS run
// beside it. A quarter of the exponentials goes to the FMA pipe: forward and backward of
// 1 x 16001 tokens, 12 heads over 2, window 1000, 16 sinks take 526 us against 540 with none
// and 532 with half (532 with the waits between products, which came later). dQ
// takes all of P from the special-function unit: up to 7.5e-5 from these, where P's rounding to
// bf16 is 50 times that. Eight compute warps, P through shared memory and two groups of warps on
// 64-query steps (S^T double buffered, but products of N = 64) measured no faster.
constexpr int kDkvStages = 2;
struct WinDkvSmem {
  static constexpr int kK = 0;
  static constexpr int kV = kK + kTileBytes;
  static constexpr int kQD = kV + kTileBytes;  // stage s: Q at +0, dO at +kTileBytes
  static constexpr int kVec = kQD + kDkvStages * 2 * kTileBytes;  // stage s: nl2, D (2 x 512 B)
  static constexpr int kBar = kVec + kDkvStages * 2 * kTile * 4;
  // kv_full, full[2], empty[2], s_full, p_full, dp_full, ds_full, acc_done, dv_done, drain
  static constexpr int kNumBars = 1 + 2 * kDkvStages + 7;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kUsed = kMisc + 16;
  static constexpr int kBytes = kUsed + 1024 <= 232448 ? kUsed + 1024 : 232448;
};
static_assert(WinDkvSmem::kUsed + 128 <= 232448, "window attention dK/dV shared memory");

__global__ void __launch_bounds__(kThreads, 1)
    win_dkdv_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_k,
                    const __grid_constant__ CUtensorMap tma_v,
                    const __grid_constant__ CUtensorMap tma_do, BwdArgs a, int* err) {
  using L = WinDkvSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  if ((uint32_t)(smem - smem_raw) + L::kUsed > dynamic_smem_bytes()) {  // grid-uniform
    if (threadIdx.x == 0) atomicCAS(err, 0, kErrWinSmem);
    return;
  }
  const DkvUnit u = dkv_unit(a, blockIdx.x);
  const int total = u.nh * u.n;  // steps of all this unit's query heads
  if (total == 0) return;        // an empty segment: later tiles have fewer (it has no slot)
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::kBar;
  const uint32_t kv_full = bar0;
  auto full = [&](int st) { return bar0 + 8u * (1 + st); };
  auto empty = [&](int st) { return bar0 + 8u * (1 + kDkvStages + st); };
  constexpr int kB = 1 + 2 * kDkvStages;
  const uint32_t s_full = bar0 + 8u * kB, p_full = bar0 + 8u * (kB + 1);
  const uint32_t dp_full = bar0 + 8u * (kB + 2), ds_full = bar0 + 8u * (kB + 3);
  const uint32_t acc_done = bar0 + 8u * (kB + 4), dv_done = bar0 + 8u * (kB + 5);
  const uint32_t drain_bar = bar0 + 8u * (kB + 6);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k0 = u.kt * kTile;
  const int64_t s_pad = ((int64_t)a.S + kTile - 1) / kTile * kTile;
  const uint64_t wait_ns = a.wait_ns;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kNumBars; ++i) {
      const uint32_t bar = bar0 + 8u * i;
      mbar_init(bar, bar == p_full || bar == ds_full ? kWarps : 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc::tma_prefetch_desc(&tma_q);
    tc::tma_prefetch_desc(&tma_k);
    tc::tma_prefetch_desc(&tma_v);
    tc::tma_prefetch_desc(&tma_do);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_holder)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer ----
      mbar_arrive_expect_tx(kv_full, 2 * kTileBytes);
      tma_load_4d(sbase + L::kK, &tma_k, kv_full, 0, k0, u.hk, u.b);
      tma_load_4d(sbase + L::kK + kBox, &tma_k, kv_full, 64, k0, u.hk, u.b);
      tma_load_4d(sbase + L::kV, &tma_v, kv_full, 0, k0, u.hk, u.b);
      tma_load_4d(sbase + L::kV + kBox, &tma_v, kv_full, 64, k0, u.hk, u.b);
      int issued = 0, h = u.h0, step = u.step0;
      for (int i = 0; i < total; ++i) {
        const int st = i % kDkvStages;
        if (!bounded_wait(empty(st), ((i / kDkvStages) & 1) ^ 1, abort_flag, err, kErrWinProducer,
                          wait_ns))
          break;
        const int q0 = step * kTile;
        const uint32_t qd = sbase + L::kQD + st * 2 * kTileBytes;
        const int64_t vrow = ((int64_t)u.b * a.H + h) * s_pad + q0;
        const uint32_t vd = sbase + L::kVec + st * 2 * kTile * 4;
        mbar_arrive_expect_tx(full(st), 2 * kTileBytes + 2 * kTile * 4);
        tma_load_4d(qd, &tma_q, full(st), 0, q0, h, u.b);
        tma_load_4d(qd + kBox, &tma_q, full(st), 64, q0, h, u.b);
        tma_load_4d(qd + kTileBytes, &tma_do, full(st), 0, q0, h, u.b);
        tma_load_4d(qd + kTileBytes + kBox, &tma_do, full(st), 64, q0, h, u.b);
        bulk_load(vd, a.nl2 + vrow, kTile * 4, full(st));
        bulk_load(vd + kTile * 4, a.Dv + vrow, kTile * 4, full(st));
        ++issued;
        if (++step == u.step0 + u.n) {
          step = u.step0;
          ++h;
        }
      }
      uint64_t t0 = tc::globaltimer();
      while (!mbar_try_wait(kv_full, 0) && tc::globaltimer() - t0 < wait_ns) {
      }
      for (int i = issued > kDkvStages ? issued - kDkvStages : 0; i < issued; ++i) {
        t0 = tc::globaltimer();
        while (!mbar_try_wait(full(i % kDkvStages), (i / kDkvStages) & 1) &&
               tc::globaltimer() - t0 < wait_ns) {
        }
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------- MMA issuer ----
    auto wait = [&](uint32_t bar, int parity) {
      return warp_wait(bar, parity, abort_flag, err, kErrWinMma, wait_ns);
    };
    bool ok = wait(kv_full, 0);
    bool issued = false;
    const Desc k_desc(smem_desc_sw128(sbase + L::kK, 16, 1024));
    const Desc v_desc(smem_desc_sw128(sbase + L::kV, 16, 1024));
    const Desc qd_desc(smem_desc_sw128(sbase + L::kQD, 16, 1024));   // as K-major operands
    const Desc qd_mn(smem_desc_sw128(sbase + L::kQD, kBox, 1024));   // as MN-major operands
    // S^T (dP = 0) or dP^T (1) of step i
    auto issue_s = [&](int dP, int i) -> bool {
      const int st = i % kDkvStages;
      if (!wait(full(st), (i / kDkvStages) & 1)) return false;
      tc_fence_after();
      const uint32_t b_off = st * 2 * kTileBytes + dP * kTileBytes;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kHeadDim / 16; ++kk)
          mma_ss(tmem + dP * 128, (dP ? v_desc : k_desc).at(kmajor_step(kk, kBox)), k_desc.hi,
                 qd_desc.at(b_off + kmajor_step(kk, kBox)), qd_desc.hi, kIdescKK, kk > 0 ? 1u : 0u);
        tc_commit(dP ? dp_full : s_full);
      }
      __syncwarp();
      issued = true;
      return true;
    };
    // dV += P^T dO (dK = 0) or dK += dS^T Q (1) of step i
    auto issue_acc = [&](int dK, int i) -> bool {
      const int st = i % kDkvStages;
      if (!wait(dK ? ds_full : p_full, i & 1)) return false;
      tc_fence_after();
      const uint32_t b_off = st * 2 * kTileBytes + (dK ? 0 : kTileBytes);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kTile / 16; ++kk)
          mma_ts(tmem + 256 + dK * 128, tmem + dK * 128 + (kk >> 1) * 32 + (kk & 1) * 8,
                 qd_mn.at(b_off + mnmajor_step(kk)), qd_mn.hi, kIdescKM, (i > 0 || kk > 0) ? 1u : 0u);
      }
      __syncwarp();
      return true;
    };
    if (ok) ok = issue_s(0, 0);
    if (ok) ok = issue_s(1, 0);
    // S^T and dP^T of a step overwrite the P^T and dS^T that dV and dK of the step before
    // read: each follows its commit
    for (int i = 0; i < total && ok; ++i) {
      const bool more = i + 1 < total;
      ok = issue_acc(0, i);
      if (ok && more) {
        if (elect_one()) tc_commit(dv_done);
        __syncwarp();
        ok = wait(dv_done, i & 1) && issue_s(0, i + 1);
      }
      if (ok) ok = issue_acc(1, i);
      if (ok && elect_one()) tc_commit(empty(i % kDkvStages));
      __syncwarp();
      if (ok && more) ok = wait(empty(i % kDkvStages), (i / kDkvStages) & 1) && issue_s(1, i + 1);
    }
    if (ok && elect_one()) tc_commit(acc_done);
    __syncwarp();
    for (int i = total > kDkvStages ? total - kDkvStages : 0; i < total && ok; ++i)
      ok = wait(empty(i % kDkvStages), (i / kDkvStages) & 1);
    if (!ok && issued) {
      if (elect_one()) tc_commit(drain_bar);
      __syncwarp();
      uint64_t t0 = tc::globaltimer();
      while (!mbar_try_wait(drain_bar, 0) && tc::globaltimer() - t0 < wait_ns) {
      }
    }
  } else {
    // ------------------------------------------------------- compute ----
    const int quarter = warp & 3;
    const int part = (warp - 2) >> 2;   // queries [32 part, 32 part + 32) of each step
    const int cb = part * 32;
    const int r = quarter * 32 + lane;  // key row of this thread
    const int key = k0 + r;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_t = tmem + cb + lane_off, dp_t = s_t + 128;
    const uint64_t sl2 = f2_pack(a.scale_log2, a.scale_log2);
    bool ok = true;
    int step = u.step0;
    for (int i = 0; i < total; ++i) {
      const int st = i % kDkvStages;
      const int qs = step * kTile;
      if (++step == u.step0 + u.n) step = u.step0;
      const float* vnl = reinterpret_cast<const float*>(smem + L::kVec + st * 2 * kTile * 4) + cb;
      const float* vD = vnl + kTile;
      const bool edge = qs + kTile > a.S || qs < k0 + kTile ||
                        win_edge(qs + kTile - 1, k0, a.window, a.sinks);
      uint32_t mk = 0xffffffffu;
      int kind = 1;
      if (edge) {
        mk = queries_seeing(key, qs + cb, a.S, a.window, a.sinks);
        kind = mask_kind(mk, 0xffffffffu);
      }
      if (!(ok = warp_wait(s_full, i & 1, abort_flag, err, kErrWinSoftmax, wait_ns))) break;
      tc_fence_after();
      float p[32];
      uint32_t words[16];
      if (kind == 0) {
#pragma unroll
        for (int e = 0; e < 32; ++e) p[e] = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) words[e] = 0u;
      } else {
        tmem_ld32_async(s_t, p);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 nl = *reinterpret_cast<const float4*>(vnl + e);
          f2_unpack(f2_fma(f2_pack(p[e], p[e + 1]), sl2, f2_pack(nl.x, nl.y)), p[e], p[e + 1]);
          f2_unpack(f2_fma(f2_pack(p[e + 2], p[e + 3]), sl2, f2_pack(nl.z, nl.w)), p[e + 2], p[e + 3]);
          if (e % 8 == 0) {
            exp2_fma(p[e], p[e + 1]);
          } else {
            p[e] = fast_exp2(p[e]);
            p[e + 1] = fast_exp2(p[e + 1]);
          }
          p[e + 2] = fast_exp2(p[e + 2]);
          p[e + 3] = fast_exp2(p[e + 3]);
        }
        if (kind == 2) {  // hidden and padding rows may hold anything: select, do not scale
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(mk & (1u << e))) p[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) words[e] = pack_bf16(p[2 * e], p[2 * e + 1]);
      }
      tmem_st16u(s_t, words);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      if (!(ok = warp_wait(dp_full, i & 1, abort_flag, err, kErrWinSoftmax, wait_ns))) break;
      tc_fence_after();
      if (kind != 0) {
        float dp[32];
        tmem_ld32_async(dp_t, dp);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 dd = *reinterpret_cast<const float4*>(vD + e);
          float d[4];
          f2_unpack(f2_mul(f2_pack(p[e], p[e + 1]),
                           f2_add(f2_pack(dp[e], dp[e + 1]), f2_pack(-dd.x, -dd.y))), d[0], d[1]);
          f2_unpack(f2_mul(f2_pack(p[e + 2], p[e + 3]),
                           f2_add(f2_pack(dp[e + 2], dp[e + 3]), f2_pack(-dd.z, -dd.w))), d[2], d[3]);
          if (kind == 2) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (!(mk & (1u << (e + v)))) d[v] = 0.f;
          }
          words[e >> 1] = pack_bf16(d[0], d[1]);
          words[(e >> 1) + 1] = pack_bf16(d[2], d[3]);
        }
      }
      tmem_st16u(dp_t, words);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok) {
      bool w = true;
      if (lane == 0) w = bounded_wait(acc_done, 0, abort_flag, err, kErrWinSoftmax, wait_ns);
      ok = warp_ok(w);
    }
    if (ok) {
      tc_fence_after();
      const int db = part * 32;  // this warp's 32 of the 128 head dims
      float v[32], g[32];
      tmem_ld32_async(tmem + 256 + db + lane_off, v);
      tmem_ld32_async(tmem + 384 + db + lane_off, g);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; ++e) g[e] *= a.scale;
      if (key < a.S) {
        if (u.slot >= 0) {
          float* pk = a.part + ((int64_t)u.slot * 2 * kTile + r) * kHeadDim + db;
          float* pv = pk + (int64_t)kTile * kHeadDim;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            *reinterpret_cast<float4*>(pk + e) = make_float4(g[e], g[e + 1], g[e + 2], g[e + 3]);
            *reinterpret_cast<float4*>(pv + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        } else {
          const int64_t o = (((int64_t)u.b * a.S + key) * a.Hk + u.hk) * kHeadDim + db;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            *reinterpret_cast<uint4*>(a.dk + o + e) =
                make_uint4(pack_bf16(g[e], g[e + 1]), pack_bf16(g[e + 2], g[e + 3]),
                           pack_bf16(g[e + 4], g[e + 5]), pack_bf16(g[e + 6], g[e + 7]));
            *reinterpret_cast<uint4*>(a.dv + o + e) =
                make_uint4(pack_bf16(v[e], v[e + 1]), pack_bf16(v[e + 2], v[e + 3]),
                           pack_bf16(v[e + 4], v[e + 5]), pack_bf16(v[e + 6], v[e + 7]));
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

// dk, dv of the key tiles whose sums are in slots: the sink tiles, and with groups > 1
// all tiles. Slots are added in a fixed order. Four elements per thread; one block
// takes 8 key rows of one tile.
__global__ void __launch_bounds__(256) win_dkdv_sum_kernel(BwdArgs a, int tiles) {
  const int nq = (a.S + kTile - 1) / kTile;
  const int rows8 = blockIdx.x % (kTile / 8);
  const int i = blockIdx.x / (kTile / 8);
  const int kt = i % tiles, bhk = i / tiles;
  const int r = rows8 * 8 + (threadIdx.x >> 5);
  const int key = kt * kTile + r;
  if (key >= a.S) return;
  int slot0, n;
  if (kt < a.n_sink) {
    slot0 = (bhk * a.sink_slots + segments_before(kt, nq, a.seg_steps)) * a.groups;
    n = a.groups * segments_of(kt, nq, a.seg_steps);
  } else {
    slot0 = (a.B * a.Hk * a.sink_slots + (kt - a.n_sink) * a.B * a.Hk + bhk) * a.groups;
    n = a.groups;
  }
  const int d = (threadIdx.x & 31) * 4;
  float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
  for (int s = 0; s < n; ++s) {
    const float* p = a.part + ((int64_t)(slot0 + s) * 2 * kTile + r) * kHeadDim + d;
    const float4 x = *reinterpret_cast<const float4*>(p);
    const float4 y = *reinterpret_cast<const float4*>(p + kTile * kHeadDim);
    k.x += x.x; k.y += x.y; k.z += x.z; k.w += x.w;
    v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
  }
  const int64_t o = (((int64_t)(bhk / a.Hk) * a.S + key) * a.Hk + bhk % a.Hk) * kHeadDim + d;
  *reinterpret_cast<uint2*>(a.dk + o) = make_uint2(pack_bf16(k.x, k.y), pack_bf16(k.z, k.w));
  *reinterpret_cast<uint2*>(a.dv + o) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// dQ of one query tile, keys in blocks of 64, two CTAs an SM (one fills the tensor pipe while
// the other's compute warps work, starts or ends): 204 us with D at 1 x 16001 tokens, 12 heads
// over 2, window 1000, 16 sinks, against 206 + 31 us of one CTA an SM with 128-key tiles and a
// kernel for D; 76 against 76 + 20 us at 4 x 2048 tokens, window 512. A persistent CTA that
// loads the next tile's operands early measured 212 and 85 us. Bound by the products: N = 64
// ones take as long as N = 128 ones.
// TMEM (256 columns): S 0, dP 64, dQ 128. dS overwrites the dP columns that it was computed
// from (bf16 pairs, the 32 keys of a compute warp in the first 16 of its own 32 columns) and
// is the A operand of dQ += dS K read from TMEM. Issue order
//   S(i + 1), dQ(i), dP(i + 1), S(i + 2), ...
// Shared memory: Q and dO (32 KB each), two K blocks and a V block of 16 KB. A compute thread
// owns 32 keys of one query row of each block.
// The compute warps first form D = dO . O of the tile's rows, and store it with
// -lse log2(e) for the dK / dV kernel, which follows: no kernel of its own reads out and dout.
constexpr int kDqWarps = 8;
constexpr int kDqThreads = 64 + 32 * kDqWarps;
struct WinDqSmem {
  static constexpr int kQ = 0;
  static constexpr int kDO = kQ + kTileBytes;
  static constexpr int kK = kDO + kTileBytes;
  static constexpr int kV = kK + 2 * kStepTile;
  static constexpr int kBar = kV + kStepTile;
  // qdo_full, k_full[2], k_empty[2], v_full, v_empty, s_full, s_empty, dp_full, ds_full, d_full,
  // acc_done, drain
  static constexpr int kNumBars = 14;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kD = kMisc + 16;  // D of the rows
  static constexpr int kUsed = kD + kTile * 4;
  static constexpr int kBytes = 115712;  // half of an SM's 228 KB less 1 KB a CTA
};
static_assert(WinDqSmem::kUsed + 256 <= WinDqSmem::kBytes, "window attention dQ shared memory");

__global__ void __launch_bounds__(kDqThreads, 2)
    win_dq_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_k,
                  const __grid_constant__ CUtensorMap tma_v,
                  const __grid_constant__ CUtensorMap tma_do, BwdArgs a, int* err) {
  using L = WinDqSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  if ((uint32_t)(smem - smem_raw) + L::kUsed > dynamic_smem_bytes()) {  // grid-uniform
    if (threadIdx.x == 0) atomicCAS(err, 0, kErrWinSmem);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::kBar;
  const uint32_t qdo_full = bar0;
  auto k_full = [&](int i) { return bar0 + 8u * (1 + (i & 1)); };
  auto k_empty = [&](int i) { return bar0 + 8u * (3 + (i & 1)); };
  const uint32_t v_full = bar0 + 8u * 5, v_empty = bar0 + 8u * 6;
  const uint32_t s_full = bar0 + 8u * 7, s_empty = bar0 + 8u * 8;
  const uint32_t dp_full = bar0 + 8u * 9, ds_full = bar0 + 8u * 10, d_full = bar0 + 8u * 11;
  const uint32_t acc_done = bar0 + 8u * 12, drain_bar = bar0 + 8u * 13;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nq = (a.S + kTile - 1) / kTile;
  const int bh = blockIdx.x % (a.B * a.H);
  const int qt = nq - 1 - blockIdx.x / (a.B * a.H);  // late query tiles first
  const int b = bh / a.H, h = bh % a.H;
  const int hk = h / (a.H / a.Hk);
  const int q0 = qt * kTile;
  const KeyBlocks kb = key_blocks(qt, a.S, a.window, a.sinks);
  const int n = kb.n;
  const uint64_t wait_ns = a.wait_ns;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kNumBars; ++i) {
      const uint32_t bar = bar0 + 8u * i;
      mbar_init(bar, bar == s_empty || bar == ds_full || bar == d_full ? kDqWarps : 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc::tma_prefetch_desc(&tma_q);
    tc::tma_prefetch_desc(&tma_k);
    tc::tma_prefetch_desc(&tma_v);
    tc::tma_prefetch_desc(&tma_do);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_holder)),
                 "r"(256)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer ----
      mbar_arrive_expect_tx(qdo_full, 2 * kTileBytes);
      tma_load_4d(sbase + L::kQ, &tma_q, qdo_full, 0, q0, h, b);
      tma_load_4d(sbase + L::kQ + kBox, &tma_q, qdo_full, 64, q0, h, b);
      tma_load_4d(sbase + L::kDO, &tma_do, qdo_full, 0, q0, h, b);
      tma_load_4d(sbase + L::kDO + kBox, &tma_do, qdo_full, 64, q0, h, b);
      int issued_k = 0, issued_v = 0;
      for (int i = 0; i < n; ++i) {
        const int key0 = kb.at(i) * kBlk;
        if (!bounded_wait(k_empty(i), ((i >> 1) & 1) ^ 1, abort_flag, err, kErrWinProducer, wait_ns))
          break;
        const uint32_t kd = sbase + L::kK + (i & 1) * kStepTile;
        mbar_arrive_expect_tx(k_full(i), kStepTile);
        tma_load_4d(kd, &tma_k, k_full(i), 0, key0, hk, b);
        tma_load_4d(kd + kStepBox, &tma_k, k_full(i), 64, key0, hk, b);
        ++issued_k;
        if (!bounded_wait(v_empty, (i & 1) ^ 1, abort_flag, err, kErrWinProducer, wait_ns)) break;
        mbar_arrive_expect_tx(v_full, kStepTile);
        tma_load_4d(sbase + L::kV, &tma_v, v_full, 0, key0, hk, b);
        tma_load_4d(sbase + L::kV + kStepBox, &tma_v, v_full, 64, key0, hk, b);
        ++issued_v;
      }
      uint64_t t0 = tc::globaltimer();
      while (!mbar_try_wait(qdo_full, 0) && tc::globaltimer() - t0 < wait_ns) {
      }
      for (int i = issued_k > 2 ? issued_k - 2 : 0; i < issued_k; ++i) {
        t0 = tc::globaltimer();
        while (!mbar_try_wait(k_full(i), (i >> 1) & 1) && tc::globaltimer() - t0 < wait_ns) {
        }
      }
      t0 = tc::globaltimer();
      while (issued_v > 0 && !mbar_try_wait(v_full, (issued_v - 1) & 1) &&
             tc::globaltimer() - t0 < wait_ns) {
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------- MMA issuer ----
    auto wait = [&](uint32_t bar, int parity) {
      return warp_wait(bar, parity, abort_flag, err, kErrWinMma, wait_ns);
    };
    bool ok = wait(qdo_full, 0);
    bool issued = false;
    const Desc q_desc(smem_desc_sw128(sbase + L::kQ, 16, 1024));
    const Desc do_desc(smem_desc_sw128(sbase + L::kDO, 16, 1024));
    const Desc k_desc(smem_desc_sw128(sbase + L::kK, 16, 1024));
    const Desc k_mn(smem_desc_sw128(sbase + L::kK, kStepBox, 1024));
    const Desc v_desc(smem_desc_sw128(sbase + L::kV, 16, 1024));
    auto issue_s = [&](int i) -> bool {  // S = Q K^T
      if (!wait(k_full(i), (i >> 1) & 1)) return false;
      if (i > 0 && !wait(s_empty, (i - 1) & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kHeadDim / 16; ++kk)
          mma_ss(tmem, q_desc.at(kmajor_step(kk, kBox)), q_desc.hi,
                 k_desc.at((i & 1) * kStepTile + kmajor_step(kk, kStepBox)), k_desc.hi, kIdescKK64,
                 kk > 0 ? 1u : 0u);
        tc_commit(s_full);
      }
      __syncwarp();
      issued = true;
      return true;
    };
    auto issue_dp = [&](int i) -> bool {  // dP = dO V^T
      if (!wait(v_full, i & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kHeadDim / 16; ++kk)
          mma_ss(tmem + 64, do_desc.at(kmajor_step(kk, kBox)), do_desc.hi,
                 v_desc.at(kmajor_step(kk, kStepBox)), v_desc.hi, kIdescKK64, kk > 0 ? 1u : 0u);
        tc_commit(dp_full);
        tc_commit(v_empty);
      }
      __syncwarp();
      return true;
    };
    if (ok) ok = issue_s(0);
    if (ok) ok = issue_dp(0);
    for (int i = 0; i < n && ok; ++i) {
      if (i + 1 < n && !(ok = issue_s(i + 1))) break;
      if (!(ok = wait(ds_full, i & 1))) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kBlk / 16; ++kk)  // dQ += dS K
          mma_ts(tmem + 128, tmem + 64 + (kk >> 1) * 32 + (kk & 1) * 8,
                 k_mn.at((i & 1) * kStepTile + mnmajor_step(kk)), k_mn.hi, kIdescKM,
                 (i > 0 || kk > 0) ? 1u : 0u);
        tc_commit(k_empty(i));
        if (i + 1 == n) tc_commit(acc_done);
      }
      __syncwarp();
      // dP(i + 1) overwrites the dS that dQ has read
      if (i + 1 < n) ok = wait(k_empty(i), (i >> 1) & 1) && issue_dp(i + 1);
    }
    // the last arrivals of the rings
    for (int i = n > 2 ? n - 2 : 0; i < n && ok; ++i) ok = wait(k_empty(i), (i >> 1) & 1);
    if (ok) ok = wait(v_empty, (n - 1) & 1);
    if (!ok && issued) {
      if (elect_one()) tc_commit(drain_bar);
      __syncwarp();
      uint64_t t0 = tc::globaltimer();
      while (!mbar_try_wait(drain_bar, 0) && tc::globaltimer() - t0 < wait_ns) {
      }
    }
  } else {
    // ------------------------------------------------------- compute ----
    const int quarter = warp & 3;
    const int part = (warp - 2) >> 2;   // keys [32 part, 32 part + 32) of each block
    const int r = quarter * 32 + lane;  // query row of this thread
    const int q = q0 + r;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint64_t sl2 = f2_pack(a.scale_log2, a.scale_log2);
    const uint32_t s_t = tmem + part * 32 + lane_off, dp_t = s_t + 64;
    const int64_t vrow = ((int64_t)b * a.H + h) * ((int64_t)nq * kTile);
    float* d_rows = reinterpret_cast<float*>(smem + L::kD);
    bool ok = true, w = true;
    const float nl = q < a.S ? -a.lse[vrow + q] * kLog2e : 0.f;
    {  // D: 16 lanes a row (16 bytes each), four rows of a half-warp in flight
      const int sub = lane & 15;
#pragma unroll 1
      for (int r0 = ((warp - 2) * 2 + (lane >> 4)) * 4; r0 < kTile; r0 += 8 * kDqWarps) {
        uint4 x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = y[e] = make_uint4(0, 0, 0, 0);
          if (q0 + r0 + e < a.S) {
            const int64_t o = (((int64_t)b * a.S + q0 + r0 + e) * a.H + h) * kHeadDim + sub * 8;
            x[e] = *reinterpret_cast<const uint4*>(a.dout + o);
            y[e] = *reinterpret_cast<const uint4*>(a.out + o);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __nv_bfloat162* xp = reinterpret_cast<const __nv_bfloat162*>(&x[e]);
          const __nv_bfloat162* yp = reinterpret_cast<const __nv_bfloat162*>(&y[e]);
          float acc = 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float2 f = __bfloat1622float2(xp[v]), g = __bfloat1622float2(yp[v]);
            acc = fmaf(f.x, g.x, fmaf(f.y, g.y, acc));
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
          if (sub == 0) d_rows[r0 + e] = acc;
        }
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(d_full);
        w = bounded_wait(d_full, 0, abort_flag, err, kErrWinSoftmax, wait_ns);
      }
      ok = warp_ok(w);
      __syncwarp();
    }
    const float nd = ok ? -d_rows[r] : 0.f;
    if (ok && part == 0 && q < a.S) {
      a.Dv[vrow + q] = -nd;
      a.nl2[vrow + q] = nl;
    }
    const uint64_t nl2 = f2_pack(nl, nl), nd2 = f2_pack(nd, nd);
    for (int i = 0; i < n && ok; ++i) {
      const int k0 = kb.at(i) * kBlk;
      uint32_t mk = 0xffffffffu;
      int kind = 1;
      if (block_edge(k0, q0, a.S, a.window, a.sinks)) {
        mk = keys_seen(q, k0 + part * 32, a.S, a.window, a.sinks);
        kind = mask_kind(mk, 0xffffffffu);
      }
      if (!(ok = warp_wait(s_full, i & 1, abort_flag, err, kErrWinSoftmax, wait_ns))) break;
      tc_fence_after();
      float p[32];
      tmem_ld32_async(s_t, p);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_empty);  // the next block's S may overwrite it
      if (kind != 0) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          f2_unpack(f2_fma(f2_pack(p[e], p[e + 1]), sl2, nl2), p[e], p[e + 1]);
          p[e] = fast_exp2(p[e]);
          p[e + 1] = fast_exp2(p[e + 1]);
        }
      }
      if (!(ok = warp_wait(dp_full, i & 1, abort_flag, err, kErrWinSoftmax, wait_ns))) break;
      tc_fence_after();
      float dp[32];
      tmem_ld32_async(dp_t, dp);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; e += 2)
        f2_unpack(f2_mul(f2_pack(p[e], p[e + 1]), f2_add(f2_pack(dp[e], dp[e + 1]), nd2)), p[e],
                  p[e + 1]);
      if (kind != 1) {  // hidden keys may hold anything: select, do not scale
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(mk & (1u << e))) p[e] = 0.f;
      }
      uint32_t dw[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) dw[e] = pack_bf16(p[2 * e], p[2 * e + 1]);
      tmem_st16u(dp_t, dw);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok) {
      if (lane == 0) w = bounded_wait(acc_done, 0, abort_flag, err, kErrWinSoftmax, wait_ns);
      ok = warp_ok(w);
    }
    if (ok) {
      tc_fence_after();
      bf16* orow = a.dq + (((int64_t)b * a.S + q) * a.H + h) * kHeadDim + part * 64;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float o[32];
        tmem_ld32(tmem + 128 + part * 64 + c * 32 + lane_off, o);
        if (q < a.S) {
          const float sc = a.scale;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint4*>(orow + c * 32 + 8 * g) =
                make_uint4(pack_bf16(o[8 * g] * sc, o[8 * g + 1] * sc),
                           pack_bf16(o[8 * g + 2] * sc, o[8 * g + 3] * sc),
                           pack_bf16(o[8 * g + 4] * sc, o[8 * g + 5] * sc),
                           pack_bf16(o[8 * g + 6] * sc, o[8 * g + 7] * sc));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256)
                 : "memory");
  }
}

// ----------------------------------------------------------------- host ----
void fn_error(const char* fn, const char* text) {
  char msg[256];
  snprintf(msg, sizeof(msg), "%s: %s", fn, text);
  set_last_error(msg);
}

bool sizes_ok(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq) {
  return batch > 0 && heads > 0 && kv_heads > 0 && seq > 0 && heads % kv_heads == 0 &&
         batch * heads <= (1 << 20) && seq <= (1 << 24) &&
         batch * heads * ((seq + kTile - 1) / kTile) <= (1 << 28);
}

// The visible keys in the form that the kernels run fastest: a window and sinks that
// together reach every key (window + sinks >= seq) are the plain causal case.
struct Visible {
  int window, sinks;
};
Visible visible(int64_t seq, int64_t window, int64_t sinks) {
  if (window > seq) window = seq;
  if (sinks > seq) sinks = seq;
  if (window + sinks >= seq) return {(int)seq, 0};
  return {(int)window, (int)sinks};
}

// How the dK / dV work is cut: the query heads of a KV head into `groups` CTAs when
// one CTA per key tile would leave SMs idle, the sink tiles' steps into segments as
// long as an ordinary tile's, or, with many sinks, a quarter of an SM's share of all steps
// (each segment costs 128 KB of partials, and shorter ones no longer even out the SMs).
struct DkvPlan {
  int groups, heads_per, n_sink, segs, seg_steps, sink_slots;
  int64_t units, slots;
};
DkvPlan dkv_plan(int64_t B, int64_t H, int64_t Hk, int64_t S, int64_t window, int64_t sinks) {
  DkvPlan p;
  const int64_t nt = (S + kTile - 1) / kTile;
  const Visible vis = visible(S, window, sinks);
  p.n_sink = (vis.sinks + kTile - 1) / kTile;
  const int64_t steps = (kTile + vis.window - 2) / kTile + 1;  // of an ordinary tile
  const int64_t rep = H / Hk;
  const int64_t tiles = B * Hk * nt;
  // one CTA per key tile if that fills most SMs, else the fewest head groups that do
  int64_t g = (num_sms() * 4 / 5 + tiles - 1) / tiles;
  if (g > rep) g = rep;
  if (g < 1) g = 1;
  p.heads_per = (int)((rep + g - 1) / g);
  p.groups = (int)((rep + p.heads_per - 1) / p.heads_per);
  const int64_t ns = p.n_sink, tile_steps = steps < nt ? steps : nt;
  const int64_t all = B * Hk * p.groups * (ns * nt - ns * (ns - 1) / 2 + (nt - ns) * tile_steps);
  const int64_t share = (all + 4 * num_sms() - 1) / (4 * num_sms());
  int64_t seg = share > tile_steps ? share : tile_steps;
  if (seg > nt) seg = nt;
  p.seg_steps = (int)(seg < 4 ? 4 : seg);
  p.segs = (int)((nt + p.seg_steps - 1) / p.seg_steps);
  p.sink_slots = segments_before(p.n_sink, (int)nt, p.seg_steps);
  const int64_t sink_units = B * Hk * p.n_sink * p.groups * p.segs;
  const int64_t rest = B * Hk * (nt - p.n_sink) * p.groups;
  p.units = sink_units + rest;
  p.slots = B * Hk * p.sink_slots * p.groups + (p.groups > 1 ? rest : 0);
  return p;
}
size_t vec_bytes(int64_t B, int64_t H, int64_t S) {
  const size_t s_pad = (size_t)((S + kTile - 1) / kTile * kTile);
  return ((size_t)B * H * s_pad * 4 + 255) / 256 * 256;
}

}  // namespace
}  // namespace attn
}  // namespace soup

using namespace soup;
using namespace soup::attn;

extern "C" {

int soup_attention_window_fwd(const void* q, const int64_t* q_strides, const void* k,
                              const int64_t* k_strides, const void* v, const int64_t* v_strides,
                              int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq,
                              int64_t head_dim, float scale, int64_t window, int64_t sinks,
                              void* out, float* lse, void* stream) {
  const char* fn = "soup_attention_window_fwd";
  if (!sizes_ok(batch, heads, kv_heads, seq) || !out || !lse || !(scale > 0.f)) {
    fn_error(fn, "bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (window <= 0 || sinks < 0) {
    fn_error(fn, "window must be positive and sinks not negative");
    return SOUP_ERR_INVALID;
  }
  if (head_dim != kHeadDim) {
    fn_error(fn, "head_dim must be 128");
    return SOUP_ERR_UNSUPPORTED;
  }
  if (!bhsd_ok(q, q_strides) || !bhsd_ok(k, k_strides) || !bhsd_ok(v, v_strides) ||
      !aligned16(out)) {
    fn_error(fn, "q/k/v need 16-byte aligned bases and strides that are multiples of 8 elements "
                 "(last dimension contiguous)");
    return SOUP_ERR_UNSUPPORTED;
  }
  int* err = device_err_ptr();
  if (!err) {
    set_last_error("device error word unavailable");
    return SOUP_ERR_CUDA;
  }
  CUtensorMap mq, mk, mv;
  int rc;
  if ((rc = make_bhsd_map(&mq, q, q_strides, batch, heads, seq, "q"))) return rc;
  if ((rc = make_bhsd_map(&mk, k, k_strides, batch, kv_heads, seq, "k", kBlk))) return rc;
  if ((rc = make_bhsd_map(&mv, v, v_strides, batch, kv_heads, seq, "v", kBlk))) return rc;
  static bool smem_set_done[64] = {false};
  if ((rc = set_smem(win_fwd_kernel, WinFwdSmem::kBytes, smem_set_done))) return rc;
  const Visible vis = visible(seq, window, sinks);
  FwdArgs a{(int)batch, (int)heads, (int)kv_heads, (int)seq, scale * 1.4426950408889634f, vis.window,
            vis.sinks, static_cast<bf16*>(out), lse, wait_limit_ns() ? wait_limit_ns() : tc::kWaitNs};
  const int64_t nq = (seq + kTile - 1) / kTile;
  win_fwd_kernel<<<(unsigned)(batch * heads * nq), kFwdThreads, WinFwdSmem::kBytes,
                   as_stream(stream)>>>(mq, mk, mv, a, err);
  return launch_status();
}

size_t soup_attention_window_bwd_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads,
                                                 int64_t seq, int64_t window, int64_t sinks) {
  if (!sizes_ok(batch, heads, kv_heads, seq) || window <= 0 || sinks < 0) return 0;
  const DkvPlan p = dkv_plan(batch, heads, kv_heads, seq, window, sinks);
  return 2 * vec_bytes(batch, heads, seq) + (size_t)p.slots * 2 * kTile * kHeadDim * 4;
}

int soup_attention_window_bwd(const void* q, const int64_t* q_strides, const void* k,
                              const int64_t* k_strides, const void* v, const int64_t* v_strides,
                              const void* out, const void* dout, const float* lse, int64_t batch,
                              int64_t heads, int64_t kv_heads, int64_t seq, int64_t head_dim,
                              float scale, int64_t window, int64_t sinks, void* dq, void* dk,
                              void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "soup_attention_window_bwd";
  if (!sizes_ok(batch, heads, kv_heads, seq) || !out || !dout || !lse || !dq || !dk || !dv ||
      !workspace || !(scale > 0.f)) {
    fn_error(fn, "bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (window <= 0 || sinks < 0) {
    fn_error(fn, "window must be positive and sinks not negative");
    return SOUP_ERR_INVALID;
  }
  if (head_dim != kHeadDim) {
    fn_error(fn, "head_dim must be 128");
    return SOUP_ERR_UNSUPPORTED;
  }
  if (!bhsd_ok(q, q_strides) || !bhsd_ok(k, k_strides) || !bhsd_ok(v, v_strides) ||
      !aligned16(out) || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
      !aligned16(lse)) {
    fn_error(fn, "operands need 16-byte aligned bases and strides that are multiples of 8 elements");
    return SOUP_ERR_UNSUPPORTED;
  }
  const DkvPlan p = dkv_plan(batch, heads, kv_heads, seq, window, sinks);
  const size_t vbytes = vec_bytes(batch, heads, seq);
  if (workspace_bytes < soup_attention_window_bwd_workspace_bytes(batch, heads, kv_heads, seq, window,
                                                                  sinks) ||
      !aligned16(workspace)) {
    fn_error(fn, "workspace too small or misaligned");
    return SOUP_ERR_WORKSPACE;
  }
  if (p.units > 0x7fffffff) {
    fn_error(fn, "too many key tiles");
    return SOUP_ERR_UNSUPPORTED;
  }
  int* err = device_err_ptr();
  if (!err) {
    set_last_error("device error word unavailable");
    return SOUP_ERR_CUDA;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* dvec = reinterpret_cast<float*>(ws);
  float* nl2 = reinterpret_cast<float*>(ws + vbytes);
  float* part = reinterpret_cast<float*>(ws + 2 * vbytes);
  CUtensorMap mq, mk, mv, mkb, mvb, mdo;  // tiles of 128 keys (dK, dV) and blocks of 64 (dQ)
  int rc;
  const int64_t do_strides[3] = {seq * heads * kHeadDim, kHeadDim, heads * kHeadDim};
  if ((rc = make_bhsd_map(&mq, q, q_strides, batch, heads, seq, "q"))) return rc;
  if ((rc = make_bhsd_map(&mk, k, k_strides, batch, kv_heads, seq, "k"))) return rc;
  if ((rc = make_bhsd_map(&mv, v, v_strides, batch, kv_heads, seq, "v"))) return rc;
  if ((rc = make_bhsd_map(&mkb, k, k_strides, batch, kv_heads, seq, "k", kBlk))) return rc;
  if ((rc = make_bhsd_map(&mvb, v, v_strides, batch, kv_heads, seq, "v", kBlk))) return rc;
  if ((rc = make_bhsd_map(&mdo, dout, do_strides, batch, heads, seq, "dout"))) return rc;
  static bool dkdv_set[64] = {false}, dq_set[64] = {false};
  if ((rc = set_smem(win_dkdv_kernel, WinDkvSmem::kBytes, dkdv_set))) return rc;
  if ((rc = set_smem(win_dq_kernel, WinDqSmem::kBytes, dq_set))) return rc;
  cudaStream_t st = as_stream(stream);
  const int B = (int)batch, H = (int)heads, Hk = (int)kv_heads, S = (int)seq;
  const Visible vis = visible(seq, window, sinks);
  BwdArgs a{B, H, Hk, S, scale, scale * 1.4426950408889634f, vis.window, vis.sinks, dvec, nl2,
            static_cast<const bf16*>(out), static_cast<const bf16*>(dout), lse,
            static_cast<bf16*>(dq), static_cast<bf16*>(dk), static_cast<bf16*>(dv), part, p.groups,
            p.heads_per, p.n_sink, p.segs, p.seg_steps, p.sink_slots,
            wait_limit_ns() ? wait_limit_ns() : tc::kWaitNs};
  const int nt = (S + kTile - 1) / kTile;
  win_dq_kernel<<<(unsigned)(B * H * nt), kDqThreads, WinDqSmem::kBytes, st>>>(mq, mkb, mvb, mdo, a,
                                                                              err);
  if ((rc = launch_status())) return rc;
  win_dkdv_kernel<<<(unsigned)p.units, kThreads, WinDkvSmem::kBytes, st>>>(mq, mk, mv, mdo, a, err);
  if ((rc = launch_status())) return rc;
  const int tiles = p.groups > 1 ? nt : p.n_sink;  // key tiles whose sums are in slots
  if (tiles == 0) return SOUP_OK;
  win_dkdv_sum_kernel<<<(unsigned)(B * Hk * tiles * (kTile / 8)), 256, 0, st>>>(a, tiles);
  return launch_status();
}

}  // extern "C"
