// A shared projection with low-rank adapters of many requests beside it.
//
//   y_t = W x_t + b + B_a u_t,   u_t = s_a A_a x_t,   a = adapter of token t (or none)
// backward:
//   v_t = s_a B_a^T dy_t,  dx_t = W^T dy_t + A_a^T v_t,
//   dA_a = sum over its tokens of v_t x_t^T,  dB_a = sum over its tokens of dy_t u_t^T
//
// The adapters lie side by side: A [R, K] and B [N, R] with R = adapters x rank. With
// U [T, R] holding u_t in the columns of token t's adapter and 0 elsewhere, all of it
// is plain products, y = x W^T + U B^T, U = mask(x A^T), and so on, of which only a few
// blocks of 64 rank columns (64 / rank adapters) have anything for a given tile of
// tokens: requests are runs of tokens. So each 64-token block keeps a 64-bit word with
// one bit per rank block (R <= 4096), and
//   - U and V are formed for the rank blocks of a 256-token tile (rank_tile_kernel),
//   - the base product reads, after its own k blocks, the k blocks of U and B that the
//     tile's word names, into the same accumulator (gemm_pair_kernel, Sched::k2_mask),
//   - dA and dB of a rank block run over the token blocks whose word has its bit.
// Nothing is sorted or gathered, and no host round trip is needed for the ids.
//
// The rank products move one large operand (x or dy) against a few KB, so they are
// HBM-bound: a 128-row tile of it streams through a 4-stage TMA ring into tcgen05.mma
// (M 128, N 64), the k range split over a cluster whose CTAs add their partial tiles
// in rank order through distributed shared memory (bitwise reproducible).
//
// Few tokens (next tokens of many requests): the base product is W's bytes.
// The same kernel then streams W as the 128-row operand against all tokens at once
// (N = T rounded up, at most 128 a CTA), so that every SM takes part, with U and B's
// blocks behind; it starts beside the kernel that forms U and waits for that one only
// before its rank blocks.
//
// 8192 tokens, 1536 -> 17920 features, 4 adapters of rank 16: U 17 us, y 322 (309 without
// adapters), V 68 (dy's 294 MB at 4.3 TB/s), dx 330 (328), dA 17, dB 53 (5.5 TB/s). 48 tokens
// and 64 adapters: 21 us for 55 MB of weights; 8 tokens of 18944 -> 3584 27 us, 5 TB/s.
//
// u and v are rounded to bf16 between the two products: tcgen05 multiplies operands of one
// type, and the factors are bf16. Beside the outputs' own rounding (0.00166 of the norm of
// bf16 values) that is a second one of the same size in every term of dA and dB, 0.00235 by
// the root of two and as measured, and a small part of y and dx (0.0017 to 0.0018). Held to
// 16 bits, as a second set of rank columns for the remainders, u and v would take about what
// twice the columns do: 8192 tokens trained 791 -> 811 us, 2999 ragged ones 193 -> 211, 48
// tokens of as many adapters up to 17.5 -> 27 (with the factors' bytes doubled too). A step's
// gradients, which the moments average, are not worth that.
//
//   warp 0     TMA producer (one lane)
//   warp 1     TMEM allocator + MMA issuer (one lane; for gradients it also clears rows)
//   warps 2-5  epilogue: tcgen05.ld of lane quarter (warp % 4), cluster reduction, stores
//
// Every mbarrier wait is bounded (soup_set_wait_limit_ns); on expiry the code goes to
// the device error word, the CTA stops issuing, drains what it issued, still takes part
// in both cluster barriers, skips its stores and frees its TMEM.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include <stdio.h>

#include <mutex>

#include "multi_lora.cuh"
#include "soup_common.cuh"
#include "tc_gemm.cuh"

namespace soup {
namespace {

using bf16 = __nv_bfloat16;
using namespace tc;

constexpr int kThreads = 192;
constexpr int kRankBlock = 64;     // rank columns of a block
constexpr int kMaxRank = 4096;     // adapters x rank: one bit per block in 64 bits
constexpr int kFewTokens = 256;    // at most, of kModeFew: one word of rank blocks
constexpr int kFewTile = 128;      // of them in a CTA's columns
constexpr int kMaxTokens = 1 << 21;
constexpr int kErrProducer = 0x141;
constexpr int kErrMma = 0x142;
constexpr int kErrEpilogue = 0x143;
constexpr int kErrSmem = 0x144;

// What a launch computes (C [128-row tiles of the large operand, NP columns]):
constexpr int kModeRank = 0;  // U or V: rows are tokens, k is K or N, one rank block a CTA
constexpr int kModeGrad = 1;  // dA or dB: rows are features, k the token blocks of a rank block
constexpr int kModeFew = 2;   // y of few tokens: rows are features, columns tokens

template <int NP>
struct Smem {
  // two CTAs an SM
  static constexpr int kStages = NP > 64 ? 3 : 4;
  static constexpr int kABytes = 128 * 64 * 2;
  static constexpr int kBBytes = NP * 64 * 2;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kPartStride = NP + 4;  // [row][column]
  static constexpr int kPartStrideT = 132;    // [column][row]
  static_assert(128 * kPartStride * 4 <= kStages * kStage && NP * kPartStrideT * 4 <= kStages * kStage,
                "the partial tile reuses the stages");
  static constexpr int kBar = kStages * kStage;
  static constexpr int kNumBars = 2 * kStages + 1;  // full[S], empty[S], acc_full
  static constexpr int kMisc = kBar + kNumBars * 8;  // tmem, abort, words[8]
  static constexpr int kBits = kMisc + 16 + 64;      // kModeGrad: two bits per token block
  static constexpr int kBytesFor(int token_blocks) { return kBits + ((token_blocks + 31) / 32 + 1) * 8 + 1024; }
};

struct Args {
  int rows;          // rows of C (tokens or features)
  int k;             // its k extent in elements
  int kb_total;      // k blocks of the first segment
  int ks;            // CTAs of a cluster
  int tokens, rank_cols, rank;
  int adapters;
  uint64_t wait_ns;
  // token -> adapter
  const void* ids;
  int ids_64;
  int per;           // tokens of one id
  const float* scales;
  uint64_t* mask64;  // words of 64-token blocks: rank blocks that any of their tokens has
  uint64_t* all64;   // and that all of them have
  uint64_t* mask256; // words of 256-token tiles
  int write_masks;
  // outputs
  bf16* u;           // kModeRank [tokens, rank_cols]
  void* grad;        // kModeGrad: [rows, rank_cols], or transposed
  int grad_f32, grad_trans;
  bf16* y;           // kModeFew [tokens, rows]
  int64_t ldy;
  const bf16* bias;
};

__device__ __forceinline__ uint32_t dynamic_smem() {
  uint32_t v;
  asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(v));
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}
// 32 lanes x 16 consecutive fp32 columns (no wait; tcgen05.wait::ld follows).
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ uint2 pack_bf16x4(float4 f) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(f.x, f.y), hi = __floats2bfloat162_rn(f.z, f.w);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
__device__ __forceinline__ void store_grad(const Args& a, int64_t at, float4 f) {
  if (a.grad_f32) *reinterpret_cast<float4*>(static_cast<float*>(a.grad) + at) = f;
  else *reinterpret_cast<uint2*>(static_cast<bf16*>(a.grad) + at) = pack_bf16x4(f);
}

// Adapter of token t: -1 for none, for an id outside [0, adapters) and behind the last token.
__device__ __forceinline__ int adapter_of(const Args& a, int t) {
  if (t >= a.tokens) return -1;
  const int64_t i = t / a.per;
  const int64_t id = a.ids_64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int*>(a.ids)[i];
  return id >= 0 && id < a.adapters ? (int)id : -1;
}
// Bits of the rank blocks that an adapter's columns lie in.
__device__ __forceinline__ uint64_t adapter_bits(const Args& a, int id) {
  if (id < 0) return 0;
  const int lo = id * a.rank / kRankBlock, hi = (id * a.rank + a.rank - 1) / kRankBlock;
  const uint64_t upto = hi == 63 ? ~0ull : (1ull << (hi + 1)) - 1;
  return upto & ~((1ull << lo) - 1);
}
__device__ __forceinline__ uint64_t warp_or64(uint64_t v) {
  const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)v);
  const uint32_t hi = __reduce_or_sync(0xffffffffu, (uint32_t)(v >> 32));
  return ((uint64_t)hi << 32) | lo;
}
// The words of 64 tokens, formed by a warp: rank blocks that any of them has, that all have.
__device__ __forceinline__ uint64_t block_words(const Args& a, int t0, int lane, uint64_t& all) {
  uint64_t any = 0, none = 0;
#pragma unroll
  for (int t = t0 + lane; t < t0 + 64; t += 32) {
    const uint64_t b = adapter_bits(a, adapter_of(a, t));
    any |= b;
    none |= t < a.tokens ? ~b : 0;
  }
  all = ~warp_or64(none);
  return warp_or64(any);
}

// The k blocks of a CTA: a run of blocks and (kModeFew) behind it its share of the rank
// blocks of the tokens' word; or (kModeGrad) the set bits [lo, hi) of a bit list.
// Producer and MMA issuer walk the same.
struct KWalk {
  int kb, end;             // run
  const uint64_t* pending; // the word, not read yet
  int rank, ks;
  uint64_t word;           // rank blocks still to come
  const uint32_t* bits;    // or: bit list
  int skip, left;
  int w;
  uint32_t cur;
  __device__ __forceinline__ bool next(int& k_block, bool& second) {
    second = false;
    if (bits) {
      if (left == 0) return false;
      while (true) {
        if (cur == 0) {
          cur = bits[++w];
          const int n = __popc(cur);
          if (skip >= n) {
            skip -= n;
            cur = 0;
          }
          continue;
        }
        const int b = __ffs(cur) - 1;
        cur &= cur - 1;
        if (skip > 0) {
          --skip;
          continue;
        }
        k_block = w * 32 + b;
        --left;
        return true;
      }
    }
    if (kb < end) {
      k_block = kb++;
      return true;
    }
    if (pending) {
      // the word and U are of the kernel before, whose end is waited for only here: the
      // run's operands were complete before that kernel let this one start
      pdl_wait();
      uint64_t all = *pending;
      pending = nullptr;
      const int n = __popcll(all);
      const int lo = n * rank / ks, hi = n * (rank + 1) / ks;
      for (int i = 0; i < hi; ++i) {
        if (i >= lo) word |= all & (~all + 1);
        all &= all - 1;
      }
    }
    if (word) {
      k_block = __ffsll((long long)word) - 1;
      word &= word - 1;
      second = true;
      return true;
    }
    return false;
  }
};

// Grid: (tiles of 128 rows) x ks, rank blocks (kModeRank, kModeGrad) or token tiles
// (kModeFew); clusters of ks.
// A K-major: map {k, rows}, box {64, 128}; MN-major (kModeGrad): map {rows, k}, box {64, 64}.
// B K-major: map {k, columns}, box {64, NP}; MN-major: map {columns, k}, box {64, 64}.
template <int MODE, bool B_MN, int NP>
__global__ void __launch_bounds__(kThreads, 2)
    rank_tile_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                     const __grid_constant__ CUtensorMap tma_a2, const __grid_constant__ CUtensorMap tma_b2,
                     const Args a, int* err) {
  using L = Smem<NP>;
  constexpr bool A_MN = MODE == kModeGrad;
  constexpr uint32_t kCols = NP <= 32 ? 32 : NP;
  constexpr uint32_t kIdesc = idesc_bf16(NP, A_MN, B_MN, 128);
  static_assert(!B_MN || NP == 64, "an MN-major factor is read 64 columns at a time");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int token_blocks = (a.tokens + 63) / 64;
  const uint32_t used = MODE == kModeGrad ? L::kBits + ((token_blocks + 31) / 32 + 1) * 8 : L::kBits;
  if ((uint32_t)(smem - smem_raw) + used > dynamic_smem()) {  // grid-uniform
    if (threadIdx.x == 0) atomicCAS(err, 0, kErrSmem);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + L::kBar;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (L::kStages + s); };
  const uint32_t acc_bar = bar0 + 8u * (2 * L::kStages);
  float* part = reinterpret_cast<float*>(smem);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  uint64_t* words = reinterpret_cast<uint64_t*>(smem + L::kMisc + 16);
  uint32_t* bits = reinterpret_cast<uint32_t*>(smem + L::kBits);
  uint32_t* mixed = bits + (token_blocks + 31) / 32 + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ks = a.ks;
  const int rank = ks > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int mt = blockIdx.x / ks;
  const int rb = blockIdx.y;
  const uint64_t wait_ns = a.wait_ns ? a.wait_ns : kWaitNs;

  if constexpr (MODE != kModeFew) {
    pdl_wait();
    pdl_trigger();
  }
  bool mine = true;  // kModeRank: this tile's 128 tokens have the rank block
  if constexpr (MODE == kModeRank) {
    // words of the 256 tokens around this tile, from the ids; cluster-uniform
    if (warp < 4) {
      uint64_t all;
      const uint64_t w = block_words(a, (mt >> 1) * 256 + warp * 64, lane, all);
      if (lane == 0) {
        words[warp] = w;
        words[4 + warp] = all;
      }
    }
    __syncthreads();
    const uint64_t here = words[(mt & 1) * 2] | words[(mt & 1) * 2 + 1];
    const uint64_t tile = words[0] | words[1] | words[2] | words[3];
    if (a.write_masks && rb == 0 && rank == 0 && threadIdx.x < 2) {
      const int blk = mt * 2 + threadIdx.x;
      if (blk < token_blocks) {
        a.mask64[blk] = words[(mt & 1) * 2 + threadIdx.x];
        a.all64[blk] = words[4 + (mt & 1) * 2 + threadIdx.x];
      }
      if (threadIdx.x == 0 && (mt & 1) == 0) a.mask256[mt >> 1] = tile;
    }
    if (!((tile >> rb) & 1)) return;
    mine = (here >> rb) & 1;
  }
  if constexpr (MODE == kModeGrad) {
    for (int w = warp; w * 32 < token_blocks; w += kThreads / 32) {
      const int blk = w * 32 + lane;
      const uint64_t any = blk < token_blocks ? a.mask64[blk] : 0, all = blk < token_blocks ? a.all64[blk] : 0;
      const uint32_t b = __ballot_sync(0xffffffffu, (any >> rb) & 1);
      const uint32_t m = __ballot_sync(0xffffffffu, ((any & ~all) >> rb) & 1);
      if (lane == 0) {
        bits[w] = b;
        mixed[w] = m;
      }
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kNumBars; ++i) mbar_init(bar0 + 8u * i, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tma_prefetch_desc(&tma_a);
    tma_prefetch_desc(&tma_b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_holder)),
                 "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  auto walk = [&]() {
    KWalk k{};
    if constexpr (MODE == kModeGrad) {
      int count = 0;
      const int n_words = (token_blocks + 31) / 32;
      for (int w = 0; w < n_words; ++w) count += __popc(bits[w]);
      k.bits = bits;
      k.skip = (int)((int64_t)count * rank / ks);
      k.left = (int)((int64_t)count * (rank + 1) / ks) - k.skip;
      k.w = -1;
    } else {
      k.kb = (int)((int64_t)a.kb_total * rank / ks);
      k.end = (int)((int64_t)a.kb_total * (rank + 1) / ks);
      if (MODE == kModeRank && !mine) k.end = k.kb;
      if (MODE == kModeFew) {
        k.pending = a.mask256;
        k.rank = rank;
        k.ks = ks;
      }
    }
    return k;
  };

  // The result's rows follow one another in memory (else its columns do): the partial tile
  // is kept in that order too, for whole sectors between peers and wide stores. With lanes
  // a row apart a cluster of 6 took 9 us to add up 128 x 128, a third of it now.
  const bool by_column = MODE == kModeFew || (MODE == kModeGrad && a.grad_trans);
  bool any = false;  // epilogue: this CTA has a partial tile
  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer ----
      KWalk k = walk();
      int it = 0, kb;
      bool second;
      while (k.next(kb, second)) {
        const int s = it % L::kStages;
        const uint32_t ph = (it / L::kStages) & 1u;
        if (!bounded_wait(empty_bar(s), ph ^ 1u, abort_flag, err, kErrProducer, wait_ns)) break;
        const uint32_t a_dst = sbase + s * L::kStage;
        const uint32_t b_dst = a_dst + L::kABytes;
        mbar_arrive_expect_tx(full_bar(s), L::kStage);
        const CUtensorMap* ma = MODE == kModeFew && second ? &tma_a2 : &tma_a;
        const CUtensorMap* mb = MODE == kModeFew && second ? &tma_b2 : &tma_b;
        if (A_MN) {
          tma_load_2d(a_dst, ma, full_bar(s), mt * 128, kb * 64);
          tma_load_2d(a_dst + 8192, ma, full_bar(s), mt * 128 + 64, kb * 64);
        } else {
          tma_load_2d(a_dst, ma, full_bar(s), kb * 64, mt * 128);
        }
        const int col0 = rb * (MODE == kModeFew ? kFewTile : kRankBlock);
        if (B_MN) tma_load_2d(b_dst, mb, full_bar(s), col0, kb * 64);
        else tma_load_2d(b_dst, mb, full_bar(s), kb * 64, col0);
        ++it;
      }
      // let the copies still in flight land before the CTA may leave (bounded)
      const int n_wait = it < L::kStages ? it : L::kStages;
      for (int i = 1; i <= n_wait; ++i) {
        const int j = it - i;
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(full_bar(j % L::kStages), (j / L::kStages) & 1u) && globaltimer() - t0 < wait_ns) {
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------- MMA issuer ----
    // (kModeGrad: the whole warp, which clears tokens; else one lane)
    if (MODE == kModeGrad || lane == 0) {
      KWalk k = walk();
      int it = 0, kb;
      bool second;
      while (k.next(kb, second)) {
        const int s = it % L::kStages;
        const uint32_t ph = (it / L::kStages) & 1u;
        const uint32_t a_addr = sbase + s * L::kStage;
        const uint32_t b_addr = a_addr + L::kABytes;
        bool ok = bounded_wait(full_bar(s), ph, abort_flag, err, kErrMma, wait_ns);
        if constexpr (MODE == kModeGrad) {
          ok = __all_sync(0xffffffffu, ok);
          if (ok && (mixed[kb >> 5] >> (kb & 31)) & 1) {  // warp-uniform
            // Tokens without an adapter of this rank block, whose row of U or V is 0: their
            // rows of x or dy are cleared, or a NaN in a masked row would reach every sum. A
            // token is a row of 128 bytes in each box; swizzling stays within it. (By the ids
            // it would be a global load for each such block: dA of 2999 x 8960 28 us, 22 so.)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint8_t* row = smem + s * L::kStage + (h * 32 + lane) * 128;
              uint32_t any = 0;
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const uint4 q = *reinterpret_cast<const uint4*>(row + L::kABytes + (c ^ (lane & 7)) * 16);
                any |= q.x | q.y | q.z | q.w;
              }
              if (any == 0) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                  const int at = (c ^ (lane & 7)) * 16;
                  *reinterpret_cast<uint4*>(row + at) = make_uint4(0, 0, 0, 0);
                  *reinterpret_cast<uint4*>(row + 8192 + at) = make_uint4(0, 0, 0, 0);
                }
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
        }
        if (!ok) break;
        if (lane == 0) {
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint64_t ad = A_MN ? smem_desc_sw128(a_addr + kk * 2048, 8192, 1024)
                                     : smem_desc_sw128(a_addr + kk * 32, 16, 1024);
            const uint64_t bd = B_MN ? smem_desc_sw128(b_addr + kk * 2048, 8192, 1024)
                                     : smem_desc_sw128(b_addr + kk * 32, 16, 1024);
            tc_mma_bf16(tmem, ad, bd, kIdesc, (it > 0 || kk > 0) ? 1u : 0u);
          }
          tc_commit(empty_bar(s));
        }
        ++it;
      }
      if (lane != 0) {
      } else if (it > 0) {
        tc_commit(acc_bar);
        // the MMAs are done before TMEM can be freed, also when the epilogue
        // stopped waiting for them (bounded)
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(acc_bar, 0) && globaltimer() - t0 < wait_ns) {
        }
      } else {
        mbar_arrive(acc_bar);
      }
    }
  } else {
    // ------------------------------------------------------ epilogue ----
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    if constexpr (MODE == kModeFew) {
      any = true;  // the run is at least four blocks
      pdl_wait();  // y may be memory that the kernels before this one still used
      pdl_trigger();
    } else {
      KWalk k = walk();
      int kb;
      bool second;
      any = k.next(kb, second);
    }
    bool ok = true;
    if (lane == 0) ok = bounded_wait(acc_bar, 0, abort_flag, err, kErrEpilogue, wait_ns);
    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    tc_fence_after();
    float v[NP];
    if (ok && any) {
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
      __syncwarp();
#pragma unroll
      for (int c = 0; c < NP; c += 16) tmem_ld16_nowait(taddr + c, v + c);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    } else {
#pragma unroll
      for (int c = 0; c < NP; ++c) v[c] = 0.f;
    }
    if (by_column) {
#pragma unroll
      for (int c = 0; c < NP; ++c) part[c * L::kPartStrideT + row] = v[c];
    } else {
      float* prow = part + row * L::kPartStride;
#pragma unroll
      for (int c = 0; c < NP; c += 4)
        *reinterpret_cast<float4*>(prow + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
    }
  }

  // every thread of every CTA of the cluster: the partial tiles are complete
  __syncwarp();
  if (ks > 1) cluster_sync_all();
  else __syncthreads();

  if (!*abort_flag) {
    const uint32_t part_addr = smem_u32(part);
    uint32_t peer[8];
    if (ks > 1) {
#pragma unroll
      for (int p = 0; p < 8; ++p) peer[p] = p < ks ? cluster_addr(part_addr, p) : 0u;
    }
    // partials in rank order, all of them in flight
    auto reduce = [&](int off) {
      if (ks == 1) return *reinterpret_cast<const float4*>(part + off);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f), q[8];
#pragma unroll
      for (int p = 0; p < 8; ++p)
        if (p < ks) q[p] = ld_cluster_f4(peer[p] + off * 4);
#pragma unroll
      for (int p = 0; p < 8; ++p)
        if (p < ks) {
          sum.x += q[p].x;
          sum.y += q[p].y;
          sum.z += q[p].z;
          sum.w += q[p].w;
        }
      return sum;
    };
    if (by_column) {
      // this CTA adds up and writes its share of the columns, a warp one at a time, a lane
      // four rows (rows are a multiple of 8)
      const int r = lane * 4, row = mt * 128 + r;
      const int col0 = rb * (MODE == kModeFew ? kFewTile : kRankBlock);
      const int cols = min(NP, (MODE == kModeFew ? a.tokens : a.rank_cols) - col0);
      const int end = row < a.rows ? cols * (rank + 1) / ks : 0;
      int col = cols * rank / ks + warp;
      if constexpr (MODE == kModeFew) {
        float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (a.bias && col < end)
          b = make_float4(__bfloat162float(a.bias[row]), __bfloat162float(a.bias[row + 1]),
                          __bfloat162float(a.bias[row + 2]), __bfloat162float(a.bias[row + 3]));
#pragma unroll 2
        for (; col < end; col += kThreads / 32) {
          const float4 f = reduce(col * L::kPartStrideT + r);
          *reinterpret_cast<uint2*>(a.y + (int64_t)(col0 + col) * a.ldy + row) =
              pack_bf16x4(make_float4(f.x + b.x, f.y + b.y, f.z + b.z, f.w + b.w));
        }
      } else {
#pragma unroll 2
        for (; col < end; col += kThreads / 32)
          store_grad(a, (int64_t)(col0 + col) * a.rows + row, reduce(col * L::kPartStrideT + r));
      }
    } else {
      // its share of the rows, a thread four columns of every (kThreads / G)-th
      // (rank_cols is a multiple of 8)
      const int r0 = 128 * rank / ks, rs = 128 * (rank + 1) / ks - r0;
      constexpr int G = NP / 4;
      const int col = (int)threadIdx.x % G * 4, c0 = rb * kRankBlock + col;
      const int rows = c0 < a.rank_cols ? min(rs, a.rows - mt * 128 - r0) : 0;
#pragma unroll 2
      for (int i = (int)threadIdx.x / G; i < rows; i += kThreads / G) {
        const int r = r0 + i, row = mt * 128 + r;
        float4 f = reduce(r * L::kPartStride + col);
        const int64_t at = (int64_t)row * a.rank_cols + c0;
        if constexpr (MODE == kModeRank) {
          // 0 outside the token's adapter, whatever the product of the others' columns is
          const int id = adapter_of(a, row);
          const float sc = id < 0 ? 0.f : a.scales[id];
          const int lo = id * a.rank, hi = id < 0 ? lo : lo + a.rank;
          f.x = c0 >= lo && c0 < hi ? f.x * sc : 0.f;
          f.y = c0 + 1 >= lo && c0 + 1 < hi ? f.y * sc : 0.f;
          f.z = c0 + 2 >= lo && c0 + 2 < hi ? f.z * sc : 0.f;
          f.w = c0 + 3 >= lo && c0 + 3 < hi ? f.w * sc : 0.f;
          *reinterpret_cast<uint2*>(a.u + at) = pack_bf16x4(f);
        } else {
          store_grad(a, at, f);
        }
      }
    }
  }

  // peers may still read this CTA's partial tile until here
  tc_fence_before();
  if (ks > 1) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

// U of few tokens: `split` warps a (token, rank column), each its part of k, 16 bytes of x
// and of A's row a lane and step, kFewSteps steps in flight. The projection's kernel streams
// the weights meanwhile, so that each round trip waits behind those: a call of 8 tokens of
// 18944 -> 3584 features took 53 us with one warp a column (48 of them in this kernel, which
// takes 19 alone), 27 so.
constexpr int kFewWarps = 8;
constexpr int kFewSteps = 4;
constexpr int kFewFull = 4096;
__global__ void __launch_bounds__(32 * kFewWarps) few_rank_kernel(const bf16* __restrict__ x, int64_t ldx,
                                                                  const bf16* __restrict__ lora_a, const Args a,
                                                                  int split) {
  __shared__ float parts[kFewWarps];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x, j = (blockIdx.y * kFewWarps + warp) / split;
  const int id = adapter_of(a, t);
  float dot = 0.f;
  if (id >= 0 && j < a.rank) {
    const uint4* row = reinterpret_cast<const uint4*>(lora_a + ((int64_t)id * a.rank + j) * a.k);
    const uint4* xr = reinterpret_cast<const uint4*>(x + (int64_t)t * ldx);
    uint64_t sum = 0;
    const int all = a.k / 8, part = warp % split;
    const int end = all * (part + 1) / split;
    for (int i = all * part / split + lane; i - lane < end; i += 32 * kFewSteps) {
      uint4 u[kFewSteps], v[kFewSteps];
#pragma unroll
      for (int q = 0; q < kFewSteps; ++q) {
        const bool in = i + 32 * q < end;
        u[q] = in ? xr[i + 32 * q] : make_uint4(0, 0, 0, 0);
        v[q] = in ? row[i + 32 * q] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < kFewSteps; ++q) {
        const uint32_t us[4] = {u[q].x, u[q].y, u[q].z, u[q].w}, vs[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
        for (int h = 0; h < 4; ++h)
          sum = f2_fma(f2_pack(__uint_as_float(us[h] << 16), __uint_as_float(us[h] & 0xffff0000u)),
                       f2_pack(__uint_as_float(vs[h] << 16), __uint_as_float(vs[h] & 0xffff0000u)), sum);
      }
    }
    float lo, hi;
    f2_unpack(sum, lo, hi);
    dot = warp_sum(lo + hi);
  }
  if (split > 1) {
    if (lane == 0) parts[warp] = dot;
    __syncthreads();
    if (warp % split == 0)
      for (int p = 1; p < split; ++p) dot += parts[warp + p];
  }
  if (id >= 0 && j < a.rank && warp % split == 0 && lane == 0)
    a.u[(int64_t)t * a.rank_cols + id * a.rank + j] = __float2bfloat16_rn(dot * a.scales[id]);
  if (blockIdx.y != 0 || warp != 0) return;
  // the word of all tokens, and 0 in its blocks' columns of other adapters
  uint64_t word = 0;
  for (int b = 0; b * 64 < a.tokens; ++b) {
    uint64_t all;
    const uint64_t w = block_words(a, b * 64, lane, all);
    if (t == 0 && lane == 0) {
      a.mask64[b] = w;
      a.all64[b] = all;
    }
    word |= w;
  }
  if (t == 0 && lane == 0) a.mask256[0] = word;
  const int own0 = id * a.rank, own1 = id < 0 ? own0 : own0 + a.rank;
  bf16* u = a.u + (int64_t)t * a.rank_cols;
  for (uint64_t w = word; w; w &= w - 1) {
    const int c0 = (__ffsll((long long)w) - 1) * kRankBlock;
#pragma unroll
    for (int c = c0 + lane; c < c0 + kRankBlock; c += 32)
      if (c < a.rank_cols && (c < own0 || c >= own1)) u[c] = __float2bfloat16_rn(0.f);
  }
}

// ------------------------------------------------------------------- host --
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::lock_guard<std::mutex> lock(cache_mutex());
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// bf16 matrix [outer, inner] with row stride ld: box {64, box_outer}, 128-byte
// swizzle, zero fill out of bounds.
int map2d(CUtensorMap* map, const void* ptr, int64_t inner, int64_t outer, int64_t ld, int box_outer) {
  auto fn = encode_fn();
  if (!fn) {
    set_last_error("cuTensorMapEncodeTiled is not available from the driver");
    return SOUP_ERR_CUDA;
  }
  if (int rc = bind_context()) return rc;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled failed for an adapter operand");
    return SOUP_ERR_UNSUPPORTED;
  }
  return SOUP_OK;
}

// `busy`: clusters of the grid that have work, as far as the host can tell. The k
// range is split until one wave of two CTAs an SM is full, at least four k blocks each;
// into more than four parts only where each has sixteen blocks, eight at most: peers add up
// and place slower than they save (8 tokens of 1536 columns: 8960 features 17.7 us split
// four ways, 12.2 eight; 4096 x 4096 13.8 and 14.8).
template <int MODE, bool B_MN, int NP>
int launch(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& ma2, const CUtensorMap& mb2, Args args,
           int k_blocks, int rank_blocks, int busy, cudaStream_t stream) {
  using L = Smem<NP>;
  auto kern = rank_tile_kernel<MODE, B_MN, NP>;
  constexpr int kMost = 110 * 1024;  // two CTAs an SM
  static_assert(L::kBytesFor(kMaxTokens / 64) <= kMost, "shared memory of a CTA");
  static bool attr_done[64] = {false};
  static int max_clusters[64][9] = {};  // by cluster size; -1: none fits
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cuda_status(cudaErrorInvalidDevice);
  int* err = device_err_ptr();
  if (!err) {
    set_last_error("device error word unavailable");
    return SOUP_ERR_CUDA;
  }
  const int sms = num_sms();
  const int m_tiles = (args.rows + 127) / 128;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kBytesFor(MODE == kModeGrad ? (args.tokens + 63) / 64 : 0);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  {
    std::lock_guard<std::mutex> lock(cache_mutex());
    if (!attr_done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
      if (e != cudaSuccess) return cuda_status(e);
      attr_done[dev] = true;
    }
  }
  int ks = 2 * sms / (busy > 0 ? busy : 1);
  const int most = k_blocks >= 128 ? 8 : k_blocks >= 80 ? k_blocks / 16 : 4;
  if (ks > most) ks = most;
  if (ks > k_blocks / 4) ks = k_blocks / 4;
  if (ks < 1) ks = 1;
  for (; ks > 1; --ks) {
    std::lock_guard<std::mutex> lock(cache_mutex());
    if (max_clusters[dev][ks] == 0) {
      int n = 0;
      attr[0].val.clusterDim.x = ks;
      cfg.gridDim = dim3(ks * (sms / ks));
      const size_t bytes = cfg.dynamicSmemBytes;
      cfg.dynamicSmemBytes = kMost;
      cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
      cfg.dynamicSmemBytes = bytes;
      if (e != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      max_clusters[dev][ks] = n > 0 ? n : -1;
    }
    if (max_clusters[dev][ks] > 0) break;
  }
  args.ks = ks;
  attr[0].val.clusterDim.x = ks;
  cfg.gridDim = dim3(m_tiles * ks, rank_blocks);
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, ma, mb, ma2, mb2, args, err));
}

struct Layout {
  int64_t mask64, all64, mask256, u, bytes;  // byte offsets into the state
};
Layout layout_of(int64_t tokens, int64_t rank_cols) {
  Layout l;
  l.mask64 = 0;
  l.all64 = (tokens + 63) / 64 * 8;
  l.mask256 = (2 * l.all64 + 15) / 16 * 16;
  l.u = l.mask256 + ((tokens + 255) / 256 * 8 + 127) / 128 * 128;
  l.u = (l.u + 127) / 128 * 128;
  l.bytes = l.u + tokens * rank_cols * 2;
  return l;
}

bool operand_ok(const void* p, int64_t ld) { return aligned16(p) && ld > 0 && (ld * 2) % 16 == 0; }

int check_sizes(const char* fn, int64_t tokens, int64_t n, int64_t k, int64_t adapters, int64_t rank, int64_t per) {
  char msg[160];
  if (tokens <= 0 || tokens > kMaxTokens || n <= 0 || k <= 0 || n > (1 << 24) || k > (1 << 24) || adapters <= 0 ||
      rank <= 0 || per <= 0 || adapters > kMaxRank || rank > kMaxRank || adapters * rank > kMaxRank) {
    snprintf(msg, sizeof(msg), "%s: bad sizes (at most %d tokens, adapters x rank at most %d)", fn, kMaxTokens,
             kMaxRank);
    set_last_error(msg);
    return SOUP_ERR_INVALID;
  }
  if (n % 8 || k % 8 || adapters * rank % 8) {
    snprintf(msg, sizeof(msg), "%s: widths and adapters x rank must be multiples of 8", fn);
    set_last_error(msg);
    return SOUP_ERR_UNSUPPORTED;
  }
  return SOUP_OK;
}

// U = mask(x A^T) [tokens, R], or V = mask(dy B): `large` [tokens, k] against the factor.
int rank_product(const void* large, int64_t ld, int64_t k, const void* factor, bool factor_mn, const Args& base,
                 bf16* out, bool write_masks, cudaStream_t st) {
  Args a = base;
  a.rows = base.tokens;
  a.k = (int)k;
  a.kb_total = (int)((k + 63) / 64);
  a.u = out;
  a.write_masks = write_masks ? 1 : 0;
  const int blocks = (a.rank_cols + kRankBlock - 1) / kRankBlock;
  CUtensorMap ma, mb;
  int rc;
  if ((rc = map2d(&ma, large, k, a.tokens, ld, 128))) return rc;
  if ((rc = factor_mn ? map2d(&mb, factor, a.rank_cols, k, a.rank_cols, 64) : map2d(&mb, factor, k, a.rank_cols, k, 64)))
    return rc;
  // few tokens may each have a rank block of their own, many lie in runs of one
  const int tiles = (a.tokens + 127) / 128;
  const int busy = tiles < 4 ? tiles * blocks : tiles * (blocks < 2 ? blocks : 2);
  return factor_mn ? launch<kModeRank, true, 64>(ma, mb, ma, mb, a, a.kb_total, blocks, busy, st)
                   : launch<kModeRank, false, 64>(ma, mb, ma, mb, a, a.kb_total, blocks, busy, st);
}

// dB = dy^T U [n, R], or dA = (x^T V)^T [R, k].
int grad_product(const void* large, int64_t ld, int64_t features, const void* u, const Args& base, void* grad,
                 bool f32, bool trans, cudaStream_t st) {
  Args a = base;
  a.rows = (int)features;
  a.k = base.tokens;
  a.grad = grad;
  a.grad_f32 = f32 ? 1 : 0;
  a.grad_trans = trans ? 1 : 0;
  const int blocks = (a.rank_cols + kRankBlock - 1) / kRankBlock;
  CUtensorMap ma, mb;
  int rc;
  if ((rc = map2d(&ma, large, features, a.tokens, ld, 64))) return rc;
  if ((rc = map2d(&mb, u, a.rank_cols, a.tokens, a.rank_cols, 64))) return rc;
  const int tiles = (a.rows + 127) / 128;
  const int token_blocks = (a.tokens + 63) / 64;
  return launch<kModeGrad, true, 64>(ma, mb, ma, mb, a, token_blocks, blocks, tiles * (blocks < 4 ? blocks : 4), st);
}

template <int NP>
int few_product(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* lora_b, int64_t n, int64_t k,
                const bf16* u, const Args& base, cudaStream_t st) {
  Args a = base;
  a.rows = (int)n;
  a.k = (int)k;
  a.kb_total = (int)((k + 63) / 64);
  CUtensorMap ma, mb, ma2, mb2;
  int rc;
  if ((rc = map2d(&ma, w, k, n, ldw, 128))) return rc;
  if ((rc = map2d(&mb, x, k, a.tokens, ldx, NP))) return rc;
  if ((rc = map2d(&ma2, lora_b, a.rank_cols, n, a.rank_cols, 128))) return rc;
  if ((rc = map2d(&mb2, u, a.rank_cols, a.tokens, a.rank_cols, NP))) return rc;
  const int token_tiles = (a.tokens + kFewTile - 1) / kFewTile;
  return launch<kModeFew, false, NP>(ma, mb, ma2, mb2, a, a.kb_total, token_tiles, (a.rows + 127) / 128 * token_tiles,
                                     st);
}

Args base_args(const void* ids, int ids_64, int64_t per, const float* scales, int64_t tokens, int64_t adapters,
               int64_t rank, uint8_t* state, const Layout& l) {
  Args a{};
  a.tokens = (int)tokens;
  a.adapters = (int)adapters;
  a.rank = (int)rank;
  a.rank_cols = (int)(adapters * rank);
  a.wait_ns = wait_limit_ns();
  a.ids = ids;
  a.ids_64 = ids_64;
  a.per = (int)(per > tokens ? tokens : per);
  a.scales = scales;
  a.mask64 = reinterpret_cast<uint64_t*>(state + l.mask64);
  a.all64 = reinterpret_cast<uint64_t*>(state + l.all64);
  a.mask256 = reinterpret_cast<uint64_t*>(state + l.mask256);
  return a;
}

}  // namespace
}  // namespace soup

using namespace soup;

extern "C" {

size_t soup_multi_lora_state_bytes(int64_t tokens, int64_t adapters, int64_t rank) {
  if (tokens <= 0 || adapters <= 0 || rank <= 0) return 0;
  return (size_t)layout_of(tokens, adapters * rank).bytes;
}

int soup_multi_lora_fwd(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias,
                        const void* lora_a, const void* lora_b, const float* scales, const void* ids, int ids_64,
                        int64_t tokens_per_id, int64_t tokens, int64_t n, int64_t k, int64_t adapters, int64_t rank,
                        void* y, int64_t ldy, void* state, size_t state_bytes, void* stream) {
  const char* fn = "soup_multi_lora_fwd";
  if (int rc = check_sizes(fn, tokens, n, k, adapters, rank, tokens_per_id)) return rc;
  if (!x || !weight || !lora_a || !lora_b || !scales || !ids || !y || ldx < k || ldw < k || ldy < n) {
    set_last_error("soup_multi_lora_fwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (!operand_ok(x, ldx) || !operand_ok(weight, ldw) || !aligned16(lora_a) || !aligned16(lora_b) ||
      !operand_ok(y, ldy)) {
    set_last_error("soup_multi_lora_fwd: operands need 16-byte aligned rows");
    return SOUP_ERR_UNSUPPORTED;
  }
  const Layout l = layout_of(tokens, adapters * rank);
  if (!state || !aligned16(state) || state_bytes < (size_t)l.bytes) {
    set_last_error("soup_multi_lora_fwd: state missing, unaligned or too small");
    return SOUP_ERR_WORKSPACE;
  }
  uint8_t* s = static_cast<uint8_t*>(state);
  Args a = base_args(ids, ids_64, tokens_per_id, scales, tokens, adapters, rank, s, l);
  bf16* u = reinterpret_cast<bf16*>(s + l.u);
  cudaStream_t st = as_stream(stream);
  // up to 128 tokens always; up to 256 where the 256-row tiles of the pair GEMM would leave
  // half of the SMs idle (256 tokens: 3584 -> 3584 features 24.5 us and 35.4 by that, 1536 ->
  // 8960 21.3 and 23.9, 3584 -> 18944 46.4 and 40.1)
  if (tokens <= kFewTile || (tokens <= kFewTokens && (n + 255) / 256 * 2 < num_sms())) {
    a.k = (int)k;
    a.u = u;
    // warps a rank column: until one round of loads is all, or as many warps as the SMs hold
    int split = 1;
    while (split < kFewWarps && k > (int64_t)split * kFewSteps * 256 && tokens * a.rank * split < kFewFull) split *= 2;
    const int columns = kFewWarps / split;
    if (int rc = cuda_status(launch_pdl(few_rank_kernel, dim3((unsigned)tokens, (a.rank + columns - 1) / columns),
                                        dim3(32 * kFewWarps), 0, st, static_cast<const bf16*>(x), ldx,
                                        static_cast<const bf16*>(lora_a), a, split)))
      return rc;
    a.y = static_cast<bf16*>(y);
    a.ldy = ldy;
    a.bias = static_cast<const bf16*>(bias);
    if (tokens <= 16) return few_product<16>(x, ldx, weight, ldw, lora_b, n, k, u, a, st);
    if (tokens <= 32) return few_product<32>(x, ldx, weight, ldw, lora_b, n, k, u, a, st);
    if (tokens <= 64) return few_product<64>(x, ldx, weight, ldw, lora_b, n, k, u, a, st);
    return few_product<128>(x, ldx, weight, ldw, lora_b, n, k, u, a, st);
  }
  if (int rc = rank_product(x, ldx, k, lora_a, false, a, u, true, st)) return rc;
  return gemm_bf16_masked_k2(x, ldx, weight, ldw, false, u, a.rank_cols, lora_b, a.rank_cols, a.rank_cols, a.mask256,
                             bias, y, ldy, tokens, n, k, st);
}

size_t soup_multi_lora_bwd_workspace_bytes(int64_t tokens, int64_t adapters, int64_t rank) {
  if (tokens <= 0 || adapters <= 0 || rank <= 0) return 0;
  return (size_t)(tokens * adapters * rank * 2);
}

int soup_multi_lora_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight, int64_t ldw,
                        const void* lora_a, const void* lora_b, const float* scales, const void* ids, int ids_64,
                        int64_t tokens_per_id, int64_t tokens, int64_t n, int64_t k, int64_t adapters, int64_t rank,
                        const void* state, size_t state_bytes, void* dx, int64_t lddx, void* da, int da_dtype,
                        void* db, int db_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "soup_multi_lora_bwd";
  if (int rc = check_sizes(fn, tokens, n, k, adapters, rank, tokens_per_id)) return rc;
  auto grad_ok = [](void* p, int dt) { return !p || dt == SOUP_F32 || dt == SOUP_BF16; };
  if (!dy || !weight || !lora_a || !lora_b || !scales || !ids || lddy < n || ldw < k || (dx && lddx < k) ||
      (da && (!x || ldx < k)) || !grad_ok(da, da_dtype) || !grad_ok(db, db_dtype)) {
    set_last_error("soup_multi_lora_bwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (!operand_ok(dy, lddy) || !operand_ok(weight, ldw) || (da && !operand_ok(x, ldx)) ||
      (dx && !operand_ok(dx, lddx)) || !aligned16(lora_a) || !aligned16(lora_b) || !aligned16(da) || !aligned16(db)) {
    set_last_error("soup_multi_lora_bwd: operands need 16-byte aligned rows");
    return SOUP_ERR_UNSUPPORTED;
  }
  const Layout l = layout_of(tokens, adapters * rank);
  if (!state || !aligned16(state) || state_bytes < (size_t)l.bytes) {
    set_last_error("soup_multi_lora_bwd: state missing, unaligned or too small");
    return SOUP_ERR_WORKSPACE;
  }
  if ((dx || da) && (!workspace || !aligned16(workspace) ||
                     workspace_bytes < soup_multi_lora_bwd_workspace_bytes(tokens, adapters, rank))) {
    set_last_error("soup_multi_lora_bwd: workspace missing, unaligned or too small");
    return SOUP_ERR_WORKSPACE;
  }
  uint8_t* s = static_cast<uint8_t*>(const_cast<void*>(state));
  const Args a = base_args(ids, ids_64, tokens_per_id, scales, tokens, adapters, rank, s, l);
  const bf16* u = reinterpret_cast<const bf16*>(s + l.u);
  bf16* v = static_cast<bf16*>(workspace);
  cudaStream_t st = as_stream(stream);
  int rc;
  if (dx || da)
    if ((rc = rank_product(dy, lddy, n, lora_b, true, a, v, false, st))) return rc;
  if (dx)
    if ((rc = gemm_bf16_masked_k2(dy, lddy, weight, ldw, true, v, a.rank_cols, lora_a, k, a.rank_cols, a.mask256,
                                  nullptr, dx, lddx, tokens, k, n, st)))
      return rc;
  if (da)
    if ((rc = grad_product(x, ldx, k, v, a, da, da_dtype == SOUP_F32, true, st))) return rc;
  if (db)
    if ((rc = grad_product(dy, lddy, n, u, a, db, db_dtype == SOUP_F32, false, st))) return rc;
  return SOUP_OK;
}

}  // extern "C"
