// Pieces shared by the attention kernels (attention.cu, attention_window.cu): TMA
// tile loads, TMEM loads and stores, operand descriptors, the backward's row dot
// products and the tensor maps.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include <stdio.h>

#include <mutex>

#include "soup_common.cuh"
#include "tc_gemm.cuh"

namespace soup {
namespace attn {

using bf16 = __nv_bfloat16;
using tc::bounded_wait;
using tc::mbar_arrive;
using tc::mbar_arrive_expect_tx;
using tc::mbar_init;
using tc::mbar_try_wait;
using tc::smem_desc_sw128;
using tc::smem_u32;
using tc::tc_commit;
using tc::tc_fence_after;
using tc::tc_fence_before;
using tc::tc_mma_bf16;
using tc::tmem_ld32;

constexpr int kHeadDim = 128;
constexpr int kTile = 128;             // query rows per CTA and keys per tile
constexpr int kBox = kTile * 128;      // one [128 rows x 64 cols] bf16 box: 16 KB
constexpr int kTileBytes = 2 * kBox;   // a 128 x 128 bf16 tile (two 64-column boxes)

constexpr int kErrAttnProducer = 0x111;
constexpr int kErrAttnMma = 0x112;
constexpr int kErrAttnSoftmax = 0x113;
constexpr int kErrAttnSmem = 0x114;  // dynamic shared memory too small after 1 KB alignment

// 4-D TMA tile load (coordinates innermost first) into this CTA's shared memory.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int32_t c0, int32_t c1, int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// 32 lanes x 32 consecutive fp32 columns from registers into TMEM (the
// inverse of tmem_ld32); the caller waits with tmem_st_wait.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
      "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
      "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])), "r"(__float_as_uint(v[8])),
      "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
      "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])),
      "r"(__float_as_uint(v[15])), "r"(__float_as_uint(v[16])), "r"(__float_as_uint(v[17])),
      "r"(__float_as_uint(v[18])), "r"(__float_as_uint(v[19])), "r"(__float_as_uint(v[20])),
      "r"(__float_as_uint(v[21])), "r"(__float_as_uint(v[22])), "r"(__float_as_uint(v[23])),
      "r"(__float_as_uint(v[24])), "r"(__float_as_uint(v[25])), "r"(__float_as_uint(v[26])),
      "r"(__float_as_uint(v[27])), "r"(__float_as_uint(v[28])), "r"(__float_as_uint(v[29])),
      "r"(__float_as_uint(v[30])), "r"(__float_as_uint(v[31]))
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 32 lanes x 32 fp32 columns from TMEM without waiting: several loads are
// issued back to back and completed by one tmem_ld_wait (the registers may
// not be read before it).
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t dynamic_smem_bytes() {
  uint32_t v;
  asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(v));
  return v;
}
// One bool from lane 0 to the warp.
__device__ __forceinline__ bool warp_ok(bool v) { return __shfl_sync(0xffffffffu, v ? 1 : 0, 0) != 0; }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// K-major operand tile of 128 rows x 128 bf16 columns in shared memory: two
// 16 KB boxes (columns 0-63, 64-127), rows of 128 B, 128-byte swizzle. The
// descriptor of k-step kk (16 columns) for tcgen05.mma.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t base, int kk) {
  return smem_desc_sw128(base + (kk >> 2) * kBox + (kk & 3) * 32, 16, 1024);
}
// The same bytes read as an MN-major operand whose MN dimension is the tile's
// 128 columns and whose K dimension is its 128 rows: k-step kk covers rows
// [16 kk, 16 kk + 16); the two 64-column boxes are the MN atoms (LBO 16 KB).
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t base, int kk) {
  return smem_desc_sw128(base + kk * 2048, kBox, 1024);
}

// Byte offset of the 16-byte chunk c (columns 8c..8c+7 of a 64-column box) of
// row r in a 128-byte-swizzled box: the layout TMA writes and the descriptors read.
__device__ __forceinline__ uint32_t swz_off(int r, int c) {
  return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4));
}

// Instruction descriptors (fp32 accumulate, bf16 operands, M = N = 128).
constexpr uint32_t kIdescKK = tc::idesc_bf16(128, false, false, 128);  // A, B K-major
constexpr uint32_t kIdescKM = tc::idesc_bf16(128, false, true, 128);   // B MN-major

// D (TMEM) [+]= A (TMEM, M rows in lanes, two bf16 of K per 32-bit column) x B (smem descriptor).
__device__ __forceinline__ void tc_mma_bf16_tmem_a(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                                   uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 32 consecutive 32-bit columns from registers into TMEM.
__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t (&v)[32]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns from TMEM (waits for the load).
__device__ __forceinline__ void tmem_ld16u(uint32_t taddr, uint32_t (&v)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns from registers into TMEM.
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15])
      : "memory");
}

// ------------------------------------------------------------ backward ----
constexpr int kQStep = 64;                 // queries per dK / dV step
constexpr int kStepBox = kQStep * 128;     // a [64 rows x 64 cols] bf16 box: 8 KB
constexpr int kStepTile = 2 * kStepBox;    // a 64 x 128 bf16 tile: 16 KB
constexpr int kPTBytes = kTile * 128;      // P^T / dS^T: 128 rows x 64 bf16 = 16 KB

// D[b, h, q] = sum_d dO[b, q, h, d] * O[b, q, h, d] (fp32) and nl2[b, h, q] =
// -lse[b, h, q] * log2(e) (the exponent offset of P in base 2); rows padded
// like lse ([B, H, S_pad]). dO and O are [B, S, H, D] contiguous. Sixteen lanes
// per row (16 bytes each), rows taken in the output's (b, h, q) order so the
// stores are contiguous, four rows per half-warp with all loads issued first.
constexpr int kDotRows = 4;
static __global__ void __launch_bounds__(256) attn_bwd_dot_kernel(const bf16* __restrict__ dO,
                                                           const bf16* __restrict__ O,
                                                           const float* __restrict__ lse, int B,
                                                           int H, int S, float* __restrict__ Dv,
                                                           float* __restrict__ nl2) {
  pdl_wait();
  pdl_trigger();
  const int64_t nrows = (int64_t)B * H * S;
  const int sub = threadIdx.x & 15;
  const int64_t half = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4;
  const int64_t nhalves = ((int64_t)gridDim.x * blockDim.x) >> 4;
  const int64_t s_pad = (int64_t)(S + kTile - 1) / kTile * kTile;
  for (int64_t base = half * kDotRows; base < nrows; base += nhalves * kDotRows) {
    uint4 a[kDotRows], c[kDotRows];
#pragma unroll
    for (int u = 0; u < kDotRows; ++u) {
      const int64_t i = base + u;  // (b, h, q) row-major
      if (i < nrows) {
        const int q = (int)(i % S);
        const int64_t bh = i / S;
        const int h = (int)(bh % H), b = (int)(bh / H);
        const int64_t row = ((int64_t)b * S + q) * H + h;
        a[u] = *reinterpret_cast<const uint4*>(dO + row * kHeadDim + sub * 8);
        c[u] = *reinterpret_cast<const uint4*>(O + row * kHeadDim + sub * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < kDotRows; ++u) {
      const int64_t i = base + u;
      const __nv_bfloat162* ap = reinterpret_cast<const __nv_bfloat162*>(&a[u]);
      const __nv_bfloat162* cp = reinterpret_cast<const __nv_bfloat162*>(&c[u]);
      float acc = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = __bfloat1622float2(ap[e]), y = __bfloat1622float2(cp[e]);
        acc = fmaf(x.x, y.x, fmaf(x.y, y.y, acc));
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      if (sub == 0 && i < nrows) {
        const int q = (int)(i % S);
        const int64_t v = (i / S) * s_pad + q;
        Dv[v] = acc;
        nl2[v] = -lse[v] * kLog2e;
      }
    }
  }
}

// Descriptors of a 64-row step tile (two 8 KB boxes of 64 columns): as a K-major
// operand with N = 64 rows (k-step kk: 16 columns), and as an MN-major operand
// whose K dimension is its 64 rows (k-step kk: rows 16 kk..16 kk + 15; LBO 8 KB).
__device__ __forceinline__ uint64_t desc_kmajor64(uint32_t base, int kk) {
  return smem_desc_sw128(base + (kk >> 2) * kStepBox + (kk & 3) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t desc_mnmajor64(uint32_t base, int kk) {
  return smem_desc_sw128(base + kk * 2048, kStepBox, 1024);
}
// P^T / dS^T (128 rows x 64 columns, one box) as the K-major A operand.
__device__ __forceinline__ uint64_t desc_kmajor_box(uint32_t base, int kk) {
  return smem_desc_sw128(base + kk * 32, 16, 1024);
}
constexpr uint32_t kIdescKK64 = tc::idesc_bf16(64, false, false, 128);  // M 128, N 64

// Untiled bulk copy global -> this CTA's shared memory (16-byte aligned
// addresses, size a multiple of 16), completing on an mbarrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}

// ----------------------------------------------------------------- host ----
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::lock_guard<std::mutex> lock(cache_mutex());
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// 4-D map over a bf16 [B, heads, S, D] tensor with element strides (b, h, s)
// and a contiguous last dimension: dims {D, S, heads, B}, box {64, 128, 1, 1},
// 128-byte swizzle, zero fill outside.
static int make_bhsd_map(CUtensorMap* map, const void* ptr, const int64_t* strides, int64_t B,
                         int64_t heads, int64_t S, const char* what, int box_rows = kTile) {
  auto fn = encode_fn();
  if (!fn) {
    set_last_error("cuTensorMapEncodeTiled is not available from the driver");
    return SOUP_ERR_CUDA;
  }
  if (int rc = bind_context()) return rc;
  cuuint64_t dims[4] = {(cuuint64_t)kHeadDim, (cuuint64_t)S, (cuuint64_t)heads, (cuuint64_t)B};
  cuuint64_t gstr[3] = {(cuuint64_t)strides[2] * 2, (cuuint64_t)strides[1] * 2,
                        (cuuint64_t)strides[0] * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, gstr, box,
                  estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    char msg[200];
    snprintf(msg, sizeof(msg), "attention: cuTensorMapEncodeTiled failed (%d) for %s", (int)r, what);
    set_last_error(msg);
    return SOUP_ERR_UNSUPPORTED;
  }
  return SOUP_OK;
}

// Strides of a [B, heads, S, 128] bf16 operand usable by TMA: 16-byte aligned
// base, every stride a multiple of 8 elements.
static bool bhsd_ok(const void* p, const int64_t* st) {
  return p && aligned16(p) && st && st[0] > 0 && st[1] > 0 && st[2] > 0 && st[0] % 8 == 0 &&
         st[1] % 8 == 0 && st[2] % 8 == 0;
}

template <typename K>
static int set_smem(K kern, int bytes, bool* done) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cuda_status(cudaErrorInvalidDevice);
  std::lock_guard<std::mutex> lock(cache_mutex());
  if (!done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return cuda_status(e);
    done[dev] = true;
  }
  return SOUP_OK;
}

}  // namespace attn
}  // namespace soup
