// Losses over per-token log-probabilities: the paired log-ratio (preference)
// loss and the clipped importance-ratio (policy) loss with a KL term, forward
// and backward.
//
// Both are masked reductions over [sequences, tokens] fp32 arrays: a first
// kernel sums each sequence (one block per sequence and chunk of tokens) into
// one record per block, a second, one block, joins the records in a fixed
// order (no atomics: the same inputs give the same bits) and writes the loss,
// the metrics and one gradient factor per sequence; when the blocks fit a
// cluster, one launch does both. The backward is one elementwise pass. Labels equal to
// ignore_index mark masked tokens: their values are selected away, never multiplied, so
// infinities and NaN there do not reach a sum. Sums over tokens run in 64 bits: thousands of terms of
// either sign leave a difference that 32 bits would round away, and the adds
// are free beside the loads.
#include "soup_common.cuh"

namespace soup {
namespace {

constexpr int kThreads = 256;
// Tokens per block of the summing kernels: forward of the policy loss over 2 x 16384 tokens
// 8.5 us (4096: 11.1, 1024: 7.1), over 2048 x 2048 25.3 us (4096: 25.9, 1024: 31.8).
constexpr int kChunk = 2048;
constexpr int kUnroll = 4;    // tokens per thread whose loads are in flight together

// v[i] = its sum over the block, in every thread; sh: N doubles a warp. At most 32 warps.
template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (lane == 0) sh[warp * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lane < warps ? sh[lane * N + i] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  __syncthreads();
}

// Few blocks (the usual step: a handful of sequences) sum and join in one launch: the
// blocks form one cluster, whose first block joins the records after a cluster barrier.
// 4 x 512 tokens, in a graph: preference 3.3 us against 3.7 with two launches, policy 3.9
// against 7.5; eager calls save the launch (3 us of host time).
constexpr int kClusterBlocks = 8;
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), unsigned blocks, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = blocks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// ------------------------------------------------------------ preference ----
struct PrefArgs {
  const float* logps;
  int64_t lp_ld;
  const float* ref;  // [2P, S] per token, or [2P] sums, or nullptr
  int64_t ref_ld;
  int ref_mode;
  const int64_t* labels;
  int64_t lab_ld;
  int64_t pairs, seq;
  int64_t ignore;
  double beta, smoothing;
  int loss_type;
};

// records[n][c] = (sum of log ratios, labelled tokens) of sequence n, chunk c
__device__ __forceinline__ void pref_sum(const PrefArgs& a, int chunks, double2* records) {
  __shared__ double sh[2 * kThreads / 32];
  const int64_t n = blockIdx.x / chunks;
  const int c = blockIdx.x % chunks;
  const int64_t s0 = (int64_t)c * kChunk;
  const int64_t s1 = s0 + kChunk < a.seq ? s0 + kChunk : a.seq;
  const float* lp = a.logps + n * a.lp_ld;
  const float* rf = a.ref_mode == 1 ? a.ref + n * a.ref_ld : nullptr;
  const int64_t* lab = a.labels + n * a.lab_ld;
  double sum = 0.0;
  int cnt = 0;
  for (int64_t i = s0 + threadIdx.x; i < s1; i += kThreads * kUnroll) {
    int64_t t[kUnroll];
    float x[kUnroll], r[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t j = i + u * kThreads;
      const bool in = j < s1;
      t[u] = in ? lab[j] : a.ignore;
      x[u] = in ? lp[j] : 0.f;
      r[u] = in && rf ? rf[j] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (t[u] != a.ignore) {
        sum += (double)x[u] - (double)r[u];
        ++cnt;
      }
    }
  }
  double v[2] = {sum, (double)cnt};
  block_sums(v, sh);
  if (threadIdx.x == 0) records[blockIdx.x] = make_double2(v[0], v[1]);
}

// Per pair p: h = score(chosen) - score(rejected), the loss and dL/dh; then the
// mean loss. rewards[n] = beta * log ratio, coef[n] = dL/d(log prob of a
// labelled token of sequence n). softplus(x) = max(x, 0) + log1p(exp(-|x|)). In
// 64 bits: label smoothing subtracts nearly equal terms, and one thread does one
// pair, so the wider arithmetic hides behind the launch.
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

__device__ __forceinline__ void pref_join(const PrefArgs& a, int chunks, const double2* records,
                                          float* loss, float* rewards, float* coef) {
  __shared__ double sh[kThreads / 32];
  double total = 0.0;
  for (int64_t p = threadIdx.x; p < a.pairs; p += kThreads) {
    double d[2], per[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int64_t n = p + w * a.pairs;
      double sum = 0.0, cnt = 0.0;
      for (int c = 0; c < chunks; ++c) {
        const double2 r = __ldcg(records + n * chunks + c);  // another block's writes
        sum += r.x;
        cnt += r.y;
      }
      if (a.ref_mode == 2) sum -= (double)a.ref[n];
      d[w] = sum;
      per[w] = cnt > 1.0 ? 1.0 / cnt : 1.0;
      rewards[n] = (float)(a.beta * sum);
    }
    const bool ipo = a.loss_type == SOUP_PREF_IPO;
    const double h = ipo ? d[0] * per[0] - d[1] * per[1] : d[0] - d[1];
    const double bh = a.beta * h;
    double l, g;
    if (a.loss_type == SOUP_PREF_SIGMOID) {
      // dL/dh = -beta ((1 - e) sigmoid(-bh) - e sigmoid(bh)) = -beta (sigmoid(-bh) - e)
      l = (1.0 - a.smoothing) * softplus(-bh) + (a.smoothing > 0.0 ? a.smoothing * softplus(bh) : 0.0);
      g = -a.beta * (1.0 / (1.0 + exp(bh)) - a.smoothing);
    } else if (a.loss_type == SOUP_PREF_HINGE) {
      // the comparisons are written so that a NaN margin stays NaN
      const double m = 1.0 - bh;
      l = m < 0.0 ? 0.0 : m;
      g = m <= 0.0 ? 0.0 : m == m ? -a.beta : m;
    } else {
      const double t = h - 0.5 / a.beta;
      l = t * t;
      g = 2.0 * t;
    }
    total += l;
    g /= (double)a.pairs;
    coef[p] = (float)(ipo ? g * per[0] : g);
    coef[p + a.pairs] = (float)(ipo ? -g * per[1] : -g);
  }
  double v[1] = {total};
  block_sums(v, sh);
  if (threadIdx.x == 0) loss[0] = (float)(v[0] / (double)a.pairs);
}

__global__ void __launch_bounds__(kThreads) pref_sum_kernel(PrefArgs a, int chunks, double2* records) {
  pdl_wait();
  pdl_trigger();
  pref_sum(a, chunks, records);
}
__global__ void __launch_bounds__(kThreads) pref_join_kernel(PrefArgs a, int chunks,
                                                             const double2* records, float* loss,
                                                             float* rewards, float* coef) {
  pdl_wait();
  pdl_trigger();
  pref_join(a, chunks, records, loss, rewards, coef);
}
__global__ void __launch_bounds__(kThreads) pref_cluster_kernel(PrefArgs a, int chunks, double2* records,
                                                                float* loss, float* rewards, float* coef) {
  pdl_wait();
  pdl_trigger();
  pref_sum(a, chunks, records);
  cluster_sync();
  if (blockIdx.x == 0) pref_join(a, chunks, records, loss, rewards, coef);
}

// dlogps[n, s] = labelled ? grad_loss * factor[n] * (per_token ? tok[n, s] : 1) : 0
// (tok may be dlogps itself)
__global__ void __launch_bounds__(kThreads) loss_bwd_kernel(const float* __restrict__ grad_loss,
                                                            const float* __restrict__ factor,
                                                            const float* tok,
                                                            const int64_t* __restrict__ labels,
                                                            int64_t lab_ld, int64_t seq, int chunks,
                                                            int64_t ignore, float* dlogps) {
  pdl_wait();
  pdl_trigger();
  const int64_t n = blockIdx.x / chunks;
  const int64_t s0 = (int64_t)(blockIdx.x % chunks) * kChunk;
  const int64_t s1 = s0 + kChunk < seq ? s0 + kChunk : seq;
  const float f = grad_loss[0] * factor[n];
  float* out = dlogps + n * seq;
  const float* tk = tok ? tok + n * seq : nullptr;
  const int64_t* lab = labels ? labels + n * lab_ld : nullptr;
  for (int64_t i = s0 + threadIdx.x; i < s1; i += kThreads * kUnroll) {
    float v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t j = i + u * kThreads;
      if (j >= s1) break;
      if (tk) {
        const float t = tk[j];
        v[u] = t == 0.f ? 0.f : t * f;  // masked tokens hold an exact 0
      } else {
        v[u] = lab[j] != ignore ? f : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t j = i + u * kThreads;
      if (j < s1) out[j] = v[u];
    }
  }
}

// ---------------------------------------------------------------- policy ----
struct PolicyArgs {
  const float* logps;
  int64_t lp_ld;
  const float* old_logps;  // nullptr: the ratio is 1 (its gradient is not)
  int64_t old_ld;
  const float* ref_logps;  // nullptr: no KL term
  int64_t ref_ld;
  const float* adv;        // [B], or [B, S] with adv_ld > 0
  int64_t adv_ld;
  const int64_t* labels;
  int64_t lab_ld;
  int64_t batch, seq, ignore;
  double log_lo, log_hi;   // log(1 - clip_low), log(1 + clip_high)
  float lo, hi;            // 1 - clip_low, 1 + clip_high
  float kl_coef;
  int reduction;
};

// e^d - d - 1 and e^d - 1. A policy near its reference has small d, where expm1(d) - d would
// cancel (off by 2e-4 of itself at 1e-4); the series' omitted terms are below 2^-28 of it at
// 1/2, and above that the difference keeps 2^-20.
__device__ __forceinline__ float kl_term(float d, float& em) {
  em = expm1f(d);
  if (!(fabsf(d) < 0.5f)) return em - d;
  float s = 1.f / 362880.f;
  s = fmaf(s, d, 1.f / 40320.f);
  s = fmaf(s, d, 1.f / 5040.f);
  s = fmaf(s, d, 1.f / 720.f);
  s = fmaf(s, d, 1.f / 120.f);
  s = fmaf(s, d, 1.f / 24.f);
  s = fmaf(s, d, 1.f / 6.f);
  s = fmaf(s, d, 0.5f);
  return d * d * s;
}

// Records of two double2 per (sequence, chunk): loss and KL sums, clipped and labelled tokens.
// Per token: r = exp(x - old), L = -min(r A, clip(r) A) + c (e^d - d - 1) with
// d = ref - x, and dL/dx = -A r (0 where the clipped branch is the smaller one)
// + c (1 - e^d), stored for the backward. Which side of a clip border a ratio
// lies on is decided on x - old in 64 bits (exact there) against the border's
// logarithm, so the gradient's jump does not depend on exp's rounding.
__device__ __forceinline__ void policy_sum(const PolicyArgs& a, int chunks, double2* records,
                                           float* __restrict__ tok_grad) {
  __shared__ double sh[4 * kThreads / 32];
  const int64_t n = blockIdx.x / chunks;
  const int64_t s0 = (int64_t)(blockIdx.x % chunks) * kChunk;
  const int64_t s1 = s0 + kChunk < a.seq ? s0 + kChunk : a.seq;
  const float* lp = a.logps + n * a.lp_ld;
  const float* od = a.old_logps ? a.old_logps + n * a.old_ld : nullptr;
  const float* rf = a.ref_logps ? a.ref_logps + n * a.ref_ld : nullptr;
  const float* av = a.adv_ld ? a.adv + n * a.adv_ld : nullptr;
  const float arow = av ? 0.f : a.adv[n];
  const int64_t* lab = a.labels + n * a.lab_ld;
  double loss = 0.0, kl = 0.0;
  int clipped = 0, cnt = 0;
  for (int64_t i = s0 + threadIdx.x; i < s1; i += kThreads * kUnroll) {
    int64_t t[kUnroll];
    float x[kUnroll], o[kUnroll], r[kUnroll], ad[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t j = i + u * kThreads;
      const bool in = j < s1;
      t[u] = in ? lab[j] : a.ignore;
      x[u] = in ? lp[j] : 0.f;
      o[u] = in && od ? od[j] : x[u];
      r[u] = in && rf ? rf[j] : x[u];
      ad[u] = in && av ? av[j] : arow;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t j = i + u * kThreads;
      if (j >= s1) continue;
      float g = 0.f;
      if (t[u] != a.ignore) {
        const float A = ad[u];
        // without old_logps x - x: 0, or NaN for a log-probability that is none
        const double delta = (double)x[u] - (double)o[u];
        const float ratio = od ? expf((float)delta) : 1.f + (float)delta;
        const bool cut = (A > 0.f && delta > a.log_hi) || (A < 0.f && delta < a.log_lo);
        float l = cut ? -(A > 0.f ? a.hi : a.lo) * A : -ratio * A;
        g = cut ? 0.f : -A * ratio;
        if (rf) {
          const float d = r[u] - x[u];
          float em;
          const float k = kl_term(d, em);
          kl += (double)k;
          if (a.kl_coef != 0.f) {  // without a coefficient the term is the metric's alone: 0 x inf is NaN
            l += a.kl_coef * k;
            g -= a.kl_coef * em;
          }
        }
        loss += (double)l;
        clipped += cut ? 1 : 0;
        ++cnt;
      }
      if (tok_grad) tok_grad[n * a.seq + j] = g;
    }
  }
  double v[4] = {loss, kl, (double)clipped, (double)cnt};
  block_sums(v, sh);
  if (threadIdx.x == 0) {
    records[2 * blockIdx.x] = make_double2(v[0], v[1]);
    records[2 * blockIdx.x + 1] = make_double2(v[2], v[3]);
  }
}

// out[0] = loss, out[1] = mean KL, out[2] = clipped share; factor[n] = weight of
// a labelled token of sequence n in the loss.
template <int kWarps>
__device__ __forceinline__ void policy_join(const PolicyArgs& a, int chunks, const double2* records,
                                            float* out_loss, float* out_kl, float* out_clipped,
                                            float* factor) {
  __shared__ double sh[4 * kWarps];
  double loss = 0.0, kl = 0.0, clipped = 0.0, count = 0.0;
  const bool by_seq = a.reduction == SOUP_POLICY_SEQUENCE;
  for (int64_t n = threadIdx.x; n < a.batch; n += blockDim.x) {
    double l = 0.0, c = 0.0;
    for (int i = 0; i < chunks; ++i) {
      const double2 x = __ldcg(records + 2 * (n * chunks + i));  // another block's writes
      const double2 y = __ldcg(records + 2 * (n * chunks + i) + 1);
      l += x.x;
      kl += x.y;
      clipped += y.x;
      c += y.y;
    }
    count += c;
    if (by_seq) {
      const double w = 1.0 / ((c > 1.0 ? c : 1.0) * (double)a.batch);
      factor[n] = (float)w;
      loss += l * w;
    } else {
      loss += l;
    }
  }
  double v[4] = {loss, kl, clipped, count};
  block_sums(v, sh);
  const double inv = 1.0 / (v[3] > 1.0 ? v[3] : 1.0);
  if (!by_seq)
    for (int64_t n = threadIdx.x; n < a.batch; n += blockDim.x) factor[n] = (float)inv;
  if (threadIdx.x == 0) {
    out_loss[0] = (float)(by_seq ? v[0] : v[0] * inv);
    out_kl[0] = (float)(v[1] * inv);
    out_clipped[0] = (float)(v[2] * inv);
  }
}

__global__ void __launch_bounds__(kThreads) policy_sum_kernel(PolicyArgs a, int chunks, double2* records,
                                                              float* tok_grad) {
  pdl_wait();
  pdl_trigger();
  policy_sum(a, chunks, records, tok_grad);
}
__global__ void __launch_bounds__(1024) policy_join_kernel(PolicyArgs a, int chunks,
                                                           const double2* records, float* loss,
                                                           float* kl, float* clipped, float* factor) {
  pdl_wait();
  pdl_trigger();
  policy_join<32>(a, chunks, records, loss, kl, clipped, factor);
}
__global__ void __launch_bounds__(kThreads) policy_cluster_kernel(PolicyArgs a, int chunks,
                                                                  double2* records, float* tok_grad,
                                                                  float* loss, float* kl,
                                                                  float* clipped, float* factor) {
  pdl_wait();
  pdl_trigger();
  policy_sum(a, chunks, records, tok_grad);
  cluster_sync();
  if (blockIdx.x == 0)
    policy_join<kThreads / 32>(a, chunks, records, loss, kl, clipped, factor);
}

int64_t chunks_of(int64_t seq) { return (seq + kChunk - 1) / kChunk; }

bool sizes_ok(int64_t n, int64_t seq) {
  return n > 0 && seq > 0 && n <= (int64_t(1) << 30) && seq <= (int64_t(1) << 40) &&
         n * chunks_of(seq) <= 0x7fffffff;
}

}  // namespace
}  // namespace soup

using namespace soup;

extern "C" {

size_t soup_preference_loss_workspace_bytes(int64_t pairs, int64_t seq) {
  if (!sizes_ok(2 * pairs, seq)) return 0;
  return (size_t)(2 * pairs * chunks_of(seq)) * sizeof(double2);
}

int soup_preference_loss_fwd(const float* logps, int64_t lp_ld, const float* ref, int64_t ref_ld,
                             int ref_mode, const int64_t* labels, int64_t lab_ld, int64_t pairs,
                             int64_t seq, int64_t ignore_index, double beta, double label_smoothing,
                             int loss_type, float* loss, float* rewards, float* coef,
                             void* workspace, size_t workspace_bytes, void* stream) {
  if (!logps || !labels || !loss || !rewards || !coef || !workspace || !sizes_ok(2 * pairs, seq) ||
      lp_ld < seq || lab_ld < seq || ref_mode < 0 || ref_mode > 2 || (ref_mode != 0 && !ref) ||
      (ref_mode == 1 && ref_ld < seq)) {
    set_last_error("soup_preference_loss_fwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (!(beta > 0.0) || isinf(beta) || !(label_smoothing >= 0.0 && label_smoothing < 0.5) ||
      loss_type < SOUP_PREF_SIGMOID || loss_type > SOUP_PREF_IPO ||
      (label_smoothing != 0.0 && loss_type != SOUP_PREF_SIGMOID)) {
    set_last_error("soup_preference_loss_fwd: beta must be positive and finite, label_smoothing in [0, 0.5) "
                   "and only with the sigmoid loss, loss_type one of the SOUP_PREF codes");
    return SOUP_ERR_INVALID;
  }
  if (workspace_bytes < soup_preference_loss_workspace_bytes(pairs, seq) || !aligned16(workspace)) {
    set_last_error("soup_preference_loss_fwd: workspace too small or misaligned");
    return SOUP_ERR_WORKSPACE;
  }
  const int chunks = (int)chunks_of(seq);
  PrefArgs a{logps, lp_ld, ref, ref_ld, ref_mode, labels, lab_ld, pairs, seq, ignore_index, beta,
             label_smoothing, loss_type};
  double2* rec = static_cast<double2*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (2 * pairs * chunks <= kClusterBlocks)
    return cuda_status(launch_cluster(pref_cluster_kernel, (unsigned)(2 * pairs * chunks), st, a, chunks,
                                      rec, loss, rewards, coef));
  int rc = cuda_status(launch_pdl(pref_sum_kernel, dim3((unsigned)(2 * pairs * chunks)),
                                  dim3(kThreads), 0, st, a, chunks, rec));
  if (rc) return rc;
  return cuda_status(launch_pdl(pref_join_kernel, dim3(1), dim3(kThreads), 0, st, a, chunks,
                                (const double2*)rec, loss, rewards, coef));
}

int soup_preference_loss_bwd(const float* grad_loss, const float* coef, const int64_t* labels,
                             int64_t lab_ld, int64_t pairs, int64_t seq, int64_t ignore_index,
                             float* dlogps, void* stream) {
  if (!grad_loss || !coef || !labels || !dlogps || !sizes_ok(2 * pairs, seq) || lab_ld < seq) {
    set_last_error("soup_preference_loss_bwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  const int chunks = (int)chunks_of(seq);
  return cuda_status(launch_pdl(loss_bwd_kernel, dim3((unsigned)(2 * pairs * chunks)),
                                dim3(kThreads), 0, as_stream(stream), grad_loss, coef,
                                (const float*)nullptr, labels, lab_ld, seq, chunks, ignore_index,
                                dlogps));
}

size_t soup_policy_loss_workspace_bytes(int64_t batch, int64_t seq) {
  if (!sizes_ok(batch, seq)) return 0;
  return (size_t)(batch * chunks_of(seq)) * 2 * sizeof(double2);
}

int soup_policy_loss_fwd(const float* logps, int64_t lp_ld, const float* old_logps, int64_t old_ld,
                         const float* ref_logps, int64_t ref_ld, const float* advantages,
                         int64_t adv_ld, const int64_t* labels, int64_t lab_ld, int64_t batch,
                         int64_t seq, int64_t ignore_index, double clip_low, double clip_high,
                         float kl_coef, int reduction, float* loss, float* kl, float* clipped,
                         float* factor, float* tok_grad, void* workspace, size_t workspace_bytes,
                         void* stream) {
  if (!logps || !advantages || !labels || !loss || !kl || !clipped || !factor || !workspace ||
      !sizes_ok(batch, seq) || lp_ld < seq || lab_ld < seq || (old_logps && old_ld < seq) ||
      (ref_logps && ref_ld < seq) || (adv_ld != 0 && adv_ld < seq)) {
    set_last_error("soup_policy_loss_fwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  if (!(clip_low >= 0.0 && clip_low < 1.0) || !(clip_high >= 0.0) || isinf(clip_high) ||
      !(kl_coef >= 0.f) || isinf(kl_coef) ||
      (reduction != SOUP_POLICY_TOKEN && reduction != SOUP_POLICY_SEQUENCE)) {
    set_last_error("soup_policy_loss_fwd: clip_low must be in [0, 1), clip_high and kl_coef finite "
                   "and not negative, reduction one of the SOUP_POLICY codes");
    return SOUP_ERR_INVALID;
  }
  if (workspace_bytes < soup_policy_loss_workspace_bytes(batch, seq) || !aligned16(workspace)) {
    set_last_error("soup_policy_loss_fwd: workspace too small or misaligned");
    return SOUP_ERR_WORKSPACE;
  }
  const int chunks = (int)chunks_of(seq);
  PolicyArgs a{logps, lp_ld, old_logps, old_ld, ref_logps, ref_ld, advantages, adv_ld, labels,
               lab_ld, batch, seq, ignore_index, log(1.0 - clip_low), log(1.0 + clip_high),
               (float)(1.0 - clip_low), (float)(1.0 + clip_high), kl_coef, reduction};
  double2* rec = static_cast<double2*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (batch * chunks <= kClusterBlocks)
    return cuda_status(launch_cluster(policy_cluster_kernel, (unsigned)(batch * chunks), st, a, chunks,
                                      rec, tok_grad, loss, kl, clipped, factor));
  int rc = cuda_status(launch_pdl(policy_sum_kernel, dim3((unsigned)(batch * chunks)),
                                  dim3(kThreads), 0, st, a, chunks, rec, tok_grad));
  if (rc) return rc;
  return cuda_status(launch_pdl(policy_join_kernel, dim3(1), dim3(1024), 0, st, a, chunks,
                                (const double2*)rec, loss, kl, clipped, factor));
}

int soup_policy_loss_bwd(const float* grad_loss, const float* factor, const float* tok_grad,
                         int64_t batch, int64_t seq, float* dlogps, void* stream) {
  if (!grad_loss || !factor || !tok_grad || !dlogps || !sizes_ok(batch, seq)) {
    set_last_error("soup_policy_loss_bwd: bad arguments");
    return SOUP_ERR_INVALID;
  }
  const int chunks = (int)chunks_of(seq);
  return cuda_status(launch_pdl(loss_bwd_kernel, dim3((unsigned)(batch * chunks)), dim3(kThreads), 0,
                                as_stream(stream), grad_loss, factor, tok_grad,
                                (const int64_t*)nullptr, int64_t(0), seq, chunks, int64_t(0),
                                dlogps));
}

}  // extern "C"
