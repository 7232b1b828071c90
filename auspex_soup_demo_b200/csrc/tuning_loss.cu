// Losses over per-token log-probabilities: the paired log-ratio (preference)
// loss and the clipped importance-ratio (policy) loss with a KL term, forward
// and backward.
//
// Both are masked reductions over [sequences, tokens] fp32 arrays: a first
// kernel sums each sequence (one block per sequence and chunk of tokens) into
// one record per block, a second, one block, joins the records in a fixed
// order (no atomics: the same inputs give the same bits) and writes the loss,
// the metrics and one gradient factor per sequence; the backward is one
// elementwise pass. Labels equal to ignore_index mark masked tokens: their
// values are selected away, never multiplied, so infinities and NaN there do
// not reach a sum. Sums over tokens run in 64 bits: thousands of terms of
// either sign leave a difference that 32 bits would round away, and the adds
// are free beside the loads.
#include "soup_common.cuh"

namespace soup {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;  // tokens per block of the summing kernels
constexpr int kUnroll = 4;    // tokens per thread whose loads are in flight together

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += sh[i];
  __syncthreads();
  return t;
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
__global__ void __launch_bounds__(kThreads) pref_sum_kernel(PrefArgs a, int chunks,
                                                            double2* __restrict__ records) {
  __shared__ double sh[kThreads / 32];
  pdl_wait();
  pdl_trigger();
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
  sum = block_sum(sum, sh);
  const double n_lab = block_sum((double)cnt, sh);
  if (threadIdx.x == 0) records[blockIdx.x] = make_double2(sum, n_lab);
}

// Per pair p: h = score(chosen) - score(rejected), the loss and dL/dh; then the
// mean loss. rewards[n] = beta * log ratio, coef[n] = dL/d(log prob of a
// labelled token of sequence n). softplus(x) = max(x, 0) + log1p(exp(-|x|)). In
// 64 bits: label smoothing subtracts nearly equal terms, and one thread does one
// pair, so the wider arithmetic hides behind the launch.
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

__global__ void __launch_bounds__(kThreads) pref_join_kernel(PrefArgs a, int chunks,
                                                             const double2* __restrict__ records,
                                                             float* __restrict__ loss,
                                                             float* __restrict__ rewards,
                                                             float* __restrict__ coef) {
  __shared__ double sh[kThreads / 32];
  pdl_wait();
  pdl_trigger();
  double total = 0.0;
  for (int64_t p = threadIdx.x; p < a.pairs; p += kThreads) {
    double d[2], per[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int64_t n = p + w * a.pairs;
      double sum = 0.0, cnt = 0.0;
      for (int c = 0; c < chunks; ++c) {
        const double2 r = records[n * chunks + c];
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
  total = block_sum(total, sh);
  if (threadIdx.x == 0) loss[0] = (float)(total / (double)a.pairs);
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

struct PolicyRecord {
  double loss, kl;
  double clipped, count;
};

// Per token: r = exp(x - old), L = -min(r A, clip(r) A) + c (e^d - d - 1) with
// d = ref - x, and dL/dx = -A r (0 where the clipped branch is the smaller one)
// + c (1 - e^d), stored for the backward. Which side of a clip border a ratio
// lies on is decided on x - old in 64 bits (exact there) against the border's
// logarithm, so the gradient's jump does not depend on exp's rounding.
__global__ void __launch_bounds__(kThreads) policy_sum_kernel(PolicyArgs a, int chunks,
                                                              PolicyRecord* __restrict__ records,
                                                              float* __restrict__ tok_grad) {
  __shared__ double sh[kThreads / 32];
  pdl_wait();
  pdl_trigger();
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
        const double delta = od ? (double)x[u] - (double)o[u] : 0.0;
        const float ratio = od ? expf((float)delta) : 1.f;
        const bool cut = (A > 0.f && delta > a.log_hi) || (A < 0.f && delta < a.log_lo);
        float l = cut ? -(A > 0.f ? a.hi : a.lo) * A : -ratio * A;
        g = cut ? 0.f : -A * ratio;
        if (rf) {
          const float d = r[u] - x[u];
          const float em = expm1f(d);
          const float k = em - d;
          kl += (double)k;
          l += a.kl_coef * k;
          g -= a.kl_coef * em;
        }
        loss += (double)l;
        clipped += cut ? 1 : 0;
        ++cnt;
      }
      if (tok_grad) tok_grad[n * a.seq + j] = g;
    }
  }
  loss = block_sum(loss, sh);
  kl = block_sum(kl, sh);
  const double nc = block_sum((double)clipped, sh);
  const double nl = block_sum((double)cnt, sh);
  if (threadIdx.x == 0) records[blockIdx.x] = PolicyRecord{loss, kl, nc, nl};
}

// out[0] = loss, out[1] = mean KL, out[2] = clipped share; factor[n] = weight of
// a labelled token of sequence n in the loss.
__global__ void __launch_bounds__(1024) policy_join_kernel(PolicyArgs a, int chunks,
                                                           const PolicyRecord* __restrict__ records,
                                                           float* __restrict__ out_loss,
                                                           float* __restrict__ out_kl,
                                                           float* __restrict__ out_clipped,
                                                           float* __restrict__ factor) {
  __shared__ double sh[32];
  pdl_wait();
  pdl_trigger();
  double loss = 0.0, kl = 0.0, clipped = 0.0, count = 0.0;
  const bool by_seq = a.reduction == SOUP_POLICY_SEQUENCE;
  for (int64_t n = threadIdx.x; n < a.batch; n += blockDim.x) {
    double l = 0.0, c = 0.0;
    for (int i = 0; i < chunks; ++i) {
      const PolicyRecord r = records[n * chunks + i];
      l += r.loss;
      c += r.count;
      kl += r.kl;
      clipped += r.clipped;
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
  loss = block_sum(loss, sh);
  kl = block_sum(kl, sh);
  clipped = block_sum(clipped, sh);
  count = block_sum(count, sh);
  const double inv = 1.0 / (count > 1.0 ? count : 1.0);
  if (!by_seq)
    for (int64_t n = threadIdx.x; n < a.batch; n += blockDim.x) factor[n] = (float)inv;
  if (threadIdx.x == 0) {
    out_loss[0] = (float)(by_seq ? loss : loss * inv);
    out_kl[0] = (float)(kl * inv);
    out_clipped[0] = (float)(clipped * inv);
  }
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
  return (size_t)(batch * chunks_of(seq)) * sizeof(PolicyRecord);
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
  PolicyRecord* rec = static_cast<PolicyRecord*>(workspace);
  cudaStream_t st = as_stream(stream);
  int rc = cuda_status(launch_pdl(policy_sum_kernel, dim3((unsigned)(batch * chunks)),
                                  dim3(kThreads), 0, st, a, chunks, rec, tok_grad));
  if (rc) return rc;
  return cuda_status(launch_pdl(policy_join_kernel, dim3(1), dim3(1024), 0, st, a, chunks,
                                (const PolicyRecord*)rec, loss, kl, clipped, factor));
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
