// Verification of drafted tokens against the target's logits, from given uniform numbers.
//
// Per sequence, with p_j = softmax(target_j / T), q_j = softmax(draft_j / T) (without draft logits: all on the drafted
// token x_j) and uniform numbers u in [0, 1): the drafts are accepted in order while u_j q_j(x_j) < p_j(x_j); at the first
// rejection j the next token is drawn from max(p_j - q_j, 0), normalised, and when all n are accepted from p_n.  The draw
// is the inverse of the cumulative sum: the first token whose cumulative weight passes u_t times their sum.  T <= 0 is the
// greedy limit: a draft is accepted if it is the target's largest logit (the lowest token among equal ones), which is the
// next token otherwise.  The tokens emitted are then distributed as the target's own (T > 0), or equal to its greedy ones.
#include "agens_kernels.h"
#include "wq_common.h"

namespace agq {
namespace {

constexpr int kVerThreads = 1024;

struct VerifyArgs {
  const uint16_t *target, *draft;
  const int *ids, *counts;
  const float *u, *temp;
  int* tokens;
  int* accepted;
  float* logp;
  long ldt, ldd;
  int b, t, vocab;
};

// NaN counts as -inf
__device__ __forceinline__ float logit(uint16_t b) {
  const float f = bf2f(b);
  return f != f ? -INFINITY : f;
}

struct RowStat {
  float top;     // largest logit
  int best;      // its lowest index
  double total;  // sum of weights
};

__device__ __forceinline__ float weight(float l, float top, float heat) {
  return top == -INFINITY ? 0.0f : l == top ? 1.0f : expf((l - top) / heat);
}

__device__ RowStat row_stat(const uint16_t* row, int vocab, float heat, double* red, int* ired) {
  float top = -INFINITY;
  for (int i = threadIdx.x; i < vocab; i += kVerThreads) top = fmaxf(top, logit(row[i]));
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  for (int w = 0; w < kVerThreads / 64; ++w) top = fmaxf(top, (float)red[w]);
  __syncthreads();
  int best = vocab;
  double sum = 0.0;
  for (int i = threadIdx.x; i < vocab; i += kVerThreads) {
    const float l = logit(row[i]);
    if (l == top && top > -INFINITY && best == vocab) best = i;
    sum += weight(l, top, heat);
  }
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d), best = min(best, __shfl_xor(best, d));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum, ired[threadIdx.x >> 6] = best;
  __syncthreads();
  RowStat r{top, vocab, 0.0};
  for (int w = 0; w < kVerThreads / 64; ++w) r.total += red[w], r.best = min(r.best, ired[w]);
  if (r.best == vocab) r.best = -1;
  return r;
}

__global__ void __launch_bounds__(kVerThreads) spec_verify_kernel(const VerifyArgs a) {
  __shared__ double red[kVerThreads + 1];
  __shared__ int ired[kVerThreads / 64], pick;
  const int seq = blockIdx.x, V = a.vocab;
  const int n = a.counts ? min(max(a.counts[seq], 0), a.t) : a.t;
  const float temp = a.temp ? a.temp[seq] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  const float heat = greedy ? 1.0f : temp;
  int* const tok = a.tokens + (size_t)seq * (a.t + 1);
  float* const lp = a.logp ? a.logp + (size_t)seq * (a.t + 1) : nullptr;
  for (int j = 0;; ++j) {
    const uint16_t* const row = a.target + ((size_t)seq * (a.t + 1) + j) * a.ldt;
    const RowStat P = row_stat(row, V, heat, red, ired);
    const int x = j < n ? a.ids[(size_t)seq * a.t + j] : -1;
    const bool known = x >= 0 && x < V;
    const uint16_t* const drow = a.draft && j < n ? a.draft + ((size_t)seq * a.t + j) * a.ldd : nullptr;
    RowStat Q{0.0f, 0, 1.0};
    if (drow && !greedy) Q = row_stat(drow, V, heat, red, ired);
    if (known) {
      const double p = P.total > 0 ? weight(logit(row[x]), P.top, heat) / P.total : 0.0;
      const double q = drow ? (Q.total > 0 ? weight(logit(drow[x]), Q.top, heat) / Q.total : 0.0) : 1.0;
      if (greedy ? x == P.best : a.u[(size_t)seq * (a.t + 1) + j] * q < p) {
        if (threadIdx.x == 0) {
          tok[j] = x;
          if (lp) lp[j] = (float)((logit(row[x]) == P.top ? 0.0 : (double)(logit(row[x]) - P.top) / heat) - log(P.total));
        }
        continue;
      }
    }
    // the next token: weights p - q of a rejection (p where nothing is left of it), p otherwise
    if (threadIdx.x == 0) pick = greedy ? P.best : -1;
    __syncthreads();
    for (int pass = j < n ? 0 : 1; pass < 2 && pick < 0 && P.total > 0 && !greedy; ++pass) {
      const int each = (V + kVerThreads - 1) / kVerThreads, lo = min(V, (int)threadIdx.x * each), hi = min(V, lo + each);
      auto w = [&](int i) {
        const double p = weight(logit(row[i]), P.top, heat) / P.total;
        if (pass == 1) return p;
        const double q = drow ? (Q.total > 0 ? weight(logit(drow[i]), Q.top, heat) / Q.total : 0.0) : (i == x ? 1.0 : 0.0);
        return p > q ? p - q : 0.0;
      };
      double sum = 0.0;
      for (int i = lo; i < hi; ++i) sum += w(i);
      red[threadIdx.x + 1] = sum;
      __syncthreads();
      if (threadIdx.x == 0) {
        red[0] = 0.0;
        for (int i = 1; i <= kVerThreads; ++i) red[i] += red[i - 1];
        if (red[kVerThreads] > 0) {
          const double at = (double)a.u[(size_t)seq * (a.t + 1) + a.t] * red[kVerThreads];
          int last = -1;
          for (int c = 0; c < kVerThreads && pick < 0; ++c) {
            if (red[c + 1] <= at && c + 1 < kVerThreads) {
              continue;
            }
            double s = red[c];
            for (int i = c * each; i < min(V, c * each + each); ++i) {
              const double wi = w(i);
              s += wi;
              if (wi > 0) last = i;
              if (s > at) {
                pick = i;
                break;
              }
            }
          }
          if (pick < 0) pick = last;
        }
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      tok[j] = pick;
      if (lp)
        lp[j] = pick < 0 ? 0.0f
                         : (float)((logit(row[pick]) == P.top ? 0.0 : (double)(logit(row[pick]) - P.top) / heat) -
                                   log(P.total));
      for (int i = j + 1; i <= a.t; ++i) {
        tok[i] = -1;
        if (lp) lp[i] = 0.0f;
      }
      a.accepted[seq] = j;
    }
    return;
  }
}

}  // namespace
}  // namespace agq

extern "C" int ak_spec_verify(const void* target, long ldt, const void* draft, long ldd, const int* ids,
                              const int* counts, const float* u, const float* temperature, int b, int t, int vocab,
                              int* tokens, int* accepted, float* logp, void* stream) {
  if (b < 0 || t < 0 || t > AK_VERIFY_MAX_DRAFTS || vocab < 1 || ldt < vocab || (draft && t && ldd < vocab))
    return AK_INVALID;
  if (!b) return 0;
  if (!target || (t && !ids) || !u || !tokens || !accepted) return AK_INVALID;
  const agq::VerifyArgs a{static_cast<const uint16_t*>(target), t ? static_cast<const uint16_t*>(draft) : nullptr, ids,
                          counts, u, temperature, tokens, accepted, logp, ldt, ldd, b, t, vocab};
  hipLaunchKernelGGL(agq::spec_verify_kernel, dim3((unsigned)b), dim3(agq::kVerThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return (int)hipGetLastError();
}
