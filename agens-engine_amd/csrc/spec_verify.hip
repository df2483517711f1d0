// Verification of drafted tokens against the target's logits, from given uniform numbers.
//
// Per sequence, with p_j = softmax(target_j / T), q_j = softmax(draft_j / T) (without draft logits: all on the drafted
// token x_j) and uniform numbers u in [0, 1): the drafts are accepted in order while u_j q_j(x_j) < p_j(x_j); at the first
// rejection j the next token is drawn from max(p_j - q_j, 0), normalised, and when all n are accepted from p_n.  The draw
// is the inverse of the cumulative sum: the first token whose cumulative weight passes u_t times their sum.  T <= 0 is the
// greedy limit: a draft is accepted if it is the target's largest logit (the lowest token among equal ones), which is the
// next token otherwise.  The tokens emitted are then distributed as the target's own (T > 0), or equal to its greedy ones.
//
// Bound by the logits' bytes, each read once: verify_rows_kernel gives every workgroup kChunk logits of one row, which it
// holds in registers for both their largest and the sum of their weights relative to it.  What follows needs little of it:
//   verify_decide_kernel  puts the chunks of a sequence's rows together and decides on its drafts in order; without draft
//                         logits it also draws the next token, for which the chunks' sums say in which chunk it lies, and
//                         only that one is read again;
//   with draft logits     its workgroups, one a chunk, each come to the same decision and add up their chunk of the
//                         weights p - q, which are known only now; verify_draw_kernel draws the next token.
// (Joined by the launches' order: counters and fences between workgroups cost more than a launch here.)
// Without scratch (a capture before any other call), verify_whole_kernel does all of it in one workgroup a sequence, in the
// same order, so with the same bits.
//
// Measured: 32 sequences of 5 looked-up drafts, 152064 logits (58 MB) 22 us: rows 16, 3.7 TB/s (a wave instead of a workgroup
// for 4096 logits, without barriers, or 32 logits a thread: no faster), decision and draw 8, a chain of dependent loads; one
// sequence with 4 drafts and their logits 14 us, of which rows 4, decision 5, draw 4.  (LDS atomics for the picks cost 5 us
// each, exchanges through LDS instead of DPP 2.)
//
// Weights are fp32 (the hardware's exp2 of the scaled difference to the largest logit), as are the sums of the 16 that a
// thread holds; all larger sums are 64 bits, in an order that only a row's length decides.
#include "agens_kernels.h"
#include "wq_common.h"

#include <cfloat>

namespace agq {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kEach = 16, kChunk = kThreads * kEach;
constexpr int kMaxChunks = kThreads;  // of a row: a thread looks at one
constexpr int kMaxVocab = kMaxChunks * kChunk;
static_assert(kMaxVocab == AK_VERIFY_MAX_VOCAB, "the header's limit");
constexpr size_t kMaxScratch = (size_t)64 << 20;  // of a launch; more sequences take several

// A row, or a chunk of one: its largest logit, the lowest token that has it (-1: nothing above -inf), the sum of the
// weights relative to it.
struct RowStat {
  float top;
  int best;
  double total;
};

// The next token of a sequence is drawn for place j, whose rows' sums are p and q (residual: from p - q).
struct Decision {
  int j, residual;
  RowStat p, q;
};

struct VerifyArgs {
  const uint16_t *target, *draft;
  const int *ids, *counts;
  const float *u, *temp;
  int* tokens;
  int* accepted;
  float* logp;
  long ldt, ldd;
  int t, vocab, chunks, rows;  // rows: of a sequence, target rows first
  // scratch
  RowStat* stats;  // [b][rows][chunks]
  double* sums;    // [b][chunks]: of max(p - q, 0) in the rejected draft's place
  double* rest;    // [b][t], without draft logits: the sum of the draft's chunk without the draft
  Decision* plan;  // [b]
};

// What a workgroup shares
struct Shared {
  double red[kWaves];
  int ired[kWaves];
  double before[kWaves];
  RowStat p[kWaves], q[kWaves];
  int ok[kWaves];
};

struct Seq {
  int id, n;  // n: drafts
  bool greedy;
  float heat;
  // log2(e) / T in two parts: one of 24 bits alone shifts all exponents the same way, so the row's sum by up to 2^-24 times
  // the mean exponent.  T counts as at least fp32's smallest normal number, and as 1.44e30 at most.
  float scale, scale_lo;
  float least;  // a difference of logits whose weight is 0 (2^-300), as is that of all below: its products are numbers at any T
  float next_u;
};
__device__ __forceinline__ Seq seq_of(const VerifyArgs& a, int id) {
  Seq s;
  s.id = id;
  s.n = a.counts ? min(max(a.counts[id], 0), a.t) : a.t;
  const float temp = a.temp ? a.temp[id] : 1.0f;
  s.greedy = !(temp > 0.0f);
  s.heat = s.greedy ? 1.0f : temp;
  const float heat = fminf(fmaxf(s.heat, FLT_MIN), 1.44e30f);
  const double scale = 1.44269504088896340736 / (double)heat;
  s.scale = (float)scale;
  s.scale_lo = (float)(scale - (double)s.scale);
  s.least = -208.0f * heat;
  s.next_u = a.u[(size_t)id * (a.t + 1) + a.t];
  return s;
}
__device__ __forceinline__ const uint16_t* target_row(const VerifyArgs& a, int seq, int j) {
  return a.target + ((size_t)seq * (a.t + 1) + j) * a.ldt;
}
__device__ __forceinline__ const uint16_t* draft_row(const VerifyArgs& a, int seq, int j) {
  return a.draft + ((size_t)seq * a.t + j) * a.ldd;
}

// The weight of logit l in a row whose largest is top (not +inf).  The clamp takes a masked logit's -inf, and NaN, to a
// difference whose weight is 0.
__device__ __forceinline__ float weight(const Seq& s, float l, float top) {
  const float d = fmaxf(l - (top == -INFINITY ? 0.0f : top), s.least);
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, s.scale, d * s.scale_lo));
}
// Of any row: where the largest is +inf, all that are it weigh the same.
__device__ __forceinline__ float any_weight(const Seq& s, float l, float top) {
  return top == INFINITY ? (l == top ? 1.0f : 0.0f) : weight(s, l, top);
}
__device__ __forceinline__ void weigh16(const Seq& s, float top, float (&l)[kEach]) {
  if (top == INFINITY) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) l[i] = l[i] == top ? 1.0f : 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) l[i] = weight(s, l[i], top);
  }
}

// 8 logits from token k on, -inf past the end.  Rows begin at any even address.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
__device__ __forceinline__ void load8(const uint16_t* row, int k, int vocab, float* l) {
  if (k + 8 <= vocab) {
    const u32x4 v = *reinterpret_cast<const u32x4_any*>(row + k);
#pragma unroll
    for (int i = 0; i < 8; ++i) l[i] = __uint_as_float(i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) l[i] = k + i < vocab ? bf2f(row[k + i]) : -INFINITY;
  }
}

__device__ __forceinline__ double sum16(const float (&w)[kEach]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) s += w[i];
  return (double)s;
}

// Over the lanes of a wave, by DPP (an LDS exchange takes several times as long): x of the lane `ctrl` names, `none` where
// there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t x, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xF, false);
}
// op over the lanes up to each one: row_shr 1, 2, 4, 8 within the rows of 16, then the rows' last lanes
template <class T, class Op>
__device__ __forceinline__ T wave_scan(T x, Op op) {
  x = op.template step<0x111, 0xF>(x);
  x = op.template step<0x112, 0xF>(x);
  x = op.template step<0x114, 0xF>(x);
  x = op.template step<0x118, 0xF>(x);
  x = op.template step<0x142, 0xA>(x);  // row_bcast 15
  return op.template step<0x143, 0xC>(x);  // row_bcast 31
}
struct Add {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ double step(double x) const {
    const uint64_t v = (uint64_t)__double_as_longlong(x);
    return x + __longlong_as_double((long long)((uint64_t)dpp<CTRL, ROWS>((uint32_t)(v >> 32), 0) << 32 |
                                                dpp<CTRL, ROWS>((uint32_t)v, 0)));
  }
};
struct Max {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ float step(float x) const {
    return fmaxf(x, __uint_as_float(dpp<CTRL, ROWS>(__float_as_uint(x), 0xFF800000u)));
  }
};
struct Min {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ int step(int x) const {
    return min(x, (int)dpp<CTRL, ROWS>((uint32_t)x, 0x7FFFFFFFu));
  }
};
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
__device__ __forceinline__ double wave_sum(double x) {
  const uint64_t v = (uint64_t)__double_as_longlong(wave_scan(x, Add()));
  return __longlong_as_double((long long)((uint64_t)last_lane((uint32_t)(v >> 32)) << 32 | last_lane((uint32_t)v)));
}
__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(last_lane(__float_as_uint(wave_scan(x, Max()))));
}
__device__ __forceinline__ int wave_min(int x) { return (int)last_lane((uint32_t)wave_scan(x, Min())); }

// The sum over the workgroup, in every thread.
__device__ __forceinline__ double block_sum(double x, Shared& sh) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) s += sh.red[i];
  return s;
}

// A chunk of a row, by a workgroup: thread t holds 8 logits from 8 t on in either half (whole cache lines a wave).
// Where it holds token `skip`, its sum without that token also goes to *rest.
__device__ __forceinline__ RowStat chunk_stat(const Seq& s, const uint16_t* row, int chunk, int vocab, int skip, double* rest,
                                              Shared& sh) {
  const int t = threadIdx.x, at0 = chunk * kChunk + 8 * t, at1 = at0 + kChunk / 2;
  float l[kEach];
  load8(row, at0, vocab, l);
  load8(row, at1, vocab, l + 8);
  float mine = l[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) mine = fmaxf(mine, l[i]);
  float top = wave_max(mine);
  __syncthreads();
  if ((t & 63) == 0) sh.red[t >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) top = fmaxf(top, (float)sh.red[i]);
  // the lowest token with it: in the first half before the second, there in the first wave, lane and place
  int best0 = -1, best1 = -1;
  if (mine == top && top > -INFINITY) {
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      if (l[i] == top) best0 = at0 + i;
      if (l[i + 8] == top) best1 = at1 + i;
    }
  }
  const uint64_t in0 = __ballot(best0 >= 0), in1 = __ballot(best1 >= 0);
  if (in0 | in1) {
    const int best = __shfl(in0 ? best0 : best1, __builtin_ctzll(in0 ? in0 : in1));
    if ((t & 63) == 0) sh.ired[t >> 6] = best;
  } else if ((t & 63) == 0) {
    sh.ired[t >> 6] = 0x7FFFFFFF;
  }
  weigh16(s, top, l);
  const double total = block_sum(sum16(l), sh);
  int best = sh.ired[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) best = min(best, sh.ired[i]);
  if (skip >= 0 && skip / kChunk == chunk) {  // (summed anew: nothing is left of a difference where it has nearly all)
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if ((i < 8 ? at0 : at1 - 8) + i == skip) l[i] = 0.0f;
    const double x = block_sum(sum16(l), sh);
    if (t == 0) *rest = x;
  }
  return RowStat{top, best == 0x7FFFFFFF ? -1 : best, total};
}
// The draft that its row's weights are drawn without if it is rejected (-1: none): with nothing else known of the draft model.
__device__ __forceinline__ int lone_draft(const VerifyArgs& a, const Seq& s, int j) {
  if (a.draft || s.greedy || j >= s.n) return -1;
  const int x = a.ids[(size_t)s.id * a.t + j];
  return x < a.vocab ? x : -1;
}

// How much a chunk's sum counts in its row.
__device__ __forceinline__ double chunk_share(const Seq& s, const RowStat& c, float top) {
  return c.total * (double)any_weight(s, c.top, top);
}

// A row from its chunks, by one wave: their loads (the lane's chunks), then the rest.
struct Chunks {
  RowStat c[kMaxChunks / 64];
};
__device__ __forceinline__ Chunks load_chunks(const RowStat* st, int chunks) {
  const int lane = threadIdx.x & 63;
  Chunks x;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 64; ++i) {
    x.c[i] = RowStat{-INFINITY, 0x7FFFFFFF, 0.0};
    if (lane + 64 * i < chunks) x.c[i] = st[lane + 64 * i];
  }
  return x;
}
__device__ __forceinline__ RowStat row_stat(const Seq& s, const Chunks& x) {
  const RowStat(&c)[kMaxChunks / 64] = x.c;
  RowStat r{-INFINITY, 0x7FFFFFFF, 0.0};
#pragma unroll
  for (int i = 0; i < kMaxChunks / 64; ++i)
    if (c[i].top > r.top) r.top = c[i].top, r.best = c[i].best;
  const float mine = r.top;
  r.top = wave_max(mine);
  r.best = r.top == -INFINITY ? -1 : wave_min(mine == r.top ? r.best : 0x7FFFFFFF);
  if (r.best < 0) return r;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 64; ++i) r.total += chunk_share(s, c[i], r.top);
  r.total = wave_sum(r.total);
  return r;
}

// The first thread at which the sum of the threads' x (>= 0) passes `at`; the last with any x if rounding lets none pass;
// -1 without any.  *before: the sum of the threads before it.
__device__ __forceinline__ int pick_thread(double x, double at, Shared& sh, double* before) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const double inc = wave_scan(x, Add());
  __syncthreads();
  if (lane == 63) sh.red[w] = inc;
  __syncthreads();
  double b = inc - x;
#pragma unroll
  for (int i = 0; i < kWaves; ++i)
    if (i < w) b += sh.red[i];
  const uint64_t past = __ballot(x > 0.0 && b + x > at), any = __ballot(x > 0.0);
  const int mine = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : -1;  // of the wave
  if (lane == mine) sh.before[w] = b;
  if (lane == 0) sh.ired[w] = mine < 0 ? -1 : 64 * w + mine, sh.ok[w] = past != 0;
  __syncthreads();
  int pick = -1;
  for (int i = 0; i < kWaves; ++i) {
    if (sh.ired[i] < 0) continue;
    pick = sh.ired[i], *before = sh.before[i];
    if (sh.ok[i]) break;
  }
  __syncthreads();
  return pick;
}

// The next token: chunk c weighs share (of thread c); weigh(k, w) gives the weights of the 16 tokens from k on.  -1: none.
template <class Weigh>
__device__ __forceinline__ int find_token(const VerifyArgs& a, float u, double share, Weigh weigh, Shared& sh) {
  const double all = block_sum(share, sh);
  if (!(all > 0.0)) return -1;
  double at = (double)u * all, before;
  const int chunk = pick_thread(share, at, sh, &before);
  at = fmax(at - before, 0.0);  // (the chunks before may sum to a rounding more than they did one by one)
  const int k = chunk * kChunk + (int)threadIdx.x * kEach;
  float w[kEach];
  weigh(k, w);
  const int who = pick_thread(sum16(w), at, sh, &before);
  int token = -1;
  if ((int)threadIdx.x == who) {
    double c = before;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {  // the last with any weight at worst; likewise the first
      if (w[i] > 0.0f && (token < 0 || c <= at)) token = k + i;
      c += (double)w[i];
    }
    sh.ired[0] = token;
  }
  __syncthreads();
  return who < 0 ? -1 : sh.ired[0];
}

// From the target's weights, without token `skip` (-1: all), where its chunk's sum is `rest`.
__device__ __forceinline__ int draw_target(const VerifyArgs& a, const Seq& s, int j, const RowStat* st, const RowStat& p,
                                           int skip, double rest, Shared& sh) {
  const uint16_t* const row = target_row(a, s.id, j);
  auto weigh = [&](int k, float(&w)[kEach]) {
    load8(row, k, a.vocab, w);
    load8(row, k + 8, a.vocab, w + 8);
    weigh16(s, p.top, w);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (k + i == skip) w[i] = 0.0f;
  };
  const int c = threadIdx.x;
  RowStat mine{-INFINITY, -1, 0.0};
  if (c < a.chunks) mine = st[c];
  if (skip >= 0 && c == skip / kChunk) mine.total = rest;
  return find_token(a, s.next_u, chunk_share(s, mine, p.top), weigh, sh);
}

// The weights max(p - q, 0) of the 16 tokens from k on, with p and q normalised: in 64 bits, since the two may be close.
__device__ __forceinline__ void residual16(const VerifyArgs& a, const Seq& s, const Decision& d, float (&lp)[kEach],
                                           float (&lq)[kEach], float (&w)[kEach]) {
  weigh16(s, d.p.top, lp);
  weigh16(s, d.q.top, lq);
  const double pi = 1.0 / d.p.total, qi = 1.0 / d.q.total;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    w[i] = (float)fmax(lp[i] * pi - lq[i] * qi, 0.0);
}
__device__ __forceinline__ double residual_sum(const VerifyArgs& a, const Seq& s, const Decision& d, int chunk, Shared& sh) {
  const uint16_t *const p = target_row(a, s.id, d.j), *const q = draft_row(a, s.id, d.j);
  const int at = chunk * kChunk + 8 * (int)threadIdx.x;
  float lp[kEach], lq[kEach], w[kEach];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load8(p, at + h * kChunk / 2, a.vocab, lp + 8 * h);
    load8(q, at + h * kChunk / 2, a.vocab, lq + 8 * h);
  }
  residual16(a, s, d, lp, lq, w);
  return block_sum(sum16(w), sh);
}

__device__ __forceinline__ float log_prob(const Seq& s, const RowStat& p, uint16_t bits) {
  const float l = bf2f(bits);
  return (float)((l == p.top ? 0.0 : (double)(l - p.top) / (double)s.heat) - log(p.total));
}

// The weight of one token, also below what fp32 holds: two that are both too small for it still compare.
__device__ __forceinline__ double token_weight(const Seq& s, float l, float top) {
  const float w = any_weight(s, l, top);
  return w >= 0x1p-100f || !(l > -INFINITY) || top == INFINITY ? (double)w : exp((double)(l - top) / (double)s.heat);
}

// What the decision on draft j needs besides the sums: loaded before they are there.
struct Draft {
  int x;
  float u, lp, lq;
};
__device__ __forceinline__ Draft load_draft(const VerifyArgs& a, const Seq& s, int j) {
  Draft d{a.ids[(size_t)s.id * a.t + j], a.u[(size_t)s.id * (a.t + 1) + j], -INFINITY, -INFINITY};
  if (d.x >= 0 && d.x < a.vocab) {
    d.lp = bf2f(target_row(a, s.id, j)[d.x]);
    if (a.draft) d.lq = bf2f(draft_row(a, s.id, j)[d.x]);
  } else {
    d.x = -1;
  }
  return d;
}
__device__ __forceinline__ bool accept(const VerifyArgs& a, const Seq& s, const Draft& d, const RowStat& p, const RowStat& q) {
  if (d.x < 0 || p.best < 0) return false;
  if (s.greedy) return d.x == p.best;
  double qx = 1.0;
  if (a.draft) qx = q.best < 0 ? 0.0 : token_weight(s, d.lq, q.top) / q.total;
  return d.u * qx < token_weight(s, d.lp, p.top) / p.total;
}
__device__ __forceinline__ void put_accepted(const VerifyArgs& a, const Seq& s, int j, const RowStat& p) {
  const int x = a.ids[(size_t)s.id * a.t + j];
  a.tokens[(size_t)s.id * (a.t + 1) + j] = x;
  if (a.logp) a.logp[(size_t)s.id * (a.t + 1) + j] = log_prob(s, p, target_row(a, s.id, j)[x]);
}
__device__ __forceinline__ Decision decision(const VerifyArgs& a, const Seq& s, int j, const RowStat& p, const RowStat& q) {
  return Decision{j, j < s.n && a.draft && !s.greedy && p.best >= 0 && q.best >= 0, p, q};
}

// Draws and stores the next token and that nothing follows it.  st: the chunks of target row d.j; sum: thread c's chunk of
// the residual weights, where the decision asks for them; rest: see draw_target, of a rejected lone_draft.
__device__ __forceinline__ void finish(const VerifyArgs& a, const Seq& s, const Decision& d, const RowStat* st, double sum,
                                       double rest, Shared& sh) {
  int token = -1;
  if (s.greedy || d.p.best < 0) {
    token = d.p.best;
  } else {
    if (d.residual) {
      const uint16_t *const p = target_row(a, s.id, d.j), *const q = draft_row(a, s.id, d.j);
      auto weigh = [&](int k, float(&w)[kEach]) {
        float lp[kEach], lq[kEach];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load8(p, k + 8 * h, a.vocab, lp + 8 * h);
          load8(q, k + 8 * h, a.vocab, lq + 8 * h);
        }
        residual16(a, s, d, lp, lq, w);
      };
      token = find_token(a, s.next_u, sum, weigh, sh);
    } else {
      const int x = lone_draft(a, s, d.j);
      if (x >= 0) token = draw_target(a, s, d.j, st, d.p, x, rest, sh);
    }
    if (token < 0) token = draw_target(a, s, d.j, st, d.p, -1, 0.0, sh);  // also where nothing is left of p - q
  }
  const size_t at = (size_t)s.id * (a.t + 1);
  for (int i = d.j + (int)threadIdx.x; i <= a.t; i += kThreads) {
    a.tokens[at + i] = i == d.j ? token : -1;
    if (a.logp) a.logp[at + i] = i == d.j && token >= 0 ? log_prob(s, d.p, target_row(a, s.id, d.j)[token]) : 0.0f;
  }
  if (threadIdx.x == 0) a.accepted[s.id] = d.j;
}

// One chunk of one row that its sequence's decision may need.
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const VerifyArgs a) {
  __shared__ Shared sh;
  const int chunk = blockIdx.x, row = blockIdx.y;
  const Seq s = seq_of(a, blockIdx.z);
  const bool of_target = row <= a.t;
  if (of_target ? row > s.n : s.greedy || row - a.t - 1 >= s.n) return;
  const RowStat r =
      chunk_stat(s, of_target ? target_row(a, s.id, row) : draft_row(a, s.id, row - a.t - 1), chunk, a.vocab,
                 of_target ? lone_draft(a, s, row) : -1, a.rest + (size_t)s.id * a.t + row, sh);
  if (threadIdx.x == 0) a.stats[((size_t)s.id * a.rows + row) * a.chunks + chunk] = r;
}

// A sequence's drafts in order, as many at a time as the workgroup has waves; then its next token (DRAFT: one chunk of the
// weights that it may be drawn from).
template <bool DRAFT>
__global__ void __launch_bounds__(kThreads) verify_decide_kernel(const VerifyArgs a) {
  __shared__ Shared sh;
  const int chunk = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const Seq s = seq_of(a, blockIdx.y);
  const RowStat* const st = a.stats + (size_t)s.id * a.rows * a.chunks;
  Decision d;
  for (int j0 = 0;; j0 += kWaves) {
    const int j = j0 + w;
    if (j <= s.n) {
      const bool drafted = DRAFT && !s.greedy && j < s.n;
      const Chunks pc = load_chunks(st + (size_t)j * a.chunks, a.chunks);
      const Chunks qc = load_chunks(st + (size_t)(drafted ? a.t + 1 + j : j) * a.chunks, DRAFT ? a.chunks : 0);
      const Draft x = j < s.n ? load_draft(a, s, j) : Draft{-1, 0.0f, 0.0f, 0.0f};
      const RowStat p = row_stat(s, pc), q = drafted ? row_stat(s, qc) : p;
      if (lane == 0) sh.p[w] = p, sh.q[w] = q, sh.ok[w] = accept(a, s, x, p, q);
    }
    __syncthreads();
    int n = 0;  // place j0 + n is the first that is not an accepted draft (place s.n never is)
    while (n < kWaves && sh.ok[n]) ++n;
    if ((!DRAFT || chunk == 0) && lane == 0 && w < n) put_accepted(a, s, j, sh.p[w]);
    if (n < kWaves) {
      d = decision(a, s, j0 + n, sh.p[n], sh.q[n]);
      break;
    }
    __syncthreads();
  }
  if (!DRAFT) {
    finish(a, s, d, st + (size_t)d.j * a.chunks, 0.0, d.j < s.n ? a.rest[(size_t)s.id * a.t + d.j] : 0.0, sh);
    return;
  }
  if (chunk == 0 && threadIdx.x == 0) a.plan[s.id] = d;
  if (!d.residual) return;
  const double sum = residual_sum(a, s, d, chunk, sh);
  if (threadIdx.x == 0) a.sums[(size_t)s.id * a.chunks + chunk] = sum;
}

__global__ void __launch_bounds__(kThreads) verify_draw_kernel(const VerifyArgs a) {
  __shared__ Shared sh;
  const Seq s = seq_of(a, blockIdx.x);
  const int c = threadIdx.x;
  const double sum = c < a.chunks ? a.sums[(size_t)s.id * a.chunks + c] : 0.0;  // (nothing yet, and unused, without a residual)
  const Decision d = a.plan[s.id];
  finish(a, s, d, a.stats + ((size_t)s.id * a.rows + d.j) * a.chunks, sum, 0.0, sh);
}

// All of a sequence in one workgroup, row after row.
__global__ void __launch_bounds__(kThreads) verify_whole_kernel(const VerifyArgs a) {
  __shared__ Shared sh;
  __shared__ RowStat st[2][kMaxChunks];
  __shared__ double rest;
  const Seq s = seq_of(a, blockIdx.x);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  Decision d;
  for (int j = 0;; ++j) {
    const bool drafted = a.draft && !s.greedy && j < s.n;
    for (int c = 0; c < a.chunks; ++c) {
      const RowStat r = chunk_stat(s, target_row(a, s.id, j), c, a.vocab, lone_draft(a, s, j), &rest, sh);
      if (threadIdx.x == 0) st[0][c] = r;
      if (!drafted) continue;
      const RowStat q = chunk_stat(s, draft_row(a, s.id, j), c, a.vocab, -1, nullptr, sh);
      if (threadIdx.x == 0) st[1][c] = q;
    }
    __syncthreads();
    if (w == 0) {
      const RowStat p = row_stat(s, load_chunks(st[0], a.chunks));
      const RowStat q = drafted ? row_stat(s, load_chunks(st[1], a.chunks)) : p;
      const Draft x = j < s.n ? load_draft(a, s, j) : Draft{-1, 0.0f, 0.0f, 0.0f};
      if (lane == 0) {
        sh.p[0] = p, sh.q[0] = q, sh.ok[0] = accept(a, s, x, p, q);
        if (sh.ok[0]) put_accepted(a, s, j, p);
      }
    }
    __syncthreads();
    if (!sh.ok[0]) {
      d = decision(a, s, j, sh.p[0], sh.q[0]);
      break;
    }
  }
  double sum = 0.0;
  for (int c = 0; d.residual && c < a.chunks; ++c) {
    const double x = residual_sum(a, s, d, c, sh);
    if (c == (int)threadIdx.x) sum = x;
  }
  finish(a, s, d, st[0], sum, rest, sh);
}

VerifyArgs from(VerifyArgs a, int seq) {
  const size_t i = (size_t)seq;
  a.target += i * (a.t + 1) * a.ldt;
  if (a.draft) a.draft += i * a.t * a.ldd;
  if (a.ids) a.ids += i * a.t;
  if (a.counts) a.counts += i;
  if (a.temp) a.temp += i;
  if (a.logp) a.logp += i * (a.t + 1);
  a.u += i * (a.t + 1), a.tokens += i * (a.t + 1), a.accepted += i;
  return a;
}

int launch(VerifyArgs a, int b, hipStream_t st) {
  a.chunks = (a.vocab + kChunk - 1) / kChunk;
  a.rows = a.t + 1 + (a.draft ? a.t : 0);
  const size_t per = (size_t)a.chunks * (a.rows * sizeof(RowStat) + sizeof(double)) + sizeof(Decision) + a.t * sizeof(double);
  const size_t most = kMaxScratch / per < 65535 ? kMaxScratch / per : 65535;  // (per <= 1.1 MB; a grid's y and z axes)
  const int each = b < (int)most ? b : (int)most;
  std::lock_guard<std::mutex> lock(scratch_mutex(st));  // the launches that share the scratch stay together
  uint8_t* const z = call_scratch(st, per * each, ScratchOf::kOperators).data;
  if (!z) {
    hipLaunchKernelGGL(verify_whole_kernel, dim3((unsigned)b), dim3(kThreads), 0, st, a);
    return (int)hipGetLastError();
  }
  a.stats = reinterpret_cast<RowStat*>(z);
  a.plan = reinterpret_cast<Decision*>(a.stats + (size_t)each * a.rows * a.chunks);
  a.sums = reinterpret_cast<double*>(a.plan + each);
  a.rest = a.sums + (size_t)each * a.chunks;
  for (int i = 0; i < b; i += each) {
    const VerifyArgs l = from(a, i);
    const unsigned n = (unsigned)(b - i < each ? b - i : each), chunks = (unsigned)a.chunks;
    hipLaunchKernelGGL(verify_rows_kernel, dim3(chunks, (unsigned)a.rows, n), dim3(kThreads), 0, st, l);
    if (const int e = (int)hipGetLastError()) return e;
    if (a.draft) {
      hipLaunchKernelGGL(verify_decide_kernel<true>, dim3(chunks, n), dim3(kThreads), 0, st, l);
      if (const int e = (int)hipGetLastError()) return e;
      hipLaunchKernelGGL(verify_draw_kernel, dim3(n), dim3(kThreads), 0, st, l);
    } else {
      hipLaunchKernelGGL(verify_decide_kernel<false>, dim3(1, n), dim3(kThreads), 0, st, l);
    }
    if (const int e = (int)hipGetLastError()) return e;
  }
  return 0;
}

}  // namespace
}  // namespace agq

extern "C" int ak_spec_verify(const void* target, long ldt, const void* draft, long ldd, const int* ids,
                              const int* counts, const float* u, const float* temperature, int b, int t, int vocab,
                              int* tokens, int* accepted, float* logp, void* stream) {
  if (b < 0 || t < 0 || t > AK_VERIFY_MAX_DRAFTS || vocab < 1 || vocab > AK_VERIFY_MAX_VOCAB || ldt < vocab ||
      (draft && t && ldd < vocab))
    return AK_INVALID;
  if (!b) return 0;
  if (!target || (t && !ids) || !u || !tokens || !accepted) return AK_INVALID;
  agq::VerifyArgs a{};
  a.target = static_cast<const uint16_t*>(target);
  a.draft = t ? static_cast<const uint16_t*>(draft) : nullptr;
  a.ids = ids, a.counts = counts, a.u = u, a.temp = temperature;
  a.tokens = tokens, a.accepted = accepted, a.logp = logp;
  a.ldt = ldt, a.ldd = ldd, a.t = t, a.vocab = vocab;
  try {  // (the scratch's bookkeeping allocates host memory)
    return agq::launch(a, b, static_cast<hipStream_t>(stream));
  } catch (...) {
    return AK_OOM;
  }
}
