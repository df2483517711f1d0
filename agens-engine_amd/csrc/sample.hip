// One token of each row of logits after temperature, top-k, top-p and min-p, from given uniform numbers.
//
// Weights are exp((l - top) / T), top the row's largest logit.  The tokens stand in order of falling logit, the lower token
// first among equal ones; top-k keeps the first k of them; top-p the fewest of these, from the front, whose weights reach
// top_p of theirs all; min-p drops those below min_p of the largest.  So what is kept is a front of that order, and the token
// is the first, in order of tokens, at which the sum of the kept weights passes u times their total.
//
// A logit has 16 bits, so equal ones are many and its bits, made to ascend with the value (`key`), index everything: a
// histogram of a row's keys holds all counts, and all weights as counts times the weight of a key.  The weights enter sums as
// whole numbers of 2^-42 of the largest, 2^20 of which fit 64 bits: sums are exact, in any order, so which way they were
// reached does not show in the tokens.
//
//   sample_keys_kernel   a chunk of 16384 logits a workgroup: its largest, its lowest token with that, the sum of its weights
//                        (16 in 32 bits, then 64), and how often each of the kWindow keys up to its largest occurs;
//   sample_draw_kernel   a row a workgroup: the chunks' windows, shifted to the row's largest key, give the border of what is
//                        kept, and what each chunk has of it; then the chunk that the draw falls into is read again.  Where
//                        the border is below the window, it goes over the row itself, kWide keys at a time.
// Without scratch sample_draw_kernel takes the chunks' statistics itself and does without their windows: the same tokens.
#include "agens_kernels.h"
#include "logits.h"

namespace agq {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kEach = 16, kChunk = kThreads * kEach;
constexpr int kMaxChunks = 64;  // of a row: a lane of a wave each
static_assert(kMaxChunks * kChunk == AK_SAMPLE_MAX_VOCAB, "the header's limit");
constexpr int kWindow = 1024, kWide = 8 * kThreads;
constexpr float kMaxHeat = 1.44e30f;  // (see heat_of)
constexpr float kUnit = 0x1p42f;
constexpr size_t kMaxScratch = (size_t)64 << 20;
constexpr uint32_t kLowest = 0x007F;  // key of -inf, and of NaN

struct ChunkStat {
  float top;
  int best;  // the lowest token with it; -1: nothing above -inf
  double total;
};

struct SampleArgs {
  const uint16_t* logits;
  long ld;
  const float *temp, *top_p, *min_p, *u;
  const int* top_k;
  int* tokens;
  float* logp;
  int b, vocab, chunks;
  ChunkStat* stats;  // [b][chunks]
  uint16_t* counts;  // [b][chunks][kWindow]: key of the chunk's largest - i
};

__device__ __forceinline__ uint32_t key_of(uint32_t bits) {
  if ((bits & 0x7FFFu) > 0x7F80u) return kLowest;  // NaN
  if (bits == 0x8000u) bits = 0;                   // -0 equals 0
  return bits & 0x8000u ? 0xFFFFu - bits : bits + 0x8000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return bf2f(key & 0x8000u ? key - 0x8000u : 0xFFFFu - key);
}
__device__ __forceinline__ uint32_t key_of_value(float l) { return key_of(__float_as_uint(l) >> 16); }

// in whole numbers of 2^-42
__device__ __forceinline__ uint64_t units(float w) { return (uint64_t)(w * kUnit); }
__device__ __forceinline__ float key_weight(const Heat& s, uint32_t key, float top) {
  return any_weight(s, logit_of(key), top);
}

struct Shared {
  double red[kWaves], before[kWaves];
  uint64_t sum[kWaves];
  int ired[kWaves], ok[kWaves];
  uint64_t mass[kMaxChunks];  // of the chunks: what is kept
  uint32_t at_border[kMaxChunks];
  uint32_t bins[kWide];
  uint32_t next;  // the largest key below the window
  uint64_t border;
  int chunk;
  double at;
};

template <class T>
__device__ __forceinline__ T shfl_up64(T x, int d) {
  return (T)__shfl_up((unsigned long long)x, d);
}
// The sum over the threads up to this one; *total over all.
__device__ __forceinline__ uint64_t scan(uint64_t x, Shared& sh, uint64_t* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t y = shfl_up64(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) sh.sum[w] = x;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) x += sh.sum[i];
    all += sh.sum[i];
  }
  *total = all;
  return x;
}

// A chunk: see ChunkStat.  bins: where to count its keys (kWindow, zeros), or null.
__device__ __forceinline__ ChunkStat chunk_stat(const Heat& s, const uint16_t* row, int chunk, int vocab, uint32_t* bins,
                                                Shared& sh) {
  const int t = threadIdx.x, at0 = chunk * kChunk + 8 * t, at1 = at0 + kChunk / 2;
  float l[kEach];
  load8(row, at0, vocab, l);
  load8(row, at1, vocab, l + 8);
  float mine = l[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) mine = fmaxf(mine, l[i]);
  const float wtop = wave_max(mine);
  __syncthreads();
  if ((t & 63) == 0) sh.red[t >> 6] = wtop;
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) top = fmaxf(top, (float)sh.red[i]);
  int best = 0x7FFFFFFF;
  if (mine == top && top > -INFINITY) {
#pragma unroll
    for (int i = kEach - 1; i >= 0; --i)
      if (l[i] == top) best = (i < 8 ? at0 : at1 - 8) + i;
  }
  best = wave_min(best);
  if (bins && top > -INFINITY) {
    const uint32_t high = key_of_value(top);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint32_t key = key_of_value(l[i]), d = high - key;
      if (d < kWindow && key != kLowest) atomicAdd(&bins[d], 1u);  // (-inf weighs nothing)
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += any_weight(s, l[i], top);
  const double wsum = wave_sum((double)sum);
  __syncthreads();
  if ((t & 63) == 0) sh.red[t >> 6] = wsum, sh.ired[t >> 6] = best;
  __syncthreads();
  ChunkStat r{top, 0x7FFFFFFF, 0.0};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) r.total += sh.red[i], r.best = min(r.best, sh.ired[i]);
  if (r.best == 0x7FFFFFFF) r.best = -1;
  return r;
}

__global__ void __launch_bounds__(kThreads) sample_keys_kernel(const SampleArgs a) {
  __shared__ Shared sh;
  const int chunk = blockIdx.x, id = blockIdx.y;
  const Heat s = heat_of(a.temp ? a.temp[id] : 1.0f);
  sh.bins[threadIdx.x] = 0;  // (a barrier follows before the first count)
  const ChunkStat r = chunk_stat(s, a.logits + (size_t)id * a.ld, chunk, a.vocab, sh.bins, sh);
  const size_t at = (size_t)id * a.chunks + chunk;
  if (threadIdx.x == 0) a.stats[at] = r;
  a.counts[at * kWindow + threadIdx.x] = (uint16_t)sh.bins[threadIdx.x];
}

// What is kept: keys above `key` and the first `n` tokens with it, of weights from `least` on.
struct Border {
  uint32_t key, n;
  float least;
};

struct Row {
  Heat s;
  const uint16_t* logits;
  const ChunkStat* stats;   // (in LDS)
  const uint16_t* counts;   // null: none
  float top;
  int best, vocab, chunks;
  double total;
  uint32_t high;            // key of top
};

// Keys high - first, high - first - 1, ...: how often they occur.  `each` of them a thread, in its place of n.
// The chunks' windows:
__device__ __forceinline__ uint32_t count_window(const Row& r) {
  uint32_t n = 0;
  for (int c = 0; c < r.chunks; ++c) {
    const float top = r.stats[c].top;
    if (top == -INFINITY) continue;
    const int i = (int)threadIdx.x - (int)(r.high - key_of_value(top));
    if (i >= 0) n += r.counts[(size_t)c * kWindow + i];
  }
  return n;
}
// the row itself, into sh.bins; sh.next: the largest key below
__device__ __forceinline__ void count_wide(const Row& r, uint32_t high, Shared& sh) {
  __syncthreads();
  for (int i = threadIdx.x; i < kWide; i += kThreads) sh.bins[i] = 0;
  if (threadIdx.x == 0) sh.next = 0;
  __syncthreads();
  uint32_t next = 0;
  for (int k = 8 * threadIdx.x; k < r.vocab; k += 8 * kThreads) {
    float l[8];
    load8(r.logits, k, r.vocab, l);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t key = key_of_value(l[i]);
      const int d = (int)high - (int)key;
      if (d < 0 || key == kLowest) continue;
      if (d < kWide)
        atomicAdd(&sh.bins[d], 1u);
      else
        next = max(next, key);
    }
  }
  if (next) atomicMax(&sh.next, next);
  __syncthreads();
}

// The place in the order where a sum reaches `goal` (> 0): over counts (by_weight false) or weights; tokens past `limit` (a
// border) count as not there.  key 0: nowhere.  Whole workgroup; the same in every thread.
__device__ Border find(const Row& r, bool by_weight, uint64_t goal, const Border& limit, Shared& sh) {
  uint64_t done = 0;
  const bool quick = r.counts != nullptr;
  uint32_t high = r.high;
  for (bool first = quick;; first = false) {
    const int each = first ? 1 : kWide / kThreads;
    uint32_t n[kWide / kThreads];
    if (first) {
      n[0] = count_window(r);
    } else {
      count_wide(r, high, sh);
      for (int i = 0; i < each; ++i) n[i] = sh.bins[threadIdx.x * each + i];
    }
    uint64_t mine = 0;
    const uint32_t k0 = high - threadIdx.x * each;
    auto amount = [&](int i) {  // of key k0 - i
      const uint32_t key = k0 - i;
      uint32_t m = n[i];
      if (!m) return (uint64_t)0;
      if (key < limit.key) m = 0;
      if (key == limit.key) m = min(m, limit.n);
      return by_weight ? m * units(key_weight(r.s, key, r.top)) : (uint64_t)m;
    };
    for (int i = 0; i < each; ++i) mine += amount(i);
    uint64_t total;
    const uint64_t upto = scan(mine, sh, &total);
    if (done + total >= goal) {
      uint64_t sum = done + upto - mine;
      if (sum < goal && sum + mine >= goal) {
        for (int i = 0; i < each; ++i) {
          const uint64_t w = amount(i);
          if (sum + w >= goal) {
            const uint64_t one = by_weight ? units(key_weight(r.s, k0 - i, r.top)) : 1;
            sh.border = (uint64_t)((goal - sum + one - 1) / one) << 32 | (k0 - i);
            break;
          }
          sum += w;
        }
      }
      __syncthreads();
      const uint64_t b = sh.border;
      __syncthreads();
      return Border{(uint32_t)b, (uint32_t)(b >> 32), limit.least};
    }
    done += total;
    if (first) {  // the next window begins below this one
      if (high < kWindow) return Border{0, 0, limit.least};
      high -= kWindow;
    } else {
      high = sh.next;
      __syncthreads();
      if (!high) return Border{0, 0, limit.least};
    }
  }
}

// Each chunk's part of what is kept, to sh.mass, and how many tokens with the border's key it may keep, to sh.at_border.
__device__ void chunk_masses(const Row& r, const Border& b, Shared& sh) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // whether the chunks' windows hold all that is kept
  const bool quick = r.counts && r.high >= kWindow &&
                     (b.key > r.high - kWindow || key_weight(r.s, r.high - kWindow, r.top) < b.least);
  __syncthreads();
  if (quick) {
    for (int c = w; c < r.chunks; c += kWaves) {
      const float top = r.stats[c].top;
      const int shift = top == -INFINITY ? kWindow : (int)(r.high - key_of_value(top));
      uint64_t sum = 0;
      uint32_t same = 0;
      for (int j = lane; j < kWindow; j += 64) {
        const uint32_t key = r.high - j;
        if (j < shift || key < b.key) continue;
        const uint32_t n = r.counts[(size_t)c * kWindow + j - shift];
        if (!n) continue;
        if (key == b.key) {
          same = n;
          continue;
        }
        const float x = key_weight(r.s, key, r.top);
        if (x >= b.least) sum += n * units(x);
      }
      for (int d = 32; d; d /= 2) {
        sum += (uint64_t)__shfl_xor((unsigned long long)sum, d);
        same += __shfl_xor(same, d);
      }
      if (lane == 0) sh.mass[c] = sum, sh.at_border[c] = same;
    }
    __syncthreads();
  } else {
    for (int c = 0; c < r.chunks; ++c) {
      uint64_t sum = 0;
      int same = 0;
      for (int h = 0; h < 2; ++h) {
        float l[8];
        load8(r.logits, c * kChunk + h * kChunk / 2 + 8 * threadIdx.x, r.vocab, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t key = key_of_value(l[i]);
          same += key == b.key;
          if (key <= b.key) continue;
          const float x = key_weight(r.s, key, r.top);
          if (x >= b.least) sum += units(x);
        }
      }
      uint64_t total, equal;
      scan(sum, sh, &total);
      scan((uint64_t)same, sh, &equal);
      if (threadIdx.x == 0) sh.mass[c] = total, sh.at_border[c] = (uint32_t)equal;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float x = b.key ? key_weight(r.s, b.key, r.top) : 0.0f;
    uint32_t left = x >= b.least ? b.n : 0;
    for (int c = 0; c < r.chunks; ++c) {
      const uint32_t n = min(sh.at_border[c], left);
      left -= n;
      sh.at_border[c] = n;
      sh.mass[c] += n * units(x);
    }
  }
  __syncthreads();
}

// The first thread at which the sum of the threads' x (>= 0) passes `at`, the last with any x if none does, -1 without any;
// *before: the sum of the threads before it.
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
  const int mine = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : -1;
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

// The token of a chunk at which the kept weights pass `at`; n: how many tokens with the border's key it may keep.
__device__ __forceinline__ int draw_in(const Row& r, int chunk, const Border& b, uint32_t n, double at, Shared& sh) {
  const int k = chunk * kChunk + kEach * (int)threadIdx.x;
  float l[kEach];
  load8(r.logits, k, r.vocab, l);
  load8(r.logits, k + 8, r.vocab, l + 8);
  int same = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) same += key_of_value(l[i]) == b.key;
  uint64_t all;
  uint64_t rank = scan((uint64_t)same, sh, &all) - same;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const uint32_t key = key_of_value(l[i]);
    const float x = any_weight(r.s, l[i], r.top);
    bool keep = key > b.key && x >= b.least;
    if (key == b.key) keep = rank++ < n;
    l[i] = keep ? x : 0.0f;
    sum += l[i];
  }
  double before;
  const int who = pick_thread((double)sum, at, sh, &before);
  if (who < 0) return -1;
  if ((int)threadIdx.x == who) {
    int token = -1;
    double c = before;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (l[i] > 0.0f && (token < 0 || c <= at)) token = k + i;
      c += (double)l[i];
    }
    sh.ired[0] = token;
  }
  __syncthreads();
  return sh.ired[0];
}

__global__ void __launch_bounds__(kThreads) sample_draw_kernel(const SampleArgs a) {
  __shared__ Shared sh;
  __shared__ ChunkStat st[kMaxChunks];
  const int id = blockIdx.x, t = threadIdx.x;
  Row r;
  r.s = heat_of(a.temp ? a.temp[id] : 1.0f);
  r.logits = a.logits + (size_t)id * a.ld;
  r.vocab = a.vocab, r.chunks = a.chunks;
  r.counts = a.counts ? a.counts + (size_t)id * a.chunks * kWindow : nullptr;
  if (a.stats) {
    if (t < a.chunks) st[t] = a.stats[(size_t)id * a.chunks + t];
  } else {
    for (int c = 0; c < a.chunks; ++c) {
      const ChunkStat x = chunk_stat(r.s, r.logits, c, a.vocab, nullptr, sh);
      if (t == 0) st[c] = x;
    }
  }
  __syncthreads();
  r.stats = st;
  r.top = -INFINITY, r.best = -1, r.total = 0.0;
  for (int c = 0; c < a.chunks; ++c)
    if (st[c].top > r.top) r.top = st[c].top, r.best = st[c].best;
  for (int c = 0; c < a.chunks; ++c) r.total += st[c].total * (double)any_weight(r.s, st[c].top, r.top);
  int token = r.best;
  if (!r.s.greedy && r.best >= 0) {
    r.high = key_of_value(r.top);
    const int k = a.top_k ? a.top_k[id] : 0;
    const float p = a.top_p ? a.top_p[id] : 1.0f, least = a.min_p ? a.min_p[id] : 0.0f;
    Border b{0, 0, least > 0.0f ? fminf(least, 1.0f) : 0.0f};
    bool limited = b.least > 0.0f;
    if (k > 0 && k < a.vocab) {
      b = find(r, false, (uint64_t)k, b, sh);
      limited |= b.key != 0;
    }
    if (p < 1.0f) {
      double all = r.total * (double)kUnit;
      if (b.key) {
        chunk_masses(r, Border{b.key, b.n, 0.0f}, sh);
        uint64_t sum = 0;
        for (int c = 0; c < a.chunks; ++c) sum += sh.mass[c];
        all = (double)sum;
        __syncthreads();
      }
      const double goal = (double)fmaxf(p, 0.0f) * all;
      const Border q = find(r, true, goal > 1.0 ? (uint64_t)ceil(goal) : 1, b, sh);
      if (q.key) b = q, limited = true;
    }
    const float u = a.u[id];
    double at = 0.0, before = 0.0;
    int chunk = -1;
    if (limited) {
      chunk_masses(r, b, sh);
      uint64_t all = 0, sum = 0;
      for (int c = 0; c < a.chunks; ++c) all += sh.mass[c];
      at = (double)u * (double)all;
      for (int c = 0; c < a.chunks; ++c) {
        const uint64_t x = sh.mass[c];
        if (!x) continue;
        chunk = c, before = (double)sum;
        sum += x;
        if ((double)sum > at) break;
      }
      at = fmax(at - before, 0.0) * (1.0 / (double)kUnit);
    } else {
      double sum = 0.0;
      at = (double)u * r.total;
      for (int c = 0; c < a.chunks; ++c) {
        const double x = st[c].total * (double)any_weight(r.s, st[c].top, r.top);
        if (!(x > 0.0)) continue;
        chunk = c, before = sum;
        sum += x;
        if (sum > at) break;
      }
      at = fmax(at - before, 0.0);
    }
    const uint32_t n = limited && chunk >= 0 ? sh.at_border[chunk] : 0;
    if (chunk >= 0) token = draw_in(r, chunk, b, n, at, sh);
  }
  if (t == 0) {
    a.tokens[id] = token;
    if (a.logp) {
      float lp = 0.0f;
      if (token >= 0) {
        const float l = bf2f(r.logits[token]);
        lp = (float)((l == r.top ? 0.0 : (double)(l - r.top) / (double)fminf(r.s.heat, kMaxHeat)) - log(r.total));
      }
      a.logp[id] = lp;
    }
  }
}

SampleArgs from(SampleArgs a, int row) {
  a.logits += (size_t)row * a.ld;
  if (a.temp) a.temp += row;
  if (a.top_k) a.top_k += row;
  if (a.top_p) a.top_p += row;
  if (a.min_p) a.min_p += row;
  if (a.logp) a.logp += row;
  a.u += row, a.tokens += row;
  return a;
}

int launch(SampleArgs a, hipStream_t st) {
  a.chunks = (a.vocab + kChunk - 1) / kChunk;
  const size_t per = (size_t)a.chunks * (sizeof(ChunkStat) + kWindow * sizeof(uint16_t));
  const size_t most = kMaxScratch / per < 65535 ? kMaxScratch / per : 65535;  // (a grid's y axis)
  const int each = a.b < (int)most ? a.b : (int)most;
  std::lock_guard<std::mutex> lock(scratch_mutex(st));  // the launches that share the scratch stay together
  uint8_t* const z = call_scratch(st, per * each, ScratchOf::kOperators).data;
  if (!z) {
    hipLaunchKernelGGL(sample_draw_kernel, dim3((unsigned)a.b), dim3(kThreads), 0, st, a);
    return (int)hipGetLastError();
  }
  a.stats = reinterpret_cast<ChunkStat*>(z);
  a.counts = reinterpret_cast<uint16_t*>(a.stats + (size_t)each * a.chunks);
  for (int i = 0; i < a.b; i += each) {
    const SampleArgs l = from(a, i);
    const unsigned n = (unsigned)(a.b - i < each ? a.b - i : each);
    hipLaunchKernelGGL(sample_keys_kernel, dim3((unsigned)a.chunks, n), dim3(kThreads), 0, st, l);
    if (const int e = (int)hipGetLastError()) return e;
    hipLaunchKernelGGL(sample_draw_kernel, dim3(n), dim3(kThreads), 0, st, l);
    if (const int e = (int)hipGetLastError()) return e;
  }
  return 0;
}

}  // namespace
}  // namespace agq

extern "C" int ak_sample(const void* logits, long ld, const float* temperature, const int* top_k, const float* top_p,
                         const float* min_p, const float* u, int b, int vocab, int* tokens, float* logp, void* stream) {
  if (b < 0 || vocab < 1 || vocab > AK_SAMPLE_MAX_VOCAB || ld < vocab) return AK_INVALID;
  if (!b) return 0;
  if (!logits || !u || !tokens) return AK_INVALID;
  agq::SampleArgs a{};
  a.logits = static_cast<const uint16_t*>(logits);
  a.ld = ld, a.temp = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p, a.u = u;
  a.b = b, a.vocab = vocab, a.tokens = tokens, a.logp = logp;
  try {  // (the scratch's bookkeeping allocates host memory)
    return agq::launch(a, static_cast<hipStream_t>(stream));
  } catch (...) {
    return AK_OOM;
  }
}
