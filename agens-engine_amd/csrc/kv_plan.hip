// Pages for a batch's new tokens off a free list, and where every token goes: positions, cache slots, ranges.
//
// The sequences are one workgroup's work, a thread a sequence: exclusive sums of the new tokens (their ranges), of the pages
// that ended sequences give back, and of the pages wanted; a sequence gets its pages if those wanted up to it are there, so
// the first that goes short leaves all later ones without new pages too.  Pages move as one flat list each way, a thread a
// page, which finds its sequence by bisecting the sums.  So do tokens.
//
// All of it is a chain of round trips to memory and barriers: 2.2 us for one sequence, 7.3 and 3.4 for 200 with 20000 new tokens,
// whose 0.2 MB are nothing.  Few sequences with few pages take four waves instead of sixteen, whose barriers are shorter.  Inputs and
// outputs may be the same arrays: every thread has read its sequence's numbers before the first barrier, and nothing is written
// before it.
#include "agens_kernels.h"
#include "kv_page.h"
#include "logits.h"

namespace agq {
namespace {

constexpr int kPlanThreads = 1024, kFewThreads = 256;
static_assert(kPlanThreads >= AK_PLAN_MAX_SEQS, "a thread a sequence");

struct PlanArgs {
  const int *counts, *drop, *cached, *held, *free_count;
  int *free_pages, *table, *lens, *held_out, *free_out, *qstart, *pos, *slots, *refused;
  int b, m, npages, page_log2, ldt;
};

struct AddInt {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ int step(int x) const {
    return x + (int)dpp<CTRL, ROWS>((uint32_t)x, 0);
  }
};
// the sum of x over the threads up to this one; *total: over all.  Sums below 2^31.  One barrier; red: this scan's own.
template <int WAVES>
__device__ __forceinline__ int block_scan(int x, int* red, int* total) {
  const int w = threadIdx.x >> 6;
  x = wave_scan(x, AddInt());
  if ((threadIdx.x & 63) == 63) red[w] = x;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i < w) x += red[i];
    all += red[i];
  }
  *total = all;
  return x;
}

// the last of n entries of the ascending `at` (at[0] = 0) that is not above e
__device__ __forceinline__ int range_of(const int* at, int n, int e) {
  int lo = 0;
  for (int hi = n; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= e)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void put_token(const PlanArgs& a, int t, int i, int first, int p) {
  int slot = -1;
  if (p >= 0) {
    const int pg = a.table[(size_t)i * a.ldt + (p >> a.page_log2)];
    if (pg >= 0 && pg < a.npages) slot = (pg << a.page_log2) + (p & ((1 << a.page_log2) - 1));
  }
  a.pos[t] = p;
  a.slots[t] = slot;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) plan_seqs_kernel(const PlanArgs a, int tokens_too) {
  constexpr int kWaves = THREADS / 64;
  __shared__ int red[3][kWaves], granted;
  __shared__ int at[THREADS], from[THREADS];
  const int i = threadIdx.x;
  const bool mine = i < a.b, pages = a.free_pages != nullptr;
  int count = 0, n = 0, h = 0, back = 0;
  if (mine) {
    count = min(max(a.counts[i], 0), a.m + 1);  // (more than m is refused, however many)
    n = max(a.cached[i], 0);
    if (pages) h = min(max(a.held[i], 0), a.ldt);
    if (a.drop && a.drop[i]) back = h, n = 0, h = 0;
  }
  const int stack = pages ? min(max(a.free_count[0], 0), a.npages) : 0;
  if (i == 0) granted = 0;
  int total, total_back = 0;
  const int end = block_scan<kWaves>(count, red[0], &total), start = end - count;
  if (pages && a.drop) {  // what ended sequences held
    const int up = block_scan<kWaves>(back, red[1], &total_back);
    if (total_back) {
      at[i] = up - back;
      __syncthreads();
      for (int e0 = i; e0 < total_back; e0 += 4 * THREADS) {  // four on their way at a time
        int page[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = min(e0 + j * THREADS, total_back - 1), s = range_of(at, a.b, e);
          page[j] = a.table[(size_t)s * a.ldt + e - at[s]];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = e0 + j * THREADS;
          if (e < total_back && stack + e < a.npages) a.free_pages[stack + e] = page[j];
        }
      }
    }
  }
  const int avail = min(stack + total_back, a.npages);
  const long room = (long)a.ldt << a.page_log2, after = (long)n + count;
  bool no = after > room || after > 0x7FFFFFFF || end > a.m;
  int want = 0, taken = 0;
  if (pages) {
    if (!no) want = max((int)((after + (1 << a.page_log2) - 1) >> a.page_log2) - h, 0);
    int all;
    const int upto = block_scan<kWaves>(want, red[2], &all);  // (its barrier: the pages given back are in the list)
    if (all) {
      at[i] = upto - want, from[i] = h;
      no = no || (want > 0 && upto > avail);
      if (no)
        want = 0;
      else if (want)
        atomicMax(&granted, upto);  // (those refused for want of pages come after)
      __syncthreads();
      taken = granted;
      for (int e = i; e < taken; e += THREADS) {
        const int s = range_of(at, a.b, e);
        a.table[(size_t)s * a.ldt + from[s] + e - at[s]] = a.free_pages[avail - 1 - e];
      }
    }
  }
  if (mine) {
    a.lens[i] = (int)(no ? n : after);
    a.refused[i] = no;
    a.qstart[i] = min(start, a.m);
    if (pages) a.held_out[i] = h + want;
  }
  if (i == 0) {
    a.qstart[a.b] = min(total, a.m);
    if (pages) a.free_out[0] = avail - taken;
  }
  if (!tokens_too) return;
  __syncthreads();
  at[i] = min(start, a.m), from[i] = no ? -1 : n;
  __syncthreads();
  for (int t = i; t < a.m; t += THREADS) {
    const int s = a.b ? range_of(at, a.b, t) : 0;
    const bool there = t < total && from[s] >= 0;
    put_token(a, t, s, at[s], there ? from[s] + t - at[s] : -1);
  }
}

// The tokens, from what the sequences' kernel wrote.
__global__ void __launch_bounds__(256) plan_tokens_kernel(const PlanArgs a) {
  __shared__ int at[kPlanThreads + 1];
  for (int i = threadIdx.x; i <= a.b; i += 256) at[i] = a.qstart[i];
  __syncthreads();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.m) return;
  const int s = a.b ? range_of(at, a.b, t) : 0;
  int p = -1;
  if (t < at[a.b] && !a.refused[s]) p = a.lens[s] - (at[s + 1] - t);
  put_token(a, t, s, at[s], p);
}

constexpr int kTokensInOne = 4096;

}  // namespace
}  // namespace agq

extern "C" int ak_kv_plan(int b, int m, const int* counts, const int* drop, const int* cached, const int* held,
                          const int* free_count, int* free_pages, int npages, int page, int* table, int ldt, int* lens,
                          int* held_out, int* free_out, int* qstart, int* pos, int* slots, int* refused, void* stream) {
  if (b < 0 || b > AK_PLAN_MAX_SEQS || m < 0 || m > AK_PLAN_MAX_TOKENS || page < agq::kPageMin || page > agq::kPageMax ||
      page & (page - 1) || npages < 1 || (long)npages * page > 0x7FFFFFFFL || ldt < 1 || (long)b * ldt > 1L << 30)
    return AK_INVALID;
  if (!qstart || (b && (!counts || !cached || !table || !lens || !refused)) || (m && (!pos || !slots))) return AK_INVALID;
  if (free_pages && (!free_count || !free_out || (b && (!held || !held_out)))) return AK_INVALID;
  const agq::PlanArgs a{counts, drop, cached, held, free_count, free_pages, table, lens, held_out, free_out, qstart, pos,
                        slots, refused, b, m, npages, __builtin_ctz((unsigned)page), ldt};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool one = m <= agq::kTokensInOne;
  // Four waves: shorter barriers, but fewer pages and tokens at a time.  One sequence of 8192 new tokens, 512 pages, 5.5 us and
  // 5.9 with sixteen; 16 of 4096, 4096 pages, 12.2 and 8.3; 64 of 8192, 32768 pages, 76 and 27.  How many pages come back nobody
  // knows here: an eighth of what the rows can hold counts (64 rows of 1024 pages, some of them ended, 17 and 11 us), in steps of
  // few tokens none.
  const bool few = one ? m <= 4 * agq::kFewThreads : m / page + (drop ? (long)b * ldt / 8 : 0) <= 4 * agq::kFewThreads;
  if (b <= 64 && few)
    hipLaunchKernelGGL(agq::plan_seqs_kernel<agq::kFewThreads>, dim3(1), dim3(agq::kFewThreads), 0, s, a, one ? 1 : 0);
  else
    hipLaunchKernelGGL(agq::plan_seqs_kernel<agq::kPlanThreads>, dim3(1), dim3(agq::kPlanThreads), 0, s, a, one ? 1 : 0);
  if (const int e = (int)hipGetLastError()) return e;
  if (one) return 0;
  hipLaunchKernelGGL(agq::plan_tokens_kernel, dim3((unsigned)(m + 255) / 256), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
