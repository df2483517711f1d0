// Pages for a batch's new tokens off a free list, and where every token goes: positions, cache slots, ranges.
//
// The sequences are one workgroup's work, a thread a sequence: exclusive sums of the new tokens (their ranges), of the pages
// that ended sequences give back, and of the pages wanted; a sequence gets its pages if those wanted up to it are there, so
// the first that goes short leaves all later ones without new pages too.  Pages move as one flat list each way, a thread a
// page, which finds its sequence by bisecting the sums.  So do tokens.
//
// All of it is a chain of round trips.  Inputs and outputs may be the same arrays: every thread has read its sequence's
// numbers before the first barrier, and nothing is written before it.
#include "agens_kernels.h"
#include "kv_page.h"

namespace agq {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
static_assert(kPlanThreads >= AK_PLAN_MAX_SEQS, "a thread a sequence");

struct PlanArgs {
  const int *counts, *drop, *cached, *held, *free_count;
  int *free_pages, *table, *lens, *held_out, *free_out, *qstart, *pos, *slots, *refused;
  int b, m, npages, page_log2, ldt;
};

// the sum of x over the threads up to this one; *total: over all.  Sums below 2^31.
__device__ __forceinline__ int block_scan(int x, int* red, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) red[w] = x;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
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

__global__ void __launch_bounds__(kPlanThreads) plan_seqs_kernel(const PlanArgs a, int tokens_too) {
  __shared__ int red[kPlanWaves];
  __shared__ int at[kPlanThreads + 1], from[kPlanThreads], to[kPlanThreads];
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
  // what ended sequences held
  int total_back = 0;
  if (pages) {
    const int up = block_scan(back, red, &total_back);
    at[i] = up - back;
    __syncthreads();
    for (int e = i; e < total_back; e += kPlanThreads) {
      const int s = range_of(at, a.b, e);
      if (stack + e < a.npages) a.free_pages[stack + e] = a.table[(size_t)s * a.ldt + e - at[s]];
    }
  }
  const int avail = min(stack + total_back, a.npages);
  int total;
  const int end = block_scan(count, red, &total), start = end - count;
  const long room = (long)a.ldt << a.page_log2, after = (long)n + count;
  bool no = after > room || end > a.m;
  int want = 0;
  if (pages && !no) want = max((int)((after + (1 << a.page_log2) - 1) >> a.page_log2) - h, 0);
  int all;
  const int upto = block_scan(want, red, &all);
  no = no || (want > 0 && upto > avail);
  const int take = no ? 0 : want;
  int taken;
  const int base = block_scan(take, red, &taken) - take;  // (= upto - want: those refused come after)
  // (block_scan's barriers lie between the pages' way back and their way out)
  at[i] = base, from[i] = h;
  __syncthreads();
  for (int e = i; e < taken; e += kPlanThreads) {
    const int s = range_of(at, a.b, e);
    a.table[(size_t)s * a.ldt + from[s] + e - at[s]] = a.free_pages[avail - 1 - e];
  }
  if (mine) {
    a.lens[i] = (int)(no ? n : after);
    a.refused[i] = no;
    a.qstart[i] = min(start, a.m);
    if (pages) a.held_out[i] = h + take;
  }
  if (i == 0) {
    a.qstart[a.b] = min(total, a.m);
    if (pages) a.free_out[0] = avail - taken;
  }
  if (!tokens_too) return;
  __syncthreads();
  at[i] = min(start, a.m), to[i] = no ? -1 : n;
  __syncthreads();
  for (int t = i; t < a.m; t += kPlanThreads) {
    const int s = a.b ? range_of(at, a.b, t) : 0;
    const bool there = t < total && to[s] >= 0;
    put_token(a, t, s, at[s], there ? to[s] + t - at[s] : -1);
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
  hipLaunchKernelGGL(agq::plan_seqs_kernel, dim3(1), dim3(agq::kPlanThreads), 0, s, a, one ? 1 : 0);
  if (const int e = (int)hipGetLastError()) return e;
  if (one) return 0;
  hipLaunchKernelGGL(agq::plan_tokens_kernel, dim3((unsigned)(m + 255) / 256), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
