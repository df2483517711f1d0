// One token of each row of logits after temperature, top-k, top-p and min-p, from given uniform numbers.
//
// Weights are exp((l - top) / T), top the row's largest logit.  The tokens stand in order of falling logit, the lower token
// first among equal ones; top-k keeps the first k of them; top-p the fewest of these, from the front, whose weights reach
// top_p of theirs all; min-p drops those below min_p of the largest.  So what is kept is a front of that order, and the token
// is the first, in order of tokens, at which the sum of the kept weights passes u times their total.
//
// A logit has 16 bits, so equal ones are many and its bits, made to ascend with the value (`key`), index everything: a
// histogram of a row's keys holds all counts, and all weights as counts times the weight of a key.  The weights enter sums as
// whole numbers of 2^-40 of the largest (2^20 of them fit 64 bits, 2^12 a double's 53): sums are exact, in any
// order, so which way they were reached does not show in the tokens.
//
//   sample_keys_kernel   a chunk of 4096 logits a workgroup, held in registers: its largest, its lowest token with that, the
//                        sum of its weights (16 in 32 bits, then 64), and how often each of the kWindow keys up to its
//                        largest, or to the one above where that is even, occurs: windows are shifted by whole pairs;
//   sample_draw_kernel   a row a workgroup: the chunks' windows, shifted to the row's largest key and summed, give the border of
//                        what is kept (one scan of counts and weights serves top-k and top-p, since top-p's border is not
//                        behind top-k's), and what each chunk has of it; then the chunk that the draw falls into is read again.
//                        A window goes down to 2^-4 of a positive largest logit.  Where the border is below it, a sample of the
//                        row leaves few keys for it and one pass lists the logits with these (find_sampled); where that does not
//                        do, the row's keys are counted anew, all at once, and the chunks' shares summed up in another pass.
// Without scratch sample_draw_kernel takes the chunks' statistics itself and does without their windows: the same tokens.
//
// What bounds them: latency, of loads, barriers and one wave's instructions one after another (1 row of 152064: 3.7 us, and then 4.2
// without a filter, 8.6 with one, of which 1.4 the first loads, 1.3 the windows, 1.1 the border, 1.4 the chunks' shares and 2 the
// draw; 32 rows: 5.8 + 11 us, where 9.7 MB at 7 TB/s are 1.4); and instructions where a border is far down: 25 a logit by one
// workgroup, 1 row of 152064 with top-k 50000 52 us where counting all keys in LDS takes 88 (40 cycles for 64 counts), 250 flat rows
// of 100277 63 us and 87 (59 with settings of which a part reaches so far down).
#include "agens_kernels.h"
#include "logits.h"

namespace agq {
namespace {

constexpr int kEach = 16, kGroupThreads = 256, kChunk = kGroupThreads * kEach;
constexpr int kDraw = 512, kWaves = kDraw / 64, kGroups = kDraw / kGroupThreads;
constexpr int kMaxChunks = 256, kLaneChunks = kMaxChunks / 64;  // of a row
static_assert(kMaxChunks * kChunk == AK_SAMPLE_MAX_VOCAB, "the header's limit");
constexpr int kWindow = 512;
static_assert(kWindow == kDraw && kChunk == 8 * kDraw, "a bin of the window and eight logits of a chunk a thread");
static_assert(kWindow == 2 * kGroupThreads, "two bins a thread");
// Bins of all keys that matter: kSpan from the largest down, zero's, and the rest up from the least with any weight.
constexpr int kSpan = 4096, kBins = 2 * kSpan, kBinsEach = kBins / kDraw;
// Where a sample narrows the border down: its logits and its bins, and how many logits a wave lists.
constexpr int kSample = 16 * kDraw, kSampleBins = 4 * kDraw, kPiece = kChunk / 2, kList = 2048 - 64, kListed = kList - 512,
              kPool = kBins + kWaves * (kList + 64) / 2;
constexpr float kMaxHeat = 1.44e30f;  // (see heat_of)
constexpr float kUnit = 0x1p40f;
constexpr size_t kMaxScratch = (size_t)64 << 20;
constexpr uint32_t kLowest = 0x007F, kHighest = 0xFF80;  // keys of -inf and inf
constexpr uint32_t kZero = 0x8000, kMinusZero = 0x7FFF;

// 8 logits from token k on as pairs of bits, -inf past the end.
__device__ __forceinline__ u32x4 load_bits(const uint16_t* row, int k, int vocab) {
  u32x4 v;
  if (k + 8 <= vocab) {
    v = *reinterpret_cast<const u32x4_any*>(row + k);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = (k + 2 * i < vocab ? row[k + 2 * i] : 0xFF80u) | (k + 2 * i + 1 < vocab ? row[k + 2 * i + 1] : 0xFF80u) << 16;
  }
  return v;
}
__device__ __forceinline__ float value(const u32x4& v, int i) {
  return __uint_as_float(i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16);
}

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
  uint32_t* counts;  // [b][chunks][kWindow / 2]: pairs of 16 bits, of keys from the chunk's largest down, the first one odd
};

// A row's.
struct Settings {
  float temp, p, least;
  int limit;     // of top-k; 0: none
  bool filters;  // any
};
__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int id) {
  const int k = a.top_k ? a.top_k[id] : 0;
  Settings s{a.temp ? a.temp[id] : 1.0f, a.top_p ? a.top_p[id] : 1.0f, a.min_p ? a.min_p[id] : 0.0f, k > 0 && k < a.vocab ? k : 0, false};
  s.filters = s.temp > 0.0f && (s.limit || s.p < 1.0f || s.least > 0.0f);
  return s;
}

typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
// Keys of two logits: their bits, all inverted where the sign is set, else the sign alone.  -0 has a key of its own, kMinusZero,
// which counts as kZero; NaN are above +inf's key or below -inf's, and never counted.
__device__ __forceinline__ uint32_t two_keys(uint32_t bits) {
  const uint32_t sign = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, bits) >> 15);
  return bits ^ (sign | 0x80008000u);
}
__device__ __forceinline__ uint32_t key_of(uint32_t bits) {
  const uint32_t key = two_keys(bits & 0xFFFFu) & 0xFFFFu;
  return key > kHighest ? kLowest : max(key == kMinusZero ? kZero : key, kLowest);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return bf2f(key & 0x8000u ? key - 0x8000u : 0xFFFFu - key);
}
__device__ __forceinline__ uint32_t key_of_value(float l) { return key_of(__float_as_uint(l) >> 16); }
// in whole numbers of 2^-40
__device__ __forceinline__ uint64_t units(float w) {
  const float x = w * kUnit, hi = __builtin_truncf(x * 0x1p-32f);
  return (uint64_t)(uint32_t)hi << 32 | (uint32_t)__builtin_fmaf(hi, -0x1p32f, x);
}
__device__ __forceinline__ float key_weight(const Heat& s, uint32_t key, float top) {
  return any_weight(s, logit_of(key), top);
}

// What a chunk's sum counts in its row's: in 64 bits, since 32 would move all of the chunk's tokens the same way (by 2^-22 of their
// weight, 2 10^-8 of a row's in all, within which one row of 10^4 has its draw).  0 where its tokens' own weights are.
__device__ __forceinline__ double chunk_weight(const Heat& s, float l, float top) {
  const float x = any_weight(s, l, top);
  return x > 0.0f && l < top ? exp2(((double)l - (double)top) * ((double)s.scale + (double)s.scale_lo)) : (double)x;
}

struct AddUnits {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ uint64_t step(uint64_t x) const {
    return x + ((uint64_t)dpp<CTRL, ROWS>((uint32_t)(x >> 32), 0) << 32 | dpp<CTRL, ROWS>((uint32_t)x, 0));
  }
};
struct AddCounts {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ uint32_t step(uint32_t x) const {
    return x + dpp<CTRL, ROWS>(x, 0);
  }
};
struct MaxCounts {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ uint32_t step(uint32_t x) const {
    return max(x, dpp<CTRL, ROWS>(x, 0));
  }
};
__device__ __forceinline__ uint64_t last_lane64(uint64_t x) {
  return (uint64_t)last_lane((uint32_t)(x >> 32)) << 32 | last_lane((uint32_t)x);
}
__device__ __forceinline__ uint64_t units_sum(uint64_t x) { return last_lane64(wave_scan(x, AddUnits())); }
__device__ __forceinline__ uint32_t counts_sum(uint32_t x) { return last_lane(wave_scan(x, AddCounts())); }

// What kGroupThreads threads share over a chunk
struct Group {
  uint32_t high[kGroupThreads / 64];
  double red[kGroupThreads / 64];
  int best[kGroupThreads / 64];
};

// A chunk, by a group of kGroupThreads threads: see ChunkStat.  bins: where to count its keys (kWindow + 1 zeros), or null.  All
// threads of the workgroup come here together; a chunk past the last is empty.
struct ChunkBits {
  u32x4 v[2];
};
__device__ __forceinline__ ChunkBits load_chunk(const uint16_t* row, int chunk, int vocab) {
  const int at = chunk * kChunk + 8 * (threadIdx.x % kGroupThreads);
  return ChunkBits{{load_bits(row, at, vocab), load_bits(row, at + kChunk / 2, vocab)}};
}
__device__ __forceinline__ ChunkStat chunk_stat(const Heat& s, const ChunkBits& bits, int chunk, uint32_t* bins, Group& g) {
  const int t = threadIdx.x % kGroupThreads, w = t >> 6, at0 = chunk * kChunk + 8 * t, at1 = at0 + kChunk / 2;
  const u32x4 (&v)[2] = bits.v;
  float l[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) l[i] = value(v[i >> 3], i & 7);
  // the largest by its key, with what is above an infinity's, NaN, wrapped to the lowest (fmaxf loses what it has to a signalling
  // NaN)
  u16x2 keys = {0, 0};
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i)
    keys = __builtin_elementwise_max(keys, __builtin_bit_cast(u16x2, two_keys(v[i >> 2][i & 3])) + (uint16_t)kLowest);
  uint32_t high = last_lane(wave_scan((uint32_t)max(keys.x, keys.y), MaxCounts()));
  __syncthreads();
  const uint32_t mine = high;
  if ((t & 63) == 0) g.high[w] = high;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kGroupThreads / 64; ++i) high = max(high, g.high[i]);
  const float top = high <= 2 * kLowest ? -INFINITY : logit_of(high - kLowest);
  int best = 0x7FFFFFFF;
  // (whole waves; where it is 0, a wave with -0 alone has it too)
  if (top > -INFINITY && (mine == high || top == 0.0f)) {
#pragma unroll
    for (int i = kEach - 1; i >= 0; --i)
      if (l[i] == top) best = (i < 8 ? at0 : at1 - 8) + i;
    best = wave_min(best);
  }
  if (bins && top > -INFINITY) {
    const uint32_t first = key_of_value(top), even = ~first & 1;
    const uint32_t span = min((uint32_t)kWindow + 1 - even, first - kLowest);  // (-inf weighs nothing)
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) {
      const uint32_t keys = two_keys(v[i >> 2][i & 3]), d0 = first - (keys & 0xFFFFu), d1 = first - (keys >> 16);
      if (d0 < span) atomicAdd(&bins[even + d0], 1u);
      if (d1 < span) atomicAdd(&bins[even + d1], 1u);
    }
  }
  float sum = 0.0f;
  if (top == INFINITY) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += l[i] == top ? 1.0f : 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += weight(s, l[i], top);
  }
  const double wsum = wave_sum((double)sum);
  __syncthreads();
  if ((t & 63) == 0) g.red[w] = wsum, g.best[w] = best;
  __syncthreads();
  ChunkStat r{top, 0x7FFFFFFF, 0.0};
#pragma unroll
  for (int i = 0; i < kGroupThreads / 64; ++i) r.total += g.red[i], r.best = min(r.best, g.best[i]);
  if (r.best == 0x7FFFFFFF) r.best = -1;
  return r;
}

__global__ void __launch_bounds__(kGroupThreads) sample_keys_kernel(const SampleArgs a) {
  __shared__ Group g;
  __shared__ __attribute__((aligned(16))) uint32_t bins[kWindow + 1];  // (one more: -0 behind 0)
  const int chunk = blockIdx.x, id = blockIdx.y, t = threadIdx.x;
  const ChunkBits v = load_chunk(a.logits + (size_t)id * a.ld, chunk, a.vocab);
  const Settings set = settings_of(a, id);
  const Heat s = heat_of(set.temp);  // (a division in 64 bits, while these are on their way)
  *reinterpret_cast<uint2*>(bins + 2 * t) = make_uint2(0, 0);  // (a barrier follows before the first count)
  if (t == 0) bins[kWindow] = 0;
  const ChunkStat r = chunk_stat(s, v, chunk, set.filters ? bins : nullptr, g);
  const size_t at = (size_t)id * a.chunks + chunk;
  if (t == 0) a.stats[at] = r;
  if (!set.filters) return;  // (nobody reads counts)
  if (t == 0) {
    const uint32_t d = (key_of_value(r.top) | 1) - kZero;  // the counts of -0
    if (r.top >= 0.0f && d < kWindow) bins[d] += bins[d + 1], bins[d + 1] = 0;
  }
  __syncthreads();
  const uint2 n = *reinterpret_cast<const uint2*>(bins + 2 * t);
  a.counts[at * (kWindow / 2) + t] = n.x | n.y << 16;
}

// What is kept: keys above `key` and the first `n` tokens with it, of weights from `least` on.
struct Border {
  uint32_t key, n;
  float least;
};
struct Shared {
  Group g[kGroups];
  ChunkStat stats[kMaxChunks];  // without scratch
  uint32_t count[kWaves];
  uint64_t mass[kWaves];
  double sum[kWaves];
  uint32_t same[kWaves];
  Border border;
  uint64_t border_mass;  // in front of it, its own tokens included
  uint32_t between;
  int after, upto;            // bins of a sample
  float low[kWaves];
  double square[kWaves];
  uint16_t ends[2 * kMaxChunks];  // of the pieces' parts of their waves' lists
  uint64_t kept[kMaxChunks];  // the chunks' weights above the border's key
  uint32_t equal[kMaxChunks]; // and their tokens with it
  __attribute__((aligned(16))) double weight[kWindow + 2];  // of the window's keys, in units; the last two are 0
  __attribute__((aligned(16))) uint32_t bins[kPool];  // (lists behind the bins)
};

struct Row {
  Heat s;
  const uint16_t* logits;
  const uint32_t* counts;  // null: none
  float top;
  int best, vocab, chunks;
  double total;
  uint32_t first;  // the key of top
  uint32_t base;   // the first of the window: that, or the one above where that is even
  uint32_t least;  // the lowest key that weighs anything
  uint32_t low;    // the first key of the bins past zero's
  bool straight;   // or the bins go on below kSpan without a gap, and without a bin for zero alone
};

// Bins in order: one of the window a thread, or kBinsEach of all keys'.
template <bool WIDE>
struct Bins {
  static constexpr int kCount = WIDE ? kBinsEach : 1;
  uint32_t n;
  __device__ __forceinline__ uint32_t count(const Shared& sh, int i) const {
    if constexpr (WIDE)
      return sh.bins[threadIdx.x * kBinsEach + i];
    else
      return n;
  }
  __device__ __forceinline__ uint32_t key(const Row& r, int i) const {
    const int at = (int)threadIdx.x * kCount + i;
    if (!WIDE) return r.base - at;
    if (at < kSpan || r.straight) return r.first - at;
    return at == kSpan ? kZero : r.low - (at - kSpan - 1);
  }
  __device__ __forceinline__ uint64_t mass(const Row& r, const Shared& sh, int i) const {
    const uint32_t m = count(sh, i);
    return m ? m * units(key_weight(r.s, key(r, i), r.top)) : 0;
  }
};

// The chunks' windows, in LDS where sh.bins, which holds nothing else yet, has room for all: slots of kSlot pairs, for the banks, the
// first one unused, so that what is in front of a window can be loaded too.
constexpr int kSlot = kWindow / 2 + 4, kStaged = kPool / kSlot - 1;
static_assert(kStaged < 64 && kSlot % 4 == 0 && (kStaged + 1) * kSlot <= kPool - 4, "a chunk a lane, windows of whole 16 bytes, 16 left");
struct Slot {
  int at, begin;  // of the pair that lines up with the row's first; of the window's first
};
// of the chunk of the lane, whose window begins with key `base`
__device__ __forceinline__ Slot slot_of(const Row& r, uint32_t base) {
  const int lane = threadIdx.x & 63, begin = kSlot * (min(lane, r.chunks - 1) + 1);
  return Slot{begin - (int)min(r.base - base, (uint32_t)kWindow) / 2, lane < r.chunks ? begin : INT_MAX};
}

// The thread's bin of the row's window, from the staged ones: one half of the threads adds up every other chunk's pairs.
__device__ __forceinline__ Bins<false> count_staged(const Row& r, uint32_t base, Shared& sh) {
  const int t = threadIdx.x, pair = t % (kDraw / 2), half = __builtin_amdgcn_readfirstlane(t / (kDraw / 2));
  const Slot slot = slot_of(r, base);
  uint32_t even = 0, odd = 0;
  for (int c0 = half; c0 < r.chunks; c0 += 16) {
    uint32_t v[8], sum = 0;  // (eight chunks' counts fit 16 bits)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = min(c0 + 2 * j, r.chunks - 1), at = pair + __builtin_amdgcn_readlane(slot.at, c);
      v[j] = sh.bins[at];
      v[j] = at >= (c0 + 2 * j < r.chunks ? kSlot * (c + 1) : INT_MAX) ? v[j] : 0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j];
    even += sum & 0xFFFFu, odd += sum >> 16;
  }
  uint32_t* const halves = reinterpret_cast<uint32_t*>(sh.weight);
  reinterpret_cast<uint2*>(halves)[t] = make_uint2(even, odd);
  __syncthreads();
  return Bins<false>{halves[t] + halves[kDraw + t]};
}

// and from memory
__device__ __forceinline__ Bins<false> count_window(const Row& r, const uint32_t (&base)[kLaneChunks]) {
  const uint16_t* const counts = reinterpret_cast<const uint16_t*>(r.counts);
  constexpr int kAt = 32;  // loads in flight
  Bins<false> b{0};
#pragma unroll
  for (int i = 0; i < kLaneChunks; ++i)
    for (int c0 = 0; c0 < min(r.chunks - 64 * i, 64); c0 += kAt) {
      uint32_t v[kAt];
#pragma unroll
      for (int j = 0; j < kAt; ++j) {
        const int c = min(64 * i + c0 + j, r.chunks - 1);
        // how far the window is from the row's; past the last chunk as far as can be
        const int shift = c0 + j < r.chunks - 64 * i ? (int)(r.base - (uint32_t)__builtin_amdgcn_readlane((int)base[i], c & 63)) : kWindow;
        v[j] = counts[(size_t)c * kWindow + max((int)threadIdx.x - shift, 0)];
        v[j] = (int)threadIdx.x >= shift ? v[j] : 0;
      }
#pragma unroll
      for (int j = 0; j < kAt; ++j) b.n += v[j];
    }
  return b;
}

// All keys of the row that weigh anything, into sh.bins; `window`: what is known already, or null.  False: some are between the
// bins.
template <bool STRAIGHT>
__device__ __forceinline__ bool count_keys(const Row& r, uint32_t from, Shared& sh) {
  // (the last key that weighs anything may be within the window: nothing is left then)
  const uint32_t top = r.first - from, all = (uint32_t)max((int)(r.first - r.least + 1) - (int)from, 0);
  const uint32_t span = STRAIGHT ? all : kSpan - from;
  bool between = false;
  auto add = [&](uint32_t key) {
    const uint32_t d = top - key;
    if constexpr (STRAIGHT) {
      if (d < span) atomicAdd(&sh.bins[from + d], 1u);
    } else {
      const uint32_t e = r.low - key;
      const bool second = e < kSpan - 1;
      if (d < span || second) {
        atomicAdd(&sh.bins[second ? kSpan + 1 + e : from + d], 1u);
      } else if (d < all) {  // hardly ever
        if ((key == kZero || key == kMinusZero) && r.first - kZero >= kSpan)
          atomicAdd(&sh.bins[kSpan], 1u);
        else
          between = true;
      }
    }
  };
  // (loading the next 32 logits during these is slower: the atomics are what takes the time)
  for (int k0 = 8 * threadIdx.x; k0 < r.vocab; k0 += 4 * 8 * kDraw) {
    u32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = load_bits(r.logits, min(k0 + j * 8 * kDraw, r.vocab), r.vocab);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t keys = two_keys(v[j][i]);
        add(keys & 0xFFFFu);
        add(keys >> 16);
      }
  }
  return between;
}
// The bin of a key that has one.
__device__ __forceinline__ uint32_t bin_of(const Row& r, uint32_t key) {
  return r.straight || r.first - key < kSpan ? r.first - key : kSpan + 1 + r.low - key;
}
// Whether 0 and -0 have neighbouring bins.
__device__ __forceinline__ bool zeros_in(const Row& r) {
  return r.first >= kZero && r.least <= kMinusZero && (r.straight || r.first - kMinusZero < kSpan || kZero <= r.low);
}
__device__ __forceinline__ bool count_all(Row& r, const Bins<false>* window, Shared& sh) {
  // what lies 31 T below the largest weighs less than 2^-44; a key less, since the value loses its low bits
  const float heat = fminf(fmaxf(r.s.heat, FLT_MIN), kMaxHeat);
  r.least = r.top == INFINITY ? r.first : max((int)key_of_value(r.top - 31.0f * heat), (int)kLowest + 2) - 1;
  r.low = r.least + (kSpan - 2);
  r.straight = r.low + kSpan >= r.first;
  const uint32_t from = window ? kWindow - (r.base - r.first) : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < kBins / 4; i += kDraw) reinterpret_cast<uint4*>(sh.bins)[i] = make_uint4(0, 0, 0, 0);
  if (threadIdx.x == 0) sh.between = 0;
  __syncthreads();
  if (window && threadIdx.x >= r.base - r.first) sh.bins[threadIdx.x - (r.base - r.first)] = window->n;
  if (r.straight ? count_keys<true>(r, from, sh) : count_keys<false>(r, from, sh)) sh.between = 1;
  __syncthreads();
  if (threadIdx.x == 0 && zeros_in(r)) {  // -0 counts as 0 (in the window, both are counted)
    const uint32_t zero = bin_of(r, kZero);
    if (zero >= from) sh.bins[zero] += sh.bins[zero + 1];
    if (zero + 1 >= from) sh.bins[zero + 1] = 0;
  } else if (threadIdx.x == 0 && !r.straight && r.low == kMinusZero) {  // and where its bin is the first past zero's own
    sh.bins[kSpan] += sh.bins[kSpan + 1];
    sh.bins[kSpan + 1] = 0;
  }
  __syncthreads();
  return sh.between == 0;
}

struct Sums {
  uint32_t count, own_count, counts;  // in front of the thread's bins; in them; all
  uint64_t mass, own_mass, masses;
};
template <bool WIDE>
__device__ __forceinline__ Sums sum_bins(const Row& r, const Bins<WIDE>& b, Shared& sh) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t n = 0;
  uint64_t m = 0;
  for (int j = 0; j < b.kCount; ++j) {
    const int i = WIDE ? (j + lane) % b.kCount : j;  // (every lane another bank)
    n += b.count(sh, i), m += b.mass(r, sh, i);
  }
  const uint32_t upto = wave_scan(n, AddCounts());
  const uint64_t mass = wave_scan(m, AddUnits());
  if (lane == 63) sh.count[w] = upto, sh.mass[w] = mass;
  __syncthreads();
  Sums s{upto - n, n, 0, mass - m, m, 0};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) s.count += sh.count[i], s.mass += sh.mass[i];
    s.counts += sh.count[i], s.masses += sh.mass[i];
  }
  return s;
}

// What top-p's front weighs at least, of a sum.
__device__ __forceinline__ uint64_t goal_of(float p, double all) {
  const double want = ceil((double)fmaxf(p, 0.0f) * all);
  return want > 1.0 ? (uint64_t)want : 1;
}

// The borders of top-k (k > 0) and top-p (p < 1) among bins that hold all in front of them, but for `counts` tokens that weigh
// `masses`.  False: these do not.
template <bool WIDE>
__device__ __forceinline__ bool find(const Row& r, const Bins<WIDE>& b, int k, float p, Border& out, Shared& sh, uint32_t counts = 0,
                                     uint64_t masses = 0) {
  Sums s = sum_bins(r, b, sh);
  s.count += counts, s.counts += counts, s.mass += masses, s.masses += masses;
  double all = r.total * (double)kUnit;
  bool found = false;
  if (k > 0 && counts < (uint32_t)k && s.counts >= (uint32_t)k) {
    uint32_t n = s.count;
    uint64_t m = s.mass;
    for (int i = 0; i < b.kCount && n < (uint32_t)k && s.count + s.own_count >= (uint32_t)k; ++i) {
      const uint32_t x = b.count(sh, i);
      if (n + x >= (uint32_t)k) {
        const uint32_t key = b.key(r, i);
        sh.border = Border{key, (uint32_t)k - n, 0.0f};
        sh.border_mass = m + ((uint32_t)k - n) * units(key_weight(r.s, key, r.top));
      }
      n += x, m += b.mass(r, sh, i);
    }
    __syncthreads();
    out.key = sh.border.key, out.n = sh.border.n;
    all = (double)sh.border_mass;
    found = true;
  } else if (k > 0 && !WIDE) {
    return false;
  }
  if (p < 1.0f) {
    const uint64_t goal = goal_of(p, all);
    if (s.masses < goal || masses >= goal) return found;
    __syncthreads();  // (border was read)
    uint64_t m = s.mass;
    for (int i = 0; i < b.kCount && m < goal && s.mass + s.own_mass >= goal; ++i) {
      const uint64_t x = b.mass(r, sh, i);
      if (m + x >= goal) {
        const uint32_t key = b.key(r, i);
        const uint64_t one = units(key_weight(r.s, key, r.top));
        sh.border = Border{key, (uint32_t)((goal - m + one - 1) / one), 0.0f};
      }
      m += x;
    }
    __syncthreads();
    // (top-k's own border where a rounding of the goal would go past it)
    if (!found || sh.border.key > out.key || (sh.border.key == out.key && sh.border.n < out.n))
      out.key = sh.border.key, out.n = sh.border.n;
    found = true;
  }
  return found;
}

// The weights of the window's keys above the border, to sh.weight: in doubles, where a chunk's counts times these are whole (4096 of
// 2^40 units), and whose products take a quarter of the time of those in 64 bits.
__device__ __forceinline__ void window_weights(const Row& r, const Border& b, Shared& sh) {
  const int t = threadIdx.x;
  const uint32_t key = r.base - t;
  const float x = key_weight(r.s, key, r.top);
  sh.weight[t] = key <= r.first && key > b.key && x >= b.least ? (double)__builtin_truncf(x * kUnit) : 0.0;
  if (t < 2) sh.weight[kWindow + t] = 0.0;
  __syncthreads();
}
// Each chunk's weights above the border's key and its tokens with it: from the staged windows, a lane a chunk, every eighth pair a
// wave;
__device__ __forceinline__ void staged_masses(const Row& r, const Border& b, uint32_t base, uint64_t& kept, uint32_t& equal, Shared& sh) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  window_weights(r, b, sh);
  const Slot slot = slot_of(r, base);
  const int down = (int)min(r.base - b.key, (uint32_t)kWindow - 1);
  double sum = 0.0;
#pragma unroll 4
  for (int pair = w; pair <= down / 2; pair += kWaves) {
    uint32_t n = sh.bins[slot.at + pair];
    n = slot.at + pair >= slot.begin ? n : 0;
    const double2 x = *reinterpret_cast<const double2*>(&sh.weight[2 * pair]);
    sum = __builtin_fma((double)(n & 0xFFFFu), x.x, sum);
    sum = __builtin_fma((double)(n >> 16), x.y, sum);
  }
  double* const parts = reinterpret_cast<double*>(sh.stats);
  static_assert(sizeof(sh.stats) >= kDraw * sizeof(double), "a part a thread");
  parts[threadIdx.x] = sum;
  const uint32_t n = sh.bins[slot.at + down / 2];
  equal = b.key && slot.at + down / 2 >= slot.begin ? n >> (16 * (down & 1)) & 0xFFFFu : 0;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) sum += parts[64 * i + lane];
  kept = (uint64_t)sum;
}
// to sh.kept and sh.equal from those in memory,
__device__ __forceinline__ void window_masses(const Row& r, const Border& b, const uint32_t (&base)[kLaneChunks], Shared& sh) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  window_weights(r, b, sh);
  // a wave kAt chunks at a time, lane by lane two neighbouring bins, 128 a step; steps past the border are not loaded
  constexpr int kAt = 5, kSteps = kWindow / 128;
  for (int c0 = w; c0 < r.chunks; c0 += kAt * kWaves) {
    uint32_t pair[kAt][kSteps];
    int shift[kAt], border[kAt];  // border: the chunk's bin of the border's key
#pragma unroll
    for (int a = 0; a < kAt; ++a) {
      const int c = min(c0 + a * kWaves, r.chunks - 1);
      uint32_t f = base[0];
#pragma unroll
      for (int i = 1; i < kLaneChunks; ++i) f = c >> 6 == i ? base[i] : f;
      shift[a] = (int)(r.base - (uint32_t)__builtin_amdgcn_readlane((int)f, c & 63));
      border[a] = (int)(r.base - b.key) - shift[a];
      const int last = min(border[a], kWindow - 1 - shift[a]);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        pair[a][j] = 0;
        if (128 * j <= last) pair[a][j] = r.counts[(size_t)c * (kWindow / 2) + 64 * j + lane];
      }
    }
    double sum[kAt];
    uint32_t same[kAt];
#pragma unroll
    for (int a = 0; a < kAt; ++a) {
      sum[a] = 0.0, same[a] = 0;
      const int last = min(border[a], kWindow - 1 - shift[a]);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        if (128 * j > last) break;
        const int in = min(128 * j + 2 * lane + shift[a], kWindow);  // (past the window the weights are 0)
        sum[a] = __builtin_fma((double)(pair[a][j] & 0xFFFFu), sh.weight[in], sum[a]);
        sum[a] = __builtin_fma((double)(pair[a][j] >> 16), sh.weight[in + 1], sum[a]);
        if (border[a] >> 7 == j)
          same[a] = (uint32_t)__builtin_amdgcn_readlane((int)pair[a][j], border[a] >> 1 & 63) >> (16 * (border[a] & 1)) & 0xFFFFu;
      }
    }
#pragma unroll
    for (int a = 0; a < kAt; ++a) sum[a] = wave_sum(sum[a]);
#pragma unroll
    for (int a = 0; a < kAt; ++a)
      if (lane == 0 && c0 + a * kWaves < r.chunks)
        sh.kept[c0 + a * kWaves] = (uint64_t)sum[a], sh.equal[c0 + a * kWaves] = b.key ? same[a] : 0;
  }
  __syncthreads();
}
// and from the row: a wave adds up a chunk's, in whole units, so exactly.  (Weights looked up in LDS by key instead: no faster.)
template <bool INF>
__device__ __forceinline__ void chunk_masses_of(const Row& r, const Border& b, Shared& sh) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const float border = b.key ? logit_of(b.key) : -INFINITY;
  for (int c = w; c < r.chunks; c += kWaves) {
    u32x4 v[kChunk / 512];
#pragma unroll
    for (int j = 0; j < kChunk / 512; ++j) v[j] = load_bits(r.logits, min(c * kChunk + 512 * j + 8 * lane, r.vocab), r.vocab);
    double sum = 0.0;
    uint32_t same = 0;
#pragma unroll
    for (int j = 0; j < kChunk / 512; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float l = value(v[j], i), x = INF ? (l == r.top ? 1.0f : 0.0f) : weight(r.s, l, r.top);
        sum += (double)(l > border && x >= b.least ? __builtin_truncf(x * kUnit) : 0.0f);
        same += l == border;
      }
    sum = wave_sum(sum), same = counts_sum(same);
    if (lane == 0) sh.kept[c] = (uint64_t)sum, sh.equal[c] = b.key ? same : 0;
  }
}
__device__ __forceinline__ void chunk_masses(const Row& r, const Border& b, Shared& sh) {
  __syncthreads();
  if (r.top == INFINITY)
    chunk_masses_of<true>(r, b, sh);
  else
    chunk_masses_of<false>(r, b, sh);
  __syncthreads();
}

// One border, top-k's or top-p's, past the window of a long row: the weights (or tokens) behind a logit, estimated by those of a
// sample, leave few keys for it, within four standard deviations.  One pass over the row adds up the weights in front of these
// and lists the logits between; that list has the border, and what is missing of the chunks' weights.
enum class Sampled { kFound, kBehind, kNot };  // kBehind: behind min-p's border, it seems; kNot: not in the list
__device__ __forceinline__ Sampled find_sampled(const Row& r, int k, float p, Border& out, Shared& sh) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  uint16_t* const list = reinterpret_cast<uint16_t*>(sh.bins + kBins) + w * (kList + 64);
  __syncthreads();
  reinterpret_cast<uint4*>(sh.bins)[t] = make_uint4(0, 0, 0, 0);
  if (t == 0) sh.after = -1, sh.upto = kSampleBins, sh.between = 0;
  if (t < kMaxChunks) sh.kept[t] = 0, sh.equal[t] = 0;
  float l[16], low = r.top;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const u32x4 v = load_bits(r.logits, (2 * t + j) * (r.vocab / 8) / (2 * kDraw) * 8, r.vocab);
#pragma unroll
    for (int i = 0; i < 8; ++i) l[8 * j + i] = value(v, i);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (l[i] > -INFINITY) low = fminf(low, l[i]);
  const float farthest = wave_max(r.top - low);
  if (lane == 0) sh.low[w] = farthest;
  __syncthreads();
  float span = 0.0f;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) span = fmaxf(span, sh.low[i]);
  span = fminf(span, 31.0f * fminf(fmaxf(r.s.heat, FLT_MIN), kMaxHeat));
  const float fine = (float)kSampleBins / span;  // bins from the least up
  if (!(span < INFINITY && fine < 0x1p100f)) return Sampled::kNot;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float at = span - (r.top - l[i]);
    if (at >= 0.0f && at <= span) atomicAdd(&sh.bins[min((int)(at * fine), kSampleBins - 1)], 1u);
  }
  __syncthreads();
  const uint4 bins = reinterpret_cast<const uint4*>(sh.bins)[t];
  const uint32_t n[4] = {bins.x, bins.y, bins.z, bins.w};
  float x[4];
  double sum = 0.0, square = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = k > 0 ? 1.0f : weight(r.s, r.top - span + (4 * t + i + 0.5f) / fine, r.top);
    sum += (double)(n[i] * x[i]), square += (double)(n[i] * x[i] * x[i]);
  }
  const double upto = wave_scan(sum, Add()), upto2 = wave_scan(square, Add());
  if (lane == 63) sh.sum[w] = upto, sh.square[w] = upto2;
  __syncthreads();
  double behind = upto - sum, behind2 = upto2 - square, all = 0.0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) behind += sh.sum[i], behind2 += sh.square[i];
    all += sh.sum[i];
  }
  const double part = (double)kSample / r.vocab;
  const float goal = (float)(k > 0 ? all - k * part : (1.0 - (double)fmaxf(p, 0.0f)) * r.total * part);
  int after = -1, end = kSampleBins;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    behind += (double)(n[i] * x[i]), behind2 += (double)(n[i] * x[i] * x[i]);
    const double var = k > 0 ? (all - behind) * (1.0 - (all - behind) / kSample) : behind2;
    const float far = 4.0f * sqrtf((float)fmax(var, 0.0)) + 2.0f * x[i], b = (float)behind;
    if (b + far < goal) after = 4 * t + i;
    if (b - far > goal) end = min(end, 4 * t + i);
  }
  after = -wave_min(-after), end = wave_min(end);
  if (lane == 0) atomicMax(&sh.after, after), atomicMin(&sh.upto, end);
  __syncthreads();
  after = sh.after, end = sh.upto;
  uint32_t count = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) count += 4 * t + i > after && 4 * t + i <= end ? n[i] : 0;
  count = counts_sum(count);
  if (lane == 0) sh.count[w] = count;
  for (int i = t; i < kBins / 4; i += kDraw) reinterpret_cast<uint4*>(sh.bins)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  count = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) count += sh.count[i];
  Row q = r;
  if (end < kSampleBins) q.first = min(r.first, key_of_value(r.top - span + (end + 1) / fine) + 1);
  if (q.first == kMinusZero) q.first = kZero;
  q.least = max(key_of_value(r.top - span + (after + 1) / fine), kLowest + 2) - 1;
  q.low = q.least + (kSpan - 2);
  q.straight = q.low + kSpan >= q.first;
  if (out.least > 1.0f / kUnit && key_weight(r.s, q.first, r.top) < out.least) return Sampled::kBehind;
  if (count > 0.8 * part * (kWaves * kListed) || q.least > q.first) return Sampled::kNot;

  const float highest = logit_of(q.first), lowest = logit_of(q.least);
  const int pieces = (r.vocab + kPiece - 1) / kPiece;
  uint32_t listed = 0;
  count = 0;
  u32x4 v[kPiece / 512], next[kPiece / 512];
  auto load = [&](int piece) {
#pragma unroll
    for (int j = 0; j < kPiece / 512; ++j) next[j] = load_bits(r.logits, min(piece * kPiece + 512 * j + 8 * lane, r.vocab), r.vocab);
  };
  load(w);
  for (int c = w; c < pieces; c += kWaves) {
#pragma unroll
    for (int j = 0; j < kPiece / 512; ++j) v[j] = next[j];
    if (c + kWaves < pieces) load(c + kWaves);
    double mass = 0.0;
#pragma unroll
    for (int j = 0; j < kPiece / 512; ++j) {
      if (listed > kListed) break;  // (the next 512 may not fit: the row is counted instead)
      float x[8];
      uint64_t over[8], in[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = value(v[j], i), d = y - r.top;  // (no clamp: what is over is near enough)
        x[i] = __builtin_truncf(__builtin_amdgcn_exp2f(__builtin_fmaf(d, r.s.scale, d * r.s.scale_lo)) * kUnit);
        over[i] = __ballot(y > highest), in[i] = __ballot(y >= lowest) & ~over[i];
        x[i] = y > highest ? x[i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mass += (double)x[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        count += __builtin_popcountll(over[i]);
        const uint32_t at = __builtin_amdgcn_mbcnt_hi((uint32_t)(in[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[i], listed));
        // (what is not listed goes behind the list: a branch takes longer)
        const uint32_t bits = v[j][i >> 1] >> (16 * (i & 1));
        list[__builtin_amdgcn_inverse_ballot_w64(in[i]) ? at : (uint32_t)kList + lane] = (uint16_t)bits;
        listed += __builtin_popcountll(in[i]);
      }
    }
    mass = wave_sum(mass);
    if (lane == 0) {
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.kept[c / 2]), (unsigned long long)mass);
      sh.ends[c] = (uint16_t)listed;
    }
  }
  bool between = listed > kListed;
  for (uint32_t i = lane; i < listed; i += 64) {
    const uint32_t key = key_of(list[i]), d = q.first - key, e = q.low - key;
    list[i] = (uint16_t)key;
    if (q.straight || d < kSpan)
      atomicAdd(&sh.bins[d], 1u);
    else if (e < kSpan - 1)
      atomicAdd(&sh.bins[kSpan + 1 + e], 1u);
    else if (key == kZero)
      atomicAdd(&sh.bins[kSpan], 1u);
    else
      between = true;
  }
  if (between) sh.between = 1;
  __syncthreads();
  if (lane == 0) sh.same[w] = count;
  uint64_t mass = 0;
#pragma unroll
  for (int i = 0; i < kLaneChunks; ++i) mass += sh.kept[64 * i + lane];
  mass = units_sum(mass);
  __syncthreads();
  if (sh.between) return Sampled::kNot;
  count = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) count += sh.same[i];
  Border b = out;
  if (!find(q, Bins<true>{}, k, p, b, sh, count, mass)) return Sampled::kNot;
  uint32_t begin = 0;
  for (int c = w; c < pieces; c += kWaves) {
    const uint32_t stop = sh.ends[c];
    uint64_t kept = 0;
    uint32_t same = 0;
    for (uint32_t i = begin + lane; i < stop; i += 64) {
      const uint32_t key = list[i];
      const float x = key_weight(r.s, key, r.top);
      kept += key > b.key && x >= b.least ? units(x) : 0;
      same += key == b.key;
    }
    kept = units_sum(kept), same = counts_sum(same);
    if (lane == 0) {
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.kept[c / 2]), (unsigned long long)kept);
      atomicAdd(&sh.equal[c / 2], same);
    }
    begin = stop;
  }
  out = b;
  __syncthreads();
  return Sampled::kFound;
}

// Keys of a row that has some between the bins: down from the largest, kBins at a time and over empty stretches at once, first to
// top-k's border, then to top-p's.  Slow, for rows with logits of 2^-31 of the largest and less.
__device__ __attribute__((noinline)) Border find_slowly(Row r, int k, float p, Border out, Shared& sh) {
  const uint32_t top = r.first;
  r.straight = true;
  double all = r.total * (double)kUnit;
  bool found = false;
  for (int turn = k > 0 ? 0 : 1; turn < (p < 1.0f ? 2 : 1); ++turn) {
    const uint64_t goal = turn ? goal_of(p, all) : (uint64_t)k;
    uint32_t counts = 0;
    uint64_t masses = 0;
    r.first = top;
    for (;;) {
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += kDraw) sh.bins[i] = 0;
      if (threadIdx.x == 0) sh.between = 0;
      __syncthreads();
      uint32_t next = 0;
      for (int k0 = 8 * threadIdx.x; k0 < r.vocab; k0 += 8 * kDraw) {
        float l[8];
        load8(r.logits, k0, r.vocab, l);
        for (int i = 0; i < 8; ++i) {
          const uint32_t key = key_of_value(l[i]);
          if (key > r.first || key == kLowest) continue;
          if (r.first - key < kBins)
            atomicAdd(&sh.bins[r.first - key], 1u);
          else
            next = max(next, key);
        }
      }
      if (next) atomicMax(&sh.between, next);
      __syncthreads();
      const Bins<true> b{};
      const Sums s = sum_bins(r, b, sh);
      if ((turn ? masses + s.masses : (uint64_t)counts + s.counts) >= goal) {
        uint32_t n = counts + s.count;
        uint64_t m = masses + s.mass;
        for (int i = 0; i < kBinsEach && (turn ? m : n) < goal; ++i) {
          const uint32_t x = b.count(sh, i), key = b.key(r, i);
          const uint64_t one = x ? units(key_weight(r.s, key, r.top)) : 0;
          if ((turn ? m + x * one : (uint64_t)n + x) >= goal) {
            const uint32_t take = turn ? (uint32_t)((goal - m + one - 1) / one) : (uint32_t)goal - n;
            sh.border = Border{key, take, 0.0f};
            sh.border_mass = m + take * one;
          }
          n += x, m += x * one;
        }
        __syncthreads();
        if (!found || sh.border.key > out.key || (sh.border.key == out.key && sh.border.n < out.n))
          out.key = sh.border.key, out.n = sh.border.n;
        all = (double)sh.border_mass;
        found = true;
        break;
      }
      counts += s.counts, masses += s.masses;
      r.first = sh.between;
      if (!r.first) break;
    }
  }
  return out;
}

__device__ __forceinline__ void store(const SampleArgs& a, int id, const Row& r, int token) {
  a.tokens[id] = token;
  if (!a.logp) return;
  float lp = 0.0f;
  if (token >= 0) {
    const float l = bf2f(r.logits[token]);
    lp = (float)((l == r.top ? 0.0 : (double)(l - r.top) / (double)fminf(fmaxf(r.s.heat, FLT_MIN), kMaxHeat)) - log(r.total));
  }
  a.logp[id] = lp;
}

// The token of a chunk at which the kept weights pass `at`; n: how many tokens with the border's key it may keep.  Its thread
// stores it.
__device__ __forceinline__ void draw_in(const SampleArgs& a, int id, const Row& r, int chunk, const Border& b, uint32_t n, double at,
                                        Shared& sh) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, k = chunk * kChunk + 8 * t;
  float l[8], x[8];
  load8(r.logits, k, r.vocab, l);
  uint32_t rank = 0;
  if (b.key) {
    uint32_t same = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) same += key_of_value(l[i]) == b.key;
    const uint32_t upto = wave_scan(same, AddCounts());
    if (lane == 63) sh.same[w] = upto;
    __syncthreads();
    rank = upto - same;
#pragma unroll
    for (int i = 0; i < kWaves; ++i)
      if (i < w) rank += sh.same[i];
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t key = key_of_value(l[i]);
    x[i] = any_weight(r.s, l[i], r.top);
    bool keep = key > b.key && x[i] >= b.least;
    if (b.key && key == b.key) keep = rank++ < n;
    x[i] = keep ? x[i] : 0.0f;
    sum += x[i];
  }
  const double mine = (double)sum, upto = wave_scan(mine, Add());
  if (lane == 63) sh.sum[w] = upto;
  __syncthreads();
  // the first wave that passes `at`, the last with any weight if none does; in it the lane likewise, and there the token
  double before = 0.0, c = 0.0;
  int wave = -1;
  bool past = false;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const double s = sh.sum[i];
    if (!past && s > 0.0) wave = i, before = c, past = c + s > at;
    c += s;
  }
  if (wave < 0) wave = 0;  // (not with any weight in the chunk)
  if (w != wave) return;
  const double to = before + upto, from = to - mine;
  const uint64_t over = __ballot(mine > 0.0 && to > at), any = __ballot(mine > 0.0);
  if (lane != (over ? __builtin_ctzll(over) : any ? 63 - __builtin_clzll(any) : 0)) return;
  int token = r.best;
  bool have = false;
  c = from;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (x[i] > 0.0f && (!have || c <= at)) token = k + i, have = true;
    c += (double)x[i];
  }
  store(a, id, r, token);
}

__global__ void __launch_bounds__(kDraw, 4) sample_draw_kernel(const SampleArgs a) {
  __shared__ Shared sh;
  const int id = blockIdx.x, t = threadIdx.x, lane = t & 63;
  Row r;
  r.logits = a.logits + (size_t)id * a.ld;
  r.vocab = a.vocab, r.chunks = a.chunks;
  r.counts = a.counts ? a.counts + (size_t)id * a.chunks * (kWindow / 2) : nullptr;
  const auto [temp, p, least, limit, filters] = settings_of(a, id);
  const float u = a.u[id];
  const bool staged = filters && r.counts && a.chunks <= kStaged;
  ChunkStat st[kLaneChunks];
  auto load_stats = [&](const ChunkStat* stats) {
#pragma unroll
    for (int i = 0; i < kLaneChunks; ++i) {
      st[i] = ChunkStat{-INFINITY, -1, 0.0};
      if (lane + 64 * i < a.chunks) st[i] = stats[lane + 64 * i];
    }
  };
  if (a.stats) load_stats(a.stats + (size_t)id * a.chunks);
  if (staged) {  // beside the statistics
    constexpr int kAt = kPool / 4 / kDraw;
    const uint4* const src = reinterpret_cast<const uint4*>(r.counts);
    const int pieces = a.chunks * (kWindow / 8);
    uint4 v[kAt];
#pragma unroll
    for (int i = 0; i < kAt; ++i) v[i] = src[min(t + i * kDraw, pieces - 1)];
    r.s = heat_of(temp);  // (a division in 64 bits, while these are on their way)
#pragma unroll
    for (int i = 0; i < kAt; ++i) {
      const int e = t + i * kDraw, c = e / (kWindow / 8);
      reinterpret_cast<uint4*>(sh.bins)[e < pieces ? (c + 1) * (kSlot / 4) + e % (kWindow / 8) : kPool / 4 - 1] = v[i];  // (or nowhere)
    }
  }
  if (!staged) r.s = heat_of(temp);
  if (!a.stats) {
    for (int c0 = 0; c0 < a.chunks; c0 += kGroups) {
      const int c = min(c0 + t / kGroupThreads, a.chunks);
      const ChunkStat x = chunk_stat(r.s, load_chunk(r.logits, c, a.vocab), c, nullptr, sh.g[t / kGroupThreads]);
      if (t % kGroupThreads == 0 && c < a.chunks) sh.stats[c] = x;
    }
    __syncthreads();
    load_stats(sh.stats);
  }
  // every wave by itself: the row from its chunks (lane by lane, then over the lanes)
  uint32_t base[kLaneChunks];
  r.top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kLaneChunks; ++i) r.top = fmaxf(r.top, st[i].top), base[i] = key_of_value(st[i].top) | 1;
  r.top = wave_max(r.top);
  if (r.top == -INFINITY) {
    if (t == 0) {
      a.tokens[id] = -1;
      if (a.logp) a.logp[id] = 0.0f;
    }
    return;
  }
  double share[kLaneChunks], total = 0.0;
  int best = 0x7FFFFFFF;
#pragma unroll
  for (int i = kLaneChunks - 1; i >= 0; --i) {
    if (st[i].top == r.top) best = st[i].best;
    share[i] = 64 * i < a.chunks ? st[i].total * chunk_weight(r.s, st[i].top, r.top) : 0.0;
  }
#pragma unroll
  for (int i = 0; i < kLaneChunks; ++i) total += share[i];
  r.total = wave_sum(total);
  r.best = wave_min(best);
  r.first = key_of_value(r.top), r.base = r.first | 1;
  if (r.s.greedy) {
    if (t == 0) store(a, id, r, r.best);
    return;
  }
  Border b{0, 0, 0.0f};
  if (!filters) {  // no filter: the chunk from their own sums
    double at = (double)u * r.total, before = 0.0, c = 0.0;
    int chunk = -1;
    bool past = false;
#pragma unroll
    for (int i = 0; i < kLaneChunks; ++i) {
      if (64 * i >= a.chunks || past) break;
      const double upto = wave_scan(share[i], Add()), from = c + upto - share[i];
      const uint64_t over = __ballot(share[i] > 0.0 && c + upto > at), any = __ballot(share[i] > 0.0);
      if (over | any) {
        const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
        chunk = 64 * i + l, before = __shfl(from, l);
        past = over != 0;
      }
      c += __shfl(upto, 63);
    }
    draw_in(a, id, r, max(chunk, 0), b, 0, fmax(at - before, 0.0), sh);  // (the largest has a weight: there is a chunk)
    return;
  }
  // (weights below a unit are nothing in the sums, so their tokens are not drawn either, whatever shares their chunk)
  b.least = fmaxf(least > 0.0f ? fminf(least, 1.0f) : 0.0f, 1.0f / kUnit);
  if (staged) __syncthreads();
  bool quick = r.counts != nullptr;
  Bins<false> window{0};
  if (quick) {
    // whether min-p's border, or the end of what weighs a unit, is within the window: then no border that is further down matters
    // (where top-p's may be within it though top-k's is not, that has to be known)
    const bool cut = r.first < kWindow || key_weight(r.s, r.base - (kWindow - 1), r.top) < b.least;
    bool found = false;
    if (limit || p < 1.0f) {
      window = staged ? count_staged(r, base[0], sh) : count_window(r, base);
      found = find(r, window, limit, p, b, sh);
    }
    quick = found || (cut && !(limit && p < 1.0f));
    if (!found) b.key = 0, b.n = 0;
  }
  uint64_t kept[kLaneChunks];
  uint32_t equal[kLaneChunks];
  if (quick && !staged) {
    window_masses(r, b, base, sh);
  } else if (quick) {
    staged_masses(r, b, base[0], kept[0], equal[0], sh);
  } else {
    const bool one = (limit != 0) != (p < 1.0f) && a.vocab >= kSample && r.top < INFINITY;
    Sampled how = one ? find_sampled(r, limit, p, b, sh) : Sampled::kNot;
    if (how == Sampled::kBehind && !limit) {  // (of top-k's, weights do not say it)
      chunk_masses(r, b, sh);
      uint64_t all = 0;
      for (int i = lane; i < a.chunks; i += 64) all += sh.kept[i];
      if (units_sum(all) < goal_of(p, r.total * (double)kUnit)) how = Sampled::kFound;  // so it is: no border but min-p's
    }
    if (how != Sampled::kFound) {
      if (limit || p < 1.0f) {
        if (count_all(r, r.counts ? &window : nullptr, sh))
          (void)find(r, Bins<true>{}, limit, p, b, sh);  // (found nowhere: there is no border)
        else
          b = find_slowly(r, limit, p, b, sh);
      }
      chunk_masses(r, b, sh);
    }
  }
  if (!(quick && staged)) {
#pragma unroll
    for (int i = 0; i < kLaneChunks; ++i) kept[i] = sh.kept[lane + 64 * i], equal[i] = sh.equal[lane + 64 * i];
  }
  // the chunk, every wave by itself
  const float border_weight = b.key ? key_weight(r.s, b.key, r.top) : 0.0f;
  const uint64_t one = units(border_weight);
  uint32_t left = border_weight >= b.least ? b.n : 0;
  uint64_t mass[kLaneChunks], all = 0;
  uint32_t mine[kLaneChunks];
#pragma unroll
  for (int i = 0; i < kLaneChunks; ++i) {
    mass[i] = 0, mine[i] = 0;
    if (64 * i >= a.chunks) continue;
    const int c = lane + 64 * i;
    const uint32_t n = c < a.chunks ? equal[i] : 0, upto = wave_scan(n, AddCounts()), from = upto - n;
    mine[i] = min(n, left > from ? left - from : 0u);
    mass[i] = (c < a.chunks ? kept[i] : 0) + mine[i] * one;
    const uint32_t used = last_lane(upto);
    left = left > used ? left - used : 0;
    all += units_sum(mass[i]);
  }
  const double at = (double)u * (double)all;
  uint64_t c = 0;
  double before = 0.0;
  int chunk = -1;
  uint32_t n = 0;
  bool past = false;
#pragma unroll
  for (int i = 0; i < kLaneChunks; ++i) {
    if (64 * i >= a.chunks || past) continue;
    const uint64_t upto = wave_scan(mass[i], AddUnits());
    const uint64_t over = __ballot(mass[i] && (double)(c + upto) > at), any = __ballot(mass[i] != 0);
    if (over | any) {
      const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
      chunk = 64 * i + l, past = over != 0;
      before = (double)(c + (uint64_t)__shfl((unsigned long long)(upto - mass[i]), l));
      n = __shfl(mine[i], l);
    }
    c += last_lane64(upto);
  }
  draw_in(a, id, r, max(chunk, 0), b, n, fmax(at - before, 0.0) * (1.0 / (double)kUnit), sh);
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
    for (int i = 0; i < a.b; i += 65535) {
      hipLaunchKernelGGL(sample_draw_kernel, dim3((unsigned)(a.b - i < 65535 ? a.b - i : 65535)), dim3(kDraw), 0, st, from(a, i));
      if (const int e = (int)hipGetLastError()) return e;
    }
    return 0;
  }
  a.stats = reinterpret_cast<ChunkStat*>(z);
  a.counts = reinterpret_cast<uint32_t*>(a.stats + (size_t)each * a.chunks);
  for (int i = 0; i < a.b; i += each) {
    const SampleArgs l = from(a, i);
    const unsigned n = (unsigned)(a.b - i < each ? a.b - i : each);
    hipLaunchKernelGGL(sample_keys_kernel, dim3((unsigned)a.chunks, n), dim3(kGroupThreads), 0, st, l);
    if (const int e = (int)hipGetLastError()) return e;
    hipLaunchKernelGGL(sample_draw_kernel, dim3(n), dim3(kDraw), 0, st, l);
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
