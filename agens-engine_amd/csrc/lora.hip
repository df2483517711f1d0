// Low-rank adapters of many requests beside a shared linear: y_t = y0_t + scale_a B_a (A_a x_t) for the tokens t of adapter a.
//
// Tokens are grouped by adapter in tiles of up to kTile (ak_lora_plan, once for all linears of a step), so that an adapter's
// weights are read once for all of its tokens of a tile.  Two launches then:
//   lora_down_kernel   s = A x of 16 tokens at a time on MFMA (bf16, sums in fp32), one wave a chunk of kChunk inputs;
//   lora_up_kernel     adds up the chunks' parts, and y = y0 + B (scale s): s enters the MFMA as two bf16 operands, which hold
//                      16 bits of it (one alone would move y by 2^-9 of what is added).
// The chunks' parts are added up first by eights, then from left to right, whoever does it: a token's bits do not depend on
// the other tokens of the call.
#include "agens_kernels.h"
#include "wq_common.h"

namespace agq {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64, kChunk = 512, kGroup = 8;
constexpr int kPlanThreads = 1024;

struct Tile {
  int adapter, start, count, pad;  // adapter -1: tokens without one
};
// A plan's memory: this, tiles, the tokens in the tiles' order, then the products' parts.
struct PlanHead {
  int m, adapters, tiles, pad;
};
struct PlanView {
  PlanHead* head;
  Tile* tiles;
  int* order;
  float* parts;  // [chunks][m][ranks]
};
__host__ __device__ inline int max_tiles(int m, int adapters) {
  const long t = (long)m / kTile + (m < adapters + 1 ? m : adapters + 1);
  return (int)(t < m ? t : m);
}
__host__ __device__ inline size_t tiles_at() { return sizeof(PlanHead); }
__host__ __device__ inline size_t order_at(int m, int adapters) {
  return tiles_at() + (size_t)max_tiles(m, adapters) * sizeof(Tile);
}
__host__ __device__ inline size_t parts_at(int m, int adapters) {
  return (order_at(m, adapters) + (size_t)m * 4 + 127) & ~(size_t)127;
}
__host__ __device__ inline PlanView view(void* plan, int m, int adapters) {
  uint8_t* const p = static_cast<uint8_t*>(plan);
  return PlanView{reinterpret_cast<PlanHead*>(p), reinterpret_cast<Tile*>(p + tiles_at()),
                  reinterpret_cast<int*>(p + order_at(m, adapters)), reinterpret_cast<float*>(p + parts_at(m, adapters))};
}
inline int chunks_of(int k) { return (k + kChunk - 1) / kChunk; }

__device__ __forceinline__ int adapter_of(const int* ids, int t, int adapters) {
  const int a = ids[t];
  return a >= 0 && a < adapters ? a : adapters;  // (the last group: none)
}

// Counts the adapters' tokens, gives each adapter its places and tiles, then the tokens their places.
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const int* ids, int m, int adapters, void* plan) {
  extern __shared__ int n[];  // [adapters + 1] counts, then the next free places
  __shared__ int red[2][kPlanThreads / 64], base[2];
  const PlanView p = view(plan, m, adapters);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  for (int i = tid; i <= adapters; i += kPlanThreads) n[i] = 0;
  if (tid == 0) base[0] = base[1] = 0;
  __syncthreads();
  for (int t = tid; t < m; t += kPlanThreads) atomicAdd(&n[adapter_of(ids, t, adapters)], 1);
  __syncthreads();
  for (int i0 = 0; i0 <= adapters; i0 += kPlanThreads) {
    const int i = i0 + tid, count = i <= adapters ? n[i] : 0, tiles = (count + kTile - 1) / kTile;
    int x = count, y = tiles;
    for (int d = 1; d < 64; d *= 2) {
      const int u = __shfl_up(x, d), v = __shfl_up(y, d);
      if (lane >= d) x += u, y += v;
    }
    if (lane == 63) red[0][w] = x, red[1][w] = y;
    __syncthreads();
    int at = base[0] + x - count, tile = base[1] + y - tiles;
    for (int j = 0; j < w; ++j) at += red[0][j], tile += red[1][j];
    for (int j = 0; j < tiles; ++j)
      p.tiles[tile + j] = Tile{i < adapters ? i : -1, at + j * kTile, min(kTile, count - j * kTile), 0};
    if (i <= adapters) n[i] = at;
    __syncthreads();
    if (tid == kPlanThreads - 1) base[0] = at + count, base[1] = tile + tiles;
    __syncthreads();
  }
  for (int t = tid; t < m; t += kPlanThreads) p.order[atomicAdd(&n[adapter_of(ids, t, adapters)], 1)] = t;
  if (tid == 0) *p.head = PlanHead{m, adapters, base[1], 0};
}

struct LoraArgs {
  void* plan;
  const uint16_t *x, *a;
  const float* scale;
  const uint16_t* b[kMaxSegs];
  const uint16_t* y0[kMaxSegs];
  uint16_t* y[kMaxSegs];
  int n[kMaxSegs], ldy[kMaxSegs], end[kMaxSegs];  // end: of the segments' blocks of output rows
  long ldx;
  int m, adapters, k, rank, ranks, nseg, each;  // each: chunks of a part
};

__device__ __forceinline__ bf16x8 frag(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

// One wave: 16 tokens of a tile (grid x: tile, sixteen), up to 64 ranks (z), the chunks of one part (y).
__global__ void __launch_bounds__(64) lora_down_kernel(const LoraArgs a) {
  const PlanView p = view(a.plan, a.m, a.adapters);
  const int tile = blockIdx.x / (kTile / 16), sub = blockIdx.x % (kTile / 16);
  const PlanHead head = *p.head;
  if (head.m != a.m || head.adapters != a.adapters || tile >= head.tiles) return;
  const Tile t = p.tiles[tile];
  if (t.adapter < 0 || 16 * sub >= t.count) return;
  const int lane = threadIdx.x, col = lane & 15, quad = lane >> 4;
  const int token = p.order[t.start + min(16 * sub + col, t.count - 1)];
  const int r0 = blockIdx.z * 64;
  const uint16_t* const x = a.x + token * a.ldx;
  const uint16_t* const w = a.a + (size_t)t.adapter * a.ranks * a.k;
  f32x4 part[4] = {}, acc[4] = {};
  const int first = blockIdx.y * a.each, last = min(first + a.each, (a.k + kChunk - 1) / kChunk);
  for (int c = first; c < last; ++c) {
    f32x4 now[4] = {};
    const int end = min((c + 1) * kChunk, a.k);
    for (int k = c * kChunk + 8 * quad; k - 8 * quad < end; k += 32) {
      const bool in = k < end;
      const uint4 xv = in ? *reinterpret_cast<const uint4*>(x + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + 16 * i + col;
        const uint4 av = in && r < a.ranks ? *reinterpret_cast<const uint4*>(w + (size_t)r * a.k + k) : make_uint4(0, 0, 0, 0);
        now[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(av), frag(xv), now[i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      part[i] += now[i];
      if (c % kGroup == kGroup - 1 || c == last - 1) acc[i] += part[i], part[i] = f32x4{};
    }
  }
  if (16 * sub + col >= t.count) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 16 * i + 4 * quad;
    if (r < a.ranks) *reinterpret_cast<f32x4*>(p.parts + ((size_t)blockIdx.y * a.m + token) * a.ranks + r) = acc[i];
  }
}

// A workgroup: a tile's tokens and 256 output rows of a segment, 64 a wave.
constexpr int kUpRows = 256;
__global__ void __launch_bounds__(256) lora_up_kernel(const LoraArgs a) {
  extern __shared__ uint16_t sv[];  // [hi, lo][kTile][rank + 8]
  const PlanView p = view(a.plan, a.m, a.adapters);
  const PlanHead head = *p.head;
  if (head.m != a.m || head.adapters != a.adapters || (int)blockIdx.y >= head.tiles) return;
  const Tile t = p.tiles[blockIdx.y];
  int seg = 0;
  while (seg < a.nseg - 1 && (int)blockIdx.x >= a.end[seg]) ++seg;
  const int n0 = ((int)blockIdx.x - (seg ? a.end[seg - 1] : 0)) * kUpRows, n = a.n[seg];
  const long ldy = a.ldy[seg];
  const uint16_t* const y0 = a.y0[seg];
  uint16_t* const y = a.y[seg];
  if (t.adapter < 0) {
    if (y0 == y) return;
    for (int e = threadIdx.x; e < t.count * kUpRows; e += 256) {
      const size_t row = (size_t)p.order[t.start + e / kUpRows] * ldy;
      const int c = n0 + e % kUpRows;
      if (c < n) y[row + c] = y0[row + c];
    }
    return;
  }
  const int stride = a.rank + 8, parts = (a.k + kChunk * a.each - 1) / (kChunk * a.each);
  const float scale = a.scale ? a.scale[t.adapter] : 1.0f;
  for (int e = threadIdx.x; e < kTile * a.rank; e += 256) {
    const int i = e / a.rank, r = e - i * a.rank;
    float s = 0.0f;
    if (i < t.count) {
      const float* const at = p.parts + (size_t)p.order[t.start + i] * a.ranks + seg * a.rank + r;
      float part = 0.0f;
      for (int c = 0; c < parts; ++c) {
        part += at[(size_t)c * a.m * a.ranks];
        if (a.each > 1 || c % kGroup == kGroup - 1 || c == parts - 1) s += part, part = 0.0f;
      }
    }
    s *= scale;
    const uint32_t hi = f2bf(s);
    const float rest = s - bf2f(hi);
    sv[i * stride + r] = (uint16_t)hi;
    sv[(kTile + i) * stride + r] = fabsf(s) < INFINITY && fabsf(bf2f(hi)) < INFINITY ? f2bf(rest) : 0;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, wn = n0 + 64 * ((int)threadIdx.x >> 6);
  if (wn >= n) return;
  const uint16_t* const w = a.b[seg] + (size_t)t.adapter * n * a.rank;
  // row of the tile's i-th product that lane col reads: four of them leave a lane 16 neighbouring outputs
  for (int sub = 0; 16 * sub < t.count; ++sub) {
    f32x4 acc[4] = {};
    for (int k = 0; k < a.rank; k += 32) {
      const int kk = k + 8 * quad;
      const bool in = kk < a.rank;
      uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
      if (in) {
        hi = *reinterpret_cast<const uint4*>(sv + (16 * sub + col) * stride + kk);
        lo = *reinterpret_cast<const uint4*>(sv + (kTile + 16 * sub + col) * stride + kk);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = wn + 16 * (col >> 2) + 4 * i + (col & 3);
        const uint4 b = in && row < n ? *reinterpret_cast<const uint4*>(w + (size_t)row * a.rank + kk) : make_uint4(0, 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(b), frag(lo), acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(b), frag(hi), acc[i], 0, 0, 0);
      }
    }
    if (16 * sub + col < t.count) {
      const size_t at = (size_t)p.order[t.start + 16 * sub + col] * ldy;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = wn + 16 * quad + 4 * i + j;
          if (c < n) y[at + c] = f2bf(bf2f(y0[at + c]) + acc[i][j]);
        }
    }
  }
}

bool sizes_ok(int m, int adapters) {
  return m >= 0 && m <= AK_LORA_MAX_TOKENS && adapters >= 1 && adapters <= AK_LORA_MAX_ADAPTERS;
}

}  // namespace
}  // namespace agq

extern "C" size_t ak_lora_plan_bytes(int m, int adapters, int ranks, int k) {
  if (!agq::sizes_ok(m, adapters) || ranks < 8 || ranks % 8 || ranks > AK_LORA_MAX_RANK * agq::kMaxSegs || k < 8 || k % 8 ||
      k > AK_LORA_MAX_INPUTS)
    return 0;
  return agq::parts_at(m, adapters) + (size_t)agq::chunks_of(k) * m * ranks * sizeof(float);
}

extern "C" int ak_lora_plan(const int* ids, int m, int adapters, void* plan, void* stream) {
  if (!agq::sizes_ok(m, adapters) || !plan || (reinterpret_cast<uintptr_t>(plan) & 15) || (m && !ids)) return AK_INVALID;
  hipLaunchKernelGGL(agq::lora_plan_kernel, dim3(1), dim3(agq::kPlanThreads), (size_t)(adapters + 1) * 4,
                     static_cast<hipStream_t>(stream), ids, m, adapters, plan);
  return (int)hipGetLastError();
}

extern "C" int ak_lora_add(void* plan, const void* x, int m, long ldx, int k, int adapters, int rank, const void* a,
                           const float* scale, int nseg, const void* const* b, const void* const* base, void* const* y,
                           const int* n, const int* ldy, void* stream) {
  if (!agq::sizes_ok(m, adapters) || nseg < 1 || nseg > agq::kMaxSegs || rank < 8 || rank > AK_LORA_MAX_RANK || rank % 8 ||
      k < 8 || k % 8 || k > AK_LORA_MAX_INPUTS || !b || !y || !n)
    return AK_INVALID;
  const auto odd = [](const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15); };
  if (!m) return 0;
  if (odd(plan) || odd(x) || odd(a) || ldx < 0 || ldx % 8) return AK_INVALID;
  agq::LoraArgs l{};
  int blocks = 0;
  for (int i = 0; i < nseg; ++i) {
    const int ld = ldy && ldy[i] ? ldy[i] : n[i];
    if (n[i] < 1 || n[i] > AK_LORA_MAX_INPUTS || odd(b[i]) || !y[i] || (base && !base[i]) || (m > 1 && ld < n[i])) return AK_INVALID;
    l.b[i] = static_cast<const uint16_t*>(b[i]);
    l.y[i] = static_cast<uint16_t*>(y[i]);
    l.y0[i] = base ? static_cast<const uint16_t*>(base[i]) : l.y[i];
    l.n[i] = n[i], l.ldy[i] = ld;
    l.end[i] = blocks += (n[i] - 1) / agq::kUpRows + 1;
  }
  l.plan = plan, l.x = static_cast<const uint16_t*>(x), l.a = static_cast<const uint16_t*>(a), l.scale = scale;
  l.ldx = ldx, l.m = m, l.adapters = adapters, l.k = k, l.rank = rank, l.ranks = rank * nseg, l.nseg = nseg;
  const int tiles = agq::max_tiles(m, adapters), chunks = agq::chunks_of(k);
  l.each = 1;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(agq::lora_down_kernel, dim3((unsigned)tiles * (agq::kTile / 16), (unsigned)((chunks - 1) / l.each + 1),
                                                 (unsigned)((l.ranks - 1) / 64 + 1)),
                     dim3(64), 0, s, l);
  if (const int e = (int)hipGetLastError()) return e;
  hipLaunchKernelGGL(agq::lora_up_kernel, dim3((unsigned)blocks, (unsigned)tiles), dim3(256),
                     (size_t)2 * agq::kTile * (rank + 8) * 2, s, l);
  return (int)hipGetLastError();
}
