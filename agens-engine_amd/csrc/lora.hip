// Low-rank adapters of many requests beside a shared linear: y_t = y0_t + scale_a B_a (A_a x_t) for the tokens t of adapter a.
//
// Tokens are grouped by adapter in tiles of up to kTile (ak_lora_plan, once for all linears of a step), so that an adapter's
// weights are read once for all of its tokens of a tile.  Then:
//   lora_down_few_kernel, lora_down_many_kernel   s = A x on MFMA (bf16, sums in fp32), a part for every kGroup chunks of kChunk
//                      inputs: 16 tokens and ranks a workgroup, or a tile and up to 64 ranks with the weights through LDS;
//   lora_join_kernel   the parts' sums, where there are many tokens and parts; otherwise
//   lora_up_kernel     adds the parts up, and y = y0 + scale (B s): s enters the MFMA as three bf16 operands, which hold all 24
//                      bits of it (one alone would move y by 2^-9 of what is added, two by 2^-17).
// A chunk's products are one chain of MFMA, the chunks' sums are added up by fours and then from left to right, whoever does it: a
// token's bits do not depend on the other tokens of the call.
//
// What bounds them.  One token of 5120 inputs, 16 ranks and 5120 outputs: three chains of loads that wait for one another (head and
// tile, token, row), 2.8 + 4.6 + 4.9 us.  64 tokens of 24 adapters beside q, k and v: the same, 2.8 + 7.3 + 6.2, where the weights'
// 16 MB are 2.3 at 7 TB/s.  4001 tokens of 27648 inputs and 64 ranks: A x reads 193 MB of x in 57 us (3.4 TB/s) and the weights from
// L2 as often; without the latter it takes 41, without x 33, and the two do not overlap fully behind one barrier a stage.  The second
// product moves 82 MB of outputs in 28 us (24 with two bf16 of a sum and not three).
#include <type_traits>

#include "agens_kernels.h"
#include "wq_common.h"

namespace agq {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64, kChunk = 512, kGroup = 4;

struct Tile {
  int adapter, count;  // adapter -1: tokens without one
};
// A plan's memory: this, tiles, kTile places for each one's tokens, then the products' parts.  (Places of their own: the tokens are
// loaded beside the tile, not after it.)
struct PlanHead {
  int m, adapters, tiles, pad;
};
struct PlanView {
  PlanHead* head;
  Tile* tiles;
  int* order;
  float* parts;  // [groups of chunks][m][ranks]
};
__host__ __device__ inline int max_tiles(int m, int adapters) {
  const long t = (long)m / kTile + (m < adapters + 1 ? m : adapters + 1);
  return (int)(t < m ? t : m);
}
__host__ __device__ inline size_t tiles_at() { return sizeof(PlanHead); }
__host__ __device__ inline size_t order_at(int m, int adapters) {
  return (tiles_at() + (size_t)max_tiles(m, adapters) * sizeof(Tile) + 127) & ~(size_t)127;
}
__host__ __device__ inline size_t parts_at(int m, int adapters) {
  return order_at(m, adapters) + (size_t)max_tiles(m, adapters) * kTile * 4;
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

// The next places of the lanes' keys (in: this lane has one).  A wave of one prompt's tokens takes them all at once.
__device__ __forceinline__ int next_place(int* n, int key, bool in) {
  const int lane = threadIdx.x & 63, k = __builtin_amdgcn_readfirstlane(key);
  if (__all(in && key == k)) {
    int base = 0;
    if (lane == 0) base = atomicAdd(&n[k], 64);
    return __builtin_amdgcn_readfirstlane(base) + lane;
  }
  return in ? atomicAdd(&n[key], 1) : 0;
}

// Counts the adapters' tokens, gives each adapter its places and tiles, then the tokens their places.  Up to kPlanEach tokens a
// thread keep the place among their adapter's that the count gave them.
constexpr int kPlanEach = 4;  // tokens of a thread at a time
template <int THREADS>
__global__ void __launch_bounds__(THREADS) lora_plan_kernel(const int* ids, int m, int adapters, void* plan) {
  extern __shared__ int n[];  // [adapters + 1] counts, then the next free places
  __shared__ int red[THREADS / 64], base;
  const PlanView p = view(plan, m, adapters);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int key[kPlanEach], place[kPlanEach];
  const bool once = m <= kPlanEach * THREADS;
  auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) {
      const int t = t0 + tid + i * THREADS;
      key[i] = t < m ? adapter_of(ids, t, adapters) : -1;
    }
  };
  load(0);
  for (int i = tid; i <= adapters; i += THREADS) n[i] = 0;
  if (tid == 0) base = 0;
  __syncthreads();
  for (int t0 = 0; t0 < m; t0 += kPlanEach * THREADS) {
    if (t0) load(t0);
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) place[i] = next_place(n, key[i], key[i] >= 0);
  }
  __syncthreads();
  for (int i0 = 0; i0 <= adapters; i0 += THREADS) {
    const int i = i0 + tid, count = i <= adapters ? n[i] : 0, tiles = (count + kTile - 1) / kTile;
    int y = tiles;
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(y, d);
      if (lane >= d) y += v;
    }
    if (lane == 63) red[w] = y;
    __syncthreads();
    int tile = base + y - tiles;
    for (int j = 0; j < w; ++j) tile += red[j];
    for (int j = 0; j < tiles; ++j) p.tiles[tile + j] = Tile{i < adapters ? i : -1, min(kTile, count - j * kTile)};
    if (i <= adapters) n[i] = tile * kTile;
    __syncthreads();
    if (tid == THREADS - 1) base = tile + tiles;
    __syncthreads();
  }
  for (int t0 = 0; t0 < m; t0 += kPlanEach * THREADS) {
    if (!once) load(t0);
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) {
      if (!once)
        place[i] = next_place(n, key[i], key[i] >= 0);
      else if (key[i] >= 0)
        place[i] += n[key[i]];
      if (key[i] >= 0) p.order[place[i]] = t0 + tid + i * THREADS;
    }
  }
  if (tid == 0) *p.head = PlanHead{m, adapters, base, 0};
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
  int m, adapters, k, rank, ranks, nseg;
  int parts;           // of the sums A x: one for each kGroup chunks
  float* sums;         // these, behind the parts, or null: lora_up_kernel adds the parts up itself
  int rows, wide;      // output rows of a workgroup; bit i: segment i's rows of y and y0 are 16-byte aligned
};

__device__ __forceinline__ uint4 load_if(bool in, const uint16_t* p) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (in) v = *reinterpret_cast<const uint4*>(p);
  return v;
}
__device__ __forceinline__ bf16x8 frag(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

// Whether a plan was made for a call of these sizes; nothing else of another one's memory is read or written, which may be shorter.
__device__ __forceinline__ bool made_for(const PlanHead& head, const LoraArgs& a) {
  return head.m == a.m && head.adapters == a.adapters;
}
// Whether it has a tile.
__device__ __forceinline__ bool has_tile(const PlanView& p, const LoraArgs& a, int tile) {
  const PlanHead head = *p.head;
  return made_for(head, a) && tile < head.tiles;
}
// The token in place i of a tile; any token's where the tile has none.
__device__ __forceinline__ int token_of(const PlanView& p, const LoraArgs& a, int tile, int i) {
  return (int)min((unsigned)p.order[tile * kTile + i], (unsigned)a.m - 1);
}

// Few tokens: a workgroup takes 16 tokens of a tile (grid x), a group of chunks (y) and 16 ranks (z), a wave a chunk, all of whose
// loads go out before its first product.  (z: the tiles' first sixteens before the second, which most tiles do not have.)
__global__ void __launch_bounds__(64 * kGroup) lora_down_few_kernel(const LoraArgs a) {
  constexpr int kSteps = kChunk / 32;
  __shared__ f32x4 sums[kGroup][64];
  const PlanView p = view(a.plan, a.m, a.adapters);
  if (!has_tile(p, a, blockIdx.x)) return;
  const Tile t = p.tiles[blockIdx.x];
  const int blocks = (a.ranks + 15) / 16, sub = blockIdx.z / blocks, r0 = (blockIdx.z - sub * blocks) * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int token = token_of(p, a, blockIdx.x, 16 * sub + col);
  if (t.adapter < 0 || 16 * sub >= t.count) return;
  const bool mine = 16 * sub + col < t.count;
  const int r = r0 + col, k0 = (blockIdx.y * kGroup + wave) * kChunk + 8 * quad;
  const uint16_t* const w = a.a + ((size_t)t.adapter * a.ranks + min(r, a.ranks - 1)) * a.k;
  const uint16_t* const x = a.x + token * a.ldx;
  uint4 av[kSteps], xv[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) av[i] = load_if(r < a.ranks && k0 + 32 * i < a.k, w + k0 + 32 * i);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) xv[i] = load_if(mine && k0 + 32 * i < a.k, x + k0 + 32 * i);
  f32x4 acc = {};
#pragma unroll
  for (int i = 0; i < kSteps; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(av[i]), frag(xv[i]), acc, 0, 0, 0);
  sums[wave][lane] = acc;
  __syncthreads();
  const int row = r0 + 4 * quad, here = min((a.k - 1) / kChunk + 1 - (int)blockIdx.y * kGroup, kGroup);
  if (wave || !mine || row >= a.ranks) return;
  f32x4 part = {};
#pragma unroll
  for (int j = 0; j < kGroup; ++j)
    if (j < here) part += sums[j][lane];
  *reinterpret_cast<f32x4*>(p.parts + ((size_t)blockIdx.y * a.m + token) * a.ranks + row) = part;
}

// Many tokens: a workgroup takes a tile (grid x), a group of chunks (y) and 16 RT ranks (z), 16 tokens a wave.  The weights go
// through LDS, kStage inputs at a time, for all four waves; the next stage's loads are in flight during a stage's products.
constexpr int kStage = 256, kStageSteps = kStage / 32, kRow = kStage * 2 + 16;  // a row's bytes: 16 more, for the banks
template <int RT>
__global__ void __launch_bounds__(256, 2) lora_down_many_kernel(const LoraArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][16 * RT * kRow];
  const PlanView p = view(a.plan, a.m, a.adapters);
  if (!has_tile(p, a, blockIdx.x)) return;
  const Tile t = p.tiles[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quad = lane >> 4, sub = tid >> 6;
  const int r0 = blockIdx.z * 16 * RT;
  const int token = token_of(p, a, blockIdx.x, 16 * sub + col);
  if (t.adapter < 0) return;
  const uint16_t* const x = a.x + token * a.ldx;
  const bool mine = 16 * sub < t.count;
  const uint16_t* const w = a.a + (size_t)t.adapter * a.ranks * a.k;
  const int first = blockIdx.y * kGroup * kChunk, last = min(first + kGroup * kChunk, a.k);
  uint4 an[2 * RT], xn[kStageSteps], xv[kStageSteps];
  auto fetch = [&](int k) {
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
      const int r = r0 + (tid >> 5) + 8 * i, kk = k + 8 * (tid & 31);
      an[i] = load_if(r < a.ranks && kk < last, w + (size_t)r * a.k + kk);
    }
#pragma unroll
    for (int i = 0; i < kStageSteps; ++i) {
      const int kk = k + 32 * i + 8 * quad;
      xn[i] = load_if(mine && kk < last, x + kk);
    }
  };
  fetch(first);
  f32x4 now[RT] = {}, sum[RT] = {};
  int buf = 0;
  for (int k = first; k < last; k += kStage, buf ^= 1) {
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i)
      *reinterpret_cast<uint4*>(lds[buf] + ((tid >> 5) + 8 * i) * kRow + 16 * (tid & 31)) = an[i];
#pragma unroll
    for (int i = 0; i < kStageSteps; ++i) xv[i] = xn[i];
    if (k + kStage < last) fetch(k + kStage);
    __syncthreads();  // (the buffer written next was read before this barrier)
    if (mine) {
#pragma unroll
      for (int i = 0; i < kStageSteps; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) {
          const uint4 av = *reinterpret_cast<const uint4*>(lds[buf] + (16 * j + col) * kRow + 64 * i + 16 * quad);
          now[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(av), frag(xv[i]), now[j], 0, 0, 0);
        }
      if ((k + kStage) % kChunk == 0 || k + kStage >= last) {
#pragma unroll
        for (int j = 0; j < RT; ++j) sum[j] += now[j], now[j] = f32x4{};
      }
    }
  }
  if (16 * sub + col >= t.count) return;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const int r = r0 + 16 * j + 4 * quad;
    if (r < a.ranks) *reinterpret_cast<f32x4*>(p.parts + ((size_t)blockIdx.y * a.m + token) * a.ranks + r) = sum[j];
  }
}

// N times four sums: their parts from left to right, kLoads loads at a time.
constexpr int kLoads = 16;
template <int N>
__device__ __forceinline__ void add_parts(const float* (&at)[N], int parts, size_t step, f32x4 (&s)[N]) {
  constexpr int kAt = kLoads / N;
  for (int c = 0; c < parts; c += kAt) {
    f32x4 x[N][kAt];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < kAt; ++j) x[i][j] = *reinterpret_cast<const f32x4*>(at[i] + min(c + j, parts - 1) * step);
#pragma unroll
    for (int j = 0; j < kAt; ++j)
      if (c + j < parts) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += x[i][j];
      }
  }
}

// What fp32 holds of four sums in kSplit bf16 each (nothing past the first beside infinities and NaN), into rows `step` apart.
constexpr int kSplit = 3;
__device__ __forceinline__ void split(f32x4 s, uint16_t* to, int step) {
#pragma unroll
  for (int j = 0; j < kSplit; ++j) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = f2bf2(s[2 * i], s[2 * i + 1]);
      const float x = bf2f(w[i] & 0xFFFFu), y = bf2f(w[i] >> 16);
      s[2 * i] = fabsf(x) < INFINITY ? s[2 * i] - x : 0.0f, s[2 * i + 1] = fabsf(y) < INFINITY ? s[2 * i + 1] - y : 0.0f;
    }
    *reinterpret_cast<uint2*>(to + j * step) = make_uint2(w[0], w[1]);
  }
}

// The sums of every token from their parts: [token][ranks].
__global__ void __launch_bounds__(256) lora_join_kernel(const LoraArgs a) {
  const PlanView p = view(a.plan, a.m, a.adapters);
  const size_t fours = a.ranks / 4, i = (size_t)blockIdx.x * 256 + threadIdx.x, token = i / fours, r = 4 * (i - token * fours);
  if (token >= (size_t)a.m || !made_for(*p.head, a)) return;
  const float* at[1] = {p.parts + token * a.ranks + r};
  f32x4 s[1] = {};
  add_parts(at, a.parts, (size_t)a.m * a.ranks, s);
  *reinterpret_cast<f32x4*>(a.sums + token * a.ranks + r) = s[0];
}

// 16 outputs of a token, 8 from c on and 8 from c + 32 on: y = y0 + scale acc.  WIDE: both rows 16-byte aligned, all 64 outputs
// of the wave within them.
template <bool WIDE>
__device__ __forceinline__ void load_out(const uint16_t* y0, int c, int n, uint32_t (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h, c += 32) {
    if constexpr (WIDE) {
      const uint4 p = *reinterpret_cast<const uint4*>(y0 + c);
      v[4 * h] = p.x, v[4 * h + 1] = p.y, v[4 * h + 2] = p.z, v[4 * h + 3] = p.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t x = c + i < n ? y0[c + i] : 0;
        v[4 * h + i / 2] = i & 1 ? v[4 * h + i / 2] | x << 16 : x;
      }
    }
  }
}
template <bool WIDE>
__device__ __forceinline__ void store_out(uint16_t* y, int c, int n, float scale, const uint32_t (&v)[8], const f32x4 (&acc)[4]) {
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    o[i] = f2bf2(bf2f(v[i] & 0xFFFFu) + scale * acc[i / 2][2 * (i & 1)], bf2f(v[i] >> 16) + scale * acc[i / 2][2 * (i & 1) + 1]);
#pragma unroll
  for (int h = 0; h < 2; ++h, c += 32) {
    if constexpr (WIDE) {
      *reinterpret_cast<uint4*>(y + c) = make_uint4(o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < n) y[c + i] = (uint16_t)(o[4 * h + i / 2] >> (16 * (i & 1)));
    }
  }
}

// 64 output rows of a segment by one wave, for all tokens of a tile: KS steps of 32 ranks.  v: the outputs before; s(sub, j, kk):
// the j-th bf16 of 8 of a token's sums.
template <int KS, bool WIDE, class S>
__device__ __forceinline__ void up_rows(const LoraArgs& a, const Tile& t, int seg, int wn, float scale, S s,
                                        const uint4 (&bv)[KS][4], const int (&tok)[kTile / 16], const uint32_t (&v)[kTile / 16][8]) {
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, n = a.n[seg], c = wn + 8 * quad;
  uint16_t* const y = a.y[seg];
  const long ldy = a.ldy[seg];
#pragma unroll
  for (int sub = 0; sub < kTile / 16; ++sub) {
    if (16 * sub >= t.count) break;
    f32x4 acc[4] = {};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      uint4 x[kSplit];
#pragma unroll
      for (int j = 0; j < kSplit; ++j) x[j] = s(sub, j, 32 * k + 8 * quad);
#pragma unroll
      for (int j = kSplit - 1; j >= 0; --j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(bv[k][i]), frag(x[j]), acc[i], 0, 0, 0);
    }
    if (16 * sub + col < t.count) store_out<WIDE>(y + tok[sub] * ldy, c, n, scale, v[sub], acc);
  }
}

// Pieces [c0, c0 + width) of a tile's rows, eight in flight a thread.
template <class T>
__device__ __forceinline__ void copy_rows(const PlanView& p, const LoraArgs& a, const Tile& t, const void* from, void* to, int c0,
                                          int width, long ld) {
  const T* const src = static_cast<const T*>(from) + c0;
  T* const dst = static_cast<T*>(to) + c0;
  const int all = t.count * width;
  for (int e0 = threadIdx.x; e0 < all; e0 += 8 * 256) {
    T v[8];
    long at[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = min(e0 + 256 * i, all - 1), row = e / width;
      at[i] = token_of(p, a, blockIdx.y, row) * ld + (e - row * width);
      v[i] = src[at[i]];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e0 + 256 * i < all) dst[at[i]] = v[i];
  }
}

// A workgroup: a tile's tokens (grid y) and a.rows output rows of a segment (x), 64 at a time a wave.  JOINED: the sums A x are
// there; otherwise it adds up their parts.  Into LDS, several loads at a time (16 bytes at a time where they are used: 31 us, not 24).
constexpr int kUpRows = 256;
template <int KS, bool JOINED>
__global__ void __launch_bounds__(256) lora_up_kernel(const LoraArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint16_t sv[];  // [kSplit][kTile][rank + 8]
  const PlanView p = view(a.plan, a.m, a.adapters);
  if (!has_tile(p, a, blockIdx.y)) return;
  const Tile t = p.tiles[blockIdx.y];
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  int tok[kTile / 16];
#pragma unroll
  for (int i = 0; i < kTile / 16; ++i) tok[i] = token_of(p, a, blockIdx.y, 16 * i + col);
  int seg = 0;
  while (seg < a.nseg - 1 && (int)blockIdx.x >= a.end[seg]) ++seg;
  const int n = a.n[seg], n0 = ((int)blockIdx.x - (seg ? a.end[seg - 1] : 0)) * a.rows, n1 = min(n0 + a.rows, n);
  const long ldy = a.ldy[seg];
  const uint16_t* const y0 = a.y0[seg];
  uint16_t* const y = a.y[seg];
  if (t.adapter < 0) {  // no products
    if (y0 != y) {
      if ((a.wide >> seg & 1) && (n1 - n0) % 8 == 0)
        copy_rows<u32x4>(p, a, t, y0, y, n0 / 8, (n1 - n0) / 8, ldy / 8);
      else
        copy_rows<uint16_t>(p, a, t, y0, y, n0, n1 - n0, ldy);
    }
    return;
  }
  const uint16_t* const w = a.b[seg] + (size_t)t.adapter * n * a.rank;
  const bool wide = a.wide >> seg & 1;
  uint4 bv[KS][4];
  uint32_t v[kTile / 16][8];
  auto load = [&](int wn) {
    // row of B for lane col of product i: two products leave a lane 8 neighbouring outputs
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = wn + 32 * (i >> 1) + 8 * (col >> 2) + 4 * (i & 1) + (col & 3), kk = 32 * k + 8 * quad;
        bv[k][i] = load_if(kk < a.rank && row < n, w + (size_t)row * a.rank + kk);
      }
#pragma unroll
    for (int i = 0; i < kTile / 16; ++i) {
      if (16 * i >= t.count) break;
      if (wide && wn + 64 <= n)
        load_out<true>(y0 + tok[i] * ldy, wn + 8 * quad, n, v[i]);
      else
        load_out<false>(y0 + tok[i] * ldy, wn + 8 * quad, n, v[i]);
    }
  };
  int wn = n0 + 64 * ((int)threadIdx.x >> 6);
  load(wn);  // (on their way while the parts are added up)
  const float scale = a.scale ? a.scale[t.adapter] : 1.0f;
  const int stride = a.rank + 8;
  if constexpr (!JOINED) {
    const size_t step = (size_t)a.m * a.ranks;
    const int fours = a.rank / 4, all = 16 * ((t.count + 15) / 16) * fours;
    auto some = [&](auto times, int e0) {  // so many times 4 ranks of a token
      constexpr int N = decltype(times)::value;
      const float* at[N];
      int to[N];
      f32x4 s[N] = {};
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int e = min(e0 + 256 * j, all - 1), i = e / fours, r = 4 * (e - i * fours);
        at[j] = p.parts + (size_t)token_of(p, a, blockIdx.y, i) * a.ranks + seg * a.rank + r;
        to[j] = i * stride + r;
      }
      add_parts(at, a.parts, step, s);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (to[j] / stride >= t.count) s[j] = f32x4{};
        split(s[j], sv + to[j], kTile * stride);
      }
    };
    // four at a time where all their parts are on their way at once: 256 tokens of 64 ranks and 3 parts 11.8 -> 7.8 us (64 of 14
    // parts would take 10 and not 8); up to 32 ranks that costs more in registers than it brings (5.9 -> 7.6).  (Of sums in two bf16.)
    if (KS == 1 || all <= 256 || a.parts > kLoads / 4) {
      for (int e0 = threadIdx.x; e0 < all; e0 += 256) some(std::integral_constant<int, 1>(), e0);
    } else if constexpr (KS > 1) {
      for (int e0 = threadIdx.x; e0 < all; e0 += 4 * 256) some(std::integral_constant<int, 4>(), e0);
    }
    __syncthreads();
  } else {
    const int fours = a.rank / 4, all = 16 * ((t.count + 15) / 16) * fours;
    for (int e0 = threadIdx.x; e0 < all; e0 += 4 * 256) {  // 4 sums of a token, four times
      f32x4 x[4];
      int to[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = min(e0 + 256 * j, all - 1), i = e / fours, r = 4 * (e - i * fours);
        to[j] = i * stride + r;
        x[j] = *reinterpret_cast<const f32x4*>(a.sums + (size_t)token_of(p, a, blockIdx.y, i) * a.ranks + seg * a.rank + r);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) split(x[j], sv + to[j], kTile * stride);
    }
    __syncthreads();
  }
  auto s = [&](int sub, int j, int kk) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (kk < a.rank) x = *reinterpret_cast<const uint4*>(sv + (j * kTile + 16 * sub + col) * stride + kk);
    return x;
  };
  for (; wn < n1; wn += kUpRows) {
    if (wn >= n0 + kUpRows) load(wn);
    if (wide && wn + 64 <= n)
      up_rows<KS, true>(a, t, seg, wn, scale, s, bv, tok, v);
    else
      up_rows<KS, false>(a, t, seg, wn, scale, s, bv, tok, v);
  }
}

template <int RT>
void down_many(const LoraArgs& l, unsigned tiles, hipStream_t s) {
  hipLaunchKernelGGL(lora_down_many_kernel<RT>,
                     dim3(tiles, (unsigned)l.parts, (unsigned)((l.ranks - 1) / (16 * RT) + 1)), dim3(256),
                     0, s, l);
}
template <int KS>
void up(const LoraArgs& l, unsigned blocks, unsigned tiles, hipStream_t s) {
  const size_t lds = (size_t)kSplit * kTile * (l.rank + 8) * 2;
  if (KS > 1 && l.sums)
    hipLaunchKernelGGL((lora_up_kernel<KS, (KS > 1)>), dim3(blocks, tiles), dim3(256), lds, s, l);
  else
    hipLaunchKernelGGL((lora_up_kernel<KS, false>), dim3(blocks, tiles), dim3(256), lds, s, l);
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
  // (and the sums, once more)
  return agq::parts_at(m, adapters) + (size_t)((agq::chunks_of(k) - 1) / agq::kGroup + 2) * m * ranks * sizeof(float);
}

extern "C" int ak_lora_plan(const int* ids, int m, int adapters, void* plan, void* stream) {
  if (!agq::sizes_ok(m, adapters) || !plan || (reinterpret_cast<uintptr_t>(plan) & 15) || (m && !ids)) return AK_INVALID;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t lds = (size_t)(adapters + 1) * 4;
  if (m <= 256 && adapters < 256)  // barriers of four waves
    hipLaunchKernelGGL(agq::lora_plan_kernel<256>, dim3(1), dim3(256), lds, s, ids, m, adapters, plan);
  else
    hipLaunchKernelGGL(agq::lora_plan_kernel<1024>, dim3(1), dim3(1024), lds, s, ids, m, adapters, plan);
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
  for (int i = 0; i < nseg; ++i) {
    const int ld = ldy && ldy[i] ? ldy[i] : n[i];
    if (n[i] < 1 || n[i] > AK_LORA_MAX_INPUTS || odd(b[i]) || !y[i] || (base && !base[i]) || (m > 1 && ld < n[i])) return AK_INVALID;
    l.b[i] = static_cast<const uint16_t*>(b[i]);
    l.y[i] = static_cast<uint16_t*>(y[i]);
    l.y0[i] = base ? static_cast<const uint16_t*>(base[i]) : l.y[i];
    l.n[i] = n[i], l.ldy[i] = ld;
    if (ld % 8 == 0 && !odd(l.y[i]) && !odd(l.y0[i])) l.wide |= 1 << i;
  }
  l.plan = plan, l.x = static_cast<const uint16_t*>(x), l.a = static_cast<const uint16_t*>(a), l.scale = scale;
  l.ldx = ldx, l.m = m, l.adapters = adapters, l.k = k, l.rank = rank, l.ranks = rank * nseg, l.nseg = nseg;
  const unsigned tiles = (unsigned)agq::max_tiles(m, adapters);
  const int chunks = agq::chunks_of(k);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // Tiles of 64 tokens and ranks read less, sixteens keep more of the GPU at work: 256 tokens of 27648 inputs and 64 ranks 36 us by
  // tiles and 42 by sixteens, 1024 of 5120 and 16 ranks 27 and 21, 2048 of 5120 and 48 ranks 44 and 45.
  l.parts = (chunks - 1) / agq::kGroup + 1;
  const bool many = (long)((m - 1) / agq::kTile + 1) * l.parts >= 52;
  if (!many)
    hipLaunchKernelGGL(agq::lora_down_few_kernel, dim3(tiles, (unsigned)l.parts, ((unsigned)(l.ranks - 1) / 16 + 1) * (agq::kTile / 16)),
                       dim3(64 * agq::kGroup), 0, s, l);
  else if (l.ranks <= 16)
    agq::down_many<1>(l, tiles, s);
  else if (l.ranks <= 32)
    agq::down_many<2>(l, tiles, s);
  else
    agq::down_many<4>(l, tiles, s);
  if (const int e = (int)hipGetLastError()) return e;
  // A launch more, but parts that are read once and not by every workgroup of outputs.  The two kernels against the one, to 5120
  // outputs: 4001 tokens of 27648 inputs and 64 ranks (14 parts) 34 us and 48, 1024 of these 16.3 and 17.6, 4000 of 9224 and 64 (5
  // parts) 33 and 45, 1500 of these 17.2 and 18.2.  Few parts are on their way at once and cost less: 3000 tokens of 5120 inputs and
  // 64 ranks (3 parts) 29 and 25, 4096 33 and 34.5, with 128 ranks 45 and 48; 1100 with 128 22 and 19.  Up to 32 ranks the parts are
  // few loads: 28 and 29 at 4096 of 27648.
  const long joined = l.parts > agq::kLoads / 4 ? 500000 : 700000;
  if (many && rank > 32 && l.parts > 1 && (long)m * l.parts * rank >= joined) {
    l.sums = agq::view(plan, m, adapters).parts + (size_t)l.parts * m * l.ranks;
    hipLaunchKernelGGL(agq::lora_join_kernel, dim3((unsigned)(((size_t)m * l.ranks / 4 - 1) / 256 + 1)), dim3(256), 0, s, l);
    if (const int e = (int)hipGetLastError()) return e;
  }
  // a workgroup adds up its tile's parts anew: more rows each where there are workgroups enough
  l.rows = agq::kUpRows;
  long rows = 0;
  for (int i = 0; i < nseg; ++i) rows += n[i];
  while (l.rows < 4 * agq::kUpRows && (long)tiles * rows / (2 * l.rows) >= 1024) l.rows *= 2;
  int blocks = 0;
  for (int i = 0; i < nseg; ++i) l.end[i] = blocks += (n[i] - 1) / l.rows + 1;
  if (rank <= 32)
    agq::up<1>(l, (unsigned)blocks, tiles, s);
  else if (rank <= 64)
    agq::up<2>(l, (unsigned)blocks, tiles, s);
  else
    agq::up<4>(l, (unsigned)blocks, tiles, s);
  return (int)hipGetLastError();
}
