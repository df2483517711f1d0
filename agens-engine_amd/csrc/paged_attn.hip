// Attention of new tokens over the pages of the cache (kv_page.h has the layout).
//
// For token t of a sequence's T new ones, query head h and its key-value head h / (heads / kv_heads):
//   z_j = scale * q . k_j,  y = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  lse = m + log sum_j exp(z_j - m),
// over the cached tokens j < len - T + t + 1 whose page is held.  exp is taken as exp2 of z * log2(e).
//
// Bound by the bytes of the cache: every one is needed once, a few flops each.  So the rows that share a key-value head (its
// query heads, times the new tokens) are the columns of one MFMA (16 rows a tile), and the cached tokens stream:
//   * a wave holds the keys and values of its TPW tokens in registers and runs the row tiles over them: S = K Q^T (keys
//     as the A operand: the lane's 16-byte load is a piece of a row, any split of the row's values over lanes and steps
//     does, so long as the queries are loaded by the same), the softmax over the wave's tokens, then O^T = V^T P^T.
//     The scores leave the first product with the row in the lane and four tokens in its registers, which is how the
//     second takes its B operand when the tokens of 32 are numbered accordingly: the weights never change lanes.  The values
//     are loaded as whole row pieces too, and transposed in the lane: a lane holds eight tokens' pieces of the same
//     values, and pairs of tokens are what a register of the A operand is;
//   * eight waves make a part of 8 TPW tokens, summed in LDS in wave order; a workgroup takes parts from a list over all
//     sequences and heads, the next part's loads in flight from the moment the registers are free.
//
// Order of summation.  What a row gives depends on its own tokens only, never on the call: parts lie at fixed places of
// the sequence, parts are added left to right into blocks of kSuper parts, blocks left to right; a part in which a row
// sees nothing adds an exact nothing.  So T tokens verified in one call have the bits of T one-token calls, in any batch.
// Who adds is free: workgroups that hold one part each write it to scratch and the last to arrive adds them
// (split 0); a workgroup that holds a whole block adds in registers (split 1), and so does one that holds a whole
// sequence's head (split 2, which needs no scratch).
#include "agens_kernels.h"
#include "kv_page.h"

namespace agq {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kSuper = 16;      // parts of a block
constexpr int kRowTiles = 8;    // row tiles of a work item (split 0)
constexpr int kArrivals = 64;   // parts written before their counters are moved
constexpr int kCounters = 1024;
constexpr size_t kMaxPartialBytes = (size_t)32 << 20;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct AttnArgs {
  KvShape s;
  const uint16_t* q;
  uint16_t* y;
  float* lse;
  const uint8_t* pool;
  const int *qstart, *lens, *table;  // of the launch's first sequence
  long ldq, ldy;
  int m, tq, q0, b, heads, g, ldt;  // tq: tokens of a sequence without qstart, from token q0 on
  float scale;
  int* cnt;
  float* part_o;   // partial rows of D sums
  float2* part_ml; // and their largest score and sum of weights
  long cap;        // partial rows that fit
};

template <int BITS, int D>
struct Geo {
  static constexpr int RB = D * BITS / 8;                // bytes of a row
  // tokens of a wave: what its registers hold of keys and values (64 each for 16 bits)
  static constexpr int TPW = BITS == 16 ? 8192 / D : BITS == 8 ? (D == 256 ? 32 : D == 128 ? 64 : 128) : D == 256 ? 64 : 128;
  static constexpr int PART = kWaves * TPW;
  static constexpr int NS = TPW / 16, NG = TPW / 32;     // subtiles of 16 tokens, groups of 32
  static constexpr int STEPS = D / 32;                   // MFMAs of a subtile's scores
  static constexpr int KLB = RB >= 64 ? 16 : 8;          // bytes of a key load
  static constexpr int KL = RB / (4 * KLB), KW = KL * KLB / 4;
  static constexpr int EPL = KLB * 8 / BITS;             // values of a key load
  static constexpr int CH = D / 16;                      // values of a lane's piece of a value row
  static constexpr int VB = RB / 16, VW = VB >= 4 ? VB / 4 : 1;
  static constexpr int kOff = BITS == 8 ? 128 : 24;      // offset of the key codes as the scores' products see them
  static constexpr int LD = D + 4;                       // of the LDS rows: the 16 rows of a tile on different banks
  // first of the 8 values that lane group g4 contributes to step s
  static __device__ __forceinline__ int dim0(int s, int g4) {
    return (s * 8 / EPL) * 4 * EPL + g4 * EPL + (s * 8) % EPL;
  }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const f32x2 x = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const f32x2 x = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}
// 1024 + n as the f16 with n in its low bits, less the offset: a code, exactly
__device__ __forceinline__ uint32_t code_f16(uint32_t n, float offset) {
  const _Float16 o = (_Float16)(-1024.0f - offset);
  const f16x2 x = __builtin_bit_cast(f16x2, n | 0x64006400u) + f16x2{o, o};
  return __builtin_bit_cast(uint32_t, x);
}
__device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b, bool high) {  // (a's half, b's half)
  return __builtin_amdgcn_perm(b, a, high ? 0x07060302u : 0x05040100u);
}
__device__ __forceinline__ bf16x8 frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const u32x4 v = {a, b, c, d};
  return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ float ubyte(uint32_t w, int i) { return (float)((w >> (8 * i)) & 255u); }

// the keys of step s (8 values of a row) as an operand
template <int BITS, int D>
__device__ __forceinline__ bf16x8 key_frag(const uint32_t (&k)[Geo<BITS, D>::KW], int s) {
  if constexpr (BITS == 16) return frag(k[4 * s], k[4 * s + 1], k[4 * s + 2], k[4 * s + 3]);
  if constexpr (BITS == 8) {
    const uint32_t a = k[2 * s], b = k[2 * s + 1];
    return frag(pack_bf16(ubyte(a, 0), ubyte(a, 1)), pack_bf16(ubyte(a, 2), ubyte(a, 3)),
                pack_bf16(ubyte(b, 0), ubyte(b, 1)), pack_bf16(ubyte(b, 2), ubyte(b, 3)));
  }
  // a nibble in the upper bits of 16.0's mantissa is 16 + it; values i and i + 4 share a register (the queries are put
  // likewise)
  const uint32_t w = k[s];
  return frag(((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
              ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u);
}

// Value tt of the lane's pieces of 8 tokens as an operand: bf16, or the codes as f16.
template <int BITS, int D>
__device__ __forceinline__ u32x4 value_frag(const uint32_t (&v)[8][Geo<BITS, D>::VW], int tt) {
  u32x4 r;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    if constexpr (BITS == 16) {
      r[a] = halves(v[2 * a][tt / 2], v[2 * a + 1][tt / 2], tt & 1);
    } else if constexpr (BITS == 8) {
      const uint32_t sel = 0x0C040C00u + 0x00010001u * (uint32_t)(tt % 4);  // (0, second's byte, 0, first's byte)
      r[a] = code_f16(__builtin_amdgcn_perm(v[2 * a + 1][tt / 4], v[2 * a][tt / 4], sel), 128.0f);
    } else {
      const uint32_t w = halves(v[2 * a][tt / 8], v[2 * a + 1][tt / 8], tt % 8 >= 4);
      r[a] = code_f16((w >> (4 * (tt % 4))) & 0x000F000Fu, 8.0f);
    }
  }
  return r;
}
// values times weights
template <int BITS>
__device__ __forceinline__ f32x4 weigh(const u32x4 v, const u32x4 p, const f32x4 c) {
  if constexpr (BITS == 16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, p), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, v), __builtin_bit_cast(f16x8, p), c, 0, 0, 0);
}

template <int BYTES>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* r) {
  if constexpr (BYTES == 2) {
    r[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (BYTES == 4) {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    r[0] = x.x, r[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[i];
      r[4 * i] = x.x, r[4 * i + 1] = x.y, r[4 * i + 2] = x.z, r[4 * i + 3] = x.w;
    }
  }
}

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// a load of the scalar unit: it does not wait for the vector loads in flight
__device__ __forceinline__ int scalar_load(const int* p) {
  return *(const __attribute__((address_space(4))) int*)(uintptr_t)p;
}

// A row's running state: largest score (in units of log2), sum of weights, and four of the weighted sums of values.
struct Sums {
  float m = -INFINITY, l = 0.0f;
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  __device__ __forceinline__ void add(const Sums& p) {
    const float mn = fmaxf(m, p.m);
    const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float b = p.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(p.m - mn);
    l = fmaf(p.l, b, l * a);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(p.o[i], b, o[i] * a);
    m = mn;
  }
};

// What every workgroup works out alike about the launch's sequences: the work list, and where partial rows and counters
// lie.  The arrays are in LDS, indexed by sequence; the first three are sums over the sequences before.
struct Plan {
  int *items, *rows, *ctrs;  // work items of one head; partial rows and counters of all heads
  int *len, *tok;            // cached tokens and new tokens
  int split, total;          // how work is split, and the work items of all heads
};

struct Seq {
  int len, tok, parts, supers, rbs;  // rbs: row blocks of an item's kind
};

template <int PART>
__device__ __forceinline__ Seq seq_shape(const AttnArgs& a, int len, int tok, int split) {
  Seq s;
  s.len = len;
  s.tok = tok;
  s.parts = max(1, (len + PART - 1) / PART);
  s.supers = (s.parts + kSuper - 1) / kSuper;
  const int tiles = (tok * a.g + 15) / 16;
  s.rbs = split ? tiles : (tiles + kRowTiles - 1) / kRowTiles;
  return s;
}
__device__ __forceinline__ int seq_items(const Seq& s, int split) {
  return s.rbs * (split == 0 ? s.parts : split == 1 ? s.supers : 1);
}
// partial rows of one head: those of the parts, then those of the blocks
__device__ __forceinline__ long seq_rows(const Seq& s, int split, int g) {
  const long r = (long)s.tok * g;
  if (split == 0) return s.parts > 1 ? r * (s.parts + (s.supers > 1 ? s.supers : 0)) : 0;
  return split == 1 && s.supers > 1 ? r * s.supers : 0;
}
__device__ __forceinline__ int seq_ctrs(const Seq& s, int split) {
  if (!s.tok) return 0;
  if (split == 0) return s.parts == 1 ? 0 : s.supers == 1 ? 1 : s.supers + 1;
  return split == 1 && s.supers > 1 ? 1 : 0;
}

template <int PART>
__device__ void make_plan(const AttnArgs& a, Plan& p, int* mem, long* red) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  p.items = mem;
  p.rows = mem + a.b + 1;
  p.ctrs = mem + 2 * (a.b + 1);
  p.len = mem + 3 * (a.b + 1);
  p.tok = mem + 4 * (a.b + 1);
  const int kv = a.s.heads;
  const int each = (a.b + kThreads - 1) / kThreads, lo = min(a.b, tid * each), hi = min(a.b, lo + each);
  long tot[4] = {0, 0, 0, 0};  // rows and counters of split 0, rows of split 1, items
  for (int i = lo; i < hi; ++i) {
    int tok = a.tq;
    if (a.qstart) {
      const int q0 = min(max(a.qstart[i], 0), a.m);
      tok = min(max(a.qstart[i + 1], q0), a.m) - q0;
    }
    const int len = (int)min((long)max(a.lens[i], 0), (long)a.ldt * a.s.page);
    p.len[i] = len;
    p.tok[i] = tok;
    const Seq s0 = seq_shape<PART>(a, len, tok, 0), s1 = seq_shape<PART>(a, len, tok, 1);
    tot[0] += seq_rows(s0, 0, a.g) * kv;
    tot[1] += seq_ctrs(s0, 0) * kv;
    tot[2] += seq_rows(s1, 1, a.g) * kv;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < 3; ++i) tot[i] += __shfl_xor(tot[i], d);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < 3; ++i) red[3 * w + i] = tot[i];
  __syncthreads();
  long sum[3] = {0, 0, 0};
#pragma unroll
  for (int j = 0; j < kWaves; ++j)
#pragma unroll
    for (int i = 0; i < 3; ++i) sum[i] += red[3 * j + i];
  p.split = sum[0] <= a.cap && sum[1] <= kCounters ? 0 : sum[2] <= a.cap ? 1 : 2;
  __syncthreads();
  int mine[3] = {0, 0, 0};
  for (int i = lo; i < hi; ++i) {
    const Seq s = seq_shape<PART>(a, p.len[i], p.tok[i], p.split);
    mine[0] += seq_items(s, p.split);
    mine[1] += (int)seq_rows(s, p.split, a.g) * kv;
    mine[2] += seq_ctrs(s, p.split) * kv;
  }
  int inc[3] = {mine[0], mine[1], mine[2]};
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int v = __shfl_up(inc[i], d);
      inc[i] += lane >= d ? v : 0;
    }
  int* const ired = reinterpret_cast<int*>(red);
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < 3; ++i) ired[3 * w + i] = inc[i];
  __syncthreads();
  int at[3] = {inc[0] - mine[0], inc[1] - mine[1], inc[2] - mine[2]};
  for (int j = 0; j < w; ++j)
#pragma unroll
    for (int i = 0; i < 3; ++i) at[i] += ired[3 * j + i];
  int all = 0;
#pragma unroll
  for (int j = 0; j < kWaves; ++j) all += ired[3 * j];
  for (int i = lo; i < hi; ++i) {
    const Seq s = seq_shape<PART>(a, p.len[i], p.tok[i], p.split);
    p.items[i] = at[0], p.rows[i] = at[1], p.ctrs[i] = at[2];
    at[0] += seq_items(s, p.split);
    at[1] += (int)seq_rows(s, p.split, a.g) * kv;
    at[2] += seq_ctrs(s, p.split) * kv;
  }
  if (tid == 0) p.items[a.b] = all;
  p.total = all * kv;
  __syncthreads();
}

// One step of a workgroup: a part of a work item.  All of it uniform.
struct Step {
  int item, seq, head, rb, part, end, len, tok;  // the item's parts end at `end`
};

template <int PART>
__device__ __forceinline__ void first_step(const AttnArgs& a, const Plan& p, int item, Step& s) {
  s.item = item;
  if (item >= p.total) return;
  const int kv = a.s.heads, at = item / kv;
  int lo = 0, hi = a.b;  // items[lo] <= at < items[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (uni(p.items[mid]) <= at)
      lo = mid;
    else
      hi = mid;
  }
  s.seq = lo;
  s.head = item - at * kv;
  s.len = uni(p.len[lo]);
  s.tok = uni(p.tok[lo]);
  const Seq q = seq_shape<PART>(a, s.len, s.tok, p.split);
  const int rem = at - uni(p.items[lo]), u = rem / q.rbs;
  s.rb = rem - u * q.rbs;
  s.part = p.split == 0 ? u : p.split == 1 ? u * kSuper : 0;
  s.end = p.split == 0 ? u + 1 : p.split == 1 ? min(q.parts, (u + 1) * kSuper) : q.parts;
}
template <int PART>
__device__ __forceinline__ void next_step(const AttnArgs& a, const Plan& p, Step& s) {
  if (s.part + 1 < s.end)
    ++s.part;
  else
    first_step<PART>(a, p, s.item + (int)gridDim.x, s);
}

// A wave's share of a step: its keys, values and scales, as they come from memory.
template <int BITS, int D>
struct Tokens {
  using G = Geo<BITS, D>;
  uint32_t k[G::NS][G::KW], v[G::NG][8][G::VW];
  uint4 sc[G::NS];
  const uint8_t* base[G::NS];  // page and slot of each subtile
  uint32_t dead;               // subtiles without tokens or page

  // the pages: first of all, one step ahead
  __device__ __forceinline__ void find(const AttnArgs& a, const Step& s, int first) {
    dead = 0;
#pragma unroll
    for (int i = 0; i < G::NS; ++i) {
      const int tok = first + 16 * i;
      int pg = -1;
      if (tok < s.len) pg = scalar_load(a.table + (size_t)s.seq * a.ldt + tok / a.s.page);
      if ((unsigned)pg >= (unsigned)a.s.npages) dead |= 1u << i, pg = 0;  // (page 0 is there to be read)
      base[i] = a.pool + a.s.bytes() * (size_t)pg;
    }
  }
  __device__ __forceinline__ void load_keys(const AttnArgs& a, const Step& s, int first, int lane) {
    const int r = lane & 15, g4 = lane >> 4;
#pragma unroll
    for (int i = 0; i < G::NS; ++i) {
      const int slot = (first + 16 * i) & (a.s.page - 1);
      const uint8_t* const p = base[i] + (size_t)(2 * s.head * a.s.page + slot) * G::RB;
#pragma unroll
      for (int j = 0; j < G::KL; ++j)
        load_bytes<G::KLB>(p + (r * G::RB + j * 4 * G::KLB + g4 * G::KLB), &k[i][j * G::KLB / 4]);
    }
  }
  __device__ __forceinline__ void load_values(const AttnArgs& a, const Step& s, int first, int lane) {
    const int r = lane & 15, g4 = lane >> 4;
    if constexpr (BITS < 16) {
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        const int slot = (first + 16 * i) & (a.s.page - 1);
        const uint8_t* const p = base[i] + a.s.scale_off() + (size_t)(s.head * a.s.page + slot) * 4;
        sc[i] = *reinterpret_cast<const uint4*>(p + 16 * g4);
      }
    }
#pragma unroll
    for (int i = 0; i < G::NS; ++i) {
      const int slot = (first + 16 * i) & (a.s.page - 1);
      const uint8_t* const p = base[i] + (size_t)((2 * s.head + 1) * a.s.page + slot) * G::RB;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        load_bytes<G::VB>(p + ((4 * g4 + j) * G::RB + r * G::VB), v[i / 2][4 * (i & 1) + j]);
    }
  }
};

template <int BITS, int D>
__global__ void __launch_bounds__(kThreads, 2) paged_attn_kernel(const AttnArgs a) {
  using G = Geo<BITS, D>;
  extern __shared__ __align__(16) uint8_t lds[];
  float* const so = reinterpret_cast<float*>(lds);                       // [waves][16][LD] sums of values
  float* const sm = so + kWaves * 16 * G::LD;                            // [waves][16] largest scores
  float* const sl = sm + kWaves * 16;                                    // [waves][16] sums of weights
  int* const list = reinterpret_cast<int*>(sl + kWaves * 16);            // [arrivals][3]
  int* const flag = list + 3 * kArrivals;                                // [arrivals + 2]
  long* const red = reinterpret_cast<long*>(flag + kArrivals + 2);       // [3 waves]
  int* const mem = reinterpret_cast<int*>(red + 3 * kWaves);
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), r16 = lane & 15, g4 = lane >> 4;

  Plan plan;
  make_plan<G::PART>(a, plan, mem, red);
  const int split = plan.split, grp = a.g;

  // where a (sequence, head)'s partial rows begin
  auto unit_row = [&](int seq, int head, const Seq& s) __attribute__((always_inline)) {
    return (long)plan.rows[seq] + head * seq_rows(s, split, grp);
  };
  auto q_first = [&](int seq) __attribute__((always_inline)) {
    return a.qstart ? min(max(uni(a.qstart[seq]), 0), a.m) : a.q0 + seq * a.tq;
  };
  // a finished row's four values, and its lse
  auto finish = [&](const Sums& s, int seq, int head, int row, int c4) __attribute__((always_inline)) {
    const int t = row / grp, h = head * grp + row - t * grp;
    const size_t tok = (size_t)(q_first(seq) + t);
    const float inv = 1.0f / s.l;
    uint2 y = make_uint2(0u, 0u);
    if (s.l != 0.0f) {
      y.x = (uint32_t)f2bf(s.o[0] * inv) | ((uint32_t)f2bf(s.o[1] * inv) << 16);
      y.y = (uint32_t)f2bf(s.o[2] * inv) | ((uint32_t)f2bf(s.o[3] * inv) << 16);
    }
    *reinterpret_cast<uint2*>(a.y + tok * a.ldy + (size_t)h * D + 4 * c4) = y;
    if (a.lse && c4 == 0)
      a.lse[tok * a.heads + h] = s.l == 0.0f ? -INFINITY : (s.m + __log2f(s.l)) * 0.69314718055994531f;
  };
  auto put_partial = [&](const Sums& s, long at, int c4) __attribute__((always_inline)) {
    uint64_t* const o = reinterpret_cast<uint64_t*>(a.part_o + at * D + 4 * c4);
    const f32x2 lo = {s.o[0], s.o[1]}, hi = {s.o[2], s.o[3]}, ml = {s.m, s.l};
    __hip_atomic_store(o, __builtin_bit_cast(uint64_t, lo), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(o + 1, __builtin_bit_cast(uint64_t, hi), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (c4 == 0)
      __hip_atomic_store(reinterpret_cast<uint64_t*>(a.part_ml + at), __builtin_bit_cast(uint64_t, ml), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
  };
  // the left-to-right sum of n partial rows `stride` apart; four at a time in flight
  auto add_partials = [&](long at, long stride, int n, int c4) __attribute__((always_inline)) {
    constexpr int U = 8;
    Sums t;
    for (int i = 0; i < n; i += U) {
      f32x2 lo[U], hi[U], ml[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long j = at + stride * min(i + u, n - 1);
        uint64_t* const o = reinterpret_cast<uint64_t*>(a.part_o + j * D + 4 * c4);
        lo[u] = __builtin_bit_cast(f32x2, __hip_atomic_load(o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        hi[u] = __builtin_bit_cast(f32x2, __hip_atomic_load(o + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        ml[u] = __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<uint64_t*>(a.part_ml + j), __ATOMIC_RELAXED,
                                                            __HIP_MEMORY_SCOPE_AGENT));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u < n) {
          Sums p;
          p.m = ml[u].x, p.l = ml[u].y;
          p.o[0] = lo[u].x, p.o[1] = lo[u].y, p.o[2] = hi[u].x, p.o[3] = hi[u].y;
          t.add(p);
        }
      }
    }
    return t;
  };

  // Parts written to scratch since the counters were last moved: moves them, and adds up what is complete.
  int arrived = 0;
  auto flush = [&]() {
    __builtin_amdgcn_s_waitcnt(0);  // every partial is acknowledged at device scope before its counter moves
    __syncthreads();
    if (tid < arrived) {
      const int seq = list[3 * tid], head = list[3 * tid + 1], sup = list[3 * tid + 2];
      const Seq s = seq_shape<G::PART>(a, plan.len[seq], plan.tok[seq], split);
      const int want = s.rbs * (split == 1 ? s.supers : min(kSuper, s.parts - sup * kSuper));
      int* const c = a.cnt + plan.ctrs[seq] + head * seq_ctrs(s, split) + (split == 0 ? sup : 0);
      const int old = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      flag[tid] = old == want - 1;
      if (old == want - 1) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    }
    __syncthreads();
    for (int i = 0; i < arrived; ++i) {
      if (!uni(flag[i])) continue;
      const int seq = uni(list[3 * i]), head = uni(list[3 * i + 1]), sup = uni(list[3 * i + 2]);
      const Seq s = seq_shape<G::PART>(a, uni(plan.len[seq]), uni(plan.tok[seq]), split);
      const int rows = s.tok * grp;
      const long base = unit_row(seq, head, s);
      bool top = split == 1 || s.supers == 1;  // the sums are the rows' own
      if (!top) {  // one block of several
        const int n = min(kSuper, s.parts - sup * kSuper);
        for (int e = tid; e < rows * (D / 4); e += kThreads) {
          const int row = e / (D / 4), c4 = e % (D / 4);
          put_partial(add_partials(base + (long)sup * kSuper * rows + row, rows, n, c4),
                      base + (long)(s.parts + sup) * rows + row, c4);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0) {
          int* const c = a.cnt + plan.ctrs[seq] + head * seq_ctrs(s, split) + s.supers;
          const int old = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          flag[kArrivals] = old == s.supers - 1;
          if (old == s.supers - 1) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        top = uni(flag[kArrivals]);
        __syncthreads();
      }
      if (!top) continue;
      const int n = s.supers > 1 ? s.supers : s.parts;
      const long from = base + (split == 0 && s.supers > 1 ? (long)s.parts * rows : 0);
      for (int e = tid; e < rows * (D / 4); e += kThreads) {
        const int row = e / (D / 4), c4 = e % (D / 4);
        finish(add_partials(from + row, rows, n, c4), seq, head, row, c4);
      }
    }
    __syncthreads();
    arrived = 0;
  };

  Step cur, nxt;
  first_step<G::PART>(a, plan, blockIdx.x, cur);
  if (cur.item >= plan.total) return;
  Tokens<BITS, D> x;
  uint32_t q[G::STEPS][4];
  // the queries of row tile rt as an operand
  auto load_q = [&](const Step& s, int rt) __attribute__((always_inline)) {
    const int row = min(rt * 16 + r16, s.tok * grp - 1), t = row / grp, h = s.head * grp + row - t * grp;
    const uint16_t* const p = a.q + (size_t)(q_first(s.seq) + t) * a.ldq + (size_t)h * D;
#pragma unroll
    for (int i = 0; i < G::STEPS; ++i) load_bytes<16>(reinterpret_cast<const uint8_t*>(p + G::dim0(i, g4)), q[i]);
  };
  auto tile0 = [&](const Step& s) __attribute__((always_inline)) { return s.rb * (split ? 1 : kRowTiles); };
  x.find(a, cur, cur.part * G::PART + w * G::TPW);
  x.load_keys(a, cur, cur.part * G::PART + w * G::TPW, lane);
  load_q(cur, tile0(cur));
  x.load_values(a, cur, cur.part * G::PART + w * G::TPW, lane);
  const float zscale = a.scale * 1.44269504088896341f;
  constexpr int kElems = (16 * D / 4 + kThreads - 1) / kThreads;  // of a tile's sums, a thread's
  Sums block[kElems], whole[kElems];

  while (cur.item < plan.total) {
    nxt = cur;
    next_step<G::PART>(a, plan, nxt);
    const bool more = nxt.item < plan.total;
    const int first = cur.part * G::PART + w * G::TPW, nfirst = nxt.part * G::PART + w * G::TPW;
    const int len = cur.len, tok = cur.tok, rows = tok * grp;
    const int rt0 = tile0(cur), rt1 = min((rows + 15) / 16, rt0 + (split ? 1 : kRowTiles));
    const uint32_t dead = x.dead;
    const bool tail = dead || first + G::TPW > len;           // slots that hold no token of this sequence
    const bool masked = tail || first + G::TPW > len - tok + 1;  // or tokens that some rows do not see
    if (more) x.find(a, nxt, nfirst);

    for (int rt = rt0; rt < rt1; ++rt) {
      const bool last = rt + 1 == rt1;
      const int row = rt * 16 + r16, limit = len - tok + 1 + row / grp;
      // ---- scores: z[i][e] of token first + 16 i + 4 g4 + e, row r16
      float z[G::NS][4];
      {
        float qsum = 0.0f;
        bf16x8 qf[G::STEPS];
#pragma unroll
        for (int s = 0; s < G::STEPS; ++s) {
          if constexpr (BITS == 4)
            qf[s] = frag(halves(q[s][0], q[s][2], false), halves(q[s][0], q[s][2], true), halves(q[s][1], q[s][3], false),
                         halves(q[s][1], q[s][3], true));
          else
            qf[s] = frag(q[s][0], q[s][1], q[s][2], q[s][3]);
          if constexpr (BITS < 16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) qsum += bf2f(q[s][i] & 0xFFFFu) + __uint_as_float(q[s][i] & 0xFFFF0000u);
          }
        }
        float init = 0.0f;
        if constexpr (BITS < 16) {  // the codes' offset, taken off before the first product is added
          qsum += __shfl_xor(qsum, 16);
          qsum += __shfl_xor(qsum, 32);
          init = -(float)G::kOff * qsum;
        }
#pragma unroll
        for (int i = 0; i < G::NS; ++i) {
          f32x4 c = {init, init, init, init};
#pragma unroll
          for (int s = 0; s < G::STEPS; ++s)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key_frag<BITS, D>(x.k[i], s), qf[s], c, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) z[i][e] = c[e];
        }
      }
      if (!last) {
        load_q(cur, rt + 1);
      } else if (more) {
        x.load_keys(a, nxt, nfirst, lane);
        load_q(nxt, tile0(nxt));
      }
      // ---- softmax over the wave's tokens
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        const uint32_t sc[4] = {x.sc[i].x, x.sc[i].y, x.sc[i].z, x.sc[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[i][e] *= BITS == 16 ? zscale : zscale * __uint_as_float(sc[e] << 16);
          if (masked) {
            const int at = first + 16 * i + 4 * g4 + e;
            if (at >= limit || at >= len || (dead >> i & 1)) z[i][e] = -INFINITY;
          }
          top = fmaxf(top, z[i][e]);
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, ptop = 0.0f;
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        const uint32_t sc[4] = {x.sc[i].x, x.sc[i].y, x.sc[i].z, x.sc[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(z[i][e] - base);
          sum += p;
          if constexpr (BITS == 16) {
            z[i][e] = p;
          } else {  // the codes' weight; where a token is not seen its scale may be anything
            z[i][e] = masked && z[i][e] == -INFINITY ? 0.0f : p * __uint_as_float(sc[e] & 0xFFFF0000u);
            ptop = fmaxf(ptop, z[i][e]);
          }
        }
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      // The weights are rounded for the product: to bf16 beside bf16 values (the range of the values needs it), to f16,
      // 8 times as fine, beside codes -- scaled such that the row's largest is in [1, 2), so what f16 cannot hold is less
      // than 2^-25 of it.
      float unscale = 1.0f;
      u32x4 pk[G::NG];
      if constexpr (BITS < 16) {
        ptop = fmaxf(ptop, __shfl_xor(ptop, 16));
        ptop = fmaxf(ptop, __shfl_xor(ptop, 32));
        const uint32_t ex = min(max(__float_as_uint(ptop) >> 23, 2u), 252u);
        unscale = __uint_as_float(ex << 23);
        const float scale = __uint_as_float((254u - ex) << 23);
#pragma unroll
        for (int i = 0; i < G::NS; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            pk[i / 2][2 * (i & 1) + e] = pack_f16(z[i][2 * e] * scale, z[i][2 * e + 1] * scale);
      } else {
#pragma unroll
        for (int i = 0; i < G::NS; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) pk[i / 2][2 * (i & 1) + e] = pack_bf16(z[i][2 * e], z[i][2 * e + 1]);
      }
      // ---- values
      uint32_t odd = 0;  // groups with a non-finite value of a token that some row does not see
      if constexpr (BITS == 16) {
        if (masked && rt == rt0) {
#pragma unroll
          for (int i = 0; i < G::NG; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at = first + 32 * i + (j < 4 ? 4 * g4 + j : 16 + 4 * g4 + j - 4);
              if (at >= len || (dead >> (2 * i + (j >> 2)) & 1))
#pragma unroll
                for (int c = 0; c < G::VW; ++c) x.v[i][j][c] = 0;  // 0 * NaN would be NaN
            }
        }
      }
      f32x4 o[G::CH];
#pragma unroll
      for (int t = 0; t < G::CH; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (BITS == 16) {
        if (masked && tok > 1) {
#pragma unroll
          for (int i = 0; i < G::NG; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at = first + 32 * i + (j < 4 ? 4 * g4 + j : 16 + 4 * g4 + j - 4);
              uint32_t bad = 0;
#pragma unroll
              for (int c = 0; c < G::VW; ++c)
                bad |= ((x.v[i][j][c] & 0x7F80u) == 0x7F80u) | ((x.v[i][j][c] & 0x7F800000u) == 0x7F800000u);
              if (__ballot(bad && at > len - tok && at < len)) odd |= 1u << i;
            }
        }
      }
#pragma unroll
      for (int i = 0; i < G::NG; ++i) {
        const u32x4 p = pk[i];
        if (BITS == 16 && (odd >> i & 1)) {
          // Rows that do not see such a token may not multiply it by their zero weight.  All rows take the finite values
          // first; then each such token alone is added, and kept by the rows that see it.
          uint32_t keep[8][G::VW];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at = first + 32 * i + (j < 4 ? 4 * g4 + j : 16 + 4 * g4 + j - 4);
#pragma unroll
            for (int c = 0; c < G::VW; ++c) {
              uint32_t v = x.v[i][j][c];
              if (at > len - tok) {
                if ((v & 0x7F80u) == 0x7F80u) v &= 0xFFFF0000u;
                if ((v & 0x7F800000u) == 0x7F800000u) v &= 0x0000FFFFu;
              }
              keep[j][c] = v;
            }
          }
#pragma unroll
          for (int t = 0; t < G::CH; ++t)
            o[t] = weigh<BITS>(value_frag<BITS, D>(keep, t), p, o[t]);
          for (int n = 0; n < 32; ++n) {
            const int one = first + 32 * i + n;
            if (one <= len - tok || one >= len) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at = first + 32 * i + (j < 4 ? 4 * g4 + j : 16 + 4 * g4 + j - 4);
#pragma unroll
              for (int c = 0; c < G::VW; ++c) {
                uint32_t v = x.v[i][j][c];
                if (at != one || (v & 0x7F80u) != 0x7F80u) v &= 0xFFFF0000u;
                if (at != one || (v & 0x7F800000u) != 0x7F800000u) v &= 0x0000FFFFu;
                keep[j][c] = v;
              }
            }
#pragma unroll
            for (int t = 0; t < G::CH; ++t) {
              const f32x4 sum1 = weigh<BITS>(value_frag<BITS, D>(keep, t), p, o[t]);
              if (one < limit) o[t] = sum1;
            }
          }
        } else {
#pragma unroll
          for (int t = 0; t < G::CH; ++t)
            o[t] = weigh<BITS>(value_frag<BITS, D>(x.v[i], t), p, o[t]);
        }
      }
      if (last && more) x.load_values(a, nxt, nfirst, lane);

      // ---- the waves' sums, in wave order
      __syncthreads();  // the LDS rows are free
      if (row < rows) {
        if (g4 == 0) sm[w * 16 + r16] = top, sl[w * 16 + r16] = sum;
        float* const dst = so + (w * 16 + r16) * G::LD + 4 * g4 * G::CH;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < G::CH; t += 4) {
            float4 v;
            v.x = o[t][i] * unscale, v.y = o[t + 1][i] * unscale, v.z = o[t + 2][i] * unscale, v.w = o[t + 3][i] * unscale;
            *reinterpret_cast<float4*>(dst + i * G::CH + t) = v;
          }
      }
      __syncthreads();
      const int tile_rows = min(16, rows - rt * 16);
      const Seq shape = seq_shape<G::PART>(a, len, tok, split);
      const int sup = cur.part / kSuper;
#pragma unroll
      for (int u = 0; u < kElems; ++u) {
        const int e = tid + u * kThreads, rr = e / (D / 4), c4 = e % (D / 4);
        if (rr >= tile_rows) continue;
        Sums s;
#pragma unroll
        for (int j = 0; j < kWaves; ++j) s.m = fmaxf(s.m, sm[j * 16 + rr]);
#pragma unroll
        for (int j = 0; j < kWaves; ++j) {
          const float mj = sm[j * 16 + rr];
          if (mj == -INFINITY && sl[j * 16 + rr] == 0.0f) continue;  // (a NaN in the sum goes on)
          const float f = __builtin_amdgcn_exp2f(mj - s.m);
          const float4 v = *reinterpret_cast<const float4*>(so + (j * 16 + rr) * G::LD + 4 * c4);
          s.l = fmaf(sl[j * 16 + rr], f, s.l);
          s.o[0] = fmaf(v.x, f, s.o[0]), s.o[1] = fmaf(v.y, f, s.o[1]);
          s.o[2] = fmaf(v.z, f, s.o[2]), s.o[3] = fmaf(v.w, f, s.o[3]);
        }
        const int grow = rt * 16 + rr;
        if (split == 0) {
          if (shape.parts == 1)
            finish(s, cur.seq, cur.head, grow, c4);
          else
            put_partial(s, unit_row(cur.seq, cur.head, shape) + (long)cur.part * rows + grow, c4);
          continue;
        }
        block[u].add(s);
        if (cur.part + 1 == cur.end || (cur.part + 1) % kSuper == 0) {  // a block's last part
          whole[u].add(block[u]);
          if (cur.part + 1 == cur.end) {
            if (split == 1 && shape.supers > 1)
              put_partial(whole[u], unit_row(cur.seq, cur.head, shape) + (long)sup * rows + grow, c4);
            else
              finish(whole[u], cur.seq, cur.head, grow, c4);
            whole[u] = Sums();
          }
          block[u] = Sums();
        }
      }
      if (last && cur.part + 1 == cur.end && (split == 0 ? shape.parts > 1 : split == 1 && shape.supers > 1)) {
        if (tid == 0) list[3 * arrived] = cur.seq, list[3 * arrived + 1] = cur.head, list[3 * arrived + 2] = sup;
        ++arrived;
      }
    }
    if (arrived == kArrivals || (arrived && !more)) flush();
    cur = nxt;
  }
}

template <int BITS, int D>
int launch(AttnArgs a, int ldt_tokens_parts, hipStream_t s) {
  using G = Geo<BITS, D>;
  static_assert(G::KW * 4 * 64 == 16 * G::RB, "");
  (void)ldt_tokens_parts;
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      return 256;
    return n;
  }();
  const long max_tokens = (long)a.ldt * a.s.page, parts = (max_tokens + G::PART - 1) / G::PART;
  const long supers = (parts + kSuper - 1) / kSuper;
  std::lock_guard<std::mutex> lock(scratch_mutex(s));
  const long m_all = a.m;
  // partial rows of all sequences at their longest; fewer where that is more than kMaxPartialBytes
  const size_t row_bytes = (size_t)D * 4 + sizeof(float2);
  double want = parts > 1 ? (double)m_all * a.heads * (double)(parts + supers) : 0.0;
  const double most = (double)(kMaxPartialBytes / row_bytes);
  if (want > most) want = most;
  a.cap = (long)want;
  if (a.cap) {
    const CallScratch c = call_scratch(s, (size_t)a.cap * row_bytes);
    a.cnt = c.cnt;
    a.part_o = reinterpret_cast<float*>(c.data);
    a.part_ml = reinterpret_cast<float2*>(c.data + (size_t)a.cap * D * 4);
    if (!c.data) a.cap = 0;
  }
  const int per = kCounters / a.s.heads, b = a.b;
  for (int i = 0; i < b; i += per) {
    AttnArgs l = a;
    l.b = b - i < per ? b - i : per;
    l.lens = a.lens + i;
    l.table = a.table + (size_t)i * a.ldt;
    l.qstart = a.qstart ? a.qstart + i : nullptr;
    l.q0 = i * a.tq;
    const size_t smem = (size_t)(kWaves * 16 * G::LD + 2 * kWaves * 16 + 3 * kArrivals + kArrivals + 2) * 4 +
                        3 * kWaves * 8 + (size_t)5 * (l.b + 1) * 4;
    const double tiles = ((double)(a.qstart ? a.m : a.tq) * a.g + 15) / 16;
    double items = (double)l.b * a.s.heads * (double)parts * tiles;
    const unsigned grid = items < cus ? (unsigned)items : (unsigned)cus;
    hipLaunchKernelGGL((paged_attn_kernel<BITS, D>), dim3(grid ? grid : 1), dim3(kThreads), smem, s, l);
    if (const int e = (int)hipGetLastError()) return e;
  }
  return 0;
}
template <int BITS>
int launch_dim(const AttnArgs& a, hipStream_t s) {
  return a.s.dim == 64 ? launch<BITS, 64>(a, 0, s) : a.s.dim == 128 ? launch<BITS, 128>(a, 0, s) : launch<BITS, 256>(a, 0, s);
}

}  // namespace
}  // namespace agq

extern "C" int ak_paged_attn(int bits, const void* q, int m, long ldq, const void* pool, int npages, int page, int heads,
                             int kv_heads, int dim, int b, const int* qstart, const int* lens, const int* table, int ldt,
                             float scale, void* y, long ldy, float* lse, void* stream) {
  const agq::KvShape s{bits, page, kv_heads, dim, npages};
  if (!s.valid() || npages < 1 || m < 0 || b < 0 || b > AK_ATTN_MAX_SEQS || heads < 1 || heads % kv_heads || ldt < 1 ||
      !(scale - scale == 0.0f) || (m && !b) || (b && !qstart && m % b))
    return AK_INVALID;
  if (!m) return 0;
  if (!q || !pool || !lens || !table || !y || !agq::aligned16(q) || !agq::aligned16(pool) || !agq::aligned16(y) ||
      ldq < 0 || ldq % 8 || ldy < 0 || ldy % 8 || (m > 1 && ldy < (long)heads * dim))
    return AK_INVALID;
  agq::AttnArgs a{};
  a.s = s;
  a.q = static_cast<const uint16_t*>(q);
  a.y = static_cast<uint16_t*>(y);
  a.lse = lse;
  a.pool = static_cast<const uint8_t*>(pool);
  a.qstart = qstart, a.lens = lens, a.table = table;
  a.ldq = ldq, a.ldy = ldy;
  a.m = m, a.tq = qstart ? 0 : m / b, a.b = b, a.heads = heads, a.g = heads / kv_heads, a.ldt = ldt;
  a.scale = scale;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return bits == 16 ? agq::launch_dim<16>(a, st) : bits == 8 ? agq::launch_dim<8>(a, st) : agq::launch_dim<4>(a, st);
}
