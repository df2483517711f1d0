// Attention of new tokens over the pages of the cache (kv_page.h has the layout).
//
// For token t of a sequence's T new ones, query head h and its key-value head h / (heads / kv_heads):
//   z_j = scale * q . k_j,  y = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  lse = m + log sum_j exp(z_j - m),
// over the cached tokens j < len - T + t + 1 whose page is held.  exp is taken as exp2 of z * log2(e).
//
// Bound by the bytes of the cache: every one is needed once, a few flops each.  So the rows that share a key-value head (its
// query heads, times the new tokens) are the columns of one MFMA (tiles of 16 rows), and the cached tokens stream through
// waves that work alone, without LDS exchange or barriers (workgroups of 8 waves that meet in LDS after each 1024 tokens: 12
// sequences of up to 6007 tokens with one key-value head 24 us instead of 15, 8 of 6000 with 4 drafts 43 instead of 36):
//   * a wave takes a chunk of TPW tokens at a time into registers: S = K Q^T (keys as the A operand: the lane's 16-byte load
//     is a piece of a row, any split of the row's values over lanes and steps does, so long as the queries are laid out by
//     the same), the softmax of the running maximum, then O^T += V^T P^T.  The scores leave the first product with the row
//     in the lane and four tokens in its registers, which is how the second takes its B operand when the tokens of 32 are
//     numbered accordingly: the weights never change lanes.  The values are loaded as whole row pieces too, and transposed
//     in the lane: a lane holds eight tokens' pieces of the same values, and pairs of tokens are what a register of the A
//     operand is.  A weight meets the values as two operands that add up to it (split_bf16, split_f16): rounded to one, equal
//     weights all move the same way and the outputs by up to 2^-9 of the values, beyond their own rounding (two cost nothing
//     in bf16 and 8 bits; 16 contexts of 32768 in 4 bits 118 -> 123 us);
//   * the next chunk's keys are loaded as soon as the scores are done with theirs, the values likewise.
//
// Order of summation.  What a row gives depends on its own tokens only, never on the call: tokens lie in parts of 128, added
// left to right into blocks of 8 parts, these into groups of 16 blocks, and these left to right; a chunk or part in which a
// row sees nothing adds an exact nothing.  So T tokens verified in one call have the bits of T one-token calls, in any
// batch.  Who adds is free (AttnSplit): a wave takes a block and writes its sums, or a part where blocks are too few to keep
// the memory busy, and a second small kernel adds up; or, where there is no scratch for that, a wave takes a sequence's head.
// Contexts of up to one block need neither plan nor second kernel: the waves of a workgroup take a part each (kShort).
//
// Measured (heads of 128 values, 40 query heads on 8): one context of 131072 tokens in bf16 89 us, 6.0 TB/s of the cache; 64 of
// 8192 in 8 bits 196 us, 5.6; 16 of up to 32768 in 4 bits 126 us, 4.2, where unpacking, some 400 instructions a chunk, is
// what the waves wait for; one of 777 tokens 13 us, of 100 8 us: a launch, a wave's loads one after the other (page table,
// then rows), and its chunks.  8 drafts of 4 sequences (40 rows a key-value head, three tiles) 42 us in 8 bits, 53 in bf16: each
// tile loads and unpacks the tokens anew.  512 tokens on 8192: 380 us in 8 bits, 220 TFLOP/s; in bf16 580, 145.
#include "agens_kernels.h"
#include "kv_page.h"

#include <cfloat>

namespace agq {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;  // of a workgroup
constexpr int kPart = 128, kBlock = 8, kGroup = 16;  // tokens of a part, parts of a block, blocks of a group
constexpr int kTable = 64;                           // work items that a wave knows ahead
constexpr size_t kMaxPartialBytes = (size_t)240 << 20;

enum AttnSplit { kByPart, kByBlock, kByHead };

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct AttnArgs {
  KvShape s;
  const uint16_t* q;
  uint16_t* y;
  float* lse;
  const uint8_t* pool;
  const int *qstart, *lens, *table;
  long ldq, ldy;
  int m, tq, b, heads, g, ldt;  // tq: tokens of a sequence without qstart
  uint32_t g_inv;               // 2^32 / g, rounded up
  int page_log2;
  size_t page_bytes, scale_off;
  float scale;
  float* part;  // partial rows: of each D sums, then of each its largest score and sum of weights; then the plan
  int cap;      // that fit
  int few;      // blocks, below which parts are the work items
  int cus;
};

template <int BITS, int D>
struct Geo {
  static constexpr int RB = D * BITS / 8;                // bytes of a row
  // workgroups on a CU: with rows of 512 bytes a wave needs more than half of the registers (two with their spills: 32
  // contexts of 4096 in bf16 of width 256 451 us, one 184)
  static constexpr int PER_CU = RB == 512 ? 1 : 2;
  static constexpr int TPW = BITS == 16 ? (D == 64 ? 64 : 32) : D == 256 ? 32 : 64;  // tokens of a chunk
  static constexpr int NS = TPW / 16, NG = TPW / 32;     // its subtiles of 16 tokens, groups of 32
  static constexpr int STEPS = D / 32;                   // MFMAs of a subtile's scores
  static constexpr int KLB = RB >= 64 ? 16 : 8;          // bytes of a key load
  static constexpr int KL = RB / (4 * KLB), KW = KL * KLB / 4;
  static constexpr int EPL = KLB * 8 / BITS;             // values of a key load
  static constexpr int CH = D / 16;                      // values of a lane's piece of a value row
  static constexpr int VB = RB / 16, VW = VB >= 4 ? VB / 4 : 1;
  // element j of lane group g4's eight of 32 tokens: the numbering in which the scores leave their product
  static __device__ __forceinline__ int token(int j, int g4) { return (j < 4 ? j : 12 + j) + 4 * g4; }
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
// Two weights x >= 0 as two operands that add up to them.  In bf16, 16 bits of each: `hi` is the largest bf16 below x, so what
// is left for `lo` is above 0 too (down to x = 2^-117), and both products with an infinite value are that infinity.  In f16, 22
// bits of each times `unit`, a power of two.
struct Split {
  uint32_t hi, lo;
};
__device__ __forceinline__ Split split_bf16(float x0, float x1) {
  const uint32_t a = __builtin_elementwise_sub_sat(__float_as_uint(x0), 1u);
  const uint32_t b = __builtin_elementwise_sub_sat(__float_as_uint(x1), 1u);
  return {__builtin_amdgcn_perm(b, a, 0x07060302u),
          pack_bf16(x0 - __uint_as_float(a & 0xFFFF0000u), x1 - __uint_as_float(b & 0xFFFF0000u))};
}
__device__ __forceinline__ Split split_f16(float x0, float x1, float unit) {
  const auto h = __builtin_amdgcn_cvt_pkrtz(x0 * unit, x1 * unit);
  return {__builtin_bit_cast(uint32_t, h),
          pack_f16(__builtin_fmaf(x0, unit, -(float)h[0]), __builtin_fmaf(x1, unit, -(float)h[1]))};
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b, bool high) {  // (a's half, b's half)
  return __builtin_amdgcn_perm(b, a, high ? 0x07060302u : 0x05040100u);
}

// Codes as operands.  A code n in the low bits of 16 is the f16 n 2^-24, a subnormal that the matrix unit takes as it is: eight
// bits cost one byte permutation for two values, four bits a mask, where a conversion to bf16 took three instructions.  The
// second of a byte's nibbles stays where it is, as 16 n.  So the queries are f16 too, in units of a power of two for each
// row.  The offset of the keys' codes comes off the scores' sums; that of the values off every value, since a sum whose
// heavy tokens hold zeros is to be as exact as any.
template <int BITS>
__device__ __forceinline__ u32x4 minus_offset() {  // -128 2^-24, or -8 2^-24 and 16 times that
  const uint32_t even = BITS == 8 ? 0x80808080u : 0x80088008u, odd = 0x80808080u;
  return u32x4{even, odd, even, odd};
}

// the keys of step s (8 values of a row) as an operand
template <int BITS, int D>
__device__ __forceinline__ u32x4 key_frag(const uint32_t (&k)[Geo<BITS, D>::KW], int s) {
  if constexpr (BITS == 16) return u32x4{k[4 * s], k[4 * s + 1], k[4 * s + 2], k[4 * s + 3]};
  if constexpr (BITS == 8) {
    const uint32_t a = k[2 * s], b = k[2 * s + 1];
    return u32x4{__builtin_amdgcn_perm(0, a, 0x0C010C00u), __builtin_amdgcn_perm(0, a, 0x0C030C02u),
                 __builtin_amdgcn_perm(0, b, 0x0C010C00u), __builtin_amdgcn_perm(0, b, 0x0C030C02u)};
  }
  const uint32_t w = k[s], u = w >> 8;  // values i and i + 4 share a register (the queries are put likewise)
  return u32x4{w & 0x000F000Fu, w & 0x00F000F0u, u & 0x000F000Fu, u & 0x00F000F0u};
}

__device__ __forceinline__ uint32_t less_offset(uint32_t n, uint32_t offset) {
  const f16x2 x = __builtin_bit_cast(f16x2, n) - __builtin_bit_cast(f16x2, offset * 0x10001u);
  return __builtin_bit_cast(uint32_t, x);
}
// Value tt of the lane's pieces of 8 tokens as an operand: bf16, or q 2^-24 (of 4 bits 16 times that where tt is odd).
template <int BITS, int D>
__device__ __forceinline__ u32x4 value_frag(const uint32_t (&v)[8][Geo<BITS, D>::VW], int tt) {
  u32x4 r;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    if constexpr (BITS == 16) {
      r[a] = halves(v[2 * a][tt / 2], v[2 * a + 1][tt / 2], tt & 1);
    } else if constexpr (BITS == 8) {
      const uint32_t sel = 0x0C040C00u + 0x00010001u * (uint32_t)(tt % 4);  // (0, second's byte, 0, first's byte)
      r[a] = less_offset(__builtin_amdgcn_perm(v[2 * a + 1][tt / 4], v[2 * a][tt / 4], sel), 128);
    } else {
      const uint32_t w = halves(v[2 * a][tt / 8], v[2 * a + 1][tt / 8], tt % 8 >= 4);
      r[a] = less_offset((tt % 4 < 2 ? w : w >> 8) & (tt % 2 ? 0x00F000F0u : 0x000F000Fu), tt % 2 ? 128 : 8);
    }
  }
  return r;
}
// a product of bf16 operands, or of f16 ones beside codes
template <int BITS>
__device__ __forceinline__ f32x4 product(const u32x4 x, const u32x4 y, const f32x4 c) {
  if constexpr (BITS == 16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

template <int BYTES>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* r) {
  if constexpr (BYTES == 2) {
    r[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (BYTES == 4) {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 8) {
    const uint2 x = ld_stream2(reinterpret_cast<const uint2*>(p));
    r[0] = x.x, r[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 x = ld_stream(reinterpret_cast<const uint4*>(p) + i);
      r[4 * i] = x.x, r[4 * i + 1] = x.y, r[4 * i + 2] = x.z, r[4 * i + 3] = x.w;
    }
  }
}

// row / g of a row of a sequence: exact while row * g is below 2^32
__device__ __forceinline__ int div_g(const AttnArgs& a, int row) {
  return a.g == 1 ? row : (int)__umulhi((uint32_t)row, a.g_inv);
}
// the largest (sum) over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max4(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// sums over the lanes up to this one
__device__ __forceinline__ int scan64(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row 0's last into 1, 2's into 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // lane 31's into the upper half
  return x;
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// order among a wave's accesses to LDS
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
}
// a load of the scalar unit: it does not wait for the vector loads in flight
__device__ __forceinline__ int scalar_load(const int* p) {
  return *(const __attribute__((address_space(4))) int*)(uintptr_t)p;
}

__device__ __forceinline__ int parts_of(int len) { return len > kPart ? (len + kPart - 1) / kPart : 1; }

// What two sums are worth side by side: the larger score, and the factors of the first's and the second's sums.
struct Fold {
  float m, a, b;
  __device__ __forceinline__ Fold(float m1, float m2) {
    m = fmaxf(m1, m2);
    a = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - m);
    b = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - m);
  }
  __device__ __forceinline__ float operator()(float x, float y) const { return fmaf(y, b, x * a); }
};

// Four values of a row's sums, its largest score (in units of log2) and its sum of weights.
struct Sums {
  float m = -INFINITY, l = 0.0f;
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  __device__ __forceinline__ void add(const Sums& p) {
    const Fold f(m, p.m);
    m = f.m, l = f(l, p.l);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = f(o[i], p.o[i]);
  }
};

// the first of a sequence's tokens in q and y
__device__ __forceinline__ int first_token(const AttnArgs& a, int seq) {
  return a.qstart ? min(max(scalar_load(a.qstart + seq), 0), a.m) : seq * a.tq;
}
// where a row of a (sequence, head) goes: its token and query head
__device__ __forceinline__ void row_place(const AttnArgs& a, int q0, int head, int row, size_t* tok, int* h) {
  const int t = div_g(a, row);
  *tok = (size_t)(q0 + t);
  *h = head * a.g + row - t * a.g;
}
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
}

// What every workgroup works out alike about the call's sequences: the work list, and where partial rows lie.  The arrays
// are in LDS, indexed by sequence; the first two are sums over the sequences before.
struct Plan {
  int *items, *rows;  // work items of one head; partial rows of all heads
  int *len, *tok;     // cached tokens and new tokens
  int split, total;   // an AttnSplit; work items of all heads
};

__device__ __forceinline__ int seq_tiles(const AttnArgs& a, int tok) { return (tok * a.g + 15) >> 4; }
// pieces that a sequence's head is split into
__device__ __forceinline__ int seq_pieces(int len, int split) {
  const int p = parts_of(len);
  return split == kByPart ? p : split == kByBlock ? (p + kBlock - 1) / kBlock : 1;
}
// Partial rows of one head.  (No more than kTooMany are told apart: it is more than fits, and the sums over all sequences
// stay in 32 bits.)
constexpr int kTooMany = 1 << 20;
static_assert((long)kTooMany * AK_ATTN_MAX_SEQS < (1l << 31), "");
__device__ __forceinline__ int seq_rows(const AttnArgs& a, int len, int tok, int split) {
  const int n = seq_pieces(len, split);
  if (n == 1) return 0;
  return (float)tok * (float)a.g * (float)n >= (float)kTooMany ? kTooMany : tok * a.g * n;
}

// Every wave works the plan out, a lane for one sequence or a few in a row.  Blocks are the work items unless they are fewer
// than `few` and parts fit; heads are where neither fits.
__device__ __forceinline__ void make_plan(const AttnArgs& a, Plan& p, int* mem) {
  const int lane = threadIdx.x & 63;
  p.items = mem;
  p.rows = mem + a.b;
  p.len = mem + 2 * a.b;
  p.tok = mem + 3 * a.b;
  const int each = (a.b + 63) >> 6, lo = min(a.b, lane * each), hi = min(a.b, lo + each);
  int len = -1, tok = 0;
  auto load = [&](int i) __attribute__((always_inline)) {
    if (each == 1 && len >= 0) return;  // (one sequence a lane stays in registers)
    tok = a.tq;
    if (a.qstart) {
      const int q0 = min(max(a.qstart[i], 0), a.m);
      tok = min(max(a.qstart[i + 1], q0), a.m) - q0;
    }
    len = (int)min((long)max(a.lens[i], 0), min((long)a.ldt << a.page_log2, 0x7FFFF000l));
  };
  const float kv = (float)a.s.heads;
  float fits[2], blocks = 0.0f;
#pragma unroll
  for (int split = 0; split < 2; ++split) {
    int rows = 0, items = 0;
    for (int i = lo; i < hi; ++i) {
      load(i);
      rows = min(rows + seq_rows(a, len, tok, split), kTooMany);
      items = min(items + seq_tiles(a, tok) * seq_pieces(len, split), kTooMany);
    }
    fits[split] = (float)__builtin_amdgcn_readlane(scan64(rows), 63) * kv;
    blocks = (float)__builtin_amdgcn_readlane(scan64(items), 63) * kv;
  }
  const float cap = (float)a.cap;
  p.split = fits[kByPart] <= cap && blocks < (float)a.few ? kByPart : fits[kByBlock] <= cap ? kByBlock : kByHead;
  int mine[2] = {0, 0};
  for (int i = lo; i < hi; ++i) {
    load(i);
    mine[0] += seq_tiles(a, tok) * seq_pieces(len, p.split);
    mine[1] += seq_rows(a, len, tok, p.split);
  }
  int at[2] = {scan64(mine[0]), scan64(mine[1])};
  p.total = __builtin_amdgcn_readlane(at[0], 63) * a.s.heads;
  at[0] -= mine[0], at[1] -= mine[1];
  if (threadIdx.x < 64)
    for (int i = lo; i < hi; ++i) {
      load(i);
      p.items[i] = at[0], p.rows[i] = at[1] * a.s.heads;
      p.len[i] = len, p.tok[i] = tok;
      at[0] += seq_tiles(a, tok) * seq_pieces(len, p.split);
      at[1] += seq_rows(a, len, tok, p.split);
    }
  __syncthreads();
}

// A wave's work item: pieces [part, end) of parts of a sequence's head, for a tile of 16 rows.  All of it uniform; end 0: no
// such item.
struct Item {
  int k, seq, head, tile, part, end, len, tok;
};

// The wave's items k .. k + 63 into its table, a lane each.
__device__ __forceinline__ void fill_table(const AttnArgs& a, const Plan& p, int* table, int k, int n, int wave, int waves) {
  const int lane = threadIdx.x & 63;
  if (lane >= n) return;
  k += lane;
  const long item = (long)wave + (long)k * waves;
  int* const e = table + (k & (kTable - 1)) * 8;
  e[3] = 0;
  if (item >= p.total) return;
  const int at = (int)item / a.s.heads;
  int lo = 0, hi = a.b;  // items[lo] <= at < items[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const bool up = p.items[mid] <= at;
    lo = up ? mid : lo;
    hi = up ? hi : mid;
  }
  const int len = p.len[lo], tok = p.tok[lo], tiles = seq_tiles(a, tok), parts = parts_of(len);
  const int rem = at - p.items[lo], u = rem / tiles;
  const int per = p.split == kByPart ? 1 : p.split == kByBlock ? kBlock : parts;
  e[0] = lo;
  e[1] = (int)item - at * a.s.heads;
  e[2] = rem - u * tiles;
  e[3] = min(parts, (u + 1) * per);
  e[4] = u * per;
  e[5] = len;
  e[6] = tok;
}
__device__ __forceinline__ void read_item(const int* table, int k, Item& s) {
  const int4* const e = reinterpret_cast<const int4*>(table + (k & (kTable - 1)) * 8);
  const int4 x = e[0], y = e[1];
  s.k = k;
  s.seq = uni(x.x), s.head = uni(x.y), s.tile = uni(x.z), s.end = uni(x.w);
  s.part = uni(y.x), s.len = uni(y.y), s.tok = uni(y.z);
}

// A chunk, as it comes from memory.
template <int BITS, int D>
struct Tokens {
  using G = Geo<BITS, D>;
  uint32_t k[G::NS][G::KW], v[G::NG][8][G::VW];
  uint4 sc[G::NS];
  const uint8_t* base[G::NS];  // page of each subtile
  uint32_t dead;               // subtiles without tokens or page

  // lane i of the result: the page of subtile i from token `first` on (-1: no tokens there)
  static __device__ __forceinline__ int load_ids(const AttnArgs& a, const Item& s, int first, int lane) {
    const int tok = first + 16 * lane;
    int id = -1;
    if (tok < min(s.len, s.end * kPart)) id = a.table[(size_t)s.seq * a.ldt + (tok >> a.page_log2)];
    return id;
  }
  __device__ __forceinline__ void find(const AttnArgs& a, int ids, int subtile) {
    dead = 0;
#pragma unroll
    for (int i = 0; i < G::NS; ++i) {
      int pg = __builtin_amdgcn_readlane(ids, subtile + i);
      if ((unsigned)pg >= (unsigned)a.s.npages) dead |= 1u << i, pg = 0;  // (page 0 is there to be read)
      base[i] = a.pool + a.page_bytes * (uint32_t)pg;
    }
  }
  // (Where there is no next chunk (live = 0) every load reads the pool's first bytes: under a condition instead, the wait
  // for the loads before these would have to hold without them, that is, wait for these too.)
  __device__ __forceinline__ void load_keys(const AttnArgs& a, int head, int first, int lane, uint32_t live) {
    const uint32_t lane_at = ((uint32_t)(lane & 15) * G::RB + (uint32_t)(lane >> 4) * G::KLB) & live;
#pragma unroll
    for (int i = 0; i < G::NS; ++i) {
      const uint32_t slot = (uint32_t)(first + 16 * i) & (a.s.page - 1);
      const uint8_t* const p = base[i] + (size_t)(2 * head * a.s.page + slot) * G::RB;
#pragma unroll
      for (int j = 0; j < G::KL; ++j) load_bytes<G::KLB>(p + (lane_at + j * 4 * G::KLB), &k[i][j * G::KLB / 4]);
    }
  }
  __device__ __forceinline__ void load_values(const AttnArgs& a, int head, int first, int lane, uint32_t live) {
    const uint32_t r = lane & 15, g4 = lane >> 4, lane_at = (g4 * 4 * G::RB + r * G::VB) & live;
    if constexpr (BITS < 16) {
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        const uint32_t slot = (uint32_t)(first + 16 * i) & (a.s.page - 1);
        sc[i] = *reinterpret_cast<const uint4*>(base[i] + a.scale_off + (size_t)(head * a.s.page + slot) * 4 +
                                                ((16u * g4) & live));
      }
    }
#pragma unroll
    for (int i = 0; i < G::NS; ++i) {
      const uint32_t slot = (uint32_t)(first + 16 * i) & (a.s.page - 1);
      const uint8_t* const p = base[i] + (size_t)((2 * head + 1) * a.s.page + slot) * G::RB;
#pragma unroll
      for (int j = 0; j < 4; ++j) load_bytes<G::VB>(p + (lane_at + (uint32_t)j * G::RB), v[i / 2][4 * (i & 1) + j]);
    }
  }
};

// Adds the non-finite values (bf16) of the 32 tokens from `first` on that the sequence's first new token does not see, one
// token at a time, to the rows that see it.  Rare, so the values are read again rather than kept.
template <int D>
__device__ __forceinline__ void add_non_finite(const AttnArgs& a, const Item& s, int first, const u32x4 hi, const u32x4 lo,
                                               int limit, int lane, f32x4 (&o)[Geo<16, D>::CH]) {
  using G = Geo<16, D>;
#pragma unroll 1
  for (int at = max(first, s.len - s.tok + 1); at < min(first + 32, s.len); ++at) {
    const int pg = scalar_load(a.table + (size_t)s.seq * a.ldt + (at >> a.page_log2));
    if ((unsigned)pg >= (unsigned)a.s.npages) continue;
    const uint16_t* const row = reinterpret_cast<const uint16_t*>(
        a.pool + a.page_bytes * (size_t)pg + (size_t)((2 * s.head + 1) * a.s.page + (at & (a.s.page - 1))) * G::RB);
    const int n = at - first, j = (n >> 4) * 4 + (n & 3);  // element j of lane group (n % 16) / 4
    const bool mine = lane >> 4 == (n & 15) >> 2;
    auto weight = [&](const u32x4 p) {
      const uint32_t w2 = j < 2 ? p.x : j < 4 ? p.y : j < 6 ? p.z : p.w;
      return u32x4{!mine ? 0u : (j & 1) ? w2 >> 16 : w2 & 0xFFFFu, 0u, 0u, 0u};
    };
#pragma unroll
    for (int t = 0; t < G::CH; ++t) {
      const uint32_t v = row[(lane & 15) * G::CH + t];
      const bool use = mine && (v & 0x7F80u) == 0x7F80u;
      const u32x4 x{use ? v : 0u, 0u, 0u, 0u};
      const f32x4 sum = product<16>(x, weight(lo), product<16>(x, weight(hi), o[t]));
      if (at < limit) o[t] = sum;
    }
  }
}

// MODE: which work items, and so what becomes of their sums.  Parts or blocks, which a plan lists; heads, likewise; or, where
// no sequence is longer than a block, a workgroup for a sequence's head and tile, its waves a part each, which meet in LDS.
enum AttnMode { kListed, kHeads, kShort };
template <int BITS, int D, int MODE>
__global__ void __launch_bounds__(MODE == kShort ? kBlock * 64 : kThreads,
                                  MODE == kShort || (MODE == kHeads && D == 256) ? 1 : (Geo<BITS, D>::PER_CU))
    paged_attn_kernel(const AttnArgs a) {
  using G = Geo<BITS, D>;
  constexpr bool HEADS = MODE == kHeads, SHORT = MODE == kShort;
  constexpr int kLevels = HEADS ? 3 : 1;
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), r16 = lane & 15, g4 = lane >> 4;
  // the wave's running sums: of a block; where it takes whole heads also of a group of blocks, and of the groups
  f32x4* const held = reinterpret_cast<f32x4*>(lds) + w * kLevels * G::CH * 64 + lane;
  const int nw = (int)blockDim.x >> 6;
  f32x4* const meet = reinterpret_cast<f32x4*>(lds);  // kShort: each wave's sums, then its rows' tops and totals
  float2* const meet_ml = reinterpret_cast<float2*>(lds + (size_t)nw * G::CH * 1024);
  int* const tables = reinterpret_cast<int*>(lds + (size_t)nw * kLevels * G::CH * 1024);
  int* const items = tables + w * kTable * 8;
  int* const mem = tables + nw * kTable * 8;

  Plan plan;
  const int grp = a.g;
  Item cur, nxt;
  int waves = 0, wave = 0;  // kListed, kHeads
  auto next_item = [&](int k, Item& s) __attribute__((always_inline)) {
    if constexpr (SHORT) {  // its part of one tile after the other
      s = cur;
      s.k = k, s.tile = (int)blockIdx.y + k * (int)gridDim.y;
      s.part = w, s.end = s.tile < seq_tiles(a, s.tok) && w < parts_of(s.len) ? w + 1 : 0;
    } else {
      read_item(items, k, s);
    }
  };
  // The tile's sums of all parts, left to right, and its outputs: a wave takes every nw-th of the lanes' values.
  auto meet_up = [&](int tile) __attribute__((always_inline)) {
    __syncthreads();
    const int rows = cur.tok * grp, row = tile * 16 + r16, parts = parts_of(cur.len);
    size_t to;
    int h;
    row_place(a, first_token(a, cur.seq), cur.head, min(row, rows - 1), &to, &h);
    uint16_t* const y = a.y + to * a.ldy + (size_t)h * D + 4 * g4 * G::CH;
    for (int t = w; t < G::CH; t += nw) {
      Sums sum;
      for (int p = 0; p < parts; ++p) {
        const f32x4 v = meet[(p * G::CH + t) * 64 + lane];
        Sums s;
        s.m = meet_ml[p * 16 + r16].x, s.l = meet_ml[p * 16 + r16].y;
#pragma unroll
        for (int i = 0; i < 4; ++i) s.o[i] = v[i];
        sum.add(s);
      }
      const float inv = 1.0f / sum.l;
      if (row < rows) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i * G::CH + t] = sum.l == 0.0f ? (uint16_t)0 : f2bf(sum.o[i] * inv);
        if (t == 0 && a.lse && g4 == 0) a.lse[to * a.heads + h] = row_lse(sum.m, sum.l);
      }
    }
    __syncthreads();
  };
  if constexpr (SHORT) {
    plan.split = kByPart;
    cur.seq = (int)blockIdx.x / a.s.heads, cur.head = (int)blockIdx.x - cur.seq * a.s.heads;
    cur.tok = a.tq;
    if (a.qstart) {
      const int q0 = first_token(a, cur.seq);
      cur.tok = min(max(scalar_load(a.qstart + cur.seq + 1), q0), a.m) - q0;
    }
    cur.len = (int)min((long)max(scalar_load(a.lens + cur.seq), 0), (long)a.ldt << a.page_log2);
    next_item(0, cur);
    next_item(1, nxt);
    if (!cur.end) {  // no such part
      if (parts_of(cur.len) == 1) return;
      for (int tile = blockIdx.y; tile < seq_tiles(a, cur.tok); tile += gridDim.y) meet_up(tile);
      return;
    }
  } else {
    make_plan(a, plan, mem);
    if (a.cap && blockIdx.x == 0 && !HEADS) {  // for the kernel that adds up
      int* const out = reinterpret_cast<int*>(a.part + (size_t)a.cap * (D + 2));
      if (tid == 0) out[0] = plan.split;
      for (int i = tid; i < a.b; i += kThreads)
        out[1 + i] = plan.rows[i], out[1 + a.b + i] = plan.len[i], out[1 + 2 * a.b + i] = plan.tok[i];
    }
    if ((plan.split == kByHead) != HEADS) return;  // the other kernel's
    // Items go to one wave of every CU before a second, and to one of every SIMD before a second: workgroup i is on CU i % cus.
    const int turn = (int)blockIdx.x / a.cus, base = turn * a.cus;
    waves = (int)gridDim.x * nw, wave = base * nw + w * min(a.cus, (int)gridDim.x - base) + (int)blockIdx.x - base;
    fill_table(a, plan, items, 0, kTable, wave, waves);
    wave_sync();

    read_item(items, 0, cur);
    if (!cur.end) return;
    read_item(items, 1, nxt);
  }
  Tokens<BITS, D> x;
  uint4 q[G::STEPS];
  auto load_queries = [&](const Item& s) __attribute__((always_inline)) {
    size_t tok;
    int h;
    row_place(a, first_token(a, s.seq), s.head, min(s.tile * 16 + r16, s.tok * grp - 1), &tok, &h);
    const uint16_t* const p = a.q + tok * a.ldq + (size_t)h * D;
#pragma unroll
    for (int i = 0; i < G::STEPS; ++i) q[i] = *reinterpret_cast<const uint4*>(p + G::dim0(i, g4));
  };
  // of the lane's row: scores in units of log2, of the products below (the smallest normal number in place of 0, the largest in
  // that of infinity: a masked score's -inf times it is -inf, 0 times it is 0)
  float zs;
  // The queries of a new item as an operand: its sign takes the scale's.  Beside codes they are f16 with the row's largest in
  // [2^14, 2^15): what f16 does not hold of the others is less than 2^-38 of it.
  auto lay_queries = [&]() __attribute__((always_inline)) {
    zs = fabsf(a.scale) * 1.44269504088896341f;
    const bool minus = a.scale < 0.0f;
    if constexpr (BITS == 16) {
      if (minus)
#pragma unroll
        for (int s = 0; s < G::STEPS; ++s)
          q[s].x ^= 0x80008000u, q[s].y ^= 0x80008000u, q[s].z ^= 0x80008000u, q[s].w ^= 0x80008000u;
    } else {
      u16x2 m = {0, 0};
#pragma unroll
      for (int s = 0; s < G::STEPS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, word(q[s], i) & 0x7FFF7FFFu));
      const float most = max4(__uint_as_float((uint32_t)(m[0] > m[1] ? m[0] : m[1]) << 16));
      const uint32_t ex = min(max(__float_as_uint(most) >> 23, 14u), 254u), past = ex > 244u ? ex - 244u : 0u;
      const float f = __uint_as_float(((268u - ex) << 23) | (minus ? 0x80000000u : 0u));
      zs = zs * __uint_as_float((ex - past + 10u) << 23) * __uint_as_float((127u + past) << 23);  // 2^(ex - 117)
#pragma unroll
      for (int s = 0; s < G::STEPS; ++s) {
        uint4 v = q[s];
        if constexpr (BITS == 4)  // values i and i + 4 share a register
          v = make_uint4(halves(v.x, v.z, false), halves(v.x, v.z, true), halves(v.y, v.w, false), halves(v.y, v.w, true));
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float g = BITS == 4 && i % 2 ? f * 0.0625f : f;  // (those codes are 16 times as large)
          r[i] = pack_f16(__uint_as_float(word(v, i) << 16) * g, __uint_as_float(word(v, i) & 0xFFFF0000u) * g);
        }
        q[s] = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
    zs = fminf(fmaxf(zs, FLT_MIN), FLT_MAX);
  };
  // of the lane's row: largest score, sum of weights (until the end of a part, of the lane's own tokens); see the product
  float top, total, ptop, unit;
  f32x4 o[G::CH];
  auto clear = [&]() __attribute__((always_inline)) {
    top = -INFINITY, total = 0.0f, ptop = 0.0f, unit = 1.0f;
#pragma unroll
    for (int t = 0; t < G::CH; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  };
  clear();
  float htop[kLevels], htotal[kLevels];  // of the sums held in LDS
  // Level i's sums, unless these are the first for it, and the sums at hand together; held there again unless they are wanted
  // `back`.
  auto hold = [&](int i, bool first, bool back) __attribute__((always_inline)) {
    if (!first) {
      const Fold f(htop[i], top);
#pragma unroll
      for (int t = 0; t < G::CH; ++t) {
        const f32x4 h = held[(i * G::CH + t) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] = f(h[e], o[t][e]);
      }
      total = f(htotal[i], total), top = f.m;
    }
    if (!back) {
#pragma unroll
      for (int t = 0; t < G::CH; ++t) held[(i * G::CH + t) * 64] = o[t];
      htop[i] = top, htotal[i] = total;
    }
  };

  // ids: the pages of 64 subtiles from token id0 on, of cur; next_ids of nxt
  int at = cur.part * kPart, id0 = at;
  int ids = x.load_ids(a, cur, at, lane), next_ids = -1;
  load_queries(cur);
  x.find(a, ids, 0);
  if (nxt.end) next_ids = x.load_ids(a, nxt, nxt.part * kPart, lane);
  // (in this order also here: the wait for the keys is the same instruction for the first chunk and all later ones)
  x.load_keys(a, cur.head, at, lane, ~0u);
  __builtin_amdgcn_sched_barrier(0);
  x.load_values(a, cur.head, at, lane, ~0u);
  __builtin_amdgcn_sched_barrier(0);

  bool fresh = true;  // the first chunk of an item
  for (;;) {
    const int len = cur.len, tok = cur.tok, rows = tok * grp, row = cur.tile * 16 + r16;
    const uint32_t dead = x.dead;
    const bool masked = dead || at + G::TPW > len - tok + 1;  // slots without a token, or that some row does not see
    const int nat0 = at + G::TPW;
    const bool same = nat0 < min(len, cur.end * kPart);  // the item goes on
    const bool more = same || nxt.end;
    const uint32_t live = more ? ~0u : 0u;
    const int nhead = same ? cur.head : more ? nxt.head : 0;
    const int nat = same ? nat0 : more ? nxt.part * kPart : 0;

    // ---- scores: z[i][e] of token at + 16 i + 4 g4 + e, row r16
    float z[G::NS][4];
    {
      if (fresh) lay_queries();
      f32x4 c[G::NS], init = {0.0f, 0.0f, 0.0f, 0.0f};
      u32x4 qf[G::STEPS];
#pragma unroll
      for (int s = 0; s < G::STEPS; ++s) {
        qf[s] = u32x4{q[s].x, q[s].y, q[s].z, q[s].w};
        if constexpr (BITS < 16)  // the offset's product with the queries comes off first
          init = product<BITS>(minus_offset<BITS>(), qf[s], init);
      }
#pragma unroll
      for (int i = 0; i < G::NS; ++i) c[i] = init;
#pragma unroll
      for (int s = 0; s < G::STEPS; ++s)
#pragma unroll
        for (int i = 0; i < G::NS; ++i) c[i] = product<BITS>(key_frag<BITS, D>(x.k[i], s), qf[s], c[i]);
#pragma unroll
      for (int i = 0; i < G::NS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[i][e] = c[i][e];
    }
    fresh = !same;
    if (!same) {
      ids = next_ids, id0 = nat;  // (-1 where there is no next item)
      next_ids = -1;
      if (more) {
        Item then;
        next_item(nxt.k + 1, then);
        if (then.end) next_ids = x.load_ids(a, then, then.part * kPart, lane);
        load_queries(nxt);
      }
    } else if (HEADS && nat - id0 == 1024) {
      ids = x.load_ids(a, cur, nat, lane), id0 = nat;
    }
    x.find(a, ids, (nat - id0) >> 4);
    x.load_keys(a, nhead, nat, lane, live);
    // ---- softmax of the running maximum
    u32x4 pk[G::NG], pl[G::NG];
    {
      const int limit = len - tok + 1 + div_g(a, row);
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        uint32_t* const sc[4] = {&x.sc[i].x, &x.sc[i].y, &x.sc[i].z, &x.sc[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BITS < 16) z[i][e] *= __uint_as_float(*sc[e] << 16);
          if (masked) {
            const int j = at + 16 * i + 4 * g4 + e;
            const bool gone = j >= limit || j >= len || (dead >> i & 1);
            if (gone) z[i][e] = -INFINITY;
            if constexpr (BITS < 16)  // (where a token is not seen its scale may be anything)
              if (gone) *sc[e] = 0;
          }
          most = fmaxf(most, z[i][e]);
        }
      }
      most = fmaxf(top, max4(most) * zs);
      float f = most == top ? 1.0f : __builtin_amdgcn_exp2f(top - most);  // what the sums so far are worth
      top = most;
      const float base = most == -INFINITY ? 0.0f : most;
      float sum = 0.0f, pmost = 0.0f;
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        const uint32_t sc[4] = {x.sc[i].x, x.sc[i].y, x.sc[i].z, x.sc[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(z[i][e] * zs - base);  // (not fused: 0 at the top, however large)
          sum += p;
          if constexpr (BITS == 16) {
            z[i][e] = p;
          } else {  // the codes' weight
            z[i][e] = p * __uint_as_float(sc[e] & 0xFFFF0000u);
            pmost = fmaxf(pmost, z[i][e]);
          }
        }
      }
      total = fmaf(total, f, sum);
      // The weights meet the values as two operands (Split), so that they keep what the sum of weights has of them.  Beside codes
      // they are in units of a power of two such that the row's largest so far is in [2^14, 2^15): what f16 cannot hold is
      // less than 2^-39 of it.  The sums are in these units.
      float inv = 1.0f;
      if constexpr (BITS < 16) {
        ptop = fmaxf(ptop * f, max4(pmost));
        const uint32_t ex = min(max(__float_as_uint(ptop) >> 23, 15u), 252u);
        inv = __uint_as_float((268u - ex) << 23);
        f = f * unit * inv;  // (in this order a number whatever the two units: f is 0 where inv is far beyond 1 / unit)
        unit = __uint_as_float((ex - 14u) << 23);
      }
#pragma unroll
      for (int i = 0; i < G::NS; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const Split w = BITS == 16 ? split_bf16(z[i][2 * e], z[i][2 * e + 1]) : split_f16(z[i][2 * e], z[i][2 * e + 1], inv);
          pk[i / 2][2 * (i & 1) + e] = w.hi, pl[i / 2][2 * (i & 1) + e] = w.lo;
        }
      if (__ballot(f != 1.0f)) {
#pragma unroll
        for (int t = 0; t < G::CH; ++t) o[t] *= f;
      }
    }
    // ---- values
    uint32_t odd = 0;  // groups with non-finite values that not all rows see
    if constexpr (BITS == 16) {
      // A zero weight does not undo a NaN: values of slots without a token are made zero, and so are non-finite values of
      // tokens that some row does not see, which are added afterwards.
      if (masked) {
#pragma unroll
        for (int i = 0; i < G::NG; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int t = at + 32 * i + G::token(j, g4);
            const bool gone = t >= len || (dead >> (2 * i + (j >> 2)) & 1), some = !gone && t > len - tok;
            bool bad = false;
#pragma unroll
            for (int c = 0; c < G::VW; ++c) {
              uint32_t v = x.v[i][j][c];
              if (gone) v = 0;
              if (some && (v & 0x7F80u) == 0x7F80u) v &= 0xFFFF0000u, bad = true;
              if (some && (v & 0x7F800000u) == 0x7F800000u) v &= 0x0000FFFFu, bad = true;
              x.v[i][j][c] = v;
            }
            if (__ballot(bad)) odd |= 1u << i;
          }
      }
    }
#pragma unroll
    for (int i = 0; i < G::NG; ++i) {
#pragma unroll
      for (int t = 0; t < G::CH; t += 2) {
        const u32x4 v = value_frag<BITS, D>(x.v[i], t), v1 = value_frag<BITS, D>(x.v[i], t + 1);
        o[t] = product<BITS>(v, pk[i], o[t]);
        o[t + 1] = product<BITS>(v1, pk[i], o[t + 1]);
        o[t] = product<BITS>(v, pl[i], o[t]);
        o[t + 1] = product<BITS>(v1, pl[i], o[t + 1]);
      }
      if constexpr (BITS == 16) {
        if (odd >> i & 1) add_non_finite<D>(a, cur, at + 32 * i, pk[i], pl[i], len - tok + 1 + div_g(a, row), lane, o);
      }
    }
    x.load_values(a, nhead, nat, lane, live);
    const int part = at / kPart;
    at = nat;
    if (same && at % kPart) continue;

    // ---- the end of a part
    total = sum4(total);
    if constexpr (BITS < 16) {
#pragma unroll
      for (int t = 0; t < G::CH; ++t) o[t] = o[t] * (BITS == 4 && t % 2 ? 0x1p20f : 0x1p24f) * unit;
    }
    if (plan.split != kByPart) {
      const bool block_ends = !same || (part + 1) % kBlock == 0;
      hold(0, part % kBlock == 0, block_ends);
      if (HEADS && block_ends) {
        const int block = part / kBlock;
        const bool group_ends = !same || (block + 1) % kGroup == 0;
        hold(1, block % kGroup == 0, group_ends);
        if (group_ends) hold(2, block < kGroup, !same);
      }
    }
    if (same) {
      clear();
      continue;
    }
    // ---- the end of an item: the lane has 4 runs of CH sums of its row
    if (SHORT && parts_of(len) > 1) {
#pragma unroll
      for (int t = 0; t < G::CH; ++t) meet[(w * G::CH + t) * 64 + lane] = o[t];
      if (g4 == 0) meet_ml[w * 16 + r16] = make_float2(top, total);
      meet_up(cur.tile);
    } else if (row < rows) {
      const int pieces = seq_pieces(len, plan.split);
      if (!SHORT && pieces > 1) {
        const int piece = part / (plan.split == kByPart ? 1 : kBlock);
        const int to = uni(plan.rows[cur.seq]) + cur.head * rows * pieces + piece * rows + cur.tile * 16;
        // four values of all the tile's rows side by side: what a store writes is in one piece
        const int n = min(16, rows - cur.tile * 16) * 16;
        float* const p = a.part + (size_t)to * D + r16 * 16 + g4 * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < G::CH; t += 4)
            *reinterpret_cast<float4*>(p + (i * G::CH + t) / 4 * n) = make_float4(o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]);
        if (g4 == 0) reinterpret_cast<float2*>(a.part + (size_t)a.cap * D)[to + r16] = make_float2(top, total);
      } else {
        size_t to;
        int h;
        row_place(a, first_token(a, cur.seq), cur.head, row, &to, &h);
        uint16_t* const p = a.y + to * a.ldy + (size_t)h * D + 4 * g4 * G::CH;
        const float inv = 1.0f / total;
        const bool none = total == 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < G::CH; t += 4) {
            uint2 v;
            v.x = none ? 0u : (uint32_t)f2bf(o[t][i] * inv) | ((uint32_t)f2bf(o[t + 1][i] * inv) << 16);
            v.y = none ? 0u : (uint32_t)f2bf(o[t + 2][i] * inv) | ((uint32_t)f2bf(o[t + 3][i] * inv) << 16);
            *reinterpret_cast<uint2*>(p + i * G::CH + t) = v;
          }
        if (a.lse && g4 == 0) a.lse[to * a.heads + h] = row_lse(top, total);
      }
    }
    if (!more) return;
    cur = nxt;
    // (items up to cur.k + 2 are read before the next one ends)
    if constexpr (!SHORT)
      if (((cur.k + 2) & (kTable / 2 - 1)) == 0 && cur.k + 2 >= kTable) {
        fill_table(a, plan, items, cur.k + 2, kTable / 2, wave, waves);
        wave_sync();
      }
    next_item(cur.k + 1, nxt);
    clear();
  }
}

// The rows whose pieces went to scratch.  A workgroup takes rows of one (sequence, head); C4 threads side by side a row's
// values, SIDE such sets the pieces: of blocks, a set adds a group; of parts, a set adds a block, and the first set then
// the blocks of a group.
template <int D>
__global__ void __launch_bounds__(kThreads) join_kernel(const AttnArgs a) {
  constexpr int C4 = D / 4, SIDE = kThreads / C4;
  __shared__ __align__(16) uint8_t lds[kGroup * C4 * sizeof(Sums)];
  Sums* const side = reinterpret_cast<Sums*>(lds);  // [up to kGroup][C4]
  const int* const plan = reinterpret_cast<const int*>(a.part + (size_t)a.cap * (D + 2));
  const int split = plan[0], seq = blockIdx.x / a.s.heads, head = blockIdx.x - seq * a.s.heads;
  const int first = plan[1 + seq], len = plan[1 + a.b + seq], tok = plan[1 + 2 * a.b + seq];
  const int pieces = seq_pieces(len, split), rows = tok * a.g;
  if (pieces == 1) return;
  const int c4 = threadIdx.x % C4, s = threadIdx.x / C4, q0 = first_token(a, seq);
  const float* const o = a.part + (size_t)(first + head * rows * pieces) * D;
  const float2* const ml = reinterpret_cast<const float2*>(a.part + (size_t)a.cap * D) + first + head * rows * pieces;
  // left to right, n pieces from p0 on
  auto add = [&](int p0, int n, int row) {
    constexpr int U = 8;
    const int tile = row & ~15, place = tile * D + c4 / 4 * min(16, rows - tile) * 16 + (row & 15) * 16 + c4 % 4 * 4;
    Sums t;
    for (int i0 = 0; i0 < n; i0 += U) {
      float4 v[U];
      float2 w[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const size_t j = (size_t)(p0 + min(i0 + i, n - 1)) * rows;
        v[i] = *reinterpret_cast<const float4*>(o + j * D + place), w[i] = ml[j + row];
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i0 + i < n) {
          Sums p;
          p.m = w[i].x, p.l = w[i].y;
          p.o[0] = v[i].x, p.o[1] = v[i].y, p.o[2] = v[i].z, p.o[3] = v[i].w;
          t.add(p);
        }
    }
    return t;
  };
  const bool fine = split == kByPart;
  const int step = fine ? kBlock : kGroup;        // pieces of a set's share
  const int at_once = fine ? kGroup : SIDE;       // shares between two meetings: a group's blocks, or as many groups as sets
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    Sums total;
    for (int from = 0; from < pieces; from += at_once * step) {
      const int n = min(at_once, (pieces - from + step - 1) / step);
      for (int i = s; i < n; i += SIDE) {
        const int p0 = from + i * step;
        side[i * C4 + c4] = add(p0, min(step, pieces - p0), row);
      }
      __syncthreads();
      if (s == 0) {
        if (fine) {
          Sums g;
          for (int i = 0; i < n; ++i) g.add(side[i * C4 + c4]);
          total.add(g);
        } else {
          for (int i = 0; i < n; ++i) total.add(side[i * C4 + c4]);
        }
      }
      __syncthreads();
    }
    if (s == 0) {
      size_t to;
      int h;
      row_place(a, q0, head, row, &to, &h);
      const float inv = 1.0f / total.l;
      uint2 y = make_uint2(0u, 0u);
      if (total.l != 0.0f) {
        y.x = (uint32_t)f2bf(total.o[0] * inv) | ((uint32_t)f2bf(total.o[1] * inv) << 16);
        y.y = (uint32_t)f2bf(total.o[2] * inv) | ((uint32_t)f2bf(total.o[3] * inv) << 16);
      }
      *reinterpret_cast<uint2*>(a.y + to * a.ldy + (size_t)h * D + c4 % 4 * (D / 4) + c4 / 4 * 4) = y;
      if (a.lse && c4 == 0) a.lse[to * a.heads + h] = row_lse(total.m, total.l);
    }
  }
}

template <int BITS, int D>
int launch(AttnArgs a, hipStream_t s) {
  using G = Geo<BITS, D>;
  static_assert(G::KW * 4 * 64 == 16 * G::RB && kPart % G::TPW == 0 && kBlock * kPart == 64 * 16, "");
  static_assert(kThreads / (D / 4) <= kGroup, "");
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      return 256;
    return n;
  }();
  const double max_tokens = (double)a.ldt * a.s.page, rows_seq = (double)a.m / a.b * a.g;  // the latter on average
  const double tiles = ((double)(a.qstart ? a.m : a.tq) * a.g + 15) / 16;
  const double items = (double)a.b * a.s.heads * (max_tokens / kPart + 1) * tiles;  // no more than these
  const int slots = G::PER_CU * cus;
  a.cus = cus;
  // Short contexts: in one launch, a workgroup for a sequence's head.  Measured with 8 key-value heads in 8 bits (us; the two
  // launches below): 1 sequence of 100 tokens 7.8 (11.1), of 600 11.1 (12.8), of 900 13.9 (13.4); 64 of 400 18 (27), 96 of
  // 900 46 (55), 128 of 900 61 (59), 256 of 900 121 (95); 1000 of 100 61 (88).  So while its waves are no more than three times
  // what the GPU holds -- beyond that the waves of a list, which load their next item beside the present one, do better --
  // or where a sequence is one part.
  if constexpr (G::PER_CU == 2) {
    const double parts = ceil(max_tokens / kPart);
    const double t = a.qstart ? rows_seq / 16 : ((double)a.tq * a.g + 15) / 16;  // tiles of a sequence, on average
    const unsigned ty = t < 1 ? 1u : t < 1024 ? (unsigned)t : 1024u;
    if (parts <= 1 || (parts <= kBlock && (double)a.b * a.s.heads * ty * parts <= 3.0 * slots * kWaves)) {
      hipLaunchKernelGGL((paged_attn_kernel<BITS, D, kShort>), dim3((unsigned)(a.b * a.s.heads), ty),
                         dim3(64 * (unsigned)parts), (size_t)parts * (G::CH * 1024 + 128), s, a);
      return (int)hipGetLastError();
    }
  }
  // A wave streams 9 to 11 GB/s (128 values a row in 8 and 16 bits), limited by its own steps, so with few blocks parts go to
  // more waves, though their starts, ends and partial rows cost as much again.  Measured (us, blocks and parts): in bf16 576
  // blocks 52 and 58; in 8 bits 256 54 and 24, 576 71 and 44, 1024 94 and 122; in 4 bits 1024 69 and 75.
  a.few = slots * (BITS == 16 ? 2 : BITS == 8 ? 3 : 4) / 2;
  const unsigned grid = items < (double)slots * kWaves ? (unsigned)((items + kWaves - 1) / kWaves) : (unsigned)slots;
  std::lock_guard<std::mutex> lock(scratch_mutex(s));
  // Partial rows: those of all blocks at the sequences' longest, and those of as many parts as are ever taken one by one
  // (the blocks are then few); no more than kMaxPartialBytes.
  const size_t row_bytes = (size_t)D * 4 + 8, plan_bytes = (size_t)(3 * a.b + 1) * 4;
  const double by_block = (double)a.m * a.heads * (max_tokens / (kBlock * kPart) + 1);
  const double by_part = (double)a.m * a.heads * (max_tokens / kPart + 1);
  const double most_rows = (double)(a.qstart ? a.m : a.tq) * a.g;  // of a sequence's head
  const double few = (double)a.few * kBlock * (most_rows < 16 ? most_rows : 16);
  const double most = (double)(kMaxPartialBytes / row_bytes);
  double want = max_tokens <= kPart ? 0.0 : by_part < few ? by_part : few < by_block ? by_block : few;
  const bool all = want <= most;
  a.cap = (int)(all ? want : most);
  if (a.cap) {
    a.part = reinterpret_cast<float*>(call_scratch(s, (size_t)a.cap * row_bytes + plan_bytes, ScratchOf::kOperators).data);
    if (!a.part) a.cap = 0;
  }
  auto smem = [&](int waves, int levels) {
    return (size_t)waves * (levels * G::CH * 1024 + kTable * 8 * 4) + (size_t)4 * a.b * 4;
  };
  hipLaunchKernelGGL((paged_attn_kernel<BITS, D, kListed>), dim3(grid), dim3(kThreads), smem(kWaves, 1), s, a);
  if (const int e = (int)hipGetLastError()) return e;
  if (a.cap) {
    const unsigned rows = rows_seq < 1 ? 1u : rows_seq < 64 ? (unsigned)rows_seq : 64u;
    hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)(a.b * a.s.heads), rows), dim3(kThreads), 0, s, a);
    if (const int e = (int)hipGetLastError()) return e;
  }
  if (max_tokens > kPart && (!a.cap || !all)) {  // the pieces may not fit: then this one does the work, by heads
    hipLaunchKernelGGL((paged_attn_kernel<BITS, D, kHeads>), dim3(2 * grid), dim3(kThreads / 2), smem(kWaves / 2, 3), s, a);
    return (int)hipGetLastError();
  }
  return 0;
}
template <int BITS>
int launch_dim(const AttnArgs& a, hipStream_t s) {
  return a.s.dim == 64 ? launch<BITS, 64>(a, s) : a.s.dim == 128 ? launch<BITS, 128>(a, s) : launch<BITS, 256>(a, s);
}

}  // namespace
}  // namespace agq

extern "C" int ak_paged_attn(int bits, const void* q, int m, long ldq, const void* pool, int npages, int page, int heads,
                             int kv_heads, int dim, int b, const int* qstart, const int* lens, const int* table, int ldt,
                             float scale, void* y, long ldy, float* lse, void* stream) {
  const agq::KvShape s{bits, page, kv_heads, dim, npages};
  if (!s.valid() || npages < 1 || m < 0 || b < 0 || b > AK_ATTN_MAX_SEQS || heads < 1 || heads % kv_heads || ldt < 1 ||
      !(scale - scale == 0.0f) || (m && !b) || (b && !qstart && m % b) ||
      (double)m * (heads / kv_heads) * (heads / kv_heads) >= 4294967296.0)
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
  a.g_inv = a.g > 1 ? (uint32_t)(((1ull << 32) + a.g - 1) / a.g) : 0;
  a.page_log2 = __builtin_ctz((unsigned)page);
  a.page_bytes = s.bytes();
  a.scale_off = s.scale_off();
  hipStream_t st = static_cast<hipStream_t>(stream);
  try {  // (the scratch's bookkeeping allocates host memory)
    return bits == 16 ? agq::launch_dim<16>(a, st) : bits == 8 ? agq::launch_dim<8>(a, st) : agq::launch_dim<4>(a, st);
  } catch (...) {
    return AK_OOM;
  }
}
