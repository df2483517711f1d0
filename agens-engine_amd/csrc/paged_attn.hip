// Attention of new tokens over the pages of the cache (kv_page.h has the layout).
//
// For token t of a sequence's T new ones, query head h and its key-value head h / (heads / kv_heads):
//   z_j = scale * q . k_j,  y = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  lse = m + log sum_j exp(z_j - m),
// over the cached tokens j < len - T + t + 1 whose page is held.  exp is taken as exp2 of z * log2(e).
//
// Bound by the bytes of the cache: every one is needed once, a few flops each.  So the rows that share a key-value head (its
// query heads, times the new tokens) are the columns of one MFMA (tiles of 16 rows), and the cached tokens stream:
//   * a wave takes TPW tokens at a time into registers: S = K Q^T (keys as the A operand: the lane's 16-byte load is a
//     piece of a row, any split of the row's values over lanes and steps does, so long as the queries are laid out by the
//     same), the softmax of the running maximum, then O^T += V^T P^T.  The scores leave the first product with the row in
//     the lane and four tokens in its registers, which is how the second takes its B operand when the tokens of 32 are
//     numbered accordingly: the weights never change lanes.  The values are loaded as whole row pieces too, and
//     transposed in the lane: a lane holds eight tokens' pieces of the same values, and pairs of tokens are what a
//     register of the A operand is;
//   * eight waves side by side make a chunk, kChunks chunks a part, whose sums the waves then add in LDS in wave order; a
//     workgroup takes parts from a list over all sequences and heads, the next chunk's loads in flight from the moment
//     the registers are free.
//
// Order of summation.  What a row gives depends on its own tokens only, never on the call: parts lie at fixed places of
// the sequence, parts are added left to right into blocks of BLOCK parts, blocks left to right; a chunk or part in which a
// row sees nothing adds an exact nothing.  So T tokens verified in one call have the bits of T one-token calls, in any
// batch.  Who adds is free: workgroups that hold one part each write it to scratch and the last to arrive adds them
// (split 0); a workgroup that holds a whole block adds in LDS (split 1), and so does one that holds a whole sequence's
// head (split 2, which needs no scratch).
#include "agens_kernels.h"
#include "kv_page.h"

namespace agq {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTable = 64;      // work items known ahead
constexpr float kEven = 1.1f;   // the longest workgroup's tokens over the average's, for whole sequences
constexpr int kNowhere = 0x7FFFFF00;  // an offset past any scratch
constexpr size_t kMaxPartialBytes = (size_t)128 << 20;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct AttnArgs {
  KvShape s;
  const uint16_t* q;
  uint16_t* y;
  float* lse;
  const uint8_t* pool;
  const int *qstart, *lens, *table;
  long ldq, ldy;
  int m, tq, b, heads, g, ldt;      // tq: tokens of a sequence without qstart
  uint32_t g_inv;                   // 2^32 / g, rounded up
  int page_log2;
  size_t page_bytes, scale_off;
  float scale;
  float* part;  // partial rows: of each D sums, then of each its largest score and sum of weights; then the plan
  int cap;      // that fit
};

// waves of a SIMD
constexpr int simd_waves(int bits, int d, int nt) { return 2; }

template <int BITS, int D>
struct Geo {
  static constexpr int RB = D * BITS / 8;                // bytes of a row
  static constexpr int TPW = BITS == 16 ? (D == 64 ? 64 : 32) : BITS == 8 ? (D == 64 ? 64 : 32) : D == 256 ? 32 : 64;
  static constexpr int CHUNK = kWaves * TPW;
  // Parts: four of 256 tokens, so that a short context has some to share out, then of 1024; blocks of 16 parts.
  static constexpr int PART = 1024, FIRST = 256, FIRSTS = PART / FIRST, BLOCK = 16;
  static constexpr int kChunks = PART / CHUNK, kFirstChunks = FIRST / CHUNK;
  static_assert(kFirstChunks >= 1, "");
  static __host__ __device__ int parts(int len) {  // of len tokens, at least one
    return len > PART ? FIRSTS + (len - 1) / PART : len > FIRST ? (len + FIRST - 1) / FIRST : 1;
  }
  static __device__ __forceinline__ int start(int part) { return part < FIRSTS ? part * FIRST : (part - FIRSTS + 1) * PART; }
  static __device__ __forceinline__ int chunks(int part) { return part < FIRSTS ? kFirstChunks : kChunks; }
  static constexpr int NS = TPW / 16, NG = TPW / 32;     // subtiles of 16 tokens, groups of 32
  static_assert(NS * kChunks <= 64, "");                 // a lane for every subtile of a wave's part
  static constexpr int STEPS = D / 32;                   // MFMAs of a subtile's scores
  static constexpr int KLB = RB >= 64 ? 16 : 8;          // bytes of a key load
  static constexpr int KL = RB / (4 * KLB), KW = KL * KLB / 4;
  static constexpr int EPL = KLB * 8 / BITS;             // values of a key load
  static constexpr int CH = D / 16;                      // values of a lane's piece of a value row
  static constexpr int VB = RB / 16, VW = VB >= 4 ? VB / 4 : 1;
  static constexpr int kOff = BITS == 8 ? 128 : 24;      // offset of the key codes as the scores' products see them
  static constexpr int kPasses = D == 256 ? 4 : D == 128 ? 2 : 1;  // in which a tile's sums go through LDS
  static constexpr int LD = D / kPasses + 4;             // of the LDS rows: the 16 rows of a tile on different banks
  static constexpr int kSums = kWaves * 16 * LD + 2 * 16 * kWaves;  // floats
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
// a barrier for what is in LDS: it does not wait for global loads in flight
__device__ __forceinline__ void block_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
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

// the first of a sequence's tokens in q and y
__device__ __forceinline__ int first_token(const AttnArgs& a, int seq) {
  return a.qstart ? min(max(scalar_load(a.qstart + seq), 0), a.m) : seq * a.tq;
}
// a finished row's four values, and its lse
template <int D>
__device__ __forceinline__ void finish_row(const AttnArgs& a, const Sums& s, int q0, int head, int row, int c4) {
  const int t = div_g(a, row), h = head * a.g + row - t * a.g;
  const size_t tok = (size_t)(q0 + t);
  const float inv = 1.0f / s.l;
  uint2 y = make_uint2(0u, 0u);
  if (s.l != 0.0f) {
    y.x = (uint32_t)f2bf(s.o[0] * inv) | ((uint32_t)f2bf(s.o[1] * inv) << 16);
    y.y = (uint32_t)f2bf(s.o[2] * inv) | ((uint32_t)f2bf(s.o[3] * inv) << 16);
  }
  *reinterpret_cast<uint2*>(a.y + tok * a.ldy + (size_t)h * D + 4 * c4) = y;
  if (a.lse && c4 == 0)
    a.lse[tok * a.heads + h] = s.l == 0.0f ? -INFINITY : (s.m + __log2f(s.l)) * 0.69314718055994531f;
}

// What every workgroup works out alike about the launch's sequences: the work list, and where partial rows and counters
// lie.  The arrays are in LDS, indexed by sequence; the first two are sums over the sequences before.
struct Plan {
  int *items, *rows;  // work items of one head; partial rows of all heads
  int *len, *tok;            // cached tokens and new tokens
  int split, total;          // parts are the work items (0) or sequences' heads (1); of all heads
};

struct Seq {
  int len, tok, parts, rbs;  // rbs: row blocks
};

template <class G, int NT>
__device__ __forceinline__ Seq seq_shape(const AttnArgs& a, int len, int tok) {
  Seq s;
  s.len = len;
  s.tok = tok;
  s.parts = G::parts(len);
  const int tiles = (tok * a.g + 15) / 16;
  s.rbs = (tiles + NT - 1) / NT;
  return s;
}
__device__ __forceinline__ int seq_items(const Seq& s, int split) { return s.rbs * (split ? 1 : s.parts); }
// Partial rows of one head.  (No more than kTooMany are told apart: it is more
// than fits, and the sums over all sequences stay in 32 bits.)
constexpr int kTooMany = 1 << 20;
static_assert((long)kTooMany * AK_ATTN_MAX_SEQS < (1l << 31), "");
__device__ __forceinline__ int seq_rows(const Seq& s, int split, int g) {
  if (split || s.parts == 1) return 0;
  return (float)s.tok * (float)g * (float)s.parts >= (float)kTooMany ? kTooMany : s.tok * g * s.parts;
}

// Every wave works the plan out, a lane for one sequence or a few in a row.
template <class G, int NT>
__device__ __forceinline__ void make_plan(const AttnArgs& a, Plan& p, int* mem) {
  const int lane = threadIdx.x & 63;
  p.items = mem;
  p.rows = mem + a.b;
  p.len = mem + 2 * a.b;
  p.tok = mem + 3 * a.b;
  const int each = (a.b + 63) >> 6, lo = min(a.b, lane * each), hi = min(a.b, lo + each);
  const bool writes = threadIdx.x < 64;
  int len = -1, tok = 0;
  auto shape = [&](int i) __attribute__((always_inline)) {
    if (each > 1 || len < 0) {  // (one sequence a lane stays in registers)
      tok = a.tq;
      if (a.qstart) {
        const int q0 = min(max(a.qstart[i], 0), a.m);
        tok = min(max(a.qstart[i + 1], q0), a.m) - q0;
      }
      len = (int)min((long)max(a.lens[i], 0), (long)a.ldt << a.page_log2);
    }
    return seq_shape<G, NT>(a, len, tok);
  };
  int split = 0;
  for (;; ++split) {
    int mine[2] = {0, 0};
    for (int i = lo; i < hi; ++i) {
      const Seq s = shape(i);
      mine[0] += seq_items(s, split);
      mine[1] = min(mine[1] + seq_rows(s, split, a.g), kTooMany);
    }
    int at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) at[i] = scan64(mine[i]);
    const int all = __builtin_amdgcn_readlane(at[0], 63);
    const float kv = (float)a.s.heads, rows = (float)__builtin_amdgcn_readlane(at[1], 63) * kv;
    if (!split) {
      if (rows > (float)a.cap) continue;
      // whole sequences also where that keeps all workgroups busy to the end, nearly
      int units = 0, most = 0;
      float sum = 0.0f;
      for (int i = lo; i < hi; ++i) {
        const Seq s = shape(i);
        units += s.rbs, most = max(most, s.rbs ? s.len : 0), sum += (float)s.rbs * (float)s.len;
      }
      units = __builtin_amdgcn_readlane(scan64(units), 63) * a.s.heads;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) most = max(most, __shfl_xor(most, d)), sum += __shfl_xor(sum, d);
      const int turns = (units + (int)gridDim.x - 1) / (int)gridDim.x;
      if (units >= (int)gridDim.x && (float)turns * (float)most * (float)gridDim.x <= kEven * sum * kv) continue;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) at[i] -= mine[i];
    for (int i = lo; writes && i < hi; ++i) {
      const Seq s = shape(i);
      p.items[i] = at[0], p.rows[i] = at[1] * a.s.heads;
      p.len[i] = len, p.tok[i] = tok;
      at[0] += seq_items(s, split);
      at[1] += seq_rows(s, split, a.g);
    }
    p.split = split;
    p.total = all * a.s.heads;
    break;
  }
  block_sync();
}

// One step of a workgroup: a part of a work item.  All of it uniform.
struct Step {
  int k, seq, head, rb, part, end, len, tok;  // the workgroup's item k; its parts end at `end` (0: no such item)
};

// Items k .. k + n - 1 of the workgroup into the table, a lane each.
template <class G, int NT>
__device__ __forceinline__ void fill_table(const AttnArgs& a, const Plan& p, int* table, int k, int n) {
  if ((int)threadIdx.x >= n) return;
  k += (int)threadIdx.x;
  const long item = (long)blockIdx.x + (long)k * gridDim.x;
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
  const Seq q = seq_shape<G, NT>(a, p.len[lo], p.tok[lo]);
  const int rem = at - p.items[lo], u = rem / q.rbs;
  e[0] = lo;
  e[1] = (int)item - at * a.s.heads;
  e[2] = rem - u * q.rbs;
  e[3] = p.split ? q.parts : u + 1;
  e[4] = u;
  e[5] = q.len;
  e[6] = q.tok;
}
__device__ __forceinline__ void read_step(const int* table, int k, Step& s) {
  const int4* const e = reinterpret_cast<const int4*>(table + (k & (kTable - 1)) * 8);
  const int4 x = e[0], y = e[1];
  s.k = k;
  s.seq = uni(x.x), s.head = uni(x.y), s.rb = uni(x.z), s.end = uni(x.w);
  s.part = uni(y.x), s.len = uni(y.y), s.tok = uni(y.z);
}

// A wave's share of a chunk, as it comes from memory.
template <int BITS, int D>
struct Tokens {
  using G = Geo<BITS, D>;
  uint32_t k[G::NS][G::KW], v[G::NG][8][G::VW];
  uint4 sc[G::NS];
  const uint8_t* base[G::NS];  // page of each subtile
  uint32_t dead;               // subtiles without tokens or page

  // lane i of the result: the page of the wave's subtile i of a part (-1: no tokens there)
  static __device__ __forceinline__ int load_ids(const AttnArgs& a, const Step& s, int w, int lane) {
    const int tok = G::start(s.part) + lane / G::NS * G::CHUNK + w * G::TPW + 16 * (lane % G::NS);
    int id = -1;
    if (lane < G::NS * G::chunks(s.part) && tok < s.len) id = a.table[(size_t)s.seq * a.ldt + (tok >> a.page_log2)];
    return id;
  }
  __device__ __forceinline__ void find(const AttnArgs& a, int ids, int chunk) {
    dead = 0;
#pragma unroll
    for (int i = 0; i < G::NS; ++i) {
      int pg = __builtin_amdgcn_readlane(ids, chunk * G::NS + i);
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
__device__ __forceinline__ void add_non_finite(const AttnArgs& a, const Step& s, int first, const u32x4 p, int limit,
                                               int lane, f32x4 (&o)[Geo<16, D>::CH]) {
  using G = Geo<16, D>;
#pragma unroll 1
  for (int at = max(first, s.len - s.tok + 1); at < min(first + 32, s.len); ++at) {
    const int pg = scalar_load(a.table + (size_t)s.seq * a.ldt + (at >> a.page_log2));
    if ((unsigned)pg >= (unsigned)a.s.npages) continue;
    const uint16_t* const row = reinterpret_cast<const uint16_t*>(
        a.pool + a.page_bytes * (size_t)pg + (size_t)((2 * s.head + 1) * a.s.page + (at & (a.s.page - 1))) * G::RB);
    const int n = at - first, j = (n >> 4) * 4 + (n & 3);  // element j of lane group (n % 16) / 4
    const bool mine = lane >> 4 == (n & 15) >> 2;
    const uint32_t w2 = j < 2 ? p.x : j < 4 ? p.y : j < 6 ? p.z : p.w, w = (j & 1) ? w2 >> 16 : w2 & 0xFFFFu;
#pragma unroll
    for (int t = 0; t < G::CH; ++t) {
      const uint32_t v = row[(lane & 15) * G::CH + t];
      const bool use = mine && (v & 0x7F80u) == 0x7F80u;
      const f32x4 sum = weigh<16>(u32x4{use ? v : 0u, 0u, 0u, 0u}, u32x4{mine ? w : 0u, 0u, 0u, 0u}, o[t]);
      if (at < limit) o[t] = sum;
    }
  }
}

template <int BITS, int D, int NT>
__global__ void __launch_bounds__(kThreads, simd_waves(BITS, D, NT)) paged_attn_kernel(const AttnArgs a) {
  using G = Geo<BITS, D>;
  extern __shared__ __align__(16) uint8_t lds[];
  float* const so = reinterpret_cast<float*>(lds);               // [waves][16][LD] the waves' sums
  float* const sm = so + kWaves * 16 * G::LD;                    // [16][waves] largest scores
  float* const sl = sm + 16 * kWaves;                            // [16][waves] sums of weights
  uint4* const sq = reinterpret_cast<uint4*>(so + G::kSums);     // [NT][STEPS][64] the queries as operands
  Sums* const state = reinterpret_cast<Sums*>(sq + NT * G::STEPS * 64);  // split > 0: [2][NT][16 D / 4] running sums
  int* const items = reinterpret_cast<int*>(state + 2 * NT * 16 * D / 4);  // [kTable][8]
  int* const mem = items + kTable * 8;
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), r16 = lane & 15, g4 = lane >> 4;

  Plan plan;
  make_plan<G, NT>(a, plan, mem);
  const int split = plan.split, grp = a.g;
  fill_table<G, NT>(a, plan, items, 0, kTable);
  if (a.cap && blockIdx.x == 0) {  // for the kernel that joins the parts
    int* const out = reinterpret_cast<int*>(a.part + (size_t)a.cap * (D + 2));
    if (tid == 0) out[0] = split;
    for (int i = tid; i < a.b; i += kThreads)
      out[1 + i] = plan.rows[i], out[1 + a.b + i] = plan.len[i], out[1 + 2 * a.b + i] = plan.tok[i];
  }
  block_sync();

  // where a (sequence, head)'s partial rows begin
  auto unit_row = [&](int seq, int head, const Seq& s) __attribute__((always_inline)) {
    return plan.rows[seq] + head * seq_rows(s, split, grp);
  };
  const __amdgpu_buffer_rsrc_t scratch =
      __builtin_amdgcn_make_buffer_rsrc(a.part, (short)0, (int)(a.cap * (D * 4 + 8)), 0x00020000);
  const uint32_t ml_at = (uint32_t)a.cap * (D * 4);
  // A part's sums are kept for a chunk and written by stores that every chunk makes, to places past the scratch's end (where
  // the hardware drops them) when there is nothing to write.  Memory operations are waited for in order, and by counts that
  // hold on every path: after a store under a condition the next wait for values would be one for the store to reach memory
  // too, several microseconds.
  Sums held[NT * G::kPasses];
  int held_o[NT * G::kPasses], held_ml[NT * G::kPasses];
  auto write_held = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT * G::kPasses; ++i) {
      const f32x4 o = {held[i].o[0], held[i].o[1], held[i].o[2], held[i].o[3]};
      const f32x2 ml = {held[i].m, held[i].l};
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), scratch, held_o[i], 0, 0);
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, ml), scratch, held_ml[i], 0, 0);
      held_o[i] = held_ml[i] = kNowhere;
    }
  };
#pragma unroll
  for (int i = 0; i < NT * G::kPasses; ++i) held_o[i] = held_ml[i] = kNowhere;
  Step cur, nxt;  // the part whose chunk is in registers, and the next one
  read_step(items, 0, cur);
  if (!cur.end) return;
  read_step(items, 1, nxt);
  if (cur.part + 1 < cur.end) nxt = cur, ++nxt.part;
  Tokens<BITS, D> x;
  int ids = x.load_ids(a, cur, w, lane), next_ids = -1;  // of cur's part, and of nxt's

  // The queries of an item, as operands in LDS: [tile][step][lane] 16 bytes, kQ a thread.  They are asked for before the
  // item's first keys, and put into LDS when the item before is done.
  constexpr int kQ = (NT * G::STEPS * 64 + kThreads - 1) / kThreads;
  uint4 qs[kQ];
  auto load_queries = [&](const Step& s) __attribute__((always_inline)) {
    const int rows = s.tok * grp, row0 = s.rb * 16 * NT;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int n = (tid + i * kThreads) & (NT * G::STEPS * 64 - 1), l = n & 63, step = (n >> 6) % G::STEPS;
      const int row = min(row0 + (n >> 6) / G::STEPS * 16 + (l & 15), rows - 1), t = div_g(a, row);
      const int h = s.head * grp + row - t * grp;
      qs[i] = *reinterpret_cast<const uint4*>(a.q + (size_t)(first_token(a, s.seq) + t) * a.ldq + (size_t)h * D +
                                              G::dim0(step, l >> 4));
    }
  };
  auto put_queries = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      uint4 v = qs[i];
      if constexpr (BITS == 4)  // values i and i + 4 share a register
        v = make_uint4(halves(v.x, v.z, false), halves(v.x, v.z, true), halves(v.y, v.w, false), halves(v.y, v.w, true));
      if (tid + i * kThreads < NT * G::STEPS * 64) sq[tid + i * kThreads] = v;
    }
    block_sync();
  };
  const float zscale = a.scale * 1.44269504088896341f;
  float top[NT], total[NT], ptop[NT], unit[NT];  // of the lane's row: largest score, sum of weights; see the product below
  f32x4 o[NT][G::CH];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      top[n] = -INFINITY, total[n] = 0.0f, ptop[n] = 0.0f, unit[n] = 1.0f;
#pragma unroll
      for (int t = 0; t < G::CH; ++t) o[n][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  };
  clear();

  int chunk = 0, at = G::start(cur.part) + w * G::TPW;  // at: the wave's first token of the chunk
  x.find(a, ids, 0);
  if (nxt.end) next_ids = x.load_ids(a, nxt, w, lane);
  load_queries(cur);
  x.load_keys(a, cur.head, at, lane, ~0u);
  x.load_values(a, cur.head, at, lane, ~0u);
  put_queries();

  for (;;) {
    const int len = cur.len, tok = cur.tok, rows = tok * grp, row0 = cur.rb * 16 * NT;
    const uint32_t dead = x.dead;
    const bool masked = dead || at + G::TPW > len - tok + 1;  // slots without a token, or that some row does not see
    const bool same = chunk + 1 < G::chunks(cur.part) && at - w * G::TPW + G::CHUNK < len;  // the part goes on
    const bool more = same || nxt.end;
    const uint32_t live = more ? ~0u : 0u;
    const int nhead = same ? cur.head : more ? nxt.head : 0;
    const int nat = same ? at + G::CHUNK : more ? G::start(nxt.part) + w * G::TPW : 0;

    // ---- scores: z[n][i][e] of token at + 16 i + 4 g4 + e, row r16 of tile n
    float z[NT][G::NS][4];
    {
      f32x4 c[NT][G::NS];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        f32x4 init = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (BITS < 16) {  // the codes' offset is taken off first: its product with the queries
          const uint32_t off = 0x00010001u * (BITS == 8 ? 0xC300u : 0xC1C0u);  // -128, -24
          static_assert(G::kOff == (BITS == 8 ? 128 : 24), "");
#pragma unroll
          for (int s = 0; s < G::STEPS; ++s)
            init = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                frag(off, off, off, off), __builtin_bit_cast(bf16x8, sq[(n * G::STEPS + s) * 64 + lane]), init, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < G::NS; ++i) c[n][i] = init;
      }
#pragma unroll
      for (int s = 0; s < G::STEPS; ++s) {
        bf16x8 q[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) q[n] = __builtin_bit_cast(bf16x8, sq[(n * G::STEPS + s) * 64 + lane]);
#pragma unroll
        for (int i = 0; i < G::NS; ++i) {
          const bf16x8 k = key_frag<BITS, D>(x.k[i], s);
#pragma unroll
          for (int n = 0; n < NT; ++n) c[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[n], c[n][i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < G::NS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) z[n][i][e] = c[n][i][e];
    }
    if (!same) {
      ids = next_ids;  // (-1 where there is no next part)
      next_ids = -1;
      if (more) {
        Step then = nxt;
        if (nxt.part + 1 < nxt.end)
          ++then.part;
        else
          read_step(items, nxt.k + 1, then);
        if (then.end) next_ids = x.load_ids(a, then, w, lane);
        load_queries(nxt);
      }
    }
    x.find(a, ids, same ? chunk + 1 : 0);
    x.load_keys(a, nhead, nat, lane, live);
    write_held();
    // ---- softmax of the running maximum
    u32x4 pk[NT][G::NG] = {};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n && row0 + n * 16 >= rows) continue;  // (the tile's sums go nowhere)
      const int limit = len - tok + 1 + div_g(a, row0 + n * 16 + r16);
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        const uint32_t sc[4] = {x.sc[i].x, x.sc[i].y, x.sc[i].z, x.sc[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[n][i][e] *= BITS == 16 ? zscale : zscale * __uint_as_float(sc[e] << 16);
          if (masked) {
            const int j = at + 16 * i + 4 * g4 + e;
            if (j >= limit || j >= len || (dead >> i & 1)) z[n][i][e] = -INFINITY;
          }
          most = fmaxf(most, z[n][i][e]);
        }
      }
      most = fmaxf(top[n], max4(most));
      float f = most == top[n] ? 1.0f : __builtin_amdgcn_exp2f(top[n] - most);  // what the sums so far are worth
      top[n] = most;
      const float base = most == -INFINITY ? 0.0f : most;
      float sum = 0.0f, pmost = 0.0f;
#pragma unroll
      for (int i = 0; i < G::NS; ++i) {
        const uint32_t sc[4] = {x.sc[i].x, x.sc[i].y, x.sc[i].z, x.sc[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(z[n][i][e] - base);
          sum += p;
          if constexpr (BITS == 16) {
            z[n][i][e] = p;
          } else {  // the codes' weight; where a token is not seen its scale may be anything
            z[n][i][e] = masked && z[n][i][e] == -INFINITY ? 0.0f : p * __uint_as_float(sc[e] & 0xFFFF0000u);
            pmost = fmaxf(pmost, z[n][i][e]);
          }
        }
      }
      total[n] = fmaf(total[n], f, sum4(sum));
      // The weights are rounded for the product: to bf16 beside bf16 values (the range of the values needs it), to f16,
      // 8 times as fine, beside codes -- in units of a power of two such that the row's largest so far is in [1, 2), so
      // what f16 cannot hold is less than 2^-25 of it.  The sums are in these units.
      if constexpr (BITS < 16) {
        ptop[n] = fmaxf(ptop[n] * f, max4(pmost));
        const uint32_t ex = min(max(__float_as_uint(ptop[n]) >> 23, 2u), 252u);
        const float inv = __uint_as_float((254u - ex) << 23);
        f *= unit[n] * inv;
        unit[n] = __uint_as_float(ex << 23);
#pragma unroll
        for (int i = 0; i < G::NS; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            pk[n][i / 2][2 * (i & 1) + e] = pack_f16(z[n][i][2 * e] * inv, z[n][i][2 * e + 1] * inv);
      } else {
#pragma unroll
        for (int i = 0; i < G::NS; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) pk[n][i / 2][2 * (i & 1) + e] = pack_bf16(z[n][i][2 * e], z[n][i][2 * e + 1]);
      }
      if (__ballot(f != 1.0f)) {
#pragma unroll
        for (int t = 0; t < G::CH; ++t) o[n][t] *= f;
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
      for (int t = 0; t < G::CH; ++t) {
        const u32x4 v = value_frag<BITS, D>(x.v[i], t);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][t] = weigh<BITS>(v, pk[n][i], o[n][t]);
      }
      if constexpr (BITS == 16) {
        if (odd >> i & 1)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            add_non_finite<D>(a, cur, at + 32 * i, pk[n][i], len - tok + 1 + div_g(a, row0 + n * 16 + r16), lane, o[n]);
      }
    }
    x.load_values(a, nhead, nat, lane, live);
    at = nat;
    if (same) {
      ++chunk;
      continue;
    }

    // ---- the end of a part: the waves' sums, in wave order
    const Seq shape = seq_shape<G, NT>(a, len, tok);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int tile0 = row0 + n * 16;
      if (tile0 >= rows) continue;
#pragma unroll
      for (int u = 0; u < G::kPasses; ++u) {
        constexpr int RUN = 4 / G::kPasses;  // of the lane's four runs of CH sums
        constexpr int C4 = D / G::kPasses / 4;
        block_sync();  // the rows in LDS are free
        if (tile0 + r16 < rows) {
          if (g4 == 0) sm[r16 * kWaves + w] = top[n], sl[r16 * kWaves + w] = total[n];
          float* const dst = so + (w * 16 + r16) * G::LD + g4 * RUN * G::CH;
#pragma unroll
          for (int i = 0; i < RUN; ++i)
#pragma unroll
            for (int t = 0; t < G::CH; t += 4) {
              const int k = u * RUN + i;
              float4 v;
              v.x = o[n][t][k] * unit[n], v.y = o[n][t + 1][k] * unit[n];
              v.z = o[n][t + 2][k] * unit[n], v.w = o[n][t + 3][k] * unit[n];
              *reinterpret_cast<float4*>(dst + i * G::CH + t) = v;
            }
        }
        block_sync();
        const int rr = tid / C4, c = tid % C4, grow = tile0 + rr;
        if (rr >= 16 || grow >= rows) continue;
        const int c4 = c / (RUN * G::CH / 4) * G::CH + u * (RUN * G::CH / 4) + c % (RUN * G::CH / 4);  // of the row
        Sums s;
        float f[kWaves], fl[kWaves];
#pragma unroll
        for (int j = 0; j < kWaves; j += 4) {
          const float4 x4 = *reinterpret_cast<const float4*>(sm + rr * kWaves + j);
          const float4 l4 = *reinterpret_cast<const float4*>(sl + rr * kWaves + j);
          f[j] = x4.x, f[j + 1] = x4.y, f[j + 2] = x4.z, f[j + 3] = x4.w;
          fl[j] = l4.x, fl[j + 1] = l4.y, fl[j + 2] = l4.z, fl[j + 3] = l4.w;
        }
#pragma unroll
        for (int j = 0; j < kWaves; ++j) s.m = fmaxf(s.m, f[j]);
        const float mx = s.m == -INFINITY ? 0.0f : s.m;
#pragma unroll
        for (int j = 0; j < kWaves; ++j) {
          f[j] = __builtin_amdgcn_exp2f(f[j] - mx);
          const float4 v = *reinterpret_cast<const float4*>(so + (j * 16 + rr) * G::LD + 4 * c);
          s.l = fmaf(fl[j], f[j], s.l);
          s.o[0] = fmaf(v.x, f[j], s.o[0]), s.o[1] = fmaf(v.y, f[j], s.o[1]);
          s.o[2] = fmaf(v.z, f[j], s.o[2]), s.o[3] = fmaf(v.w, f[j], s.o[3]);
        }
        bool done = shape.parts == 1;
        int to = -1;  // where a partial sum goes
        if (!split) {
          if (!done) to = unit_row(cur.seq, cur.head, shape) + cur.part * rows + grow;
        } else {
          Sums* const block = state + (n * G::kPasses + u) * 16 * C4 + tid;  // running sums: of the block's parts, of the blocks
          Sums* const whole = block + NT * 16 * D / 4;
          Sums b = cur.part % G::BLOCK == 0 ? Sums() : *block;
          b.add(s);
          done = cur.part + 1 == cur.end;
          if (!done && (cur.part + 1) % G::BLOCK) {
            *block = b;
            continue;
          }
          s = cur.part < G::BLOCK ? Sums() : *whole;
          s.add(b);
          if (!done) *whole = s;
        }
        if (to >= 0) {
          held[n * G::kPasses + u] = s;
          held_o[n * G::kPasses + u] = to * (D * 4) + 16 * c4;
          held_ml[n * G::kPasses + u] = c4 ? kNowhere : (int)ml_at + to * 8;
        } else if (done)
          finish_row<D>(a, s, first_token(a, cur.seq), cur.head, grow, c4);
      }
    }
    if (!more) break;
    const bool fresh = nxt.k != cur.k;
    cur = nxt;
    if (cur.part + 1 < cur.end) {
      ++nxt.part;
    } else {
      // (items up to cur.k + 2 are read before the next part ends)
      if (fresh && ((cur.k + 2) & (kTable / 2 - 1)) == 0 && cur.k + 2 >= kTable) {
        fill_table<G, NT>(a, plan, items, cur.k + 2, kTable / 2);
        block_sync();
      }
      read_step(items, cur.k + 1, nxt);
    }
    chunk = 0;
    clear();
    if (fresh) put_queries();
  }
  write_held();
}

// The rows whose parts went to scratch: blocks of parts side by side, then left to right.  A workgroup takes rows of one
// (sequence, head).
template <class G, int D>
__global__ void __launch_bounds__(kThreads) join_kernel(const AttnArgs a) {
  constexpr int C4 = D / 4, SIDE = kThreads / C4;
  __shared__ __align__(16) uint8_t lds[SIDE * C4 * sizeof(Sums)];
  Sums* const side = reinterpret_cast<Sums*>(lds);  // [SIDE][C4]
  const int* const plan = reinterpret_cast<const int*>(a.part + (size_t)a.cap * (D + 2));
  if (plan[0]) return;  // nothing was split
  const int seq = blockIdx.x / a.s.heads, head = blockIdx.x - seq * a.s.heads;
  const int first = plan[1 + seq], len = plan[1 + a.b + seq], tok = plan[1 + 2 * a.b + seq];
  const int parts = G::parts(len), rows = tok * a.g;
  if (parts == 1) return;
  const int c4 = threadIdx.x % C4, s = threadIdx.x / C4, q0 = first_token(a, seq);
  const float4* const o = reinterpret_cast<const float4*>(a.part) + (size_t)(first + head * rows * parts) * C4 + c4;
  const float2* const ml = reinterpret_cast<const float2*>(a.part + (size_t)a.cap * D) + first + head * rows * parts;
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    Sums total;
    for (int from = 0; from < parts; from += SIDE * G::BLOCK) {
      const int p0 = from + s * G::BLOCK;
      if (p0 < parts) {
        const int n = min(G::BLOCK, parts - p0);
        float4 v[G::BLOCK];
        float2 w[G::BLOCK];
#pragma unroll
        for (int i = 0; i < G::BLOCK; ++i) {
          const size_t j = (size_t)(p0 + min(i, n - 1)) * rows + row;
          v[i] = o[j * C4], w[i] = ml[j];
        }
        Sums t;
#pragma unroll
        for (int i = 0; i < G::BLOCK; ++i)
          if (i < n) {
            Sums p;
            p.m = w[i].x, p.l = w[i].y;
            p.o[0] = v[i].x, p.o[1] = v[i].y, p.o[2] = v[i].z, p.o[3] = v[i].w;
            t.add(p);
          }
        side[threadIdx.x] = t;
      }
      __syncthreads();
      if (s == 0)
        for (int i = 0; i < SIDE && from + i * G::BLOCK < parts; ++i) total.add(side[i * C4 + c4]);
      __syncthreads();
    }
    if (s == 0) finish_row<D>(a, total, q0, head, row, c4);
  }
}

template <int BITS, int D, int NT>
int launch(AttnArgs a, hipStream_t s) {
  using G = Geo<BITS, D>;
  static_assert(G::KW * 4 * 64 == 16 * G::RB, "");
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      return 256;
    return n;
  }();
  const long max_tokens = (long)a.ldt << a.page_log2;
  const long parts = G::parts((int)(max_tokens < 0x7FFFFFFF ? max_tokens : 0x7FFFFFFF));
  const double tiles = ((double)(a.qstart ? a.m : a.tq) * a.g + 15) / 16;
  const double items = (double)a.b * a.s.heads * (double)parts * tiles;
  const int slots = cus * (simd_waves(BITS, D, NT) * 4 / kWaves);
  const unsigned grid = items < slots ? (unsigned)items : (unsigned)slots;
  std::lock_guard<std::mutex> lock(scratch_mutex(s));
  // partial rows of all sequences at their longest; fewer where that is more than kMaxPartialBytes
  const size_t row_bytes = (size_t)D * 4 + 8, plan_bytes = (size_t)(3 * a.b + 1) * 4;
  double want = parts > 1 ? (double)a.m * a.heads * (double)parts : 0.0;
  const double most = (double)(kMaxPartialBytes / row_bytes);
  if (want > most) want = most;
  a.cap = (int)want;
  if (a.cap) {
    a.part = reinterpret_cast<float*>(call_scratch(s, (size_t)a.cap * row_bytes + plan_bytes).data);
    if (!a.part) a.cap = 0;
  }
  const size_t smem = (size_t)(G::kSums + kTable * 8 + 4 * a.b) * 4 + (size_t)NT * G::STEPS * 64 * 16 +
                      sizeof(Sums) * 2 * NT * 16 * D / 4;
  hipLaunchKernelGGL((paged_attn_kernel<BITS, D, NT>), dim3(grid), dim3(kThreads), smem, s, a);
  if (const int e = (int)hipGetLastError()) return e;
  if (!a.cap) return 0;
  const double rows = (double)a.m / a.b * a.g;  // of a (sequence, head), on average
  hipLaunchKernelGGL((join_kernel<G, D>), dim3((unsigned)(a.b * a.s.heads), rows < 1 ? 1u : rows < 64 ? (unsigned)rows : 64u),
                     dim3(kThreads), 0, s, a);
  return (int)hipGetLastError();
}
template <int BITS, int D>
int launch_tiles(const AttnArgs& a, hipStream_t s) {
  const double tiles = (double)a.m / a.b * a.g / 16;  // of a sequence, on average
  if constexpr (D <= 128) {
    if (tiles > 1) return launch<BITS, D, 2>(a, s);
  }
  return launch<BITS, D, 1>(a, s);
}
template <int BITS>
int launch_dim(const AttnArgs& a, hipStream_t s) {
  return a.s.dim == 64 ? launch_tiles<BITS, 64>(a, s)
                       : a.s.dim == 128 ? launch_tiles<BITS, 128>(a, s) : launch_tiles<BITS, 256>(a, s);
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
  return bits == 16 ? agq::launch_dim<16>(a, st) : bits == 8 ? agq::launch_dim<8>(a, st) : agq::launch_dim<4>(a, st);
}
