// Rotary positions: queries and keys turned by their tokens' positions, alone or on the way into the cache's pages.
//
//   pair j of a head (values j and j + rot / 2, or 2j and 2j + 1) turns by pos * freqs[j]:
//   x' = mag (x cos - y sin), y' = mag (y cos + x sin), values from `rot` on stay.
//
// Angles, their sines and cosines, and the products are 64 bits, rounded once to bf16: in 32 bits an angle of a far position
// (10^6 radians) is off by 0.03, and products off by a rounding now and then put a value on the other side of a bf16 border,
// which then moves a code in the cache.  The 64-bit vector rate of this GPU is half its 32-bit rate, and the kernels wait for
// memory.
//
// A workgroup takes a few tokens: it works out their sines and cosines once, into LDS, for all heads.  Then every group of
// dim / 8 lanes (a power of two: 80 values take 16 lanes, 10 of them at work) takes one head of one token, 16 bytes a lane; a
// lane has its pairs' other halves from the lane that loaded them (where rot is no multiple of 16, it loads them itself).  A head
// stays within one wave's instructions, so that rotating in place is safe: all of its loads come before its stores.
//
// Memory bounds long batches: 8191 tokens of 48 heads of 128, half of each, neighbours paired (201 MB) 40 us, 5.0 TB/s, as fast as a
// copy; 8192 tokens of 40 + 16 heads into pages (235 MB) 52 us, 4.5 TB/s.  One token, 2.8 us, waits for one load after another.
#include <math.h>

#include "agens_kernels.h"
#include "kv_codes.h"

namespace agq {
namespace {

constexpr int kRopeThreads = 256;

struct RopeArgs {
  const uint16_t *q, *k, *v;
  uint16_t* y;
  long ldq, ldk, ldv, ldy;
  const int *pos, *slots;
  const double* freqs;
  double mag;
  uint8_t* pool;
  KvShape s;
  int page_log2, m, heads, dim, rot, tokens;  // tokens: of a workgroup
};

// cos and sin of a = pos * f.  a = n pi / 2 + r: the product's rounding and pi's bits past 53 go into r; then Taylor's series
// for |r| <= pi / 4 up to r^16 (the next terms are below 2^-53 of the value).
__device__ __forceinline__ double2 turn(int pos, double f) {
  const double p = (double)pos, a = p * f, lost = __builtin_fma(p, f, -a);
  const double n = __builtin_rint(a * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489655800, a);
  r = __builtin_fma(-n, 6.12323399573676603587e-17, r) + lost;
  const double z = r * r;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = __builtin_fma(s, z, 1.0 / 6227020800.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(s * z, r, r);
  c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  c = __builtin_fma(c, z, 1.0 / 479001600.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int quarter = (int)(n - 4.0 * __builtin_floor(n * 0.25));
  const double u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
  return make_double2(quarter == 1 || quarter == 2 ? -u : u, quarter & 2 ? -v : v);
}

// 64 bits -> 32 on the way to bf16: the last of 15 bits kept says whether anything was cut off, so the rounding that follows sees
// the side of a border that the value is on.  (15 and not 23: of a value between 2^-134, half of bf16's least, and 2^-126 fp32
// still holds as many.  The low word may stay: five zeros are between it and that bit.)
__device__ __forceinline__ float narrow(double d) {
  const uint64_t u = (uint64_t)__double_as_longlong(d);
  const uint32_t lo = (uint32_t)u;
  uint32_t hi = (uint32_t)(u >> 32);
  hi = (hi & ~0x1Fu) | (((hi & 0x1Fu) | lo) ? 0x20u : 0u);
  return (float)__longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ uint32_t two_bf16(double x, double y) { return f2bf2(narrow(x), narrow(y)); }

__device__ __forceinline__ uint32_t value(const uint4& x, int i) {
  const uint32_t w = i < 2 ? x.x : i < 4 ? x.y : i < 6 ? x.z : x.w;
  return i & 1 ? w >> 16 : w & 0xFFFFu;
}

// Where pair j of a token lies among its sines and cosines: lanes whose pairs begin EACH apart read side by side.
template <int EACH>
__device__ __forceinline__ int spot(int j, int pairs) {
  return (j % EACH) * ((pairs + EACH - 1) / EACH) + j / EACH;
}
__host__ __device__ inline int spots(int pairs) { return (pairs + 7) / 8 * 8; }

// The lane's 8 values of a row, and those that they are paired with.  LAYOUT: 0 halves with rot % 16 == 0, 1 halves, 2
// neighbours.
struct Piece {
  uint4 x, other;
};
template <int LAYOUT>
__device__ __forceinline__ Piece load_piece(const RopeArgs& a, const uint16_t* row, int lane) {
  Piece p;
  p.x = *reinterpret_cast<const uint4*>(row + 8 * lane);
  p.other = p.x;
  const int at = 8 * lane, half = a.rot / 2;
  if (LAYOUT != 1 || at >= a.rot) return p;
  {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = min(at + i, a.rot - 1);
      o[i] = row[e < half ? e + half : e - half];
    }
    p.other = make_uint4(o[0] | o[1] << 16, o[2] | o[3] << 16, o[4] | o[5] << 16, o[6] | o[7] << 16);
  }
  return p;
}
template <int LAYOUT>
__device__ __forceinline__ uint4 rotated(const RopeArgs& a, const Piece& p, int lane, const double2* cs) {
  const int at = 8 * lane, half = a.rot / 2;
  if (at >= a.rot) return p.x;
  uint32_t out[4];
  if constexpr (LAYOUT == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double u = bf2f(value(p.x, 2 * i)), v = bf2f(value(p.x, 2 * i + 1));
      const double2 t = cs[spot<4>(min(at / 2 + i, half - 1), half)];
      out[i] = two_bf16(__builtin_fma(u, t.x, -(v * t.y)), __builtin_fma(v, t.x, u * t.y));
    }
  } else {
    uint4 other = p.other;
    if constexpr (LAYOUT == 0) {  // from the lane that has it: loaded, it would come from L2 a second time
      const int from = (int)(threadIdx.x & 63) + (at < half ? half / 8 : -half / 8);
      other = make_uint4(__shfl(p.x.x, from), __shfl(p.x.y, from), __shfl(p.x.z, from), __shfl(p.x.w, from));
    }
    double r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = LAYOUT == 0 ? at + i : min(at + i, a.rot - 1);
      const bool low = LAYOUT == 0 ? at < half : e < half;
      const double u = bf2f(value(p.x, i)), v = bf2f(value(other, i));
      const double2 t = cs[LAYOUT == 0 ? i * (half / 8) + (low ? at : at - half) / 8 : spot<8>(low ? e : e - half, half)];
      r[i] = __builtin_fma(u, t.x, low ? -(v * t.y) : v * t.y);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = two_bf16(r[2 * i], r[2 * i + 1]);
  }
  if constexpr (LAYOUT != 0) {  // a lane across rot's end
    const uint32_t x[4] = {p.x.x, p.x.y, p.x.z, p.x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + 2 * i >= a.rot) out[i] = x[i];  // (rot is even)
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// One row of keys or values (part 0 or 1) into its slot.
template <int BITS, int D>
__device__ __forceinline__ void store_row(const RopeArgs& a, const uint4 x, int slot, int head, int part, int lane) {
  const KvPlace p = kv_place(a.s, a.pool, a.page_log2, slot, head);
  uint8_t* const row = part ? p.vrow : p.krow;
  if constexpr (BITS == 16) {
    reinterpret_cast<uint4*>(row)[lane] = x;
  } else {
    uint32_t s;
    const uint64_t c = quantise8<BITS>(x, row_amax<D / 8>(x), &s);
    if constexpr (BITS == 8)
      reinterpret_cast<uint64_t*>(row)[lane] = c;
    else
      reinterpret_cast<uint32_t*>(row)[lane] = (uint32_t)c;
    if (lane == 0) reinterpret_cast<uint16_t*>(p.pair)[part] = (uint16_t)s;
  }
}

// BITS 0: heads of q alone.  Otherwise heads of q, then keys, then values of every token; grid y: `each` of these rows.
template <int BITS, int D, int LAYOUT>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a, int lanes_log2, int each) {
  extern __shared__ double2 cs[];  // [tokens][spots(rot / 2)]
  const int first = blockIdx.x * a.tokens, n = min(a.tokens, a.m - first), half = a.rot / 2, per = spots(half);
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), groups = kRopeThreads >> lanes_log2;
  const int row0 = blockIdx.y * each, rows = min(each, (BITS ? a.heads + 2 * a.s.heads : a.heads) - row0);
  struct Item {
    int t, h, pos, slot;
    Piece p;
  };
  // the e-th of the workgroup's rows: of q where h < a.heads, then keys, values.  Nothing to do: pos < 0.
  auto load = [&](int e) {
    Item x;
    const int lt = e / rows;
    x.t = first + min(lt, n - 1), x.h = row0 + e - lt * rows, x.slot = 0;
    x.pos = lt < n && 8 * lane < a.dim ? a.pos[x.t] : -1;
    if (x.pos < 0) return x;
    const size_t off = (size_t)x.h * a.dim;
    if (BITS == 0 || x.h < a.heads) {
      x.p = load_piece<LAYOUT>(a, a.q + x.t * a.ldq + off, lane);
    } else {
      const int kh = x.h - a.heads;
      x.slot = a.slots[x.t];
      if (kh < a.s.heads)
        x.p = load_piece<LAYOUT>(a, a.k + x.t * a.ldk + (size_t)kh * D, lane);
      else
        x.p.x = *reinterpret_cast<const uint4*>(a.v + x.t * a.ldv + (size_t)(kh - a.s.heads) * D + 8 * lane);
    }
    return x;
  };
  int e = threadIdx.x >> lanes_log2;
  Item x = load(e);  // (on its way while the sines and cosines are worked out)
  for (int i = threadIdx.x; i < n * half; i += kRopeThreads) {
    const int t = i / half, j = i - t * half;
    const double2 v = turn(max(a.pos[first + t], 0), a.freqs[j]);
    cs[t * per + (LAYOUT == 2 ? spot<4>(j, half) : spot<8>(j, half))] = make_double2(v.x * a.mag, v.y * a.mag);
  }
  __syncthreads();
  for (; e < n * rows; e += groups) {
    const Item now = x;
    if (e + groups < n * rows) x = load(e + groups);
    if (now.pos < 0) continue;
    const double2* const c = cs + (now.t - first) * per;
    if (BITS == 0 || now.h < a.heads) {
      *reinterpret_cast<uint4*>(a.y + now.t * a.ldy + (size_t)now.h * a.dim + 8 * lane) = rotated<LAYOUT>(a, now.p, lane, c);
    } else if constexpr (BITS != 0) {
      const int kh = now.h - a.heads, part = kh >= a.s.heads;
      if (now.slot < 0 || now.slot >> a.page_log2 >= a.s.npages) continue;  // (whole groups of lanes)
      store_row<BITS, D>(a, part ? now.p.x : rotated<LAYOUT>(a, now.p, lane, c), now.slot, part ? kh - a.s.heads : kh, part, lane);
    }
  }
}

template <int BITS, int D, int LAYOUT>
int launch(RopeArgs a, hipStream_t s) {
  int lanes_log2 = 0;
  while ((8 << lanes_log2) < a.dim) ++lanes_log2;
  const int rows = BITS ? a.heads + 2 * a.s.heads : a.heads;
  // tokens of a workgroup: three rounds of its lanes, while their sines and cosines fit 16 KB
  const int per = spots(a.rot / 2) * 16, groups = kRopeThreads >> lanes_log2;
  int tokens = 3 * groups / rows;
  tokens = tokens < 1 ? 1 : tokens;
  while (tokens > 1 && tokens * per > 16384) --tokens;
  // few tokens: one round, their sines and cosines worked out by several workgroups (one token of 48 heads 4.6 -> 3.4 us, 48 of
  // 56 6.7 -> 4.5)
  int each = rows;
  if ((long)(a.m - 1) / tokens + 1 < 512) {
    tokens = groups / rows < 1 ? 1 : groups / rows;
    while (tokens > 1 && tokens * per > 16384) --tokens;
    if (rows > groups) each = groups;
  }
  a.tokens = tokens;
  const int m = a.m, most = (1 << 23) * (tokens < 64 ? tokens : 64);  // of a launch: its lanes are counted in 32 bits
  for (int t = 0; t < m; t += a.m) {
    a.m = m - t < most ? m - t : most;
    hipLaunchKernelGGL((rope_kernel<BITS, D, LAYOUT>),
                       dim3((unsigned)((a.m - 1) / tokens + 1), (unsigned)((rows - 1) / each + 1)), dim3(kRopeThreads),
                       (size_t)tokens * per, s, a, lanes_log2, each);
    if (const int e = (int)hipGetLastError()) return e;
    a.q += a.m * a.ldq, a.k += a.m * a.ldk, a.v += a.m * a.ldv, a.y += a.m * a.ldy, a.pos += a.m;
    if (BITS) a.slots += a.m;
  }
  return 0;
}
template <int BITS, int D>
int launch_layout(const RopeArgs& a, int interleaved, hipStream_t s) {
  return interleaved ? launch<BITS, D, 2>(a, s) : a.rot % 16 ? launch<BITS, D, 1>(a, s) : launch<BITS, D, 0>(a, s);
}
template <int BITS>
int launch_dim(const RopeArgs& a, int interleaved, hipStream_t s) {
  return a.dim == 64 ? launch_layout<BITS, 64>(a, interleaved, s)
                     : a.dim == 128 ? launch_layout<BITS, 128>(a, interleaved, s) : launch_layout<BITS, 256>(a, interleaved, s);
}

bool rows_ok(const void* p, long ld, int m, long width, bool written) {
  return p && aligned16(p) && ld >= 0 && ld % 8 == 0 && (!written || m <= 1 || ld >= width);
}
bool turn_ok(const int* pos, const double* freqs, int rot, int dim, int interleaved, float mag) {
  return pos && freqs && rot >= 2 && rot <= dim && rot % 2 == 0 && (interleaved == 0 || interleaved == 1) && isfinite(mag);
}

}  // namespace
}  // namespace agq

extern "C" int ak_rope(const void* x, long ldx, void* y, long ldy, int m, int heads, int dim, const int* pos,
                       const double* freqs, int rot, int interleaved, float mag, void* stream) {
  if (m < 0 || heads < 1 || heads > 4096 || dim < 8 || dim > 512 || dim % 8) return AK_INVALID;
  if (!m) return 0;
  const long width = (long)heads * dim;
  if (!agq::rows_ok(x, ldx, m, width, false) || !agq::rows_ok(y, ldy, m, width, true) ||
      !agq::turn_ok(pos, freqs, rot, dim, interleaved, mag) || (x == y && m > 1 && ldx != ldy))
    return AK_INVALID;
  agq::RopeArgs a{};
  a.q = static_cast<const uint16_t*>(x), a.y = static_cast<uint16_t*>(y), a.ldq = ldx, a.ldy = ldy;
  a.pos = pos, a.freqs = freqs, a.mag = (double)mag, a.m = m, a.heads = heads, a.dim = dim, a.rot = rot;
  return agq::launch_layout<0, 0>(a, interleaved, static_cast<hipStream_t>(stream));
}

extern "C" int ak_rope_kv_write(int bits, const void* q, long ldq, const void* k, long ldk, const void* v, long ldv, void* y,
                                long ldy, int m, int heads, const int* pos, const double* freqs, int rot, int interleaved,
                                float mag, const int* slots, void* pool, int npages, int page, int kv_heads, int dim,
                                void* stream) {
  const agq::KvShape s{bits, page, kv_heads, dim, npages};
  if (!s.valid() || m < 0 || npages < 1 || heads < 1 || heads > 4096) return AK_INVALID;
  if (!m) return 0;
  const long width = (long)heads * dim, kv = (long)kv_heads * dim;
  if (!agq::rows_ok(q, ldq, m, width, false) || !agq::rows_ok(y, ldy, m, width, true) ||
      !agq::rows_ok(k, ldk, m, kv, false) || !agq::rows_ok(v, ldv, m, kv, false) ||
      !agq::turn_ok(pos, freqs, rot, dim, interleaved, mag) || (q == y && m > 1 && ldq != ldy) || !slots || !pool ||
      !agq::aligned16(pool))
    return AK_INVALID;
  agq::RopeArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.y = static_cast<uint16_t*>(y), a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldy = ldy;
  a.pos = pos, a.slots = slots, a.freqs = freqs, a.mag = (double)mag, a.pool = static_cast<uint8_t*>(pool), a.s = s;
  a.page_log2 = __builtin_ctz((unsigned)page), a.m = m, a.heads = heads, a.dim = dim, a.rot = rot;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return bits == 16 ? agq::launch_dim<16>(a, interleaved, st)
                    : bits == 8 ? agq::launch_dim<8>(a, interleaved, st) : agq::launch_dim<4>(a, interleaved, st);
}

// Host only.  Bands: pair j makes trained * f / 2 pi turns over the trained context; pairs of more than `fast` keep their
// frequency, pairs of fewer than `slow` have it divided, and those between are mixed in proportion.
extern "C" int ak_rope_freqs(double theta, int rot, int scaling, double factor, long trained, double slow, double fast,
                             double* freqs, float* mag) {
  if (!(theta > 0) || !isfinite(theta) || rot < 2 || rot % 2 || !freqs || !mag || scaling < AK_ROPE_PLAIN ||
      scaling > AK_ROPE_BANDS)
    return AK_INVALID;
  if (scaling != AK_ROPE_PLAIN && (!(factor >= 1) || !isfinite(factor))) return AK_INVALID;
  if (scaling == AK_ROPE_BASE && rot < 4) return AK_INVALID;
  if (scaling == AK_ROPE_BANDS && (trained < 1 || !(slow >= 0) || !(fast > slow) || !isfinite(fast))) return AK_INVALID;
  if (scaling == AK_ROPE_BASE) theta *= pow(factor, (double)rot / (rot - 2));
  for (int j = 0; j < rot / 2; ++j) {
    double f = pow(theta, -2.0 * j / rot);
    if (scaling == AK_ROPE_LINEAR) f /= factor;
    if (scaling == AK_ROPE_BANDS) {
      const double turns = (double)trained * f / 6.28318530717958647692;
      const double keep = fmin(fmax((turns - slow) / (fast - slow), 0.0), 1.0);
      f *= keep + (1.0 - keep) / factor;
    }
    freqs[j] = f;
  }
  *mag = scaling == AK_ROPE_BANDS ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
  return 0;
}
