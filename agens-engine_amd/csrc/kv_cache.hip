// Writing keys and values into the pages of the cache, and reading them back (kv_page.h has the layout).
//
// Quantisation of a row x of dim values (one token, one head, keys or values), Q = 127 (8 bits) or 7 (4 bits):
//   s = bf16(max|x| / Q), q = rint(x / s) clamped to +-Q, the value held is q * s.
// The codes are those of the rounded scale that readers multiply with, so the rounding of s costs no accuracy beyond the
// clamped end (x / s <= Q (1 + 2^-9), less than half a step).  The codes are those of exact arithmetic: two bf16's quotient is
// a half or at least 2^-11 from one, and q0 = x * (1 / s), q0 + (x - q0 s) / s is right to the last bit where it is a half.
// (Without a division: 16384 tokens of 8 heads 34 -> 24 us.)  A row whose s would lie below 2^-126 is held as zeros; one
// with a non-finite value gets the scale NaN and reads back as NaN.
//
// Both kernels are streams: dim / 8 lanes take the keys and the values of one (token, head), 16 bytes of bf16 a lane each;
// the largest magnitude is found by lane exchanges.  Consecutive groups of a workgroup take consecutive tokens of one head,
// whose slots are usually consecutive, so that a wave writes whole lines of the page.  Measured with 16384 tokens of 8 heads
// of 128, six such in turn: written in 27, 22 and 20 us in 16, 8 and 4 bits (134, 101 and 84 MB: 4.9, 4.6 and 4.2 TB/s), read in
// 27, 24 and 24 (4.9, 4.2 and 3.5); one token 3 us, a launch.
#include "agens_kernels.h"
#include "kv_page.h"

namespace agq {
namespace {

constexpr int kKvThreads = 256;

struct KvArgs {
  KvShape s;
  uint16_t *k, *v;
  long ldk, ldv;
  const int* slots;
  uint8_t* pool;
  int m, page_log2;
};

struct KvPlace {
  uint8_t *krow, *vrow;
  uint32_t* pair;  // the scales
};
__device__ __forceinline__ KvPlace place(const KvArgs& a, int slot, int head) {
  const KvShape& s = a.s;
  uint8_t* const pg = a.pool + s.bytes() * (size_t)(slot >> a.page_log2);
  const size_t off = slot & (s.page - 1);
  KvPlace p;
  p.krow = pg + s.plane() * (2 * (size_t)head) + off * s.row_bytes();
  p.vrow = p.krow + s.plane();
  p.pair = reinterpret_cast<uint32_t*>(pg + s.scale_off()) + (size_t)head * s.page + off;
  return p;
}

// The token and head of the thread's group of lanes: consecutive workgroups take the heads of the same tokens, whose rows
// are neighbours in k and v (all tokens of a head first: 16384 tokens 46 us instead of 43).
template <int LANES>
__device__ __forceinline__ void group_of(const KvArgs& a, int* t, int* head) {
  const unsigned at = blockIdx.x / (unsigned)a.s.heads;
  *head = (int)(blockIdx.x - at * (unsigned)a.s.heads);
  *t = (int)at * (kKvThreads / LANES) + (int)threadIdx.x / LANES;
}

// largest magnitude (as the bits of |bf16|: ordered as integers, NaN above Inf above all) over the lanes of one row
template <int LANES>
__device__ __forceinline__ uint32_t row_amax(const uint4 x) {
  uint32_t m = 0;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = w[i] & 0x7FFFu, hi = (w[i] >> 16) & 0x7FFFu;
    m = max(m, max(lo, hi));
  }
  auto with = [&](int other) { m = max(m, (uint32_t)other); };
  with(__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));   // quad_perm [1, 0, 3, 2]
  with(__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));   // quad_perm [2, 3, 0, 1]
  with(__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, true));  // row_half_mirror
  if constexpr (LANES >= 16) with(__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xF, 0xF, true));  // row_mirror
  if constexpr (LANES >= 32) with(__shfl_xor((int)m, 16));
  return m;
}

// 8 values -> 8 codes (64 bits of bytes, or 32 of nibbles), and the scale's bf16 bits
template <int BITS>
__device__ __forceinline__ uint64_t quantise8(const uint4 x, uint32_t amax, uint32_t* sbits) {
  constexpr float Q = BITS == 8 ? 127.0f : 7.0f;
  constexpr int kOff = BITS == 8 ? 128 : 8;
  uint32_t sb = f2bf(bf2f(amax) / Q);
  if (sb < 0x0080u) sb = 0;             // below 2^-126
  if (amax >= 0x7F80u) sb = 0x7FC0u;    // a NaN or Inf in the row
  *sbits = sb;
  const bool held = sb != 0 && sb != 0x7FC0u;
  const float up = sb < 0x2000u ? 0x1p64f : 1.0f;  // where x - q0 s would lose bits below 2^-149
  const float s = held ? bf2f(sb) * up : 1.0f, r = __builtin_amdgcn_rcpf(s);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = bf2f((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) * up;
    float q = f * r;
    q = __builtin_fmaf(__builtin_fmaf(-q, s, f), r, q);
    q = fminf(fmaxf(q, -Q), Q);
    c[i] = __float_as_uint(q + (0x1.8p23f + (float)kOff));  // rounds to the even of two; the integer is in the low bits
  }
  uint64_t out = 0;
  if constexpr (BITS == 8) {
    uint32_t h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      h[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x0C0C0400u),
                                   __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0C0C0400u), 0x05040100u);
    out = held ? (uint64_t)h[1] << 32 | h[0] : 0x8080808080808080ull;
  } else {
    uint32_t h = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) h |= (c[i] & 15u) << (4 * i);
    out = held ? h : 0x88888888u;
  }
  return out;
}

template <int BITS, int D>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(const KvArgs a) {
  constexpr int LANES = D / 8;
  const int l = threadIdx.x % LANES;
  int t, head;
  group_of<LANES>(a, &t, &head);
  if (t >= a.m) return;
  const uint4 k = *reinterpret_cast<const uint4*>(a.k + (size_t)t * a.ldk + head * D + l * 8);
  const uint4 v = *reinterpret_cast<const uint4*>(a.v + (size_t)t * a.ldv + head * D + l * 8);
  const int slot = a.slots[t];
  if (slot < 0 || slot >> a.page_log2 >= a.s.npages) return;  // (whole groups of lanes)
  const KvPlace p = place(a, slot, head);
  if constexpr (BITS == 16) {
    reinterpret_cast<uint4*>(p.krow)[l] = k;
    reinterpret_cast<uint4*>(p.vrow)[l] = v;
  } else {
    uint32_t ks, vs;
    const uint64_t kc = quantise8<BITS>(k, row_amax<LANES>(k), &ks);
    const uint64_t vc = quantise8<BITS>(v, row_amax<LANES>(v), &vs);
    if constexpr (BITS == 8) {
      reinterpret_cast<uint64_t*>(p.krow)[l] = kc;
      reinterpret_cast<uint64_t*>(p.vrow)[l] = vc;
    } else {
      reinterpret_cast<uint32_t*>(p.krow)[l] = (uint32_t)kc;
      reinterpret_cast<uint32_t*>(p.vrow)[l] = (uint32_t)vc;
    }
    if (l == 0) *p.pair = ks | (vs << 16);
  }
}

// codes -> 8 packed bf16 values q * s, rounded once (the product is exact in fp32)
template <int BITS>
__device__ __forceinline__ uint4 dequantise8(uint64_t c, float s) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t r = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t code = (uint32_t)(c >> (BITS * (2 * i + e))) & ((1u << BITS) - 1);
      r |= (uint32_t)f2bf(((float)code - (float)(1 << (BITS - 1))) * s) << (16 * e);
    }
    w[i] = r;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int BITS, int D>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const KvArgs a) {
  constexpr int LANES = D / 8;
  const int l = threadIdx.x % LANES;
  int t, head;
  group_of<LANES>(a, &t, &head);
  if (t >= a.m) return;
  const int slot = a.slots[t];
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (slot >= 0 && slot >> a.page_log2 < a.s.npages) {
    const KvPlace p = place(a, slot, head);
    if constexpr (BITS == 16) {
      k = reinterpret_cast<const uint4*>(p.krow)[l];
      v = reinterpret_cast<const uint4*>(p.vrow)[l];
    } else {
      const uint32_t pair = *p.pair;
      uint64_t kc, vc;
      if constexpr (BITS == 8) {
        kc = reinterpret_cast<const uint64_t*>(p.krow)[l];
        vc = reinterpret_cast<const uint64_t*>(p.vrow)[l];
      } else {
        kc = reinterpret_cast<const uint32_t*>(p.krow)[l];
        vc = reinterpret_cast<const uint32_t*>(p.vrow)[l];
      }
      k = dequantise8<BITS>(kc, bf2f(pair & 0xFFFFu));
      v = dequantise8<BITS>(vc, bf2f(pair >> 16));
    }
  }
  *reinterpret_cast<uint4*>(a.k + (size_t)t * a.ldk + head * D + l * 8) = k;
  *reinterpret_cast<uint4*>(a.v + (size_t)t * a.ldv + head * D + l * 8) = v;
}

template <bool WRITE, int BITS, int D>
int launch(KvArgs a, hipStream_t s) {
  constexpr int per = kKvThreads / (D / 8);
  const int m = a.m, most = (1 << 23) / a.s.heads * per;  // tokens of a launch: its lanes are counted in 32 bits
  for (int t = 0; t < m; t += a.m) {
    a.m = m - t < most ? m - t : most;
    const dim3 grid((unsigned)((a.m - 1) / per + 1) * (unsigned)a.s.heads);
    if constexpr (WRITE)
      hipLaunchKernelGGL((kv_write_kernel<BITS, D>), grid, dim3(kKvThreads), 0, s, a);
    else
      hipLaunchKernelGGL((kv_read_kernel<BITS, D>), grid, dim3(kKvThreads), 0, s, a);
    if (const int e = (int)hipGetLastError()) return e;
    a.k += (size_t)a.m * a.ldk, a.v += (size_t)a.m * a.ldv, a.slots += a.m;
  }
  return 0;
}
template <bool WRITE, int BITS>
int launch_dim(const KvArgs& a, hipStream_t s) {
  return a.s.dim == 64 ? launch<WRITE, BITS, 64>(a, s)
                       : a.s.dim == 128 ? launch<WRITE, BITS, 128>(a, s) : launch<WRITE, BITS, 256>(a, s);
}
template <bool WRITE>
int launch_bits(const KvArgs& a, hipStream_t s) {
  return a.s.bits == 16 ? launch_dim<WRITE, 16>(a, s)
                        : a.s.bits == 8 ? launch_dim<WRITE, 8>(a, s) : launch_dim<WRITE, 4>(a, s);
}

// rows of 16-byte pieces; rows written may not overlap
bool rows_ok(const void* p, long ld, int m, long width, bool written) {
  return p && aligned16(p) && ld >= 0 && ld % 8 == 0 && (!written || m <= 1 || ld >= width);
}

}  // namespace
}  // namespace agq

extern "C" size_t ak_kv_page_bytes(int bits, int page, int heads, int dim) {
  const agq::KvShape s{bits, page, heads, dim, 1};
  return s.valid() ? s.bytes() : 0;
}

extern "C" int ak_kv_write(int bits, const void* k, const void* v, int m, long ldk, long ldv, const int* slots,
                           void* pool, int npages, int page, int heads, int dim, void* stream) {
  const agq::KvShape s{bits, page, heads, dim, npages};
  if (!s.valid() || m < 0 || npages < 1) return AK_INVALID;
  if (!m) return 0;
  const long width = (long)heads * dim;
  if (!agq::rows_ok(k, ldk, m, width, false) || !agq::rows_ok(v, ldv, m, width, false) || !slots || !pool ||
      !agq::aligned16(pool))
    return AK_INVALID;
  const agq::KvArgs a{s,     const_cast<uint16_t*>(static_cast<const uint16_t*>(k)),
                      const_cast<uint16_t*>(static_cast<const uint16_t*>(v)), ldk, ldv, slots,
                      static_cast<uint8_t*>(pool), m, __builtin_ctz((unsigned)page)};
  return agq::launch_bits<true>(a, static_cast<hipStream_t>(stream));
}

extern "C" int ak_kv_read(int bits, const void* pool, int npages, int page, int heads, int dim, const int* slots, int m,
                          void* k, void* v, long ldk, long ldv, void* stream) {
  const agq::KvShape s{bits, page, heads, dim, npages};
  if (!s.valid() || m < 0 || npages < 1) return AK_INVALID;
  if (!m) return 0;
  const long width = (long)heads * dim;
  if (!agq::rows_ok(k, ldk, m, width, true) || !agq::rows_ok(v, ldv, m, width, true) || !slots || !pool ||
      !agq::aligned16(pool))
    return AK_INVALID;
  const agq::KvArgs a{s,   static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), ldk, ldv, slots,
                      const_cast<uint8_t*>(static_cast<const uint8_t*>(pool)), m, __builtin_ctz((unsigned)page)};
  return agq::launch_bits<false>(a, static_cast<hipStream_t>(stream));
}
