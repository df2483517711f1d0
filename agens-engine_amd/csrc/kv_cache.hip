// Writing keys and values into the pages of the cache, and reading them back (kv_page.h has the layout).
//
// Quantisation of a row x of dim values (one token, one head, keys or values), Q = 127 (8 bits) or 7 (4 bits):
//   s = bf16(max|x| / Q), q = rint(x / s) clamped to +-Q, the value held is q * s.
// The codes are those of the rounded scale that readers multiply with, so the rounding of s costs no accuracy beyond the
// clamped end (x / s <= Q (1 + 2^-9), less than half a step).  x / s is the fp32 quotient: bf16 over bf16 is never close
// enough to a half for that rounding to move rint, so the codes are those of exact arithmetic.  A row whose s would lie
// below 2^-126 is held as zeros; one with a non-finite value gets the scale NaN and reads back as NaN.
//
// Both kernels are streams: dim / 8 lanes take the keys and the values of one (token, head), 16 bytes of bf16 a lane each;
// the largest magnitude is found by lane exchanges.  Consecutive groups take consecutive tokens of one head, whose
// slots are usually consecutive, so that a wave writes whole lines of the page.
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
  int m;
};

struct KvPlace {
  uint8_t *krow, *vrow;
  uint32_t* pair;  // the scales
};
__device__ __forceinline__ KvPlace place(const KvArgs& a, int slot, int head) {
  const KvShape& s = a.s;
  uint8_t* const pg = a.pool + s.bytes() * (size_t)(slot / s.page);
  const size_t off = slot % s.page;
  KvPlace p;
  p.krow = pg + s.plane() * (2 * (size_t)head) + off * s.row_bytes();
  p.vrow = p.krow + s.plane();
  p.pair = reinterpret_cast<uint32_t*>(pg + s.scale_off()) + (size_t)head * s.page + off;
  return p;
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
#pragma unroll
  for (int d = LANES / 2; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
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
  const float s = bf2f(sb);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint64_t out = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = bf2f((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
    float q = rintf(f / s);
    q = fminf(fmaxf(q, -Q), Q);  // (also takes NaN, of a zero or NaN scale, to a code)
    const int code = sb == 0 || sb == 0x7FC0u ? kOff : (int)q + kOff;
    out |= (uint64_t)(uint32_t)code << (BITS * i);
  }
  return out;
}

template <int BITS, int D>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(const KvArgs a, long groups) {
  constexpr int LANES = D / 8;
  const int l = threadIdx.x % LANES;
  for (long g = (long)blockIdx.x * (kKvThreads / LANES) + threadIdx.x / LANES; g < groups;
       g += (long)gridDim.x * (kKvThreads / LANES)) {
    const int t = (int)(g % a.m), head = (int)(g / a.m);
    const int slot = a.slots[t];
    if (slot < 0 || slot / a.s.page >= a.s.npages) continue;  // (whole groups of lanes)
    const uint4 k = *reinterpret_cast<const uint4*>(a.k + (size_t)t * a.ldk + head * D + l * 8);
    const uint4 v = *reinterpret_cast<const uint4*>(a.v + (size_t)t * a.ldv + head * D + l * 8);
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
}

// codes -> 8 packed bf16 values q * s, rounded once
template <int BITS>
__device__ __forceinline__ uint4 dequantise8(uint64_t c, float s) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t r = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int code = (int)((c >> (BITS * (2 * i + e))) & ((1u << BITS) - 1)) - (1 << (BITS - 1));
      r |= (uint32_t)f2bf((float)code * s) << (16 * e);
    }
    w[i] = r;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int BITS, int D>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const KvArgs a, long groups) {
  constexpr int LANES = D / 8;
  const int l = threadIdx.x % LANES;
  for (long g = (long)blockIdx.x * (kKvThreads / LANES) + threadIdx.x / LANES; g < groups;
       g += (long)gridDim.x * (kKvThreads / LANES)) {
    const int t = (int)(g % a.m), head = (int)(g / a.m);
    const int slot = a.slots[t];
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (slot >= 0 && slot / a.s.page < a.s.npages) {
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
}

template <bool WRITE, int BITS, int D>
int launch(const KvArgs& a, hipStream_t s) {
  constexpr int per = kKvThreads / (D / 8);
  const long groups = (long)a.m * a.s.heads;
  long grid = (groups + per - 1) / per;
  if (grid > 65536) grid = 65536;
  if constexpr (WRITE)
    hipLaunchKernelGGL((kv_write_kernel<BITS, D>), dim3((unsigned)grid), dim3(kKvThreads), 0, s, a, groups);
  else
    hipLaunchKernelGGL((kv_read_kernel<BITS, D>), dim3((unsigned)grid), dim3(kKvThreads), 0, s, a, groups);
  return (int)hipGetLastError();
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
                      static_cast<uint8_t*>(pool), m};
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
                      const_cast<uint8_t*>(static_cast<const uint8_t*>(pool)), m};
  return agq::launch_bits<false>(a, static_cast<hipStream_t>(stream));
}
