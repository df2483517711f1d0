// Codes of the cache's rows (kv_cache.hip has the definition) and where they lie: shared by the kernels that write pages.
#pragma once
#include "kv_page.h"

namespace agq {

// Where a slot's rows of one head lie.
struct KvPlace {
  uint8_t *krow, *vrow;
  uint32_t* pair;  // the scales
};
__device__ __forceinline__ KvPlace kv_place(const KvShape& s, uint8_t* pool, int page_log2, int slot, int head) {
  uint8_t* const pg = pool + s.bytes() * (size_t)(slot >> page_log2);
  const size_t off = slot & (s.page - 1);
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

}  // namespace agq
