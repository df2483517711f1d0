// Attention of new tokens over the pages of the cache (kv_page.h has the layout).
//
// For token t of a sequence's T new ones, query head h and its key-value head h / (heads / kv_heads):
//   z_j = scale * q . k_j,  y = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  lse = m + log sum_j exp(z_j - m),
// over the cached tokens j < len - T + t + 1 whose page is held.
#include "agens_kernels.h"
#include "kv_page.h"

namespace agq {
namespace {

constexpr int kAttnWaves = 4;

struct AttnArgs {
  KvShape s;
  const uint16_t* q;
  uint16_t* y;
  float* lse;
  const uint8_t* pool;
  const int *qstart, *lens, *table;
  long ldq, ldy;
  int m, b, heads, ldt;
  float scale;
};

// value e of a row
template <int BITS>
__device__ __forceinline__ float value(const uint8_t* row, int e, float s) {
  if constexpr (BITS == 16) return bf2f(reinterpret_cast<const uint16_t*>(row)[e]);
  if constexpr (BITS == 8) return (float)((int)row[e] - 128) * s;
  return (float)((int)((row[e >> 1] >> (4 * (e & 1))) & 15) - 8) * s;
}

// one workgroup per (token of the sequence, query head), its waves over the cached tokens, its lanes over the values
template <int BITS, int D>
__global__ void __launch_bounds__(64 * kAttnWaves) paged_attn_kernel(const AttnArgs a) {
  constexpr int E = D / 64;
  __shared__ float sm[kAttnWaves], sl[kAttnWaves], so[kAttnWaves][D];
  const int seq = blockIdx.z, head = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int q0, q1;
  if (a.qstart) {
    q0 = min(max(a.qstart[seq], 0), a.m);
    q1 = min(max(a.qstart[seq + 1], q0), a.m);
  } else {
    q0 = seq * (a.m / a.b);
    q1 = q0 + a.m / a.b;
  }
  const int len = (int)min((long)a.lens[seq], (long)a.ldt * a.s.page), kvh = head / (a.heads / a.s.heads);
  for (int t = q0 + blockIdx.x; t < q1; t += gridDim.x) {
    const int seen = len - (q1 - 1 - t);
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      q[e] = bf2f(a.q[(size_t)t * a.ldq + head * D + lane * E + e]);
      o[e] = 0.0f;
    }
    for (int j = w; j < seen; j += kAttnWaves) {
      const int pg = a.table[(size_t)seq * a.ldt + j / a.s.page];
      if (pg < 0 || pg >= a.s.npages) continue;
      const uint8_t* const base = a.pool + a.s.bytes() * (size_t)pg;
      const uint8_t* const krow = base + a.s.plane() * (2 * (size_t)kvh) + (size_t)(j % a.s.page) * a.s.row_bytes();
      float ks = 1.0f, vs = 1.0f;
      if (BITS < 16) {
        const uint32_t pair = reinterpret_cast<const uint32_t*>(base + a.s.scale_off())[kvh * a.s.page + j % a.s.page];
        ks = bf2f(pair & 0xFFFFu);
        vs = bf2f(pair >> 16);
      }
      float z = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) z = fmaf(q[e], value<BITS>(krow, lane * E + e, ks), z);
#pragma unroll
      for (int d = 32; d; d >>= 1) z += __shfl_xor(z, d);
      z *= a.scale;
      const float mn = fmaxf(m, z);
      if (mn == -INFINITY) continue;
      const float f = expf(m - mn), p = expf(z - mn);
      l = l * f + p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(p, value<BITS>(krow + a.s.plane(), lane * E + e, vs), o[e] * f);
      m = mn;
    }
    if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
    for (int e = 0; e < E; ++e) so[w][lane * E + e] = o[e];
    __syncthreads();
    float mx = -INFINITY, lt = 0.0f;
#pragma unroll
    for (int i = 0; i < kAttnWaves; ++i) mx = fmaxf(mx, sm[i]);
    float f[kAttnWaves];
#pragma unroll
    for (int i = 0; i < kAttnWaves; ++i) {
      f[i] = sm[i] == -INFINITY ? 0.0f : expf(sm[i] - mx);
      lt += f[i] * sl[i];
    }
    for (int e = threadIdx.x; e < D; e += 64 * kAttnWaves) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < kAttnWaves; ++i) s += f[i] * so[i][e];
      a.y[(size_t)t * a.ldy + head * D + e] = lt == 0.0f ? 0 : f2bf(s / lt);
    }
    if (a.lse && threadIdx.x == 0) a.lse[(size_t)t * a.heads + head] = lt == 0.0f ? -INFINITY : mx + logf(lt);
    __syncthreads();
  }
}

template <int BITS>
int launch(const AttnArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.m + a.b - 1) / a.b), (unsigned)a.heads, (unsigned)a.b), block(64 * kAttnWaves);
  if (a.s.dim == 64)
    hipLaunchKernelGGL((paged_attn_kernel<BITS, 64>), grid, block, 0, s, a);
  else if (a.s.dim == 128)
    hipLaunchKernelGGL((paged_attn_kernel<BITS, 128>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((paged_attn_kernel<BITS, 256>), grid, block, 0, s, a);
  return (int)hipGetLastError();
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
  const agq::AttnArgs a{s,   static_cast<const uint16_t*>(q), static_cast<uint16_t*>(y), lse,
                        static_cast<const uint8_t*>(pool), qstart, lens, table, ldq, ldy, m, b, heads, ldt, scale};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return bits == 16 ? agq::launch<16>(a, st) : bits == 8 ? agq::launch<8>(a, st) : agq::launch<4>(a, st);
}
