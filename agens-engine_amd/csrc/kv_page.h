// Pages of the key-value cache: the layout that ak_kv_write, ak_kv_read and ak_paged_attn share.
//
// A page holds `page` token slots of `heads` key-value heads of `dim` values, at 16 (bf16), 8 or 4 bits a value:
//   rows    [head][keys, values][slot], each row dim * bits / 8 contiguous bytes (8 bits: q + 128 a byte; 4 bits: q + 8 a
//           nibble, the even one low -- the offsets of the int4 weight container);
//   scales  (8 and 4 bits) [head][slot] pairs of bf16 (key scale, value scale), one scale per token and head;
// and ends at a multiple of 128 bytes, so every page's rows begin on a cache line.  A head's keys, and its values, are
// contiguous over the page's slots: attention reads them in whole lines, and one 4-byte load gives both scales.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "wq_common.h"

namespace agq {

constexpr int kPageMin = 16, kPageMax = 256;  // slots of a page, powers of two
constexpr int kMaxKvHeads = 256;

struct KvShape {
  int bits, page, heads, dim, npages;
  __host__ __device__ size_t row_bytes() const { return (size_t)dim * bits / 8; }
  __host__ __device__ size_t plane() const { return row_bytes() * page; }              // one head's keys (or values)
  __host__ __device__ size_t scale_off() const { return plane() * 2 * (size_t)heads; }  // the pairs of head 0
  __host__ __device__ size_t bytes() const {
    return (scale_off() + (bits < 16 ? (size_t)heads * page * 4 : 0) + 127) & ~(size_t)127;
  }
  bool valid() const {
    return (bits == 16 || bits == 8 || bits == 4) && page >= kPageMin && page <= kPageMax && !(page & (page - 1)) &&
           heads >= 1 && heads <= kMaxKvHeads && (dim == 64 || dim == 128 || dim == 256);
  }
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace agq
