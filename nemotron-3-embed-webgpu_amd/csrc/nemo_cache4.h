// Layout of a paged cache of 4-bit floats (include/nemo.h nemo_cache4_config).
#pragma once

#include "nemo_operators.h"

namespace nemo {

// What the kernels know of a cache. A page's KV head is K codes, V codes, K
// scales and V scales, each of page * (bytes a token).
struct Cache4 {
  uint8_t* data;
  const int32_t *table, *kv_len;
  int64_t table_row, page_bytes;
  int count, pages, shift, kv_heads;  // shift: of the page's tokens

  Cache4(const nemo_cache4_config& c, const nemo_cache4_pages& p)
      : data((uint8_t*)p.data), table(p.table), kv_len(p.kv_len), table_row(p.table_row),
        page_bytes((int64_t)c.kv_heads * c.page * (c.head_dim + c.head_dim / 16)), count(p.count), pages(p.pages),
        shift(__builtin_ctz(c.page)), kv_heads(c.kv_heads) {}

  template <int D>
  __device__ __forceinline__ int64_t head(int page, int h) const {
    return page * page_bytes + ((int64_t)h << shift) * (D + D / 16);
  }
};

// Offsets in a page's KV head of D values a token, from its beginning: token t's
// K codes, piece n (of 16) of its V codes, and scale g (of D / 32) of either.
template <int D>
struct Cache4Head {
  static constexpr int kCodes = D / 2, kScales = D / 32;
  static __device__ __forceinline__ int k_codes(int t) { return t * kCodes; }
  static __device__ __forceinline__ int v_codes(int shift, int t, int n) {
    return (kCodes << shift) + (t >> 2) * (4 * kCodes) + n * (D / 8) + (t & 3) * kScales;
  }
  static __device__ __forceinline__ int scale(int shift, bool value, int t, int g) {
    return ((D + (value ? kScales : 0)) << shift) + (t >> 3) * (8 * kScales) + g * 8 + (t & 7);
  }
};

}  // namespace nemo
