// The paged key-value cache as the kernels see it (kv_cache.cu, attn_paged.cu).
#pragma once
#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace mb {
namespace kv {

struct Cache {
  void *k, *v;  // [n_pages, heads, page, D]
  float *k_scale, *v_scale;
  int64_t n_pages;
  int heads, page_log2;
};

// Index of the (position, head) row in the cache's [n_pages, heads, page] rows, 64 bits wide; -1 (and
// the device status) where the position has no page or its page is not one of the cache's.
MB_DEV int64_t row_of(const Cache& c, const int32_t* table, int table_width, int64_t pos, int h, int* status) {
  const int64_t at = pos >> c.page_log2;
  const int64_t page = at < table_width ? (int64_t)table[at] : -1;
  if (page < 0 || page >= c.n_pages) {
    atomicExch(status, kDevBadPage);
    return -1;
  }
  return (((page * c.heads + h) << c.page_log2)) + (pos & ((1 << c.page_log2) - 1));
}

// Loads of data that is read once: no line in L1.
MB_DEV uint4 ld_stream(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
MB_DEV uint2 ld_stream(const uint2* p) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

}  // namespace kv

mb_status check_kv_cache(const mb_kv_cache* c);
mb_status check_kv_table(const int32_t* table, int64_t ld_table, int table_width, int n_seqs);
kv::Cache device_cache(const mb_kv_cache* c);

}  // namespace mb
