// A key-value cache in pages (th_cache): what the kernels that write it, read
// it back (cache.hip) and attend over it (attention_paged.hip) share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "th_core.h"

namespace th {

// What th_cache holds that a kernel can address, or TH_E_ARGUMENT / TH_E_UNSUPPORTED.
int check_cache(const th_cache& c, int32_t dtype, int32_t table_pages, const char* what);

// Where a cache's rows are: element offsets, page by page.
struct Pages {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* counts;  // or null
  int64_t sh, sp, sg;     // strides along heads, positions, pages
  int32_t table_pages, page, pages;
  Divisor by_page;
};
inline Pages pages_of(const th_cache& c, int32_t table_pages, const int32_t* table, const int32_t* lengths,
                      const int32_t* counts) {
  return {table, lengths, counts, c.strides[0], c.strides[1], c.strides[2], table_pages, c.page, c.pages,
          divisor(c.page)};
}

}  // namespace th

namespace thd {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

// Positions sequence b holds, and how many of them are new.
__host__ __device__ __forceinline__ int length_of(const th::Pages& p, int b) {
  return min(max(p.lengths[b], 0), p.table_pages * p.page);
}
__host__ __device__ __forceinline__ int count_of(const th::Pages& p, int b, int seq) {
  return p.counts ? min(max(p.counts[b], 0), seq) : seq;
}

// The element at which position `at` of sequence b starts (head 0), or -1
// where no page holds it.
__host__ __device__ __forceinline__ int64_t row_of(const th::Pages& p, int b, int at) {
  const int i = quotient(at, p.by_page);
  const int page = p.table[(int64_t)p.table_pages * b + i];
  return (uint32_t)page < (uint32_t)p.pages ? page * p.sg + (at - i * p.page) * p.sp : -1;
}

// 2^(e - 127); e = 255, which stands for no number, gives infinity.
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e ? e << 23 : 0x00400000u); }

}  // namespace thd
