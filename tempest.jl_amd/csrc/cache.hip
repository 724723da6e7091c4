// A key-value cache in pages: new rows written into it and held rows read
// back, as they are (bf16, fp16) or as e4m3 codes with a scale of a power of two
// for each 32 features.  Memory-bound: each row is read once and written once
// (8 contexts of 16384 positions at the most, 8 heads of 128, from e4m3: 89 us, 5.2 TB/s; single
// positions 2.4 us, the launch).
//
// A thread moves 8 features of K and the same 8 of V (16 bytes of each on the dense side),
// neighbouring threads neighbouring features, heads, positions, so that a wave reads and
// writes whole rows; the page lookup serves both.
//
// The scale of 32 features (four lanes' worth) is 2^s for the least s with
// amax <= 448 * 2^s: of the bits of amax = 1.m * 2^x, s = x - 8, and one more
// where 1.m > 1.75.  x / 2^s is exact in fp32 (s >= -117 and |x| >= 2^-133 or 0 keep it
// normal), so the code has one rounding, v_cvt_pk_fp8_f32's to nearest
// even; a power of two also makes what is held a bf16 number, which the matrix
// cores take as it is.
#include <hip/hip_runtime.h>

#include <cmath>

#include "cache.h"

namespace {

using thd::u32x2_any;
using thd::u32x4_any;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct CacheArgs {
  uint16_t* k;   // dense rows
  uint16_t* v;
  char* ck;      // the cache's
  char* cv;
  uint8_t* cks;
  uint8_t* cvs;
  th::Pages pages;
  int64_t sh, ss, sb;           // dense strides along heads, positions, batch
  int32_t seq, heads, chunks;   // chunks of 8 features a head
  int32_t items;                // chunks * heads * seq
  th::Divisor by_heads, by_chunks;
};

template <bool F16>
__device__ __forceinline__ f32x2 widened(uint32_t w) {
  if constexpr (F16) return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
  return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}
template <bool F16>
__device__ __forceinline__ uint32_t narrowed(f32x2 x) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}

// Codes of 8 values, and their 32's scale byte (the four lanes agree on it).
template <bool F16>
__device__ __forceinline__ u32x2 codes_of(u32x4 x, uint32_t& e) {
  float f[8];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 w = widened<F16>(x[i]);
    f[2 * i] = w[0], f[2 * i + 1] = w[1];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]) < INFINITY ? fabsf(f[i]) : 0.0f);
  top = fmaxf(top, __shfl_xor(top, 1, 64));
  top = fmaxf(top, __shfl_xor(top, 2, 64));
  const uint32_t bits = __float_as_uint(top);
  const int s = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  e = (uint32_t)(min(max(s, -117), F16 ? 7 : 119) + 127);
  const float inverse = __uint_as_float((254 - e) << 23);
  u32x2 out;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = fminf(fmaxf(f[i] * inverse, -448.0f), 448.0f);
    f[i] = fabsf(f[i]) < INFINITY ? y : NAN;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
    out[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], lo, true);
  }
  return out;
}

template <bool F16>
__device__ __forceinline__ u32x4 values_of(u32x2 codes, float scale) {
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    out[2 * i] = narrowed<F16>(__builtin_amdgcn_cvt_pk_f32_fp8((int)codes[i], false) * scale);
    out[2 * i + 1] = narrowed<F16>(__builtin_amdgcn_cvt_pk_f32_fp8((int)codes[i], true) * scale);
  }
  return out;
}

// An item's head, chunk and position among the seq.
struct Item {
  int chunk, head, j;
};
__device__ __forceinline__ Item item_of(const CacheArgs& p, int i) {
  const int row = thd::quotient(i, p.by_chunks), j = thd::quotient(row, p.by_heads);
  return {i - row * p.chunks, row - j * p.heads, j};
}

template <bool E4M3, bool F16>
__global__ __launch_bounds__(256) void cache_write(CacheArgs p) {
  const int i = (int)(blockIdx.x * 256u + threadIdx.x);
  const int b = blockIdx.y;
  if (i >= p.items) return;
  const Item it = item_of(p, i);
  const int count = thd::count_of(p.pages, b, p.seq);
  const int at = thd::length_of(p.pages, b) - count + it.j;
  if (it.j >= count || at < 0) return;
  const int64_t row = thd::row_of(p.pages, b, at);
  if (row < 0) return;
  const int64_t from = b * p.sb + it.j * p.ss + it.head * p.sh + 8 * it.chunk;
  const int64_t to = row + it.head * p.pages.sh + 8 * it.chunk;
  const u32x4 k = *reinterpret_cast<const u32x4_any*>(p.k + from);
  const u32x4 v = *reinterpret_cast<const u32x4_any*>(p.v + from);
  if constexpr (!E4M3) {
    *reinterpret_cast<u32x4*>(p.ck + 2 * to) = k;
    *reinterpret_cast<u32x4*>(p.cv + 2 * to) = v;
  } else {
    uint32_t ek, ev;
    const u32x2 ck = codes_of<F16>(k, ek), cv = codes_of<F16>(v, ev);
    *reinterpret_cast<u32x2*>(p.ck + to) = ck;
    *reinterpret_cast<u32x2*>(p.cv + to) = cv;
    if (it.chunk % 4 == 0) p.cks[to / 32] = (uint8_t)ek, p.cvs[to / 32] = (uint8_t)ev;
  }
}

template <bool E4M3, bool F16>
__global__ __launch_bounds__(256) void cache_read(CacheArgs p) {
  const int i = (int)(blockIdx.x * 256u + threadIdx.x);
  const int b = blockIdx.y;
  if (i >= p.items) return;
  const Item it = item_of(p, i);
  if (it.j >= thd::length_of(p.pages, b)) return;
  const int64_t row = thd::row_of(p.pages, b, it.j);
  const int64_t to = b * p.sb + it.j * p.ss + it.head * p.sh + 8 * it.chunk;
  const int64_t from = row + it.head * p.pages.sh + 8 * it.chunk;
  u32x4 k = {}, v = {};
  if (row >= 0) {
    if constexpr (!E4M3) {
      k = *reinterpret_cast<const u32x4*>(p.ck + 2 * from);
      v = *reinterpret_cast<const u32x4*>(p.cv + 2 * from);
    } else {
      const u32x2 ck = *reinterpret_cast<const u32x2*>(p.ck + from), cv = *reinterpret_cast<const u32x2*>(p.cv + from);
      k = values_of<F16>(ck, thd::scale_of(p.cks[from / 32]));
      v = values_of<F16>(cv, thd::scale_of(p.cvs[from / 32]));
    }
  }
  // Non-temporal: a large cache read back is larger than what keeps it (458 MB in 89 us, 99
  // with ordinary stores).
  __builtin_nontemporal_store(k, reinterpret_cast<u32x4_any*>(p.k + to));
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p.v + to));
}

int build(const th_cache_desc* d, bool write, th_launch** out) {
  const char* what = write ? "cache write" : "cache read";
  TH_REQUIRE(d != nullptr, std::string(what) + ": null descriptor");
  const th_cache& c = d->cache;
  if (int r = th::check_cache(c, d->dtype, d->table_pages, what)) return r;
  TH_REQUIRE(d->batch > 0 && d->batch <= 65535, std::string(what) + ": batch must be 1..65535");
  TH_REQUIRE(d->seq > 0, std::string(what) + ": seq must be positive");
  TH_REQUIRE(d->k && d->v, std::string(what) + ": null k or v");
  TH_REQUIRE(reinterpret_cast<uintptr_t>(d->k) % 2 == 0 && reinterpret_cast<uintptr_t>(d->v) % 2 == 0,
             std::string(what) + ": k and v must be aligned to their elements");
  TH_REQUIRE(d->table && d->lengths, std::string(what) + ": null table or lengths");
  TH_REQUIRE(th::aligned4(d->table) && th::aligned4(d->lengths) && th::aligned4(d->counts),
             std::string(what) + ": table, lengths and counts must be 4-byte aligned");
  TH_REQUIRE(write || !d->counts, "cache read: counts are for writing");
  const int64_t extents[3] = {c.heads, d->seq, d->batch};
  for (int64_t s : d->strides) TH_REQUIRE(s >= 0, std::string(what) + ": strides must not be negative");
  if (!write)
    TH_REQUIRE(th::rows_apart(c.head_dim, d->strides, extents, 3), "cache read: the rows of k (and of v) overlap");
  const int64_t items = (int64_t)c.head_dim / 8 * c.heads * d->seq;
  TH_REQUIRE(items <= 0x7fffffff - 255, std::string(what) + ": head_dim * heads * seq must be under 2^34");
  if (int r = th::require_ready()) return r;
  CacheArgs a{};
  a.k = static_cast<uint16_t*>(d->k), a.v = static_cast<uint16_t*>(d->v);
  a.ck = static_cast<char*>(c.k), a.cv = static_cast<char*>(c.v);
  a.cks = c.k_scales, a.cvs = c.v_scales;
  a.pages = th::pages_of(c, d->table_pages, d->table, d->lengths, write ? d->counts : nullptr);
  a.sh = d->strides[0], a.ss = d->strides[1], a.sb = d->strides[2];
  a.seq = d->seq, a.heads = c.heads, a.chunks = c.head_dim / 8;
  a.items = (int32_t)items;
  a.by_heads = th::divisor(a.heads), a.by_chunks = th::divisor(a.chunks);
  const bool e = c.dtype == TH_E4M3, h = d->dtype == TH_F16;
  const void* fn = write ? (!e  ? (const void*)cache_write<false, false>
                            : h ? (const void*)cache_write<true, true>
                                : (const void*)cache_write<true, false>)
                         : (!e  ? (const void*)cache_read<false, false>
                            : h ? (const void*)cache_read<true, true>
                                : (const void*)cache_read<true, false>);
  const int values = write ? 9 : 8;
  th::Builder b(write ? "cache_write" : "cache_read", values);
  const unsigned blocks = (unsigned)((items + 255) / 256);
  const int k = b.kernel(fn, write ? (e ? "cache_write_e4m3" : "cache_write") : (e ? "cache_read_e4m3" : "cache_read"),
                         dim3(blocks, d->batch), dim3(256), 0, a);
  const size_t offs[9] = {TH_OFFSET(CacheArgs, k),
                          TH_OFFSET(CacheArgs, v),
                          TH_OFFSET(CacheArgs, ck),
                          TH_OFFSET(CacheArgs, cv),
                          TH_OFFSET(CacheArgs, cks),
                          TH_OFFSET(CacheArgs, cvs),
                          TH_OFFSET(CacheArgs, pages) + TH_OFFSET(th::Pages, table),
                          TH_OFFSET(CacheArgs, pages) + TH_OFFSET(th::Pages, lengths),
                          TH_OFFSET(CacheArgs, pages) + TH_OFFSET(th::Pages, counts)};
  for (int v = 0; v < values; ++v) b.ref(v, k, offs[v]);
  b.element(0, 2), b.element(1, 2);
  b.align(2, 16), b.align(3, 16);
  // Every row there is room for: how many there are only the device knows.
  const double rows = (double)d->batch * d->seq * c.heads;
  b.work(2.0 * rows * c.head_dim * (e ? 2 + 33.0 / 32 : 4), 0, (int64_t)blocks * d->batch);
  *out = b.release();
  return TH_OK;
}

}  // namespace

namespace th {

bool rows_apart(int64_t row, const int64_t* strides, const int64_t* extents, int n) {
  int order[4];
  int m = 0;
  for (int i = 0; i < n; ++i)
    if (extents[i] > 1) order[m++] = i;
  std::sort(order, order + m, [&](int a, int b) { return strides[a] < strides[b]; });
  int64_t span = row;
  for (int i = 0; i < m; ++i) {
    int64_t more;  // (an extent whose bytes pass 64 bits is taken as overlapping)
    if (strides[order[i]] < span || __builtin_mul_overflow(strides[order[i]], extents[order[i]] - 1, &more) ||
        __builtin_add_overflow(span, more, &span) || span > (int64_t)1 << 60)
      return false;
  }
  return true;
}

int check_cache(const th_cache& c, int32_t dtype, int32_t table_pages, const char* what) {
  const std::string w(what);
  if (c.dtype != TH_BF16 && c.dtype != TH_F16 && c.dtype != TH_E4M3)
    return fail(TH_E_UNSUPPORTED, w + ": the cache must be bf16, fp16 or e4m3");
  if (c.dtype == TH_E4M3 ? dtype != TH_BF16 && dtype != TH_F16 : dtype != c.dtype)
    return fail(TH_E_UNSUPPORTED, w + ": arrays beside a bf16 or fp16 cache are of its type, beside an e4m3 one bf16 or fp16");
  const int unit = c.dtype == TH_E4M3 ? 32 : 8;
  TH_REQUIRE(c.head_dim > 0 && c.head_dim <= 256 && c.head_dim % unit == 0,
             w + ": head_dim must be a multiple of 8 (of 32 for e4m3) up to 256");
  TH_REQUIRE(c.heads > 0 && c.heads <= 65535, w + ": the cache's heads must be 1..65535");
  TH_REQUIRE(c.page > 0 && c.pages > 0 && (int64_t)c.page * c.pages <= 0x7fffffff,
             w + ": page and pages must be positive, and their product under 2^31");
  TH_REQUIRE(table_pages > 0 && (int64_t)table_pages * c.page <= (1 << 30),
             w + ": table_pages must be positive, and table_pages * page at most 2^30");
  TH_REQUIRE(c.k && c.v, w + ": null cache");
  TH_REQUIRE(reinterpret_cast<uintptr_t>(c.k) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v) % 16 == 0,
             w + ": the cache's arrays must be 16-byte aligned");
  TH_REQUIRE(c.dtype != TH_E4M3 || (c.k_scales && c.v_scales), w + ": an e4m3 cache needs k_scales and v_scales");
  TH_REQUIRE(reinterpret_cast<uintptr_t>(c.k_scales) % 4 == 0 && reinterpret_cast<uintptr_t>(c.v_scales) % 4 == 0,
             w + ": the scales must be 4-byte aligned");
  for (int64_t s : c.strides)
    TH_REQUIRE(s >= 0 && s % unit == 0, w + ": the cache's strides must be multiples of 8 (of 32 for e4m3)");
  const int64_t extents[3] = {c.heads, c.page, c.pages};
  TH_REQUIRE(rows_apart(c.head_dim, c.strides, extents, 3), w + ": the cache's rows overlap");
  return TH_OK;
}

}  // namespace th

extern "C" int th_build_cache_write(const th_cache_desc* d, th_launch** out) {
  TH_REQUIRE(out != nullptr, "cache write: null result");
  *out = nullptr;
  return th::guarded([&] { return build(d, true, out); });
}

extern "C" int th_build_cache_read(const th_cache_desc* d, th_launch** out) {
  TH_REQUIRE(out != nullptr, "cache read: null result");
  *out = nullptr;
  return th::guarded([&] { return build(d, false, out); });
}
