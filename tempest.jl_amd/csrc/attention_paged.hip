// Attention over a cache in pages: its checks.  The kernels are in
// attention_paged.h, one unit for each of the head dims they are built for.
#include "cache.h"

namespace th {
int paged_attention_64(const th_paged_desc* d, th_launch** out);
int paged_attention_128(const th_paged_desc* d, th_launch** out);
int paged_attention_256(const th_paged_desc* d, th_launch** out);
}  // namespace th

namespace {

int build(const th_paged_desc* d, th_launch** out) {
  TH_REQUIRE(d != nullptr, "paged attention: null descriptor");
  if (int r = th::check_cache(d->cache, d->dtype, d->table_pages, "paged attention")) return r;
  TH_REQUIRE(d->batch > 0 && d->batch <= 65535, "paged attention: batch must be 1..65535");
  TH_REQUIRE(d->seq > 0, "paged attention: seq must be positive");
  TH_REQUIRE(d->heads > 0 && d->heads % d->cache.heads == 0,
             "paged attention: heads must be a positive multiple of the cache's heads");
  TH_REQUIRE(d->window >= 0 && (d->window == 0 || d->causal), "paged attention: a window is positive, and causal");
  TH_REQUIRE(d->q && d->o, "paged attention: null q or o");
  TH_REQUIRE(reinterpret_cast<uintptr_t>(d->q) % 2 == 0 && reinterpret_cast<uintptr_t>(d->o) % 2 == 0,
             "paged attention: q and o must be aligned to their elements");
  for (int64_t s : d->q_strides) TH_REQUIRE(s >= 0, "paged attention: strides must not be negative");
  const int64_t extents[3] = {d->heads, d->seq, d->batch};
  TH_REQUIRE(th::rows_apart(d->cache.head_dim, d->q_strides, extents, 3), "paged attention: the rows of o overlap");
  TH_REQUIRE(d->table && d->lengths, "paged attention: null table or lengths");
  TH_REQUIRE(th::aligned4(d->table) && th::aligned4(d->lengths) && th::aligned4(d->counts) && th::aligned4(d->lse),
             "paged attention: table, lengths, counts and lse must be 4-byte aligned");
  TH_REQUIRE(d->heads <= 65535 && d->seq <= 65535, "paged attention: heads and seq must be at most 65535");
  const int64_t rows = (int64_t)d->seq * (d->heads / d->cache.heads);
  const int64_t keys = (int64_t)d->table_pages * d->cache.page;
  TH_REQUIRE(rows <= 0x7fffffff - 16 && (int64_t)d->batch * d->seq * d->heads <= (1 << 22),
             "paged attention: batch * seq * heads must be at most 2^22");
  TH_REQUIRE(d->batch * ((keys + 127) / 128 * 4) < 0x7fffffff - (1 << 20),
             "paged attention: the table's room for all sequences is too large");
  if (int r = th::require_ready()) return r;
  const int n = d->cache.head_dim;
  return n <= 64 ? th::paged_attention_64(d, out) : n <= 128 ? th::paged_attention_128(d, out) : th::paged_attention_256(d, out);
}

}  // namespace

extern "C" int th_build_attention_paged(const th_paged_desc* d, th_launch** out) {
  TH_REQUIRE(out != nullptr, "paged attention: null result");
  *out = nullptr;
  return th::guarded([&] { return build(d, out); });
}
