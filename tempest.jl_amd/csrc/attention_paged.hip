// Op class (c), a cache in pages: attention forward for one or a few new
// positions a sequence over K and V in pages (bf16, fp16, or e4m3 with a scale
// of a power of two for each 32 features), head dims up to 256.
//
// The work is the cache's bytes: each (sequence, cache head) reads its K and V
// once for the 16 query rows (position, head of the group) that are the columns of one
// v_mfma_f32_16x16x32.  A wave takes 32 keys at a time, straight into
// registers: K rows as the A operand of S' = K Q', V rows transposed inside each lane
// (v_perm_b32) into the A operand of O' += V' P', whose B operand the score
// registers are as they stand (keys 4 g + i and 16 + 4 g + i of lane group g
// being slots i and 4 + i).
//   - Parts of `span` keys go to a workgroup each, a part past its sequence's
//     keys or before its window ends at once, and a second kernel joins the parts by their
//     maxima and sums.
//   - The weights are fp32's: three bf16 parts (split2_towards0), or for fp16
//     values two fp16 parts of 2^15 times the weight (22 bits, and 2^-39 of the
//     largest weight where that is more), none of them 0 unless the weight is.
//   - e4m3 becomes bf16 (v_cvt_scalef32_pk_bf16_fp8), exactly: 4 bits times a
//     power of two; fp16 queries are then two bf16 parts, exactly.
#include <hip/hip_runtime.h>

#include <cmath>

#include "attention_tiles.h"
#include "cache.h"

namespace {

using thd::u32x2_any;
using thd::u32x4_any;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = 16;   // query rows a workgroup holds
constexpr int kBlock = 32;  // keys a wave takes at a time
constexpr int kStep = 128;  // keys the four waves take at a time

struct PagedArgs {
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // natural log, [b][s][h], or null
  const char* k;
  const char* v;
  const uint8_t* ks;
  const uint8_t* vs;
  th::Pages pages;
  float* part;     // nparts > 1: unnormalised O, [part][b][s][h][D]
  float* part_ml;  // and (m, l), [part][b][s][h]
  int64_t q_sh, q_ss, q_sb;
  int32_t seq, heads, kv_heads, batch, head_dim, causal, window;
  int32_t nparts, span;  // span a multiple of kStep
  float scale;
};

// Keys [lo, hi) that new position j of a sequence sees (none where lo >= hi).
struct Range {
  int lo, hi;
};
__device__ __forceinline__ Range seen_by(const PagedArgs& p, int length, int count, int j) {
  if (j >= count) return {0, 0};
  if (!p.causal) return {0, length};
  const int at = length - count + j;
  return {p.window ? max(0, at - p.window + 1) : 0, at + 1};
}
// The parts that hold keys any of positions j0..j1 sees; one at least.
struct Parts {
  int lo, hi;
};
__device__ __forceinline__ Parts parts_of(const PagedArgs& p, int length, int count, int j0, int j1) {
  const Range a = seen_by(p, length, count, j0), z = seen_by(p, length, count, min(j1, count - 1));
  if (z.hi <= a.lo) return {0, 1};
  return {a.lo / p.span, (z.hi + p.span - 1) / p.span};
}

constexpr int kBf16 = 0, kF16 = 1, kE4m3 = 2;


// One block's operands in flight: K as A operands (key l % 16 of each half,
// features 32 s + 8 (l / 16) + (0..7)), V as rows (features E (l % 16) + ..
// of keys 16 (j / 4) + 4 (l / 16) + j % 4).
template <int D, int CT, bool EXACT>
struct Block {
  static constexpr int E = D / 16;
  static constexpr int W = CT == kE4m3 ? 4 : 2;  // features a word
  uint32_t k[2][D / 32][8 / W];
  uint32_t v[8][E / W];
  uint32_t ks[2][D / 32], vs[8];  // scale bytes (e4m3)
  uint32_t present;               // bit j: a page holds V's key j

  __device__ __forceinline__ void load(const PagedArgs& p, int b, int head, int key0, int last) {
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    constexpr int bytes = CT == kE4m3 ? 1 : 2;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t row = max(thd::row_of(p.pages, b, min(key0 + 16 * t + r, last)), (int64_t)0) + head * p.pages.sh;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        const int f = EXACT || 32 * s + 8 * g < p.head_dim ? 32 * s + 8 * g : 0;
        const char* at = p.k + (row + f) * bytes;
        if constexpr (CT == kE4m3) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(at);
          k[t][s][0] = x[0], k[t][s][1] = x[1];
          ks[t][s] = p.ks[(row + f) / 32];
        } else {
          const u32x4 x = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
          for (int i = 0; i < 4; ++i) k[t][s][i] = x[i];
        }
      }
    }
    present = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t found = thd::row_of(p.pages, b, min(key0 + 16 * (j / 4) + 4 * g + j % 4, last));
      present |= (found >= 0 ? 1u : 0u) << j;
      const int64_t row = max(found, (int64_t)0) + head * p.pages.sh;
      // Features come in eights, so the first of a lane's says for four or eight of them.
#pragma unroll
      for (int c = 0; c < (E + 7) / 8; ++c) {
        const int f = EXACT || E * r + 8 * c < p.head_dim ? E * r + 8 * c : 0;
        const char* at = p.v + (row + f) * bytes;
        constexpr int words = (E < 8 ? E : 8) / W;
        if constexpr (words == 4) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][4 * c + i] = x[i];
        } else if constexpr (words == 2) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(at);
          v[j][2 * c] = x[0], v[j][2 * c + 1] = x[1];
        } else {
          v[j][c] = *reinterpret_cast<const uint32_t*>(at);
        }
      }
      if constexpr (CT == kE4m3) {
        const int f = EXACT || E * r < p.head_dim ? E * r : 0;
        vs[j] = p.vs[(row + f) / 32];
      }
    }
  }
  __device__ __forceinline__ u32x4 k_of(int t, int s) const {
    if constexpr (CT != kE4m3) return u32x4{k[t][s][0], k[t][s][1], k[t][s][2], k[t][s][3]};
    else {
      const float scale = thd::scale_of(ks[t][s]);
      u32x4 out;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        out[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k[t][s][i], scale, false));
        out[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k[t][s][i], scale, true));
      }
      return out;
    }
  }
  // Features 2 d and 2 d + 1 of V's key j.
  __device__ __forceinline__ uint32_t v_of(int j, int d) const {
    if constexpr (CT != kE4m3) return v[j][d];
    else if (d % 2)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[j][d / 2], thd::scale_of(vs[j]), true));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[j][d / 2], thd::scale_of(vs[j]), false));
  }
};

template <bool F16>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool F16>
__device__ __forceinline__ uint32_t rounded2(float a, float b) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
  return pack2(a, b);
}

// x >= 0 (at most 2^15) in two fp16 parts, 22 bits or 2^-24, the first towards
// 0 and neither 0 unless x is: an infinite value they multiply stays one.
__device__ __forceinline__ void split2_f16(float a, float b, uint32_t& w0, uint32_t& w1) {
  const float least = 5.9604645e-8f;  // fp16's least, 2^-24
  const auto hi = __builtin_amdgcn_cvt_pkrtz(a > 0 ? fmaxf(a - least, least) : 0.0f, b > 0 ? fmaxf(b - least, least) : 0.0f);
  const float ra = a > 0 ? fmaxf(a - (float)hi[0], least) : 0.0f, rb = b > 0 ? fmaxf(b - (float)hi[1], least) : 0.0f;
  w0 = __builtin_bit_cast(uint32_t, hi);
  w1 = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{ra, rb}, f16x2));
}

template <int D, int CT, bool F16, bool EXACT>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void paged_attn_fwd(PagedArgs p) {
  constexpr int E = D / 16;  // features of V a lane holds of each key
  constexpr int LD = D + 4;  // floats a row of a wave's O in LDS
  constexpr bool kHalf = CT == kF16;              // products in fp16, not bf16
  constexpr int QP = CT == kE4m3 && F16 ? 2 : 1;  // parts of q
  constexpr int WP = kHalf ? 2 : 3;               // parts of a weight
  constexpr float kBias = kHalf ? 15.0f : 0.0f;   // weights are held times 2^kBias
  extern __shared__ __attribute__((aligned(16))) float lds[];
  float(*Os)[kRows][LD] = reinterpret_cast<float(*)[kRows][LD]>(lds);
  float(*Ms)[kRows] = reinterpret_cast<float(*)[kRows]>(lds + 4 * kRows * LD);
  float(*Ls)[kRows] = Ms + 4;
  const int group = p.heads / p.kv_heads, rows = p.seq * group, tiles = (rows + kRows - 1) / kRows;
  const int part = blockIdx.x, tile = blockIdx.y % tiles, hk = blockIdx.y / tiles, b = blockIdx.z;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
  const int length = thd::length_of(p.pages, b), count = thd::count_of(p.pages, b, p.seq);
  // The tile's rows are positions j0..j1 (position row / group, head row % group of the group).
  const int j0 = kRows * tile / group, j1 = min(min(rows, kRows * tile + kRows) - 1, count * group - 1) / group;
  if (j0 >= count) return;
  const Parts parts = parts_of(p, length, count, j0, j1);
  if (part < parts.lo || part >= parts.hi) return;
  const Range first = seen_by(p, length, count, j0), final = seen_by(p, length, count, j1);
  // Keys of this part that any row sees, and those that every row sees.
  const int k_lo = max(part * p.span, first.lo), k_hi = min(part * p.span + p.span, final.hi);
  const int all_lo = final.lo, all_hi = first.hi;
  const int row = kRows * tile + r;
  const bool live = row < count * group;
  const int j = live ? row / group : j0, h = hk * group + (live ? row % group : 0);
  const Range mine = live ? seen_by(p, length, count, j) : Range{0, 0};
  const float c = p.scale * kLog2e;
  const uint16_t* qrow = p.q + (int64_t)b * p.q_sb + (int64_t)h * p.q_sh + (int64_t)j * p.q_ss;
  u32x4 qf[QP][D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    const bool there = live && (EXACT || 32 * s + 8 * g < p.head_dim);
    const u32x4 x = there ? (u32x4) * reinterpret_cast<const u32x4_any*>(qrow + 32 * s + 8 * g) : u32x4{};
    qf[0][s] = x;
    if constexpr (QP == 2) {
      u32x4 hi = {}, lo = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t word = x[i];  // (a bit cast of a vector's element itself takes element 0)
        const f32x2 w = __builtin_convertvector(__builtin_bit_cast(f16x2, word), f32x2);
        hi[i] = pack2(w[0], w[1]);
        lo[i] = pack2(w[0] - __uint_as_float(hi[i] << 16), w[1] - __uint_as_float(hi[i] & 0xffff0000u));
      }
      qf[0][s] = hi, qf[1][s] = lo;
    }
  }
  f32x4 o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = f32x4{};
  float m = -INFINITY, l = 0.0f;
  typedef Block<D, CT, EXACT> B;
  // The block of 32 keys from key0.
  auto fold = [&](const B& x, int key0) {
    f32x4 s[2] = {f32x4{}, f32x4{}};
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        u32x4 a = x.k_of(t, i);
        if (!EXACT && 32 * i + 8 * g >= p.head_dim) a = u32x4{};  // (loaded from feature 0)
#pragma unroll
        for (int u = QP - 1; u >= 0; --u) s[t] = product<kHalf>(a, qf[u][i], s[t]);
      }
    float mb = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = key0 + 16 * (i / 4) + 4 * g + i % 4;
      const bool sees = key >= mine.lo && key < mine.hi && (x.present >> i & 1);
      s[i / 4][i % 4] = sees ? s[i / 4][i % 4] : -INFINITY;
      mb = fmaxf(mb, s[i / 4][i % 4]);
    }
    mb = fmaxf(mb, __shfl_xor(mb, 16, 64));
    mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
    const float mn = fmaxf(m, mb * c);
    const float shift = thd::lse_shift(mn);
    const float alpha = __builtin_amdgcn_exp2f(m - shift);
    m = mn;
    float w[8], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], c, kBias - shift));
      sum += w[i];
    }
    l = l * alpha + sum;
    u32x4 wp[WP];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b2, d2 = 0;
      if constexpr (kHalf) split2_f16(w[2 * i], w[2 * i + 1], a, b2);
      else split2_towards0(w[2 * i], w[2 * i + 1], a, b2, d2);
      wp[0][i] = a, wp[1][i] = b2;
      if constexpr (WP == 3) wp[2][i] = d2;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= alpha;
    // Where some row does not see some key, a value there may be anything, and 0
    // times it is not 0: the rows of one position at a time, with the values it does not
    // see taken as 0.
    const bool clean = key0 >= all_lo && key0 + kBlock <= all_hi && __all(x.present == 0xff);
    auto weigh = [&](int jj, bool mask) {
      const Range see = mask ? seen_by(p, length, count, jj) : Range{0, 0};
#pragma unroll
      for (int d2 = 0; d2 < E / 2; ++d2) {
        uint32_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = x.v_of(i, d2);
          const int key = key0 + 16 * (i / 4) + 4 * g + i % 4;
          if (mask) v[i] = key >= see.lo && key < see.hi && (x.present >> i & 1) ? v[i] : 0u;
        }
        u32x4 even, odd;  // features E (l % 16) + 2 d2 and + 1 of the eight keys
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          even[i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x05040100u);
          odd[i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x07060302u);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f32x4 t = o[2 * d2 + u];
#pragma unroll
          for (int y = WP - 1; y >= 0; --y) t = product<kHalf>(u ? odd : even, wp[y], t);
          o[2 * d2 + u] = !mask || j == jj ? t : o[2 * d2 + u];
        }
      }
    };
    if (clean) weigh(0, false);
    else
      for (int jj = j0; jj <= j1; ++jj) weigh(jj, true);
  };
  int key0 = k_lo / kBlock * kBlock + kBlock * wave;
  const int last = final.hi - 1;
  if (key0 < k_hi) {
    B even, odd;
    even.load(p, b, hk, key0, last);
    while (true) {
      if (key0 + kStep < k_hi) odd.load(p, b, hk, key0 + kStep, last);
      fold(even, key0);
      key0 += kStep;
      if (key0 >= k_hi) break;
      if (key0 + kStep < k_hi) even.load(p, b, hk, key0 + kStep, last);
      fold(odd, key0);
      key0 += kStep;
      if (key0 >= k_hi) break;
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // Lane l holds row r's features E (4 g + i) + e in o[e][i].
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < E; e += 4)
      *reinterpret_cast<f32x4*>(&Os[wave][r][E * (4 * g + i) + e]) = f32x4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
  if (g == 0) Ms[wave][r] = m, Ls[wave][r] = l;
  __syncthreads();
  // The four waves' parts in wave order: thread t takes row t / 16, features E (t % 16) + (0..E).
  const int orow = threadIdx.x / 16, col = E * (threadIdx.x % 16), all = kRows * tile + orow;
  if (all >= count * group) return;
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) mx = fmaxf(mx, Ms[w][orow]);
  const float shift = thd::lse_shift(mx);
  float sum = 0.0f;
  f32x4 acc[E / 4] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float a = __builtin_amdgcn_exp2f(Ms[w][orow] - shift);
    sum += a * Ls[w][orow];
#pragma unroll
    for (int e = 0; e < E / 4; ++e) acc[e] += a * *reinterpret_cast<const f32x4*>(&Os[w][orow][col + 4 * e]);
  }
  const int jo = all / group, ho = hk * group + all % group;
  const int64_t at = ((int64_t)b * p.seq + jo) * p.heads + ho;
  if (p.nparts > 1) {
    const int64_t to = (int64_t)part * p.batch * p.seq * p.heads + at;
#pragma unroll
    for (int e = 0; e < E / 4; ++e) *reinterpret_cast<f32x4*>(p.part + to * D + col + 4 * e) = acc[e];
    if (col == 0) reinterpret_cast<f32x2*>(p.part_ml)[to] = f32x2{mx - kBias, sum};
    return;
  }
  const float inv = mx == -INFINITY ? 0.0f : 1.0f / sum;
  uint16_t* out = p.o + (int64_t)b * p.q_sb + (int64_t)ho * p.q_sh + (int64_t)jo * p.q_ss + col;
#pragma unroll
  for (int e = 0; e < E / 4; ++e)
    if (EXACT || col + 4 * e < p.head_dim)
      *reinterpret_cast<u32x2_any*>(out + 4 * e) =
          u32x2{rounded2<F16>(acc[e][0] * inv, acc[e][1] * inv), rounded2<F16>(acc[e][2] * inv, acc[e][3] * inv)};
  if (col == 0 && p.lse) p.lse[at] = (mx - kBias + log2f(sum)) * kLn2;
}

// The parts that exist, joined in part order: a thread per four features of a
// (b, query, head) row, the parts' loads issued eight at a time.
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_attn_join(PagedArgs p) {
  constexpr int quads = D / 4;
  const int64_t rows = (int64_t)p.batch * p.seq * p.heads;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= rows * quads) return;
  const int64_t row = t / quads;
  const int c = 4 * (int)(t % quads);
  const int h = (int)(row % p.heads);
  const int pos = (int)((row / p.heads) % p.seq), b = (int)(row / ((int64_t)p.heads * p.seq));
  const int length = thd::length_of(p.pages, b), count = thd::count_of(p.pages, b, p.seq);
  if (pos >= count) return;
  const int group = p.heads / p.kv_heads, tile = (pos * group + h % group) / kRows;
  const int j1 = min(min(p.seq * group, kRows * tile + kRows) - 1, count * group - 1) / group;
  const Parts parts = parts_of(p, length, count, kRows * tile / group, j1);
  const f32x2* ml = reinterpret_cast<const f32x2*>(p.part_ml) + row;
  const f32x4* po = reinterpret_cast<const f32x4*>(p.part + row * D + c);
  const int64_t step = rows * quads;
  float m = -INFINITY, l = 0.0f;
  f32x4 acc = {};
  for (int s0 = parts.lo; s0 < parts.hi; s0 += 8) {
    f32x2 x[8];
    f32x4 y[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {  // a part past the last reads the last again, with no weight
      const int64_t s = min(s0 + u, parts.hi - 1);
      x[u] = ml[s * rows];
      y[u] = po[s * step];
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) mn = fmaxf(mn, x[u][0]);
    const float shift = thd::lse_shift(mn), alpha = __builtin_amdgcn_exp2f(m - shift);
    l *= alpha;
    acc *= alpha;
    m = mn;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (s0 + u < parts.hi) {
        const float w = __builtin_amdgcn_exp2f(x[u][0] - shift);
        l += w * x[u][1];
        acc += w * y[u];
      }
  }
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
  if (c < p.head_dim)
    *reinterpret_cast<u32x2_any*>(p.o + b * p.q_sb + h * p.q_sh + pos * p.q_ss + c) =
        u32x2{rounded2<F16>(acc[0] * inv, acc[1] * inv), rounded2<F16>(acc[2] * inv, acc[3] * inv)};
  if (c == 0 && p.lse) p.lse[row] = (m + log2f(l)) * kLn2;
}

// Keys a part: about 2048 workgroups over the whole cache; at least kStep
// (each wave one block).
int span_of(int64_t keys, int64_t sweeps) {
  const int64_t span = ((keys * sweeps + 2047) / 2048 + kStep - 1) / kStep * kStep;
  return (int)std::min<int64_t>(span, (keys + kStep - 1) / kStep * kStep);
}

template <int D, int CT, bool F16, bool EXACT>
int launch(const th_paged_desc* d, th_launch** out) {
  constexpr size_t lds = (4 * kRows * (D + 4) + 8 * kRows) * sizeof(float);
  const void* fn = (const void*)paged_attn_fwd<D, CT, F16, EXACT>;
  if (lds > 65536) TH_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const th_cache& cache = d->cache;
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(d->q), a.o = static_cast<uint16_t*>(d->o), a.lse = d->lse;
  a.k = static_cast<const char*>(cache.k), a.v = static_cast<const char*>(cache.v);
  a.ks = cache.k_scales, a.vs = cache.v_scales;
  a.pages = th::pages_of(cache, d->table_pages, d->table, d->lengths, d->counts);
  a.q_sh = d->q_strides[0], a.q_ss = d->q_strides[1], a.q_sb = d->q_strides[2];
  a.seq = d->seq, a.heads = d->heads, a.kv_heads = cache.heads, a.batch = d->batch, a.head_dim = cache.head_dim;
  a.causal = d->causal != 0, a.window = d->window;
  a.scale = d->scale > 0 ? d->scale : 1.0f / sqrtf((float)cache.head_dim);
  const int64_t keys = (int64_t)d->table_pages * cache.page;
  const int64_t rows = (int64_t)d->seq * (d->heads / cache.heads), tiles = (rows + kRows - 1) / kRows;
  a.span = span_of(keys, tiles * cache.heads * d->batch);
  a.nparts = (int)((keys + a.span - 1) / a.span);
  th::Builder b("attention_paged", 10);
  const int k = b.kernel(fn, "paged_attn_fwd", dim3(a.nparts, (unsigned)(tiles * cache.heads), d->batch), dim3(256),
                         (uint32_t)lds, a);
  int end = k;
  if (a.nparts > 1) {
    const int64_t all = (int64_t)d->batch * d->seq * d->heads;
    end = b.kernel((const void*)paged_attn_join<D, F16>, "paged_attn_join", dim3((unsigned)((all * (D / 4) + 255) / 256)),
                   dim3(256), 0, a);
    const uint64_t at_o = b.workspace((uint64_t)a.nparts * all * D * sizeof(float));
    const uint64_t at_ml = b.workspace((uint64_t)a.nparts * all * 2 * sizeof(float));
    for (int kk = k; kk <= end; ++kk) {
      b.ws_ref(kk, TH_OFFSET(PagedArgs, part), at_o);
      b.ws_ref(kk, TH_OFFSET(PagedArgs, part_ml), at_ml);
    }
  }
  const size_t pages = TH_OFFSET(PagedArgs, pages);
  const size_t offs[10] = {TH_OFFSET(PagedArgs, q),
                           TH_OFFSET(PagedArgs, o),
                           TH_OFFSET(PagedArgs, lse),
                           TH_OFFSET(PagedArgs, k),
                           TH_OFFSET(PagedArgs, v),
                           TH_OFFSET(PagedArgs, ks),
                           TH_OFFSET(PagedArgs, vs),
                           pages + TH_OFFSET(th::Pages, table),
                           pages + TH_OFFSET(th::Pages, lengths),
                           pages + TH_OFFSET(th::Pages, counts)};
  for (int v = 0; v < 10; ++v)
    for (int kk = k; kk <= end; ++kk) b.ref(v, kk, offs[v]);
  b.align(3, 16), b.align(4, 16);
  // All the cache there is room for: how much is held only the device knows.
  const double bytes = CT == kE4m3 ? 33.0 / 32 : 2, D0 = cache.head_dim;
  b.work(2.0 * d->batch * cache.heads * (double)keys * D0 * bytes + 4.0 * d->batch * d->seq * (double)d->heads * D0,
         4.0 * d->batch * d->seq * (double)d->heads * keys * D0, (int64_t)a.nparts * tiles * cache.heads * d->batch);
  *out = b.release();
  return TH_OK;
}

template <int D, bool EXACT>
int launch(const th_paged_desc* d, th_launch** out) {
  if (d->cache.dtype == TH_BF16) return launch<D, kBf16, false, EXACT>(d, out);
  if (d->cache.dtype == TH_F16) return launch<D, kF16, true, EXACT>(d, out);
  return d->dtype == TH_F16 ? launch<D, kE4m3, true, EXACT>(d, out) : launch<D, kE4m3, false, EXACT>(d, out);
}

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
  const int64_t rows = (int64_t)d->seq * (d->heads / d->cache.heads);
  TH_REQUIRE((rows + kRows - 1) / kRows * d->cache.heads <= 65535, "paged attention: seq * heads is too large");
  TH_REQUIRE((int64_t)d->batch * d->seq * d->heads <= (1 << 25), "paged attention: batch * seq * heads must be at most 2^25");
  if (int r = th::require_ready()) return r;
  const int n = d->cache.head_dim;
  return n == 64    ? launch<64, true>(d, out)
         : n == 128 ? launch<128, true>(d, out)
         : n == 256 ? launch<256, true>(d, out)
         : n < 64   ? launch<64, false>(d, out)
         : n < 128  ? launch<128, false>(d, out)
                    : launch<256, false>(d, out);
}

}  // namespace

extern "C" int th_build_attention_paged(const th_paged_desc* d, th_launch** out) {
  TH_REQUIRE(out != nullptr, "paged attention: null result");
  *out = nullptr;
  return th::guarded([&] { return build(d, out); });
}
