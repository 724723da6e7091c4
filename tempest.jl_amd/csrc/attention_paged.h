// Op class (c), a cache in pages: attention forward for one or a few new
// positions a sequence over K and V in pages (bf16, fp16, or e4m3 with a scale
// of a power of two for each 32 features), head dims up to 256.
//
// The work is the cache's bytes: each (sequence, cache head) reads its K and V
// once for the 16 query rows (position, head of the group) that are the columns of one
// v_mfma_f32_16x16x32.  A sweep is those rows' way through the sequence's keys.
//   - Only the device knows the lengths, so the workgroups divide the work
//     there: the keys of all sequences lie in one line, in blocks of 32, which
//     is cut into equal pieces, as many as let every (piece, head, tile of 16 rows) be a
//     workgroup that runs at once, whatever the lengths and the table's room.  A piece
//     that holds a whole sweep stores its result; the others leave partial results,
//     two a workgroup at most, that a second kernel joins by their maxima and sums.
//     Short tables take no pieces: eight waves a sweep, one launch (whole_sweeps).
//   - The heads of a piece, whose rows lie side by side, run on one XCD and start a few
//     workgroups apart: 8 sequences of 8 heads of 128 in e4m3 and 65536 positions 114 us, the join with it;
//     each head cut by itself 125, the heads side by side in order (all at the same line at
//     once) 130.
//   - A wave takes 32 keys at a time.  The next 32's K and V rows are under way in registers
//     meanwhile, K's from where the scores have used K, V's from where the sums have used V:
//     one set of registers, so that three workgroups of four waves fit a CU at 128 features
//     (two: 131 us in the case above, four, spilling: 156).
//   - Pages in sixteens (most): each half block lies in one page, whose entry and address
//     are scalars and the row's offset the same for all blocks.  Other pages: the entries come from LDS, where
//     they are laid once for many blocks (read from memory they would make each block wait for
//     the loads before it, which come back in order); 32 lanes work out a row's address each and
//     hand them on through LDS.
//   - K rows are the A operand of S' = K Q', V rows transposed inside each lane
//     (v_perm_b32) the A operand of O' += V' P', whose B operand the score
//     registers are as they stand (keys 4 g + i and 16 + 4 g + i of lane group g
//     being slots i and 4 + i).
//   - The weights are fp32's: three bf16 parts (split2_towards0), none of them 0 unless
//     the weight is.  Beside fp16 values, two fp16 parts of 2^15 times the weight (22 bits, half of what
//     the exponential leaves open) in the blocks where no weight is under 2^-16 of the largest so far, for
//     fp16 ends at 2^-39 of it; in the others three bf16 parts, and the values as two, exactly.  16 sequences
//     of 8 heads of 128 in fp16 38.7 us, 40.8 where all blocks hold small weights (fp16 parts alone 36.0, and
//     weights under 2^-38 wrong; bf16 parts alone 39.9, and one sequence of 600 positions 11.0 for 9.5).
//   - e4m3 becomes bf16 (v_cvt_scalef32_pk_bf16_fp8), exactly: 4 bits times a
//     power of two; fp16 queries are then two bf16 parts, exactly.
//
// Bound by memory where there is enough of it: the case above reads 530 to 660 MB at 5.5 TB/s
// (6.1 where a head's rows lie in a run); 16 sequences of 8 heads of 128 in bf16, 4096 positions at the
// most, 170 MB in 36 us, 5 of them the join.  Short ones by the steps' latency, about 1.3 us each.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "attention_tiles.h"
#include "cache.h"

namespace {

using thd::u32x2_any;
using thd::u32x4_any;
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = 16;       // query rows a sweep holds
constexpr int kBlock = 32;      // keys a wave takes at a time
constexpr int kEntries = 2048;  // table entries in LDS at a time

struct PagedArgs {
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // natural log, [b][s][h], or null
  const char* k;
  const char* v;
  const uint8_t* ks;
  const uint8_t* vs;
  th::Pages pages;
  float* part;      // unnormalised O of unfinished sweeps, [workgroup][first, last][row][D]
  float* part_ml;   // and (m, l), [workgroup][first, last][row]
  int32_t* pieces;  // of each sweep: the first piece's place in part, how many there are
  int64_t q_sh, q_ss, q_sb;
  int32_t seq, heads, kv_heads, batch, head_dim, causal, window;
  int32_t group, tiles, sweeps;  // query heads a cache head; tiles of 16 rows; sweeps a sequence
  int32_t shares;                // pieces of the line, at the most
  th::Divisor by_group, by_tiles, by_sweeps, by_shares;
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

// Sequence b's keys from the first that any new position sees, in blocks (fours of them,
// so that a short sweep fills a workgroup's waves and shares none).
struct Sequence {
  int length, count, lo, blocks;
};
__device__ __forceinline__ Sequence sequence_of(const PagedArgs& p, int length, int count) {
  const int lo = seen_by(p, length, count, 0).lo / kBlock * kBlock;
  return {length, count, lo, count > 0 ? (length - lo + 4 * kBlock - 1) / (4 * kBlock) * 4 : 0};
}
__device__ __forceinline__ Sequence sequence_of(const PagedArgs& p, int b) {
  return sequence_of(p, thd::length_of(p.pages, b), thd::count_of(p.pages, b, p.seq));
}
// The same for a b that the wave shares, by scalar loads.
typedef const __attribute__((address_space(4))) int32_t* constant_i32;
__device__ __forceinline__ Sequence sequence_of_all(const PagedArgs& p, int b) {
  const int length = min(max(((constant_i32)p.pages.lengths)[b], 0), p.pages.table_pages * p.pages.page);
  return sequence_of(p, length, p.pages.counts ? min(max(((constant_i32)p.pages.counts)[b], 0), p.seq) : p.seq);
}

// x and all of the lanes' before.
__device__ __forceinline__ int running_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr 1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // 2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // 4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // rows 1, 3 + lane 15, 47's
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // rows 2, 3 + lane 31's
  return x;
}

// The line of all sequences' blocks and the piece of it that is this workgroup's: 64
// sequences at a time, a lane each.
struct Line {
  Sequence own;            // lane's: sequence b0 + lane
  int end, b0;             // the line's length up to its end, from b0's start
  int share, start, stop;  // a piece's length; the piece
  int piece, sweep;        // which one, and of which of each sequence's sweeps
  int b, before;           // a sequence, the line's length before it

  __device__ __forceinline__ int step(const PagedArgs& p, int at) {
    const int lane = threadIdx.x % 64;
    b0 = at;
    own = at + lane < p.batch ? sequence_of(p, at + lane) : Sequence{};
    end = running_sum(own.blocks);
    return __builtin_amdgcn_readlane(end, 63);
  }
  __device__ __forceinline__ bool find(const PagedArgs& p, int least) {
    int total = 0;
    for (int at = 0; at < p.batch; at += 64) total += step(p, at);
    share = max(least, thd::quotient(total + p.shares - 1, p.by_shares));
    // A second step that only some waves take lasts as long as a full one, and fewer pieces are
    // joined: 2 sequences of one head of 256, five blocks a piece 19.9 us, eight 17.5.  (Longer pieces
    // lose more workgroups than they gain: nine to twelve, 17.5 us to 18.1.)
    if (share < 2 * least) share = (share + least - 1) & -least;
    // The sweeps of one piece are cache heads, whose rows lie side by side.  Pieces of a length
    // worth it: piece by piece for the first sweep, then for the next, so that they start soon
    // after each other, on one XCD where the pieces are in eights (workgroups go to the eight in
    // turn).  Shortest pieces: those that have work come first.
    if (share > least) sweep = thd::quotient(blockIdx.x, p.by_shares), piece = blockIdx.x - sweep * p.shares;
    else piece = thd::quotient(blockIdx.x, p.by_sweeps), sweep = blockIdx.x - piece * p.sweeps;
    start = piece * share, stop = min(total, start + share);
    if (start >= stop) return false;
    before = 0;
    if (p.batch > 64)
      for (int at = 0;; at += 64) {
        const int n = step(p, at);
        if (before + n > start) break;
        before += n;
      }
    const int at = __ffsll((unsigned long long)__ballot(before + end > start)) - 1;
    b = b0 + at;
    before += __builtin_amdgcn_readlane(end - own.blocks, at);
    return true;
  }
  // Sequence b, or one after it.
  __device__ __forceinline__ Sequence sequence(const PagedArgs& p) const {
    if (b - b0 >= 64) return sequence_of_all(p, b);
    const int at = b - b0;
    return {__builtin_amdgcn_readlane(own.length, at), __builtin_amdgcn_readlane(own.count, at),
            __builtin_amdgcn_readlane(own.lo, at), __builtin_amdgcn_readlane(own.blocks, at)};
  }
};

constexpr int kBf16 = 0, kF16 = 1, kE4m3 = 2;

// What a wave shares with itself: where the block's rows are (bytes from the
// arrays' start), and its scale bytes, K's 32 keys and then V's.
template <int D>
struct WaveLds {
  int64_t row[kBlock];
  uint32_t scale[(D + 127) / 128][2 * kBlock];
};

// The largest of the four lane groups' values, in each.
__device__ __forceinline__ float max_of_groups(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A sweep's keys: the table's row, its entries in LDS from entry `first` on
// (pages not in sixteens), the last key, the head's bytes.
struct Keys {
  const int32_t* table;
  const int32_t* entries;
  int first, last;
  int64_t at;
};

// One block's operands, in flight from load_k and load_v to the products: K as A operands
// of key l % 16 of each half, V as rows (of keys 16 (j / 4) + 4 (l / 16) + j % 4, in
// pieces of CH features, 16 bytes at the most, whole lines of memory a load: piece c from
// feature CH (l % 16 + 16 c)).  A product's slot (g, e) is feature 32 s + 8 g +
// e for 16-bit K; for e4m3, so that a lane's load is 16 bytes here too, slot
// (g, e) of products 2 s and 2 s + 1 are features 64 s + 16 g + e and + 8 + e.
// UNIFORM: pages in sixteens, so that each half block lies in one page.  The
// wave reads its entry as a scalar, and the rows are at scalar addresses and
// offsets that every block shares: no address is worked out on the vector ALU.
// STREAM: V's loads are non-temporal (16 sequences of 8 heads of 128 in bf16: 36 us, K's too, whose lines
// are each read by two loads, 39).
template <int D, int CT, bool EXACT, bool UNIFORM, bool STREAM>
struct Block {
  static constexpr int E = D / 16;
  static constexpr int bytes = CT == kE4m3 ? 1 : 2;
  static constexpr int W = 4 / bytes;                        // features a word
  static constexpr int KL = CT == kE4m3 ? D / 64 : D / 32;  // 16-byte pieces of a K row
  static constexpr int SW = (D + 127) / 128;                 // words of scale bytes a key
  static constexpr int CH = E < 16 / bytes ? E : 16 / bytes; // features of V a load
  u32x4 k[2][KL];
  uint32_t v[8][E / W];
  uint32_t scale[SW];  // key l % 32's: K's in lanes 0..31, V's in the others

  // A block's table entries: of its halves (UNIFORM), of the lane's key l % 32.
  struct Entries {
    int page[2];
  };
  // Where its rows are: of each half its first (UNIFORM), in LDS otherwise.
  struct Rows {
    int64_t half[2];
    uint32_t present;  // bit i: a page holds the block's key i
  };

  __device__ __forceinline__ static int k_feature(int s, int g) {
    return CT == kE4m3 ? 64 * s + 16 * g : 32 * s + 8 * g;
  }
  __device__ __forceinline__ void load_scale(const PagedArgs& p, int64_t row) {
    if constexpr (CT == kE4m3) {
      const uint8_t* from = (threadIdx.x % 64 < kBlock ? p.ks : p.vs) + row / 32;
      if constexpr (!EXACT) {
#pragma unroll
        for (int c = 0; c < SW; ++c) scale[c] = 0;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          if (32 * c < p.head_dim) scale[c / 4] |= (uint32_t)from[c] << (8 * (c % 4));
      } else if constexpr (D == 64) {
        scale[0] = *reinterpret_cast<const u16_any*>(from);
      } else {
#pragma unroll
        for (int c = 0; c < SW; ++c) scale[c] = reinterpret_cast<const u32_any*>(from)[c];
      }
    }
  }
  // The block at key0's keys: past the last the last one again, a half past it the
  // last one's (no row sees them).
  __device__ __forceinline__ static int key_of(const Keys& keys, int key0, int t) {
    return UNIFORM ? min(key0 + 16 * t, keys.last & ~15) : min(key0 + (int)(threadIdx.x % kBlock), keys.last);
  }
  __device__ __forceinline__ static Entries look(const PagedArgs& p, const Keys& keys, int key0) {
    Entries e;
#pragma unroll
    for (int t = 0; t < (UNIFORM ? 2 : 1); ++t) {
      const int i = thd::quotient(key_of(keys, key0, t), p.pages.by_page);
      e.page[t] = UNIFORM ? ((constant_i32)keys.table)[i] : keys.entries[i - keys.first];
    }
    return e;
  }
  // K's operands and the scales of the block at key0, whose entries are `e`.
  __device__ __forceinline__ Rows load_k(const PagedArgs& p, const Keys& keys, WaveLds<D>& w, const Entries& e, int key0) {
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    Rows rows;
    const char* row[2];
    // An entry that names no page: page 0's rows, which no row sees.
    auto place = [&](int t, bool& found) {
      const int key = key_of(keys, key0, t), at = key - thd::quotient(key, p.pages.by_page) * p.pages.page;
      found = (uint32_t)e.page[t] < (uint32_t)p.pages.pages;
      return ((found ? e.page[t] : 0) * p.pages.sg + at * p.pages.sp) * bytes + keys.at;
    };
    if constexpr (UNIFORM) {
      rows.present = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bool found;
        rows.half[t] = place(t, found);
        rows.present |= found ? 0xffffu << 16 * t : 0u;
        row[t] = p.k + rows.half[t] + (uint32_t)(r * ((int32_t)p.pages.sp * bytes));
      }
      load_scale(p, (lane % kBlock < 16 ? rows.half[0] : rows.half[1]) + r * ((int32_t)p.pages.sp * bytes));
    } else {
      bool found;
      const int64_t mine = place(0, found);
      rows.half[0] = rows.half[1] = 0;
      rows.present = (uint32_t)__ballot(found);
      if (lane < kBlock) w.row[lane] = mine;
      load_scale(p, mine);
      wave_fence();
#pragma unroll
      for (int t = 0; t < 2; ++t) row[t] = p.k + w.row[16 * t + r];
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < KL; ++s) {
        const int f = EXACT || k_feature(s, g) < p.head_dim ? k_feature(s, g) : 0;
        k[t][s] = *reinterpret_cast<const u32x4*>(row[t] + f * bytes);
      }
    return rows;
  }
  // V's rows of the block whose K was loaded last.
  __device__ __forceinline__ void load_v(const PagedArgs& p, const Rows& rows, WaveLds<D>& w) {
    const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char* row = p.v;
      if constexpr (UNIFORM) row += rows.half[j / 4] + (uint32_t)((4 * g + j % 4) * ((int32_t)p.pages.sp * bytes));
      else row += w.row[16 * (j / 4) + 4 * g + j % 4];
      // Features come in eights (e4m3 in 32s), so a piece's first says for all of it.
#pragma unroll
      for (int c = 0; c < E / CH; ++c) {
        const int f = EXACT || CH * (r + 16 * c) < p.head_dim ? CH * (r + 16 * c) : 0;
        constexpr int words = CH / W;
        if constexpr (words == 1) {
          v[j][c] = *reinterpret_cast<const uint32_t*>(row + f * bytes);
        } else {
          typedef uint32_t piece __attribute__((ext_vector_type(words)));
          const piece* from = reinterpret_cast<const piece*>(row + f * bytes);
          const piece x = STREAM ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
          for (int n = 0; n < words; ++n) v[j][words * c + n] = x[n];
        }
      }
    }
  }
};

// A block's scales as the operands need them: of K, a byte e << 23 for each half and 64
// features; of V, one for each of the lane's keys.
template <int D>
struct Scales {
  float k[2][D / 64], v[8];
  __device__ __forceinline__ void spread(WaveLds<D>& w, const uint32_t* scale, int r, int g) {
    const int lane = threadIdx.x % 64;
    constexpr int SW = (D + 127) / 128;
#pragma unroll
    for (int c = 0; c < SW; ++c) w.scale[c][lane] = scale[c];
    wave_fence();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < D / 64; ++s) {  // features 64 s + 16 g: block 2 s + g / 2
        const uint32_t word = w.scale[s / 2][16 * t + r];
        k[t][s] = __uint_as_float((word >> (16 * (s % 2) + 8 * (g / 2)) & 255u) << 23);
      }
    const int block = D / 16 * r / 32;  // of features CH r
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 words = *reinterpret_cast<const u32x4*>(&w.scale[block / 4][kBlock + 16 * h + 4 * g]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t word = words[i];
        v[4 * h + i] = __uint_as_float((word >> (8 * (block % 4)) & 255u) << 23);
      }
    }
    wave_fence();
  }
};

__device__ __forceinline__ uint32_t bf16_of(uint32_t codes, float scale, int half) {
  return __builtin_bit_cast(uint32_t, half ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
}

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

// x in 2^-1..2^15, or 0, in two fp16 parts, 22 bits, the first towards 0 and neither 0 unless x is: an
// infinite value they multiply stays one.
__device__ __forceinline__ void split2_f16(float a, float b, uint32_t& w0, uint32_t& w1) {
  const float least = 5.9604645e-8f;  // fp16's least, 2^-24
  const auto hi = __builtin_amdgcn_cvt_pkrtz(fmaxf(a - least, 0.0f), fmaxf(b - least, 0.0f));
  const float ra = a > 0 ? fmaxf(a - (float)hi[0], least) : 0.0f, rb = b > 0 ? fmaxf(b - (float)hi[1], least) : 0.0f;
  w0 = __builtin_bit_cast(uint32_t, hi);
  w1 = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{ra, rb}, f16x2));
}

// Two words of fp16 pairs (two features of two keys) as bf16 pairs of each feature: the top 8 bits of its
// 11, and the other 3, exactly.  An infinity is the first part's; the second is then finite (an
// infinity less itself is NaN, which fmaxf drops; no part that is a number reaches -256).
__device__ __forceinline__ void split_f16(uint32_t key0, uint32_t key1, uint32_t (&even)[2], uint32_t (&odd)[2]) {
  const f32x2 a = __builtin_convertvector(__builtin_bit_cast(f16x2, key0), f32x2);
  const f32x2 b = __builtin_convertvector(__builtin_bit_cast(f16x2, key1), f32x2);
  auto top = [](float x) { return __float_as_uint(x) & 0xffff0000u; };
  auto rest = [&](float x) { return __float_as_uint(fmaxf(x - __uint_as_float(top(x)), -256.0f)); };
  auto high = [](uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07060302u); };
  even[0] = high(__float_as_uint(a[0]), __float_as_uint(b[0])), even[1] = high(rest(a[0]), rest(b[0]));
  odd[0] = high(__float_as_uint(a[1]), __float_as_uint(b[1])), odd[1] = high(rest(a[1]), rest(b[1]));
}

// Waves a SIMD that the registers are kept to: as many as keep a block's K and V and the sums without
// spills (whole sweeps, whose eight waves need two, spill at 256 features and are still ahead there, 9.3 us
// against 11.5 for 64 positions).  fp16's two ways of the sums need more: with one more wave 16 sequences of 8
// heads of 128 take 39.2 us for 38.7, 46.4 for 40.8 where weights are small.
constexpr int waves_of(int D, int CT, bool SINGLE, bool WHOLE) {
  if (WHOLE) return D > 64 || !SINGLE ? 2 : 4;
  return D > 128 ? 1 : (D > 64 ? 2 : 3) + (SINGLE && CT != kF16);
}

// Whether one of a word's values is NaN or an infinity.
template <int CT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (CT == kE4m3) {  // a byte of 0x7f but for its sign
    const uint32_t x = ~w & 0x7f7f7f7fu;
    return ((x - 0x01010101u) & ~x & 0x80808080u) != 0;
  }
  constexpr uint32_t e = CT == kBf16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w >> 16 & e) == e;
}

// A word with its values that are not finite as 0.
template <int CT>
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
  if constexpr (CT == kE4m3) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 32; i += 8) out |= (w >> i & 0x7fu) == 0x7fu ? 0u : w & 0xffu << i;
    return out;
  }
  constexpr uint32_t e = CT == kBf16 ? 0x7f80u : 0x7c00u;
  return ((w & e) == e ? 0u : w & 0xffffu) | ((w >> 16 & e) == e ? 0u : w & 0xffff0000u);
}

// EXACT: head_dim is D.  SINGLE: one new position a sequence, in one tile.  WHOLE: a workgroup of
// eight waves a sweep, no pieces and nothing to join.  EARLY (WHOLE, entries by way of LDS, no window, so
// that the keys start at 0): q, the table's entries and the first blocks' rows are asked for before the
// lengths are here (what lies behind a length is some page's rows all the same): 421 positions in pages of
// five 6.8 us to 6.2.  With scalar entries, which come as soon, 9.1 both ways for 600 positions.
template <int D, int CT, bool F16, bool EXACT, bool UNIFORM, bool SINGLE, bool WHOLE, bool EARLY>
__global__ __launch_bounds__(WHOLE ? 512 : 256, waves_of(D, CT, SINGLE, WHOLE)) void paged_attn_fwd(PagedArgs p) {
  constexpr int E = D / 16;  // features of V a lane holds of each key
  constexpr int LD = D + 4;  // floats a row of a wave's O in LDS
  constexpr int NW = WHOLE ? 8 : 4;               // waves
  constexpr int kStep = kBlock * NW;              // keys they take at a time
  constexpr bool kHalf = CT == kF16;              // scores, and most weighted sums, in fp16, not bf16
  constexpr int QP = CT == kE4m3 && F16 ? 2 : 1;  // parts of q
  constexpr float kTimes = kHalf ? 32768.0f : 1.0f;  // o is held times this
  typedef Block<D, CT, EXACT, UNIFORM, SINGLE && !WHOLE> B;
  // LDS holds q's operands, what a wave shares with itself and the table's entries while a
  // sweep runs, then the waves' results.
  extern __shared__ __attribute__((aligned(16))) char lds[];
  u32x4* qs = reinterpret_cast<u32x4*>(lds);  // [part][product][lane]
  WaveLds<D>* waves = reinterpret_cast<WaveLds<D>*>(qs + QP * (D / 32) * 64);
  int32_t* entries = reinterpret_cast<int32_t*>(waves + NW);
  float(*Os)[kRows][LD] = reinterpret_cast<float(*)[kRows][LD]>(lds);
  float(*Ms)[kRows] = reinterpret_cast<float(*)[kRows]>(Os + NW);
  float(*Ls)[kRows] = Ms + NW;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
  const float c = p.scale * kLog2e;
  Line line;
  if constexpr (WHOLE) {
    line.b = thd::quotient(blockIdx.x, p.by_sweeps), line.sweep = blockIdx.x - line.b * p.sweeps;
    line.start = line.stop = 0;
  } else {
    if (!line.find(p, NW)) return;
  }
  const int sweep = line.sweep, hk = thd::quotient(sweep, p.by_tiles), tile = sweep - hk * p.tiles;
  for (int u = line.start; WHOLE || u < line.stop;) {
    const int b = line.b;
    int i0 = 0, i1, slot = -1;
    // q's operands, a product's to each wave in turn: on their way here, in LDS behind the
    // first block's loads.
    constexpr int QN = (D / 32 + NW - 1) / NW;
    u32x4 q[QN];
    const int row = kRows * tile + r;
    auto load_q = [&](bool there, int h, int j) {
      const uint16_t* qrow = p.q + (int64_t)b * p.q_sb + (int64_t)h * p.q_sh + (int64_t)j * p.q_ss;
#pragma unroll
      for (int n = 0; n < QN; ++n) {
        const int s = wave + NW * n, f = CT == kE4m3 ? B::k_feature(s / 2, g) + 8 * (s % 2) : B::k_feature(s, g);
        q[n] = there && s < D / 32 && (EXACT || f < p.head_dim) ? (u32x4) * reinterpret_cast<const u32x4_any*>(qrow + f) : u32x4{};
      }
    };
    Keys keys{p.pages.table + (int64_t)p.pages.table_pages * b, entries, 0, p.pages.table_pages * p.pages.page - 1,
              (int64_t)hk * p.pages.sh * B::bytes};
    B x;
    typename B::Rows rows;
    typename B::Entries next;  // the next block's entries
    // This wave's first block from s0: also where it has none before s1 (the last key's rows then),
    // so that what waits for q below waits for no more.
    auto begin = [&](int key0) {
      next = B::look(p, keys, key0);
      rows = x.load_k(p, keys, waves[wave], next, key0);
      x.load_v(p, rows, waves[wave]);
      next = B::look(p, keys, key0 + kStep);
    };
    if constexpr (EARLY) {
      const int at = thd::quotient(row, p.by_group);
      load_q(at < p.seq, hk * p.group + row - at * p.group, at);
      for (int i = threadIdx.x; i < p.pages.table_pages; i += 64 * NW) entries[i] = keys.table[i];
      __syncthreads();
      begin(kBlock * wave);
    }
    Sequence seq;
    if constexpr (WHOLE) {
      seq = sequence_of_all(p, b);
      i1 = seq.blocks;
    } else {
      seq = line.sequence(p);
      i0 = u - line.before;
      if (i0 >= seq.blocks) {
        line.before += seq.blocks;
        ++line.b;
        continue;
      }
      i1 = min(seq.blocks, i0 + line.stop - u);
      const bool whole = i0 == 0 && i1 == seq.blocks;
      slot = whole ? -1 : 2 * (line.piece * p.sweeps + sweep) + (u > line.start);
      // Who has a sweep's first block says where its pieces are.
      if (i0 == 0 && threadIdx.x == 0) {
        int32_t* to = p.pieces + 2 * ((int64_t)b * p.sweeps + sweep);
        to[0] = slot, to[1] = whole ? 0 : (u + seq.blocks - 1) / line.share - line.piece + 1;
      }
      u += i1 - i0;
    }
    // The tile's rows are positions j0..j1 (position row / group, head row % group of the group).
    const int length = seq.length, count = seq.count;
    const int j0 = thd::quotient(kRows * tile, p.by_group);
    if (WHOLE && j0 >= count) return;
    const int j1 = thd::quotient(min(count * p.group, kRows * tile + kRows) - 1, p.by_group);
    const Range first = seen_by(p, length, count, j0), final = seen_by(p, length, count, j1);
    // Keys of this piece that any row sees, and those that every row sees.
    const int k_lo = max(seq.lo + kBlock * i0, first.lo / kBlock * kBlock), k_hi = j0 < count ? min(seq.lo + kBlock * i1, final.hi) : 0;
    const int all_lo = final.lo, all_hi = first.hi, last = final.hi - 1;
    const bool live = row < count * p.group;
    const int j = live ? thd::quotient(row, p.by_group) : j0, h = hk * p.group + (live ? row - j * p.group : 0);
    const Range mine = live ? seen_by(p, length, count, j) : Range{0, 0};
    if constexpr (!EARLY) load_q(live, h, j);
    keys.last = last;
    auto lay_q = [&]() {
#pragma unroll
      for (int n = 0; n < QN; ++n) {
        const int s = wave + NW * n;
        if (s >= D / 32) break;
        if constexpr (QP == 1) {
          qs[64 * s + lane] = q[n];
        } else {
          u32x4 hi = {}, lo = {};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t word = q[n][i];  // (a bit cast of a vector's element itself takes element 0)
            const f32x2 w = __builtin_convertvector(__builtin_bit_cast(f16x2, word), f32x2);
            hi[i] = pack2(w[0], w[1]);
            lo[i] = pack2(w[0] - __uint_as_float(hi[i] << 16), w[1] - __uint_as_float(hi[i] & 0xffff0000u));
          }
          qs[64 * s + lane] = hi, qs[64 * (D / 32 + s) + lane] = lo;
        }
      }
    };
    f32x4 o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = f32x4{};
    float m = -INFINITY, l = 0.0f;
    // The block of 32 keys from key0, the next one's loads (`more`) issued where its
    // operands' registers are free: K's after this one's scores, V's after its sums.
    auto fold = [&](int key0, auto more) {
      Scales<D> sc;
      if constexpr (CT == kE4m3) sc.spread(waves[wave], x.scale, r, g);
      const uint32_t present = rows.present;
      f32x4 s[2] = {f32x4{}, f32x4{}};
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          u32x4 a;
          if constexpr (CT == kE4m3) {
#pragma unroll
            for (int n = 0; n < 4; ++n) a[n] = bf16_of(x.k[t][i / 2][2 * (i % 2) + n / 2], sc.k[t][i / 2], n % 2);
            if (!EXACT && B::k_feature(i / 2, g) >= p.head_dim) a = u32x4{};  // (loaded from feature 0)
          } else {
            a = x.k[t][i];
            if (!EXACT && B::k_feature(i, g) >= p.head_dim) a = u32x4{};
          }
#pragma unroll
          for (int y = QP - 1; y >= 0; --y) s[t] = product<kHalf>(a, qs[64 * (y * (D / 32) + i) + lane], s[t]);
        }
      if constexpr (more) rows = x.load_k(p, keys, waves[wave], next, key0 + kStep);
      __builtin_amdgcn_sched_barrier(0);
      // Where some row does not see some key, the value there may be anything, and 0
      // times it is not 0.  What no row sees is taken as 0; of what rows of several
      // positions differ in, values that are not finite are taken out and added to the rows that
      // see them by themselves.
      uint32_t differ = 0;  // bit i: some rows see the lane's key i, some do not
      bool apart = false;
      float low = INFINITY;  // fp16: the least score that the lane's row sees, but NaN
      if constexpr (kHalf)
#pragma unroll
        for (int i = 0; i < 8; ++i) low = fminf(low, s[i / 4][i % 4]);
      if (!(key0 >= all_lo && key0 + kBlock <= all_hi && present == 0xffffffffu)) {
        uint32_t strange = 0;
        low = INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int n = 16 * (i / 4) + 4 * g + i % 4, key = key0 + n;
          const bool held = present >> n & 1, some = held && key >= first.lo && key < final.hi;
          const bool seen = held && key >= mine.lo && key < mine.hi;
          if constexpr (kHalf) low = seen ? fminf(low, s[i / 4][i % 4]) : low;
          s[i / 4][i % 4] = seen ? s[i / 4][i % 4] : -INFINITY;
          if constexpr (CT == kE4m3) sc.v[i] = some ? sc.v[i] : 1.0f;
          if constexpr (SINGLE) {
#pragma unroll
            for (int d = 0; d < E / B::W; ++d) x.v[i][d] &= some ? 0xffffffffu : 0u;
            continue;
          }
          if (key < all_lo || key >= all_hi) differ |= 1u << i;
#pragma unroll
          for (int d = 0; d < E / B::W; ++d) {
            x.v[i][d] &= some ? 0xffffffffu : 0u;
            strange |= (differ >> i & 1) & not_finite<CT>(x.v[i][d]);
          }
          if constexpr (CT == kE4m3) strange |= (differ >> i & 1) & (sc.v[i] == INFINITY);
        }
        apart = !SINGLE && j1 > j0 && __any(strange != 0);
      }
      float mb = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) mb = fmaxf(mb, s[i / 4][i % 4]);
      mb = max_of_groups(mb);
      // (behind the scores: nothing waits for LDS until they are here)
      if constexpr (more) next = B::look(p, keys, key0 + 2 * kStep);
      const float mn = fmaxf(m, mb * c);
      const float shift = thd::lse_shift(mn);
      if (__any(mn > m)) {  // (else every factor is 1)
        const float alpha = __builtin_amdgcn_exp2f(m - shift);
        l *= alpha;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= alpha;
        m = mn;
      }
      float w[8];
      auto weights = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], c, -shift));
          l += w[i];
        }
      };
      if constexpr (!kHalf) weights();
      auto value = [&](int i, int d2) {  // features 2 d2 and 2 d2 + 1 of the lane's key i
        if constexpr (CT == kE4m3) return bf16_of(x.v[i][d2 / 2], sc.v[i], d2 % 2);
        else return x.v[i][d2];
      };
      if (apart) {
        constexpr uint32_t one = kHalf ? 0x3c00u : 0x3f80u, top = kHalf ? 0x7c00u : 0x7f80u;
        u32x4 sees;  // 1 for each key of the row's
        auto seen_weight = [&](int i) { return kHalf ? __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], c, -shift)) : w[i]; };
#pragma unroll
        for (int i = 0; i < 4; ++i) sees[i] = (seen_weight(2 * i) > 0 ? one : 0u) | (seen_weight(2 * i + 1) > 0 ? one << 16 : 0u);
#pragma unroll
        for (int d = 0; d < E; ++d)
#pragma unroll 1
          for (int kind = 0; kind < 3; ++kind) {  // infinity, -infinity, NaN
            uint32_t is[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t y = value(i, d / 2) >> (16 * (d % 2)) & 0xffffu;
              const bool that = kind == 2 ? (y & 0x7fffu) > top : y == (kind == 0 ? top : top | 0x8000u);
              is[i] = that && (differ >> i & 1) ? one : 0u;
            }
            const u32x4 a = {is[0] | is[1] << 16, is[2] | is[3] << 16, is[4] | is[5] << 16, is[6] | is[7] << 16};
            const f32x4 n = product<kHalf>(a, sees, f32x4{});
            const float there = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] += n[i] > 0 ? there : 0.0f;
          }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool whole = CT == kE4m3 && sc.v[i] == INFINITY;
#pragma unroll
          for (int d = 0; d < E / B::W; ++d)
            if (differ >> i & 1) x.v[i][d] = whole ? 0u : finite_of<CT>(x.v[i][d]);
          if (whole && (differ >> i & 1)) sc.v[i] = 1.0f;
        }
      }
      // o += V' P', in fp16 or in bf16.
      auto sums = [&](auto half) {
        constexpr int WP = half ? 2 : 3, VP = kHalf && !half ? 2 : 1;  // parts of a weight, of a value
        u32x4 wp[WP];
        if constexpr (kHalf) weights();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a, b2, d2 = 0;
          if constexpr (half) split2_f16(w[2 * i] * kTimes, w[2 * i + 1] * kTimes, a, b2);
          else split2_towards0(w[2 * i] * kTimes, w[2 * i + 1] * kTimes, a, b2, d2);
          wp[0][i] = a, wp[1][i] = b2;
          if constexpr (WP == 3) wp[2][i] = d2;
        }
#pragma unroll
        for (int d2 = 0; d2 < E / 2; ++d2) {
          uint32_t v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = value(i, d2);
          u32x4 even[VP], odd[VP];  // the two features of the eight keys
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (VP == 2) {
              uint32_t e[2], f[2];
              split_f16(v[2 * i], v[2 * i + 1], e, f);
              even[0][i] = e[0], even[1][i] = e[1], odd[0][i] = f[0], odd[1][i] = f[1];
            } else {
              even[0][i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x05040100u);
              odd[0][i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x07060302u);
            }
          }
#pragma unroll
          for (int z = WP - 1; z >= 0; --z)
#pragma unroll
            for (int y = VP - 1; y >= 0; --y) {
              o[2 * d2] = product<half>(even[y], wp[z], o[2 * d2]);
              o[2 * d2 + 1] = product<half>(odd[y], wp[z], o[2 * d2 + 1]);
            }
          if constexpr (VP == 2) __builtin_amdgcn_sched_barrier(0);  // (or the parts of many features are held at once)
        }
        if constexpr (more) x.load_v(p, rows, waves[wave]);
      };
      if constexpr (kHalf) {
        float least = fmaf(low, c, -shift);  // the least weight's exponent
        if (__builtin_expect(!__any(least < -16.0f), 1)) sums(std::true_type{});
        // (Its own branch, its condition out of the compiler's sight: of an if and its else it
        // keeps two sets of sums.)
        asm volatile("" : "+v"(least));
        if (__builtin_expect(__any(least < -16.0f), 0)) sums(std::false_type{});
      } else {
        sums(std::false_type{});
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    if (!WHOLE) __syncthreads();  // (the sweep before's results are read)
    auto go_on = [&](int key0, int s1) {
      if (key0 >= s1) return;
      for (; key0 + kStep < s1; key0 += kStep) fold(key0, std::true_type{});
      fold(key0, std::false_type{});
    };
    if constexpr (EARLY || UNIFORM) {
      if (k_lo < k_hi) {
        if constexpr (!EARLY) begin(k_lo + kBlock * wave);
        lay_q();
        __syncthreads();
        go_on(k_lo + kBlock * wave, k_hi);
      }
    } else {
      lay_q();
      for (int s0 = k_lo, s1; s0 < k_hi; s0 = s1) {
        // As many whole steps as the entries that fit in LDS reach.
        keys.first = thd::quotient(s0, p.pages.by_page);
        s1 = (int)min((int64_t)k_hi, s0 + ((int64_t)(keys.first + kEntries) * p.pages.page - s0) / kStep * kStep);
        keys.last = min(last, s1 - 1);
        const int n = thd::quotient(s1 - 1, p.pages.by_page) - keys.first + 1;
        if (s0 > k_lo) __syncthreads();  // (what was there is read)
        for (int i = threadIdx.x; i < n; i += 64 * NW) entries[i] = keys.table[keys.first + i];
        __syncthreads();
        begin(s0 + kBlock * wave);
        go_on(s0 + kBlock * wave, s1);
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // Lane l holds row r's features CH (4 g + i + 16 c) + e in o[CH c + e][i].
    __syncthreads();  // (no wave reads q any more)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<f32x4*>(&Os[wave][r][B::CH * (4 * g + i + 16 * (e / B::CH)) + e % B::CH]) = f32x4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
    if (g == 0) Ms[wave][r] = m, Ls[wave][r] = l;
    __syncthreads();
    // The waves' parts in wave order: thread t takes row t / 16, features E (t % 16) + (0..E).
    const int orow = threadIdx.x / 16, col = E * (threadIdx.x % 16), all = kRows * tile + orow;
    if (threadIdx.x >= 256 || all >= count * p.group) {
      if (WHOLE) return;
      continue;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, Ms[w][orow]);
    const float shift = thd::lse_shift(mx);
    float sum = 0.0f;
    f32x4 acc[E / 4] = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = __builtin_amdgcn_exp2f(Ms[w][orow] - shift);
      sum += a * Ls[w][orow];
#pragma unroll
      for (int e = 0; e < E / 4; ++e) acc[e] += a / kTimes * *reinterpret_cast<const f32x4*>(&Os[w][orow][col + 4 * e]);
    }
    if (slot >= 0) {
      const int64_t to = (int64_t)slot * kRows + orow;
#pragma unroll
      for (int e = 0; e < E / 4; ++e) *reinterpret_cast<f32x4*>(p.part + to * D + col + 4 * e) = acc[e];
      if (col == 0) reinterpret_cast<f32x2*>(p.part_ml)[to] = f32x2{mx, sum};
      continue;
    }
    const int jo = thd::quotient(all, p.by_group), ho = hk * p.group + all - jo * p.group;
    const float inv = mx == -INFINITY ? 0.0f : 1.0f / sum;
    uint16_t* out = p.o + (int64_t)b * p.q_sb + (int64_t)ho * p.q_sh + (int64_t)jo * p.q_ss + col;
#pragma unroll
    for (int e = 0; e < E / 4; ++e)
      if (EXACT || col + 4 * e < p.head_dim)
        *reinterpret_cast<u32x2_any*>(out + 4 * e) =
            u32x2{rounded2<F16>(acc[e][0] * inv, acc[e][1] * inv), rounded2<F16>(acc[e][2] * inv, acc[e][3] * inv)};
    if (col == 0 && p.lse) p.lse[((int64_t)b * p.seq + jo) * p.heads + ho] = (mx + log2f(sum)) * kLn2;
    if (WHOLE) return;
  }
}

// The rows whose sweep lies in several pieces, or has no keys: a workgroup for 64
// features of a row, its threads in groups of 16, each of which takes every so
// manieth piece, four loads at a time; then the groups' results in order.  Bound by
// latency: 4.8 us for 512 rows of 128 in about six pieces, 5.0 for 16 rows of 256 in 72.
template <int D, bool F16>
__global__ __launch_bounds__(1024) void paged_attn_join(PagedArgs p) {
  constexpr int slices = D / 64;
  __shared__ float Ms[64], Ls[64];
  __shared__ f32x4 Os[1024];
  const int h = blockIdx.x / slices, pos = blockIdx.y, b = blockIdx.z;
  const int hk = thd::quotient(h, p.by_group), row = pos * p.group + h - hk * p.group, tile = row / kRows;
  const constant_i32 pieces = (constant_i32)p.pieces + 2 * ((int64_t)b * p.sweeps + hk * p.tiles + tile);
  const int at0 = pieces[0], n = pieces[1];
  const Sequence seq = sequence_of_all(p, b);
  if (pos >= seq.count) return;
  const int quad = threadIdx.x % 16, mine = threadIdx.x / 16, groups = blockDim.x / 16;
  const int f = 64 * (blockIdx.x % slices) + 4 * quad;
  float m = -INFINITY, l = 0.0f;
  f32x4 acc = {};
  if (seq.blocks > 0) {
    if (n == 0) return;  // stored already
    for (int i0 = mine; i0 < n; i0 += 4 * groups) {
      f32x2 x[4];
      f32x4 y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // a piece past the last reads the last again, with no weight
        const int piece = min(i0 + i * groups, n - 1);
        // The first in either of its workgroup's places, the others in their first.
        const int64_t from = (int64_t)(piece ? (at0 & ~1) + 2 * piece * p.sweeps : at0) * kRows + row % kRows;
        x[i] = reinterpret_cast<const f32x2*>(p.part_ml)[from];
        y[i] = *reinterpret_cast<const f32x4*>(p.part + from * D + f);
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < 4; ++i) mn = fmaxf(mn, x[i][0]);
      const float shift = thd::lse_shift(mn), alpha = __builtin_amdgcn_exp2f(m - shift);
      l *= alpha;
      acc *= alpha;
      m = mn;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i0 + i * groups < n) {
          const float a = __builtin_amdgcn_exp2f(x[i][0] - shift);
          l += a * x[i][1];
          acc += a * y[i];
        }
    }
    if (groups > 1) {
      if (quad == 0) Ms[mine] = m, Ls[mine] = l;
      Os[threadIdx.x] = acc;
      __syncthreads();
      if (mine > 0) return;
      float mn = -INFINITY;
      for (int i = 0; i < groups; ++i) mn = fmaxf(mn, Ms[i]);
      const float shift = thd::lse_shift(mn);
      l = 0.0f;
      acc = f32x4{};
      for (int i = 0; i < groups; ++i) {
        const float a = __builtin_amdgcn_exp2f(Ms[i] - shift);
        l += a * Ls[i];
        acc += a * Os[i * 16 + quad];
      }
      m = mn;
    }
  }
  if (mine > 0) return;
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
  if (f < p.head_dim)
    *reinterpret_cast<u32x2_any*>(p.o + b * p.q_sb + h * p.q_sh + pos * p.q_ss + f) =
        u32x2{rounded2<F16>(acc[0] * inv, acc[1] * inv), rounded2<F16>(acc[2] * inv, acc[3] * inv)};
  if (f == 0 && p.lse) p.lse[((int64_t)b * p.seq + pos) * p.heads + h] = (m + log2f(l)) * kLn2;
}

// Whether each sweep is one workgroup's, nothing joined: a launch and its waits less, but a
// step's bytes go through one CU (about 1.3 us for 256 keys of 256 bytes), and what is left over of a
// round of workgroups waits.  Both measured, whole and in pieces, 32/8 heads of 128 in bf16: one
// sequence and a table of 500 positions 8.8 and 9.0 us, of 1000 12.7 and 10.0; 24 sequences (192 sweeps, a CU
// each) of 850 13.7 and 18.1, of 1400 21.5 and 22.6; 64 sequences of 750 28.6 and 30.7, of
// 1000 38.7 and 34.9.  A position weighs 96 and 2 for each of the kernel's D features (e4m3 1.5), which
// brings the borders of 64, 128 and 256 features, and of head dims between, together.
// Few sweeps, 52 shapes (those features, bf16, fp16 and e4m3, pages of 5, 7, 16 and 24, one to twelve
// sequences, tables and windows of 500 to 1800 positions): whole takes 0.88 of the time of pieces at a
// weight of 190000, 0.95 at 230000, 1.06 at 270000, 1.11 at 310000.  Pages in sixteens or not make no difference;
// windows, whose sweeps are all as long, cross at 270000, tables filled to all degrees at 235000.
// A CU each (10 shapes), whole takes 0.87 at 460000, 1.01 at 560000; more sweeps (10), 0.88 at 230000, 1.01 at 290000.
template <int D>
bool whole_sweeps(const th_paged_desc* d) {
  int64_t keys = (int64_t)d->table_pages * d->cache.page;
  if (d->window > 0) keys = std::min<int64_t>(keys, (int64_t)d->window + d->seq + 2 * kBlock);
  const int64_t sweeps = ((int64_t)d->seq * (d->heads / d->cache.heads) + kRows - 1) / kRows * d->cache.heads * d->batch;
  const int64_t row = 96 + D * (d->cache.dtype == TH_E4M3 ? 3 : 4) / 2;
  const int64_t cus = th::ctx().prop.multiProcessorCount;
  return keys * row <= (8 * sweeps < 3 * cus ? 15 << 14 : sweeps <= cus ? 1 << 19 : 9 << 15);
}

template <int D, int CT, bool F16, bool EXACT, bool UNIFORM, bool SINGLE, bool WHOLE, bool EARLY>
int launch(const th_paged_desc* d, th_launch** out) {
  constexpr int NW = WHOLE ? 8 : 4;
  constexpr size_t sweep_lds = (CT == kE4m3 && F16 ? 2 : 1) * kRows * D * 2 + NW * sizeof(WaveLds<D>) +
                               (UNIFORM ? 0 : kEntries * sizeof(int32_t));
  constexpr size_t result_lds = NW * kRows * (D + 4 + 2) * sizeof(float);
  constexpr size_t lds = sweep_lds > result_lds ? sweep_lds : result_lds;
  const void* fn = (const void*)paged_attn_fwd<D, CT, F16, EXACT, UNIFORM, SINGLE, WHOLE, EARLY>;
  if (lds > 65536) TH_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const th_cache& cache = d->cache;
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(d->q), a.o = static_cast<uint16_t*>(d->o), a.lse = d->lse;
  a.k = static_cast<const char*>(cache.k), a.v = static_cast<const char*>(cache.v);
  a.ks = cache.k_scales, a.vs = cache.v_scales;
  a.pages = th::pages_of(cache, d->table_pages, d->table, d->lengths, d->counts);
  a.q_sh = d->q_strides[0], a.q_ss = d->q_strides[1], a.q_sb = d->q_strides[2];
  a.seq = d->seq, a.heads = d->heads, a.kv_heads = cache.heads, a.batch = d->batch, a.head_dim = cache.head_dim;
  a.causal = d->causal != 0;
  a.window = std::min(d->window, 1 << 30);  // (a table's most positions: a wider one would pass 32 bits below position 0)
  a.scale = d->scale > 0 ? d->scale : 1.0f / sqrtf((float)cache.head_dim);
  a.group = d->heads / cache.heads;
  a.tiles = (int)(((int64_t)d->seq * a.group + kRows - 1) / kRows);
  a.sweeps = a.tiles * cache.heads;
  const int64_t keys = (int64_t)d->table_pages * cache.page, sweeps = (int64_t)a.sweeps * d->batch;
  // As many workgroups as run at once (where that cuts the line in eight or more; otherwise four
  // times as many, so that the last round counts for little), or as there are steps if that is fewer.
  const int64_t resident = (int64_t)th::ctx().prop.multiProcessorCount * waves_of(D, CT, SINGLE, WHOLE);
  int64_t shares = resident / a.sweeps;
  if (shares < 8) shares = (4 * resident + a.sweeps - 1) / a.sweeps;
  if (shares >= 64) shares -= shares % 8;
  shares = std::min(shares, d->batch * ((keys + NW * kBlock - 1) / (NW * kBlock)));
  a.shares = (int)shares;
  const int workers = WHOLE ? (int)sweeps : (int)(shares * a.sweeps);
  a.by_group = th::divisor(a.group), a.by_tiles = th::divisor(a.tiles);
  a.by_sweeps = th::divisor(a.sweeps), a.by_shares = th::divisor(a.shares);
  th::Builder b("attention_paged", 10);
  const int k = b.kernel(fn, WHOLE ? "paged_attn_fwd_whole" : "paged_attn_fwd", dim3(workers), dim3(64 * NW), (uint32_t)lds, a);
  int end = k;
  if (!WHOLE) {
    // Threads for about as many pieces as a sweep has at the most.
    int threads = 256;
    while (threads < 1024 && threads / 16 * 4 < workers / sweeps) threads *= 2;
    end = b.kernel((const void*)paged_attn_join<D, F16>, "paged_attn_join", dim3(d->heads * (D / 64), d->seq, d->batch),
                   dim3(threads), 0, a);
    const uint64_t slots = a.shares > 1 ? 2 * (uint64_t)workers : 1;  // (one piece holds every sweep whole)
    const uint64_t at_o = b.workspace(slots * kRows * D * sizeof(float));
    const uint64_t at_ml = b.workspace(slots * kRows * 2 * sizeof(float));
    const uint64_t at_pieces = b.workspace((uint64_t)sweeps * 2 * sizeof(int32_t));
    for (int kk = k; kk <= end; ++kk) {
      b.ws_ref(kk, TH_OFFSET(PagedArgs, part), at_o);
      b.ws_ref(kk, TH_OFFSET(PagedArgs, part_ml), at_ml);
      b.ws_ref(kk, TH_OFFSET(PagedArgs, pieces), at_pieces);
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
  b.element(0, 2), b.element(1, 2);
  b.align(3, 16), b.align(4, 16);
  // All the cache there is room for: how much is held only the device knows.
  const double bytes = CT == kE4m3 ? 33.0 / 32 : 2, D0 = cache.head_dim, all = (double)d->batch * d->seq * d->heads;
  b.work(2.0 * d->batch * cache.heads * (double)keys * D0 * bytes + 4.0 * all * D0, 4.0 * all * (double)keys * D0, workers);
  *out = b.release();
  return TH_OK;
}

template <int D, bool EXACT, bool UNIFORM, bool SINGLE, bool WHOLE, bool EARLY>
int launch(const th_paged_desc* d, th_launch** out) {
  if (d->cache.dtype == TH_BF16) return launch<D, kBf16, false, EXACT, UNIFORM, SINGLE, WHOLE, EARLY>(d, out);
  if (d->cache.dtype == TH_F16) return launch<D, kF16, true, EXACT, UNIFORM, SINGLE, WHOLE, EARLY>(d, out);
  return d->dtype == TH_F16 ? launch<D, kE4m3, true, EXACT, UNIFORM, SINGLE, WHOLE, EARLY>(d, out)
                            : launch<D, kE4m3, false, EXACT, UNIFORM, SINGLE, WHOLE, EARLY>(d, out);
}
template <int D, bool EXACT, bool UNIFORM, bool SINGLE>
int launch(const th_paged_desc* d, th_launch** out) {
  // Whole sweeps of several positions of 256 features lack registers, the more with the
  // scalar addresses (12.5 us and 9.3 without, 2 x 64 positions of 8 heads in bf16).
  constexpr bool scalar = UNIFORM && (SINGLE || D < 256);
  if (!whole_sweeps<D>(d)) return launch<D, EXACT, UNIFORM, SINGLE, false, false>(d, out);
  if constexpr (!scalar)
    if (d->window == 0 && d->table_pages <= kEntries) return launch<D, EXACT, scalar, SINGLE, true, true>(d, out);
  return launch<D, EXACT, scalar, SINGLE, true, false>(d, out);
}
// Pages in sixteens (and rows of a half block within 31 bits) take the scalar addresses.
template <int D>
int launch_dim(const th_paged_desc* d, th_launch** out) {
  if (d->cache.head_dim != D) return launch<D, false, false, false>(d, out);
  const bool uniform = d->cache.page % 16 == 0 && d->cache.strides[1] < (1 << 26);
  if (d->seq > 1 || d->heads / d->cache.heads > kRows)
    return uniform ? launch<D, true, true, false>(d, out) : launch<D, true, false, false>(d, out);
  return uniform ? launch<D, true, true, true>(d, out) : launch<D, true, false, true>(d, out);
}

}  // namespace
