// Rotary positions on several axes: q and k turned pair by pair, fp32, bf16
// or fp16.  Memory-bound: every element is read once and written once (537 MB of
// bf16 in 101 us, 5.3 TB/s; single positions 3.2 us, the launch).
//
// A workgroup takes a few tokens with all their heads: its threads first form
// the tokens' cosines and sines (rotary_dim / 2 a token, shared by all heads)
// in LDS, then each turns V pairs at a time, 16 bytes of either half.
//
// The angle is position * frequency, in turns t = position * (freq / 2 pi) in
// fp64 (1 / 2 pi is off by 0.56 * 2^-53 of itself, two roundings: by at most 1.28 * 2^-52 t, 2^-20 of a turn at 2^31);
// t - rint(4 t) / 4, in [-1/8, 1/8], is exact and goes on in fp32, where
// Taylor's polynomials of sin and cos on [-pi/4, pi/4] leave out under 2^-28.
#include <hip/hip_runtime.h>

#include "th_core.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct RotaryArray {
  const void* x;
  void* y;
  int64_t xh, xs, xb, yh, ys, yb;
  int32_t heads;
};

struct RotaryArgs {
  RotaryArray a[2];  // q, k
  const int32_t* positions;
  const float* freqs;
  int64_t pa, ps, pb;  // the positions' strides along axes, positions, batch
  int32_t tokens;      // seq * batch
  int32_t seq, half;   // half: pairs a head
  int32_t ends[TH_ROTARY_AXES];  // pair p turns with the first axis whose end passes it
  int32_t turning, passing;      // items of a head: turned, copied
  int32_t pass_second;           // features from a copied item's first vector to its second (0: it has one)
  int32_t per_block;             // tokens a workgroup
  th::Divisor by_seq, by_half, by_token, by_head;  // (items of a token, of a head)
  float sign;
  // LEFT: items of a head that would be copied; heads of q and k.
  int32_t left;
  th::Divisor by_left, by_heads;
};

// Whether what passes has to be copied: an array's result lies elsewhere.
__host__ __device__ __forceinline__ bool moves(const RotaryArray& q, const RotaryArray& k) {
  return q.x != q.y || (k.heads && k.x != k.y);
}

// sin and cos of 2 pi t.
__device__ __forceinline__ float2 turned(double t) {
  const double n = rint(4.0 * t);
  const float x = 6.283185307179586f * (float)(t - 0.25 * n);
  const float y = x * x;
  float s = fmaf(y, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(y, s, 8.3333333e-3f);
  s = fmaf(y, s, -1.6666667e-1f);
  s = fmaf(x * y, s, x);
  float c = fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(y, c, -1.3888889e-3f);
  c = fmaf(y, c, 4.1666667e-2f);
  c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.0f);
  const int quarter = (int)(n - 4.0 * rint(0.25 * n)) & 3;
  const float u = quarter & 1 ? c : s, v = quarter & 1 ? s : c;
  return {quarter & 2 ? -u : u, (quarter + 1) & 2 ? -v : v};
}

template <int T>  // TH_F32, TH_BF16, TH_F16
struct Element {
  typedef uint16_t type;
};
template <>
struct Element<TH_F32> {
  typedef float type;
};

template <int T>
__device__ __forceinline__ float wide(typename Element<T>::type x) {
  if constexpr (T == TH_F32) return x;
  if constexpr (T == TH_BF16) return __uint_as_float((uint32_t)x << 16);
  if constexpr (T == TH_F16) return (float)__builtin_bit_cast(_Float16, x);
}
template <int T>
__device__ __forceinline__ typename Element<T>::type narrow(float x) {
  if constexpr (T == TH_F32) return x;
  if constexpr (T == TH_BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  if constexpr (T == TH_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// V elements at the elements' own alignment, a load or a store (non-temporal:
// 61 MB in 25 us, 29 with ordinary ones; non-temporal loads were slower where the arrays
// had been in cache, 9.4 us for 7.6).
template <class E, int V>
struct Vec {
  E x[V];
};
template <int BYTES, int ALIGN>
struct Words {
  typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGN)));
};
template <int ALIGN>
struct Words<2, ALIGN> {
  typedef uint16_t type;
};
template <int V, class E>
__device__ __forceinline__ Vec<E, V> load(const E* from) {
  typedef typename Words<V * sizeof(E), sizeof(E)>::type words;
  const words w = *reinterpret_cast<const words*>(from);
  return __builtin_bit_cast(Vec<E, V>, w);
}
template <int V, class E>
__device__ __forceinline__ void store(E* to, const Vec<E, V>& x) {
  typedef typename Words<V * sizeof(E), sizeof(E)>::type words;
  __builtin_nontemporal_store(__builtin_bit_cast(words, x), reinterpret_cast<words*>(to));
}

// LEFT: built with all arrays in place, so that what passes is not among the items; the
// arrays may since have been pointed elsewhere.  (In place the test is all it costs: 8 x 2048 positions of
// 16/16 heads, 64 of 128 features turned, 25 us; apart, built so, 54.5.)
template <int T, int V, bool PAIRS, bool LEFT>
__global__ __launch_bounds__(256) void rotary(RotaryArgs p) {
  typedef typename Element<T>::type E;
  typedef Vec<E, V> W;
  extern __shared__ float2 turns[];  // [token][pair]: sin, cos
  const int first = blockIdx.x * p.per_block, tokens = min(p.per_block, p.tokens - first);
  const int per_head = p.turning + p.passing;
  const int per_token = (p.a[0].heads + p.a[1].heads) * per_head, items = tokens * per_token;
  // An item's place: its token of the workgroup's, its features of x and y.
  struct Item {
    const E* x;
    E* y;
    int t, item, f0, f1;
  };
  const RotaryArray qa = p.a[0], ka = p.a[1];
  auto item_of = [&](int i) {
    Item it;
    it.t = thd::quotient(i, p.by_token);
    const int at = i - it.t * per_token;
    int head = thd::quotient(at, p.by_head);
    it.item = at - head * per_head;
    const bool second = head >= qa.heads;
    auto of = [&](auto q, auto k) { return second ? k : q; };  // (scalars both, not loads from where the index says)
    if (second) head -= qa.heads;
    const int token = first + it.t, b = thd::quotient(token, p.by_seq), s = token - b * p.seq;
    it.x = static_cast<const E*>(of(qa.x, ka.x)) + head * of(qa.xh, ka.xh) + s * of(qa.xs, ka.xs) + b * of(qa.xb, ka.xb);
    it.y = static_cast<E*>(of(qa.y, ka.y)) + head * of(qa.yh, ka.yh) + s * of(qa.ys, ka.ys) + b * of(qa.yb, ka.yb);
    const bool turns = it.item < p.turning;
    it.f0 = turns ? (PAIRS ? 2 * V * it.item : V * it.item) : 2 * p.half + (V + p.pass_second) * (it.item - p.turning);
    it.f1 = it.f0 + (turns ? (PAIRS ? V : p.half) : p.pass_second);
    return it;
  };
  // The first items are under way while the angles are formed.
  Item it;
  W u, v;
  const int step = 256 * gridDim.y, begin = 256 * blockIdx.y + threadIdx.x;
  if (begin < items) {
    it = item_of(begin);
    u = load<V>(it.x + it.f0), v = load<V>(it.x + it.f1);
  }
  for (int i = threadIdx.x; i < tokens * p.half; i += 256) {
    const int t = thd::quotient(i, p.by_half), pair = i - t * p.half;
    const int token = first + t, b = thd::quotient(token, p.by_seq), s = token - b * p.seq;
    int axis = 0;
#pragma unroll
    for (int a = 0; a < TH_ROTARY_AXES - 1; ++a) axis += pair >= p.ends[a];
    const int position = p.positions[axis * p.pa + (int64_t)s * p.ps + b * p.pb];
    turns[i] = turned((double)position * ((double)p.freqs[pair] * 0.15915494309189535));
  }
  __syncthreads();
  for (int i = begin; i < items;) {
    const int next = i + step;
    Item it2;
    W u2, v2;
    if (next < items) {
      it2 = item_of(next);
      u2 = load<V>(it2.x + it2.f0), v2 = load<V>(it2.x + it2.f1);
    }
    if (it.item < p.turning) {
      const float2* turn = turns + it.t * p.half + V * it.item;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // Pair j: in halves element j of either, adjacent ones elements 2j and 2j + 1 of both together.
        E& lo = PAIRS ? (2 * j < V ? u.x[2 * j] : v.x[2 * j - V]) : u.x[j];
        E& hi = PAIRS ? (2 * j + 1 < V ? u.x[2 * j + 1] : v.x[2 * j + 1 - V]) : v.x[j];
        const float sin = p.sign * turn[j].x, cos = turn[j].y;
        const float g = wide<T>(lo), h = wide<T>(hi);
        lo = narrow<T>(g * cos - h * sin);
        hi = narrow<T>(g * sin + h * cos);
      }
    }
    store(it.y + it.f0, u);
    store(it.y + it.f1, v);
    it = it2, u = u2, v = v2, i = next;
  }
  if (LEFT && moves(qa, ka)) {
    const int heads = qa.heads + ka.heads;
    for (int i = begin; i < tokens * heads * p.left; i += step) {
      const int row = thd::quotient(i, p.by_left), t = thd::quotient(row, p.by_heads), head = row - t * heads;
      const int token = first + t, b = thd::quotient(token, p.by_seq), s = token - b * p.seq;
      const bool second = head >= qa.heads;
      const RotaryArray& a = second ? ka : qa;
      const int h = second ? head - qa.heads : head, f = 2 * p.half + (V + p.pass_second) * (i - row * p.left);
      const E* from = static_cast<const E*>(a.x) + h * a.xh + s * a.xs + b * a.xb + f;
      E* to = static_cast<E*>(a.y) + h * a.yh + s * a.ys + b * a.yb + f;
      u = load<V>(from), v = load<V>(from + p.pass_second);
      store(to, u);
      store(to + p.pass_second, v);
    }
  }
}

template <int T, int V>
const void* kernel_of(bool pairs, bool left) {
  return pairs ? (left ? (const void*)rotary<T, V, true, true> : (const void*)rotary<T, V, true, false>)
               : (left ? (const void*)rotary<T, V, false, true> : (const void*)rotary<T, V, false, false>);
}
template <int T>
const void* kernel_of(int v, bool pairs, bool left) {
  if constexpr (T != TH_F32)
    if (v == 8) return kernel_of<T, 8>(pairs, left);
  return v == 4 ? kernel_of<T, 4>(pairs, left) : v == 2 ? kernel_of<T, 2>(pairs, left) : kernel_of<T, 1>(pairs, left);
}

int check_array(const void* x, void* y, const int64_t* xs, const int64_t* ys, const th_rotary_desc* d, int heads,
                int size) {
  TH_REQUIRE(x && y, "rotary: null q, k, q_out or k_out");
  TH_REQUIRE(reinterpret_cast<uintptr_t>(x) % size == 0 && reinterpret_cast<uintptr_t>(y) % size == 0,
             "rotary: arrays must be aligned to their elements");
  const int64_t extents[3] = {heads, d->seq, d->batch};
  for (int i = 0; i < 3; ++i) TH_REQUIRE(xs[i] >= 0 && ys[i] >= 0, "rotary: strides must not be negative");
  TH_REQUIRE(th::rows_apart(d->head_dim, ys, extents, 3), "rotary: the output's rows overlap");
  for (int i = 0; i < 3; ++i)
    TH_REQUIRE(x != y || extents[i] == 1 || xs[i] == ys[i], "rotary: an array turned in place keeps its strides");
  return TH_OK;
}

int build(const th_rotary_desc* d, th_launch** out) {
  TH_REQUIRE(d != nullptr, "rotary: null descriptor");
  if (d->dtype != TH_F32 && d->dtype != TH_BF16 && d->dtype != TH_F16)
    return th::fail(TH_E_UNSUPPORTED, "rotary: arrays must be fp32, bf16 or fp16");
  TH_REQUIRE(d->batch > 0 && d->seq > 0 && d->heads > 0 && d->kv_heads >= 0,
             "rotary: batch, seq and heads must be positive, kv_heads not negative");
  TH_REQUIRE(d->head_dim > 0 && d->head_dim <= 1024, "rotary: head_dim must be 1..1024");
  TH_REQUIRE(d->rotary_dim > 0 && d->rotary_dim % 2 == 0 && d->rotary_dim <= d->head_dim,
             "rotary: rotary_dim must be even, positive and at most head_dim");
  TH_REQUIRE(d->axes >= 1 && d->axes <= TH_ROTARY_AXES, "rotary: axes must be 1..4");
  TH_REQUIRE((d->flags & ~(TH_ROTARY_PAIRS | TH_ROTARY_INVERSE)) == 0, "rotary: unknown flags");
  TH_REQUIRE((int64_t)d->heads + d->kv_heads <= 65535, "rotary: heads and kv_heads must be at most 65535 together");
  TH_REQUIRE(d->positions && d->freqs, "rotary: null positions or freqs");
  TH_REQUIRE(th::aligned4(d->positions) && th::aligned4(d->freqs), "rotary: positions and freqs must be 4-byte aligned");
  const int half = d->rotary_dim / 2, size = d->dtype == TH_F32 ? 4 : 2;
  RotaryArgs a{};
  int sum = 0;
  for (int i = 0; i < TH_ROTARY_AXES; ++i) {
    if (i < d->axes) {
      TH_REQUIRE(d->sections[i] >= 0 && d->sections[i] <= half, "rotary: sections must hold rotary_dim / 2 pairs together");
      sum += d->sections[i];
    }
    a.ends[i] = i + 1 < d->axes ? sum : half;
  }
  TH_REQUIRE(sum == half, "rotary: sections must hold rotary_dim / 2 pairs together");
  for (int64_t s : d->position_strides) TH_REQUIRE(s >= 0, "rotary: strides must not be negative");
  if (int r = check_array(d->q, d->q_out, d->q_strides, d->q_out_strides, d, d->heads, size)) return r;
  if (d->kv_heads)
    if (int r = check_array(d->k, d->k_out, d->k_strides, d->k_out_strides, d, d->kv_heads, size)) return r;
  a.a[0] = {d->q, d->q_out, d->q_strides[0], d->q_strides[1], d->q_strides[2],
            d->q_out_strides[0], d->q_out_strides[1], d->q_out_strides[2], d->heads};
  a.a[1] = {d->k, d->k_out, d->k_strides[0], d->k_strides[1], d->k_strides[2],
            d->k_out_strides[0], d->k_out_strides[1], d->k_out_strides[2], d->kv_heads};
  a.positions = d->positions, a.freqs = d->freqs;
  a.pa = d->position_strides[0], a.ps = d->position_strides[1], a.pb = d->position_strides[2];
  const int64_t tokens = (int64_t)d->seq * d->batch;
  TH_REQUIRE(tokens <= (1 << 30), "rotary: batch * seq must be at most 2^30");
  a.tokens = (int32_t)tokens;
  a.seq = d->seq, a.half = half;
  a.sign = d->flags & TH_ROTARY_INVERSE ? -1.0f : 1.0f;
  // The widest vector (16 bytes at most) that divides a head's pairs and what passes.
  const int pass = d->head_dim - d->rotary_dim;
  int v = 16 / size;
  while (half % v || pass % v) v /= 2;
  const bool pairs = d->flags & TH_ROTARY_PAIRS;
  a.turning = half / v, a.pass_second = pass % (2 * v) == 0 ? v : 0;
  const int copied = pass / (v + a.pass_second);
  (moves(a.a[0], a.a[1]) ? a.passing : a.left) = copied;
  const int64_t per_token = (int64_t)(d->heads + d->kv_heads) * (a.turning + a.passing);
  TH_REQUIRE(per_token <= (1 << 24), "rotary: heads * head_dim is too large");
  // About four items a thread, at most 8 KB of angles.
  a.per_block = (int)std::max<int64_t>(1, std::min<int64_t>(1024 / per_token, 1024 / half));
  const int64_t blocks = (tokens + a.per_block - 1) / a.per_block;
  TH_REQUIRE(blocks <= 0xffffff, "rotary: batch * seq is too large");  // 2^32 threads
  if (int r = th::require_ready()) return r;
  a.by_seq = th::divisor(a.seq), a.by_half = th::divisor(a.half), a.by_token = th::divisor((int)per_token);
  a.by_head = th::divisor(a.turning + a.passing);
  a.by_left = th::divisor(std::max(a.left, 1)), a.by_heads = th::divisor(d->heads + d->kv_heads);
  const void* fn = d->dtype == TH_F32    ? kernel_of<TH_F32>(v, pairs, a.left > 0)
                   : d->dtype == TH_BF16 ? kernel_of<TH_BF16>(v, pairs, a.left > 0)
                                         : kernel_of<TH_F16>(v, pairs, a.left > 0);
  // Few tokens: their items to several workgroups each.
  const int64_t slices = blocks >= 512 ? 1 : std::min<int64_t>((a.per_block * per_token + 255) / 256, 512 / blocks);
  th::Builder b("rotary", 6);
  const int k = b.kernel(fn, "rotary", dim3((unsigned)blocks, (unsigned)slices), dim3(256), (uint32_t)(a.per_block * half * sizeof(float2)), a);
  const size_t offs[6] = {TH_OFFSET(RotaryArgs, a),
                          TH_OFFSET(RotaryArgs, a) + sizeof(RotaryArray),
                          TH_OFFSET(RotaryArgs, a) + TH_OFFSET(RotaryArray, y),
                          TH_OFFSET(RotaryArgs, a) + sizeof(RotaryArray) + TH_OFFSET(RotaryArray, y),
                          TH_OFFSET(RotaryArgs, positions),
                          TH_OFFSET(RotaryArgs, freqs)};
  for (int i = 0; i < 6; ++i) b.ref(i, k, offs[i]);
  for (int i = 0; i < 4; ++i) b.element(i, size);
  const double n = (double)a.tokens * (d->heads + d->kv_heads);
  b.work(2.0 * size * n * d->head_dim + 4.0 * a.tokens * d->axes, 6.0 * n * half, blocks);
  *out = b.release();
  return TH_OK;
}

}  // namespace

extern "C" int th_build_rotary(const th_rotary_desc* d, th_launch** out) {
  TH_REQUIRE(out != nullptr, "rotary: null result");
  *out = nullptr;
  return th::guarded([&] { return build(d, out); });
}
