// Drafted tokens kept or refused by the target's probabilities and given random numbers, and the token that
// follows the last one kept (kvp_verify_drafts).
//
// With p = softmax(z / T) of a row of logits and q the draft's distribution, a draft x that was sampled from
// q is kept where u q(x) < p(x); behind a refused one the next token follows max(p - q, 0), and p behind a filler, which
// is no token and was not sampled.  A draft that was chosen (no q) is kept where u (1 - what its refused siblings have of
// p) < p(x); behind refused ones the next token follows p without them.  Either way a token of the output is
// distributed as p.
//
// In a few launches:
//   - maximum and sum of the rows of logits, in 32 bits, a segment of a row per workgroup.  Rows behind a refused draft
//     decide nothing: large batches take row 0 of every sequence first, then the rows that each can still get to.
//   - the way through the drafts, by a wave per sequence with a row per lane: siblings are ballots.
//   - the next token: the least index whose running sum of weights passes u times their sum.  A vocabulary's
//     borders lie down to 1e-9 of the sum apart, closer than 32-bit sums tell, so the weights of the one row that
//     a sequence ends at are added in 64 bits, range by range; the range with the border is taken again value by value.
//
// What bounds it: few rows, the latency of three launches and their chains of loads (a tree of 12 rows of 151936 bf16
// values: 17 us); many, HBM for the rows, then the vector ALUs for the last ones.  256 chains of 5 with a draft
// model's logits take 155 us: 34, 40 and 22 for the rows (500 of 760 MB, 5.2 TB/s), 38 for the last ones' sums, 6 for the
// tokens, and 5 or 6 for each of the three kernels between them.  With all rows read they took 223 us, with a
// workgroup per sequence that goes its way row by row 173: its longest ways were the end of the launch.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace kvp {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kRowThreads = 256;  // where rows are streamed
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kSumThreads = 256;  // where ranges are summed, each by a wave
constexpr int kSumWaves = kSumThreads / 64;
constexpr int kMaxRows = 64;  // rows of a sequence, as in kvp_tree_attention: one per lane
constexpr int kMaxSegments = 16;   // of a row: one per lane of a 16-lane row where they are joined
constexpr int kMaxRange = 512;     // chunks of a range, at most: one per thread where it is taken again
constexpr int kMostRanges = 512, kLeastRanges = 128;  // of a row, unless they would be longer or shorter than that
constexpr int kBatch = 2;          // chunks in flight per lane
constexpr int64_t kOnePass = 200 << 20;  // bytes of logits that are read in one pass, whether all of them are got to or not
constexpr int kMaxPasses = 8;
constexpr int kKnown = 64;              // sequences from which the last rows are found by a kernel of its own
constexpr float kReach = 16.f;     // binary orders that a value may lie above the reference
constexpr float kHuge = 3.4028234e38f;
// Weights relative to a row's largest: a single one below kTiny counts as 0.  Sums take them as 2^-1000 at least, so up to
// 2^30 hidden values add up to less than kNothing, and one of the 2^12 of a range that has more is no less than kTiny.
constexpr double kTiny = 0x1p-985, kNothing = 0x1p-969;
// Of p's weights: if less is left behind refused drafts, it is nothing.  It is as much as a weight may be off by, and a sequence
// gets to so little as rarely, but for decisions that 32-bit sums miss: what follows would be a token that p all but
// excludes (two siblings with all of p, the second with the last number below 1: one time in ten).
constexpr double kLeft = 0x1p-46;

// What a sequence has left to draw.
enum Mode : int32_t { kDone = 0, kAll = 1, kRest = 2, kWithout = 3, kUndefined = 4 };

struct Record {   // of a sequence
  int32_t row;    // of logits
  int32_t mode;
  int32_t count;  // drafts that stay
  float u;        // row 0's number
  double scale;   // log2(e) / T
  double top_p, top_q;  // the rows' maxima
  double lambda;  // sum of exp(p's logits) over that of q's, from 32-bit sums
  u64 gone;       // kWithout: the sequence's rows whose tokens are refused
};

struct Sums {  // of a range, relative to the maxima: of p's and q's weights, and of those where p's is larger
  // Larger by the ratio of 32-bit sums: of values that are closer to each other than it is off, p_over and q_over give the
  // difference with either sign, or nothing.  kWithout: p_over is p's without the refused tokens.
  double p, q, p_over, q_over;
};

struct VerifyParams {
  const void* logits;
  const void* draft;  // or null
  int64_t row_stride, draft_stride;  // elements
  int32_t vocab, total, num_seqs, max_rows;
  const int64_t* tokens;
  const float* uniforms;
  const float* temps;
  const int32_t* cu;
  const int64_t* masks;  // or null: a chain
  int32_t* accepted;
  int32_t* path;    // [num_seqs][max_rows]
  int64_t* out;     // [num_seqs][max_rows]
  int32_t segments; // of a row in the first pass
  int32_t range_chunks, ranges;
  float4* stats;    // [sequence][row][p, q][segment]: maximum and sum, or the greedy key
  uint4* drafts;    // [2][sequence][row]: what leave_drafts() finds
  u32* list;        // rows of a pass: sequence, row, p or q
  u32* counts;      // of them, by pass
  Record* records;
  Sums* sums;       // [sequence][range]
};

template <typename T>
struct Chunk;  // 16 bytes of logits
template <>
struct Chunk<uint16_t> {
  static constexpr int kSize = 8;
  static __device__ __forceinline__ float one(uint16_t x) { return __uint_as_float(static_cast<u32>(x) << 16); }
  static __device__ __forceinline__ void widen(uint4 w, float (&f)[8]) { unpack8(w, f); }
};
template <>
struct Chunk<float> {
  static constexpr int kSize = 4;
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ void widen(uint4 w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
  }
};

// A row of logits.  Values behind its end are -inf, weights of 0.
template <typename T>
struct Row {
  static constexpr int E = Chunk<T>::kSize;
  const T* at;
  int vocab, full;  // full chunks
  __device__ __forceinline__ Row(const T* base, int vocab) : at(base), vocab(vocab), full(vocab / E) {}
  __device__ __forceinline__ int chunks() const { return (vocab + E - 1) / E; }
  // A whole chunk; another one if c is none.
  __device__ __forceinline__ uint4 load(int c) const {
    return full > 0 ? *reinterpret_cast<const uint4*>(at + static_cast<int64_t>(E) * min(c, full - 1)) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ uint4 load_nt(int c) const {
    return full > 0 ? load16_nt(at + static_cast<int64_t>(E) * min(c, full - 1)) : make_uint4(0, 0, 0, 0);
  }
  // Chunk c, of which load() gave w.
  __device__ __forceinline__ void values(int c, uint4 w, float (&f)[E]) const {
    if (c < full) {
      Chunk<T>::widen(w, f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = E * c + e < vocab ? Chunk<T>::one(at[E * c + e]) : -INFINITY;
    }
  }
};

__device__ __forceinline__ float clamped(float m) { return fminf(fmaxf(m, -kHuge), kHuge); }

// log2(e) / T, 0 for a temperature that asks for the greedy token (0, negative, NaN).  Not below 1e-30: -inf
// stays a weight of 0 at any temperature.
__device__ __forceinline__ double scale_of(float temp) {
  return temp > 0.f ? fmax(1.4426950408889634 / static_cast<double>(temp), 1e-30) : 0.0;
}
__device__ __forceinline__ float scale32(double scale) { return fminf(static_cast<float>(scale), 3e38f); }

// 2^((x - top) scale) for x <= top, to 2e-13 of it and not below 2^-1000: t - k for the nearest integer k, which the
// addition of 1.5 * 2^52 leaves in the low bits, the Taylor series of 2^f over |f| <= 1/2, and k added to the
// exponent.  Twenty instructions at the full rate of 64-bit ones (those that round, convert to integers or scale
// are slower).
__device__ __forceinline__ double weight_floor(float x, double top, double scale) {
  const double t = fmax((static_cast<double>(x) - top) * scale, -1000.0);
  const double magic = 6755399441055744.0, r = t + magic, f = t - (r - magic);
  double y = 7.054911620801121e-9;  // ln(2)^n / n!
  y = fma(y, f, 1.0178086009239696e-7);
  y = fma(y, f, 1.3215486790144305e-6);
  y = fma(y, f, 1.5252733804059838e-5);
  y = fma(y, f, 1.5403530393381606e-4);
  y = fma(y, f, 1.3333558146428441e-3);
  y = fma(y, f, 9.618129107628477e-3);
  y = fma(y, f, 5.5504108664821576e-2);
  y = fma(y, f, 0.2402265069591007);
  y = fma(y, f, 0.6931471805599453);
  y = fma(y, f, 1.0);
  const u32 k = static_cast<u32>(__double_as_longlong(r));
  const long long bits = __double_as_longlong(y);
  return __longlong_as_double(static_cast<long long>(static_cast<u64>(static_cast<u32>(bits >> 32) + (k << 20)) << 32 |
                                                     static_cast<u32>(bits)));
}
// The same, and 0 below 2^-985.
__device__ __forceinline__ double weight(float x, double top, double scale) {
  const double w = weight_floor(x, top, scale);
  return w < kTiny ? 0.0 : w;
}

// Order of the greedy token: NaN above all, the lower index first among equals.
__device__ __forceinline__ u64 greedy_key(float x, u32 index) {
  const u32 b = __float_as_uint(x + 0.f);
  const u32 o = x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
  return static_cast<u64>(o) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ int64_t token_of(u64 key) { return 0xffffffffu - static_cast<u32>(key); }

// ---- across the lanes of a wave

// x of lane ^ S.
template <int S>
__device__ __forceinline__ u32 across(u32 x) {
  const int v = static_cast<int>(x), lane = threadIdx.x & 63;
  if constexpr (S == 1) return __builtin_amdgcn_update_dpp(0, v, kDppQuadXor1, 0xf, 0xf, false);
  if constexpr (S == 2) return __builtin_amdgcn_update_dpp(0, v, kDppQuadXor2, 0xf, 0xf, false);
  if constexpr (S == 4)  // of a half row in which the lanes of a quad are equal, as combine() leaves them
    return __builtin_amdgcn_update_dpp(0, v, kDppRowHalfMirror, 0xf, 0xf, false);
  if constexpr (S == 8)  // of a row in which half rows are
    return __builtin_amdgcn_update_dpp(0, v, kDppRowMirror, 0xf, 0xf, false);
  if constexpr (S == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return lane & 32 ? r[0] : r[1];
}
template <int S>
__device__ __forceinline__ float across(float x) {
  return __uint_as_float(across<S>(__float_as_uint(x)));
}
template <int S>
__device__ __forceinline__ u64 across(u64 x) {
  return static_cast<u64>(across<S>(static_cast<u32>(x >> 32))) << 32 | across<S>(static_cast<u32>(x));
}
template <int S>
__device__ __forceinline__ double across(double x) {
  return __longlong_as_double(static_cast<long long>(across<S>(static_cast<u64>(__double_as_longlong(x)))));
}
// x combined over LANES lanes (a power of two), the same in all of them; `op` is commutative.
template <int LANES, typename V, typename F>
__device__ __forceinline__ V combine(V x, F op) {
  x = op(x, across<1>(x));
  x = op(x, across<2>(x));
  x = op(x, across<4>(x));
  x = op(x, across<8>(x));
  if constexpr (LANES > 16) x = op(x, across<16>(x));
  if constexpr (LANES > 32) x = op(x, across<32>(x));
  return x;
}
template <int LANES = 64>
__device__ __forceinline__ float max_of(float x) {
  return combine<LANES>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int LANES = 64, typename V>
__device__ __forceinline__ V sum_of(V x) {
  return combine<LANES>(x, [](V a, V b) { return a + b; });
}
template <int LANES = 64>
__device__ __forceinline__ u64 best_of(u64 x) {
  return combine<LANES>(x, [](u64 a, u64 b) { return a > b ? a : b; });
}
// x moved CTRL (row_shr) lanes up in each row of 16, 0 where there is none.
template <int CTRL>
__device__ __forceinline__ double shifted(double x) {
  const u64 v = static_cast<u64>(__double_as_longlong(x));
  const u32 lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false);
  const u32 hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, 0xf, 0xf, false);
  return __longlong_as_double(static_cast<long long>(static_cast<u64>(hi) << 32 | lo));
}
// x of one lane, the same for all.
__device__ __forceinline__ float lane_of(float x, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(x)), lane));
}
__device__ __forceinline__ u64 lane_of(u64 x, int lane) {
  return static_cast<u64>(static_cast<u32>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane))) << 32 |
         static_cast<u32>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  return __longlong_as_double(static_cast<long long>(lane_of(static_cast<u64>(__double_as_longlong(x)), lane)));
}
// Sum of x over the lanes up to this one.
__device__ __forceinline__ double scan_f64(double x) {
  x += shifted<0x111>(x);
  x += shifted<0x112>(x);
  x += shifted<0x114>(x);
  x += shifted<0x118>(x);
  const double r0 = lane_of(x, 15), r1 = r0 + lane_of(x, 31), r2 = r1 + lane_of(x, 47);
  const int row = (threadIdx.x & 63) >> 4;
  return x + (row == 0 ? 0.0 : row == 1 ? r0 : row == 2 ? r1 : r2);
}

// ---------------------------------------------------------------- maximum and sum of a row

struct Part {  // of a row: maximum and sum of 2^((x - clamped(max)) scale); a NaN makes the sum NaN
  float max, sum;
};
__device__ __forceinline__ float rebased(const Part& part, float to, float scale) {
  return part.sum * fast_exp2((clamped(part.max) - to) * scale);
}

// a b, rounded: fused into a subtraction it would differ from itself by that rounding.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// The chunks from c0 on that the waves of a group of `waves` take, 64 at a time, up to cend; c0 is the wave's own first one.
template <typename T>
__device__ __forceinline__ Part part_of(const Row<T>& row, int c0, int waves, int cend, float scale) {
  constexpr int E = Chunk<T>::kSize;
  const int lane = threadIdx.x & 63, step = 64 * waves;
  const int whole = min(cend, row.full);
  // s is the sum of 2^(x scale - shift), one fma a value, or of 2^((x - ref) scale) where `far`: shift is
  // off by up to 2^-24 of itself, which a fma shows
  float m = -INFINITY, s = 0.f, ref = -kHuge, shift = 0.f;
  bool far = true;
  auto take = [&](auto count, const float* f) __attribute__((always_inline)) {
    constexpr int N = decltype(count)::value;
    float most = max3(f[0], f[1], f[2]);
#pragma unroll
    for (int e = 3; e < N; e += 2) most = max3(most, f[e], f[min(e + 1, N - 1)]);
    if (__any((far ? (most - ref) * scale : fmaf(most, scale, -shift)) > kReach)) {  // uniform
      const float to = clamped(max_of(most)), by = product(to, scale);
      const bool now = !(fabsf(by) < 0x1p20f);
      s *= fast_exp2(far || now ? (ref - to) * scale : shift - by);
      ref = to;
      shift = by;
      far = now;
    }
    m = max3(m, most, most);
    if (far) {
#pragma unroll
      for (int e = 0; e < N; ++e) s += fast_exp2((f[e] - ref) * scale);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) s += fast_exp2(fmaf(f[e], scale, -shift));
    }
  };
  uint4 in[kBatch];
  auto load_batch = [&](int c) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) in[u] = row.load_nt(c + u * step + lane);
  };
  load_batch(c0);
#pragma unroll 1
  for (; c0 + (kBatch - 1) * step + 64 <= whole; c0 += kBatch * step) {  // uniform
    float f[kBatch * E];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) Chunk<T>::widen(in[u], *reinterpret_cast<float(*)[E]>(f + u * E));
    load_batch(c0 + kBatch * step);
    take(std::integral_constant<int, kBatch * E>{}, f);
  }
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {  // what is left is in flight
    const int c = c0 + u * step + lane;
    if (c0 + u * step < cend) {  // uniform
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = -INFINITY;
      if (c < cend) row.values(c, in[u], f);
      take(std::integral_constant<int, E>{}, f);
    }
  }
  // divided by the weight that the largest value was added with: a sum that is this weight alone gives 1.  Times its
  // reciprocal's exponential it gave up to 2^-23 more, and a draft that has all of p could be refused.
  const float top = max_of(m), at = clamped(top);
  return {top, sum_of(s) / fast_exp2(far ? (at - ref) * scale : fmaf(at, scale, -shift))};
}

// The greedy key of the same chunks.
template <typename T>
__device__ __forceinline__ u64 key_of(const Row<T>& row, int c0, int waves, int cend) {
  constexpr int E = Chunk<T>::kSize;
  const int lane = threadIdx.x & 63, step = 64 * waves;
  u64 key = 0;
  float best = -INFINITY;  // of the lane
  bool any = false, nan = false;
  uint4 in[kBatch];
  auto load_batch = [&](int c) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) in[u] = row.load_nt(c + u * step + lane);
  };
  load_batch(c0);
#pragma unroll 1
  for (; c0 < cend; c0 += kBatch * step) {
    uint4 now[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) now[u] = in[u];
    load_batch(c0 + kBatch * step);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = c0 + u * step + lane;
      if (c >= cend) continue;
      float f[E];
      row.values(c, now[u], f);
      float most = f[0];
      bool odd = f[0] != f[0];
#pragma unroll
      for (int e = 1; e < E; ++e) {
        most = fmaxf(most, f[e]);
        odd |= f[e] != f[e];
      }
      if (nan || (any && !odd && !(most > best))) continue;  // a lane's first NaN is its last key
      any = true;
      nan = odd;
      best = most;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const u64 k = greedy_key(f[e], E * c + e);
        if (E * c + e < row.vocab && k > key) key = k;
      }
    }
  }
  return best_of(key);
}

// ---------------------------------------------------------------- the way through the drafts

// What a row's parts come to.
struct RowStats {
  float top;
  double sum;
  bool ok;  // the softmax exists: no NaN, no +inf, not -inf alone
  u64 key;  // greedy
};
__device__ __forceinline__ RowStats stats_of(float max, double sum) {
  return {clamped(max), sum, sum > 0 && sum < 1e300 && fabsf(max) <= kHuge, 0};
}

// A row of the sequence per lane.
struct Draft {
  int64_t token;
  int parent;  // -1: none
  u64 line;    // its ancestors and itself
  float u;
  float z, y;  // its logits in its parent's rows
  __device__ __forceinline__ bool inside(int vocab) const { return parent >= 0 && token >= 0 && token < vocab; }
};
// Parents and lines.
__device__ __forceinline__ Draft lines_of(const VerifyParams& p, int q0, int n) {
  const int i = threadIdx.x & 63;
  Draft d{-1, -1, 0, 0.f, 0.f, 0.f};
  if (i < n) {
    const u64 below = (1ull << i) - 1, sees = p.masks ? static_cast<u64>(p.masks[q0 + i]) & below : below;
    d.parent = sees ? 63 - __builtin_clzll(sees) : -1;
    d.line = p.masks ? (d.parent >= 0 ? 1ull << d.parent : 0) | 1ull << i : below | 1ull << i;
  }
  if (p.masks) {  // each round doubles how far back a line goes
    int back = d.parent;
#pragma unroll
    for (int round = 0; round < 6; ++round) {
      const u64 older = static_cast<u64>(__shfl(static_cast<u32>(d.line >> 32), max(back, 0))) << 32 |
                        __shfl(static_cast<u32>(d.line), max(back, 0));
      const int further = __shfl(back, max(back, 0));
      if (back >= 0) {
        d.line |= older;
        back = further;
      }
    }
  }
  return d;
}
// All of it, found once and left for the kernels behind, which then have no chain of loads to wait for.
template <typename T>
__device__ __forceinline__ void leave_drafts(const VerifyParams& p, int b, int q0, int n) {
  const int i = threadIdx.x & 63;
  const bool real = i < n;
  const int64_t token = real ? p.tokens[q0 + i] : -1;
  const float u = real ? p.uniforms[q0 + i] : 0.f;
  Draft d = lines_of(p, q0, n);
  d.token = token;
  if (d.inside(p.vocab)) {
    d.z = Chunk<T>::one(static_cast<const T*>(p.logits)[(q0 + d.parent) * p.row_stride + token]);
    if (p.draft) d.y = Chunk<T>::one(static_cast<const T*>(p.draft)[(q0 + d.parent) * p.draft_stride + token]);
  }
  if (!real) return;
  uint4* at = p.drafts + static_cast<int64_t>(b) * p.max_rows + i;
  at[0] = make_uint4(static_cast<u32>(token), static_cast<u32>(token >> 32), static_cast<u32>(d.line), static_cast<u32>(d.line >> 32));
  at[static_cast<int64_t>(p.num_seqs) * p.max_rows] =
      make_uint4(static_cast<u32>(d.parent), __float_as_uint(u), __float_as_uint(d.z), __float_as_uint(d.y));
}
__device__ __forceinline__ Draft left_drafts(const VerifyParams& p, int b, int n) {
  const int i = threadIdx.x & 63;
  const uint4* at = p.drafts + static_cast<int64_t>(b) * p.max_rows + min(i, p.max_rows - 1);
  const uint4 x = at[0], y = at[static_cast<int64_t>(p.num_seqs) * p.max_rows];
  if (i >= n) return {-1, -1, 0, 0.f, 0.f, 0.f};
  return {static_cast<int64_t>(static_cast<u64>(x.y) << 32 | x.x), static_cast<int>(y.x), static_cast<u64>(x.w) << 32 | x.z,
          __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w)};
}

// The child of a row that stays, or -1, by a whole wave; `children` are the row's.
__device__ __forceinline__ int child_that_stays(const VerifyParams& p, const Draft& d, u64 children, double scale,
                                                const RowStats& sp, const RowStats& sq) {
  if (children == 0) return -1;
  const bool in = d.inside(p.vocab);
  if (scale == 0) {
    const u64 same = __ballot(in && d.token == token_of(sp.key)) & children;
    return same ? __builtin_ctzll(same) : -1;
  }
  if (!sp.ok) return -1;
  const double px = in ? weight(d.z, sp.top, scale) / sp.sum : 0.0;
  if (p.draft) {
    if (!sq.ok) return -1;
    const double qx = in ? weight(d.y, sq.top, scale) / sq.sum : 0.0;
    const u64 passes = __ballot(in && d.u * qx < px) & children;
    return passes ? __builtin_ctzll(passes) : -1;
  }
  double left = 1;
  u64 refused = 0;
  for (u64 rest = children & __ballot(in); rest; rest &= rest - 1) {  // siblings in turn
    const int j = __builtin_ctzll(rest);
    const u64 twins = __ballot(d.token == static_cast<int64_t>(lane_of(static_cast<u64>(d.token), j)));
    if (twins & refused) continue;
    const double pj = lane_of(px, j);
    if (lane_of(d.u, j) * left < pj) return j;
    refused |= 1ull << j;
    left -= pj;
  }
  return -1;
}

__device__ __forceinline__ u64 children_of(const Draft& d, int node) { return __ballot(d.parent == node); }

struct Way {
  u64 kept;
  int node;
  bool ended;  // no child of node stays; otherwise it has not been asked
  RowStats sp, sq;
};

// Writes a sequence's results, by one wave, and gives what is left to draw.
__device__ __forceinline__ Record finish(const VerifyParams& p, int b, int q0, int n, const Draft& d, const Way& way,
                                         double scale, bool write) {
  const RowStats &sp = way.sp, &sq = way.sq;
  const u64 kept = way.kept;
  const int i = threadIdx.x & 63, count = __popcll(kept), node = way.node;
  const u64 gone = children_of(d, node), sampled = gone & __ballot(d.inside(p.vocab));  // what is no token was not sampled
  Record rec{q0 + node, kDone, count, lane_of(d.u, 0), scale, sp.top, sq.top, sp.sum / sq.sum, gone};
  if (n > 0 && scale != 0) {
    if (!sp.ok) rec.mode = kUndefined;
    else if (p.draft) rec.mode = sampled && sq.ok ? kRest : kAll;
    else rec.mode = gone ? kWithout : kAll;
  }
  if (write) {
    int32_t* path = p.path + static_cast<int64_t>(b) * p.max_rows;
    int64_t* out = p.out + static_cast<int64_t>(b) * p.max_rows;
    if (kept >> i & 1) {
      const int at = __popcll(kept & ((1ull << i) - 1));
      path[at] = i;
      out[at] = d.token;
    }
    if (i >= count && i < p.max_rows) {
      path[i] = -1;
      if (i > count || n == 0) out[i] = -1;
      else if (scale == 0) out[i] = token_of(sp.key);  // others: when it is drawn
    }
    if (i == 0) {
      p.accepted[b] = count;
      p.records[b] = rec;
    }
  }
  return rec;
}

// Rows of a sequence that is none are 0.
__device__ __forceinline__ int rows_of(const VerifyParams& p, int b, int& q0) {
  q0 = p.cu[b];
  const int end = p.cu[b + 1];
  return q0 < 0 || end <= q0 || end > p.total || end - q0 > p.max_rows ? 0 : end - q0;
}

// A row's parts: lanes 0 to 15 have p's segments, 16 to 31 q's.
__device__ __forceinline__ float4 parts_of(const VerifyParams& p, int b, int i) {
  const int lane = threadIdx.x & 63, seg = min(lane & 15, p.segments - 1);
  return p.stats[(((static_cast<int64_t>(b) * p.max_rows + i) << 1) + (p.draft ? lane >> 4 & 1 : 0)) * p.segments + seg];
}
// The way from row 0 by one wave, as far as row `depth` of it.  The statistics of the rows before that one are there; x and
// ahead are rows 0's and 1's parts, loaded together: a way that goes on mostly does so to row 1.
__device__ __forceinline__ Way way_to(const VerifyParams& p, int b, int n, const Draft& d, double scale, float4 x,
                                      float4 ahead, int depth) {
  Way way{0, 0, false, {0.f, 1, false, 0}, {0.f, 1, false, 0}};
  const int lane = threadIdx.x & 63;
  while (depth-- > 0) {
    const bool there = (lane & 15) < p.segments && (lane < 16 || (lane < 32 && p.draft && way.node < n - 1));
    if (scale == 0) {
      const u64 key = static_cast<u64>(__float_as_uint(x.y)) << 32 | __float_as_uint(x.x);
      way.sp.key = lane_of(best_of<16>(there ? key : 0), 0);
    } else {
      const Part part{there ? x.x : -INFINITY, there ? x.y : 0.f};
      const float top = max_of<16>(part.max);
      const double sum = sum_of<16>(static_cast<double>(rebased(part, clamped(top), scale32(scale))));
      way.sp = stats_of(lane_of(top, 0), lane_of(sum, 0));
      way.sq = stats_of(lane_of(top, 16), lane_of(sum, 16));
    }
    const int next = child_that_stays(p, d, children_of(d, way.node), scale, way.sp, way.sq);
    if (next < 0) {  // uniform
      way.ended = true;
      break;
    }
    way.kept |= 1ull << next;
    way.node = next;
    if (depth > 0) x = next == 1 ? ahead : parts_of(p, b, next);
  }
  return way;
}

// Maximum and sum (or greedy key) of a segment of a row, by a workgroup.
template <typename T>
__device__ __forceinline__ void row_segment(const VerifyParams& p, int b, int q0, int i, bool of_draft, int seg, double scale,
                                            Part* s_part, u64* s_key) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const Row<T> row(of_draft ? static_cast<const T*>(p.draft) + (q0 + i) * p.draft_stride
                            : static_cast<const T*>(p.logits) + (q0 + i) * p.row_stride, p.vocab);
  const int chunks = row.chunks(), per = (chunks + p.segments - 1) / p.segments;
  const int cbeg = min(seg * per, chunks), cend = min(cbeg + per, chunks);
  float4& out = p.stats[(((static_cast<int64_t>(b) * p.max_rows + i) << 1) + of_draft) * p.segments + seg];
  if (scale == 0) {  // uniform
    const u64 key = key_of(row, cbeg + 64 * wave, kRowWaves, cend);
    if (lane == 0) s_key[wave] = key;
    __syncthreads();
    if (wave != 0) return;
    const u64 best = best_of<16>(s_key[lane & (kRowWaves - 1)]);
    if (lane == 0)
      out = make_float4(__uint_as_float(static_cast<u32>(best)), __uint_as_float(static_cast<u32>(best >> 32)), 0.f, 0.f);
    return;
  }
  const Part part = part_of(row, cbeg + 64 * wave, kRowWaves, cend, scale32(scale));
  if (lane == 0) s_part[wave] = part;
  __syncthreads();
  if (wave != 0) return;
  const Part mine = s_part[lane & (kRowWaves - 1)];
  const float top = max_of<16>(mine.max);
  const float sum = sum_of<16>((lane & 15) < kRowWaves ? rebased(mine, clamped(top), scale32(scale)) : 0.f);
  if (lane == 0) out = make_float4(top, sum, 0.f, 0.f);
}

// The first rows of every sequence, as many as the grid has: a segment per workgroup.  One more workgroup for each
// sequence leaves what there is to know of its drafts, and clears the counters of the lists.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void row_stats_kernel(const VerifyParams p) {
  __shared__ Part s_part[kRowWaves];
  __shared__ u64 s_key[kRowWaves];
  const int b = blockIdx.z, item = blockIdx.y;
  const int i = p.draft ? item >> 1 : item;
  const bool of_draft = p.draft && (item & 1);
  int q0;
  const int n = rows_of(p, b, q0);
  if (item == static_cast<int>(gridDim.y) - 1) {
    if (blockIdx.x == 0 && threadIdx.x < 64) {
      leave_drafts<T>(p, b, q0, n);
      if (b == 0 && threadIdx.x < kMaxPasses) p.counts[threadIdx.x] = 0;
    }
    return;
  }
  if (i >= n - (of_draft ? 1 : 0)) return;
  const double scale = scale_of(p.temps[b]);
  if (of_draft && scale == 0) return;
  row_segment<T>(p, b, q0, i, of_draft, blockIdx.x, scale, s_part, s_key);
}

// Lists the rows `from` .. `to` - 1 steps from row 0 that the sequences can still get to, given those before them: a wave
// per sequence.
__global__ __launch_bounds__(64) void list_rows_kernel(const VerifyParams p, const int from, const int to, const int pass) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const float4 x = parts_of(p, b, 0), ahead = parts_of(p, b, min(1, p.max_rows - 1));
  int q0;
  const int n = rows_of(p, b, q0);
  const double scale = scale_of(p.temps[b]);
  const Draft d = left_drafts(p, b, n);
  if (n <= from) return;
  const Way way = way_to(p, b, n, d, scale, x, ahead, from);
  if (way.ended) return;  // uniform
  const int steps = __popcll(d.line) - 1;
  const u64 rows = __ballot((d.line >> way.node & 1) && (d.line & 1) && steps >= from && steps < to);
  const u64 rows_q = p.draft && scale != 0 ? rows & ~(1ull << (n - 1)) : 0;
  const int count = __popcll(rows), items = count + __popcll(rows_q);
  u32 at = 0;
  if (lane == 0) at = atomicAdd(&p.counts[pass], static_cast<u32>(items));  // their order changes no result
  at = __builtin_amdgcn_readfirstlane(at);
  const u64 below = (1ull << lane) - 1;
  const u32 item = static_cast<u32>(b) << 8 | static_cast<u32>(lane) << 1;
  if (rows >> lane & 1) p.list[at + __popcll(rows & below)] = item;
  if (rows_q >> lane & 1) p.list[at + count + __popcll(rows_q & below)] = item | 1;
}

// The listed rows: a unit is a segment of one, and workgroups take them in turn.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void listed_stats_kernel(const VerifyParams p, const int pass) {
  __shared__ Part s_part[2][kRowWaves];
  __shared__ u64 s_key[2][kRowWaves];
  const int units = static_cast<int>(p.counts[pass]) * p.segments;
  int turn = 0;
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x, turn ^= 1) {
    const int at = unit / p.segments, seg = unit - at * p.segments;
    const u32 item = p.list[at];
    const int b = static_cast<int>(item >> 8);
    row_segment<T>(p, b, p.cu[b], static_cast<int>(item >> 1 & 127), item & 1, seg, scale_of(p.temps[b]), s_part[turn],
                   s_key[turn]);
  }
}

// The whole way, by one wave.
__device__ __forceinline__ Record last_row(const VerifyParams& p, int b, bool write) {
  const float4 x = parts_of(p, b, 0), ahead = parts_of(p, b, min(1, p.max_rows - 1));
  int q0;
  const int n = rows_of(p, b, q0);
  const double scale = scale_of(p.temps[b]);
  const Draft d = left_drafts(p, b, n);
  const Way way = way_to(p, b, n, d, scale, x, ahead, n > 0 ? kMaxRows : 0);
  return finish(p, b, q0, n, d, way, scale, write);
}
__global__ __launch_bounds__(64) void last_row_kernel(const VerifyParams p) { last_row(p, blockIdx.x, true); }

// ---------------------------------------------------------------- sums of the last row

// The refused tokens of a sequence that lie among values [vbeg, vend), in LDS.
struct Refused {
  int count;
  int32_t token[kMaxRows];
};
__device__ __forceinline__ bool is_refused(const Refused& r, int v) {
  bool hit = false;
  for (int k = 0; k < r.count; ++k) hit |= r.token[k] == v;
  return hit;
}
// By a whole wave; a row of the sequence per lane.
__device__ __forceinline__ void find_refused(const VerifyParams& p, const Record& rec, int b, int vbeg, int vend, Refused& r) {
  const int lane = threadIdx.x & 63;
  const int64_t t = rec.gone >> lane & 1 ? p.tokens[p.cu[b] + lane] : -1;
  const bool in = t >= vbeg && t < vend;
  const u64 which = __ballot(in);
  if (in) r.token[__popcll(which & ((1ull << lane) - 1))] = static_cast<int32_t>(t);
  if (lane == 0) r.count = __popcll(which);
}

// x where `on`, otherwise a value below 2^-1022: its high word alone is cleared.
__device__ __forceinline__ double only(bool on, double x) {
  const u64 bits = static_cast<u64>(__double_as_longlong(x));
  const u32 hi = on ? static_cast<u32>(bits >> 32) : 0;
  return __longlong_as_double(static_cast<long long>(static_cast<u64>(hi) << 32 | static_cast<u32>(bits)));
}

// A range per wave.  KNOWN: last_row_kernel left the records; otherwise every wave goes the way anew.
//
// Where 64 chunks have no weight of 2^-28 of the largest or more, as most have in a row that is sure of its token, weights
// are taken in 32 bits and a chunk's 4 or 8 added there, before they go to the 64-bit sums.  The exponent t of 2^t is rounded
// three times, as a difference, in the scale and as their product, each time by 2^-24 of itself over its mantissa.  At -28,
// where the product's is 1.75, that is 2.2 * 2^-24 of t at most (1 + 1/1.75 + 1/1.75), or 42 * 2^-24 of the weight; with 2 for
// the exponential and 7 for the additions 51 * 2^-24, less than 2^-46 of the largest weight, and the less the smaller t.
// The signs differ: a row of 151936 is off by some 1e-12 of its sum, 2e-9 at worst.  256 chains with a draft model's logits:
// 38 us, 63 without.
template <typename T, bool KNOWN>
__global__ __launch_bounds__(kSumThreads) void range_sums_kernel(const VerifyParams p) {
  constexpr int E = Chunk<T>::kSize;
  __shared__ Refused s_refused[kSumWaves];
  const int b = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int range = blockIdx.x * kSumWaves + wave;
  if (range >= p.ranges) return;
  Record rec;
  if constexpr (KNOWN) rec = p.records[b];
  else rec = last_row(p, b, range == 0);
  if (rec.mode == kDone || rec.mode == kUndefined) return;
  const Row<T> row(static_cast<const T*>(p.logits) + rec.row * p.row_stride, p.vocab);
  const Row<T> row_q(rec.mode == kRest ? static_cast<const T*>(p.draft) + rec.row * p.draft_stride : row.at, p.vocab);
  const double top_p = rec.top_p, top_q = rec.top_q, scale = rec.scale;
  const float top_p32 = static_cast<float>(top_p), top_q32 = static_cast<float>(top_q), scale_f = scale32(scale);
  const float lambda32 = static_cast<float>(rec.lambda);
  const int cbeg = range * p.range_chunks, cend = min(cbeg + p.range_chunks, row.chunks());
  int c = cbeg + lane;
  uint4 in = row.load(c), in_q = row_q.load(c);
  auto small = [&](const float (&f)[E], float top) {  // of the wave's chunks
    float most = max3(f[0], f[1], f[2]);
#pragma unroll
    for (int e = 3; e < E; e += 2) most = max3(most, f[e], f[min(e + 1, E - 1)]);
    return !__any((most - top) * scale_f > -28.f);
  };
  Sums s{0, 0, 0, 0};
  if (rec.mode == kRest) {
    for (int c0 = cbeg; c0 < cend; c0 += 64, c += 64) {  // uniform
      float f[E], g[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = g[e] = -INFINITY;
      if (c < cend) {
        row.values(c, in, f);
        row_q.values(c, in_q, g);
      }
      in = row.load(c + 64);
      in_q = row_q.load(c + 64);
      if (small(f, top_p32) && small(g, top_q32)) {  // uniform
        float sp = 0.f, sq = 0.f, sp_over = 0.f, sq_over = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float x = fast_exp2((f[e] - top_p32) * scale_f), y = fast_exp2((g[e] - top_q32) * scale_f);
          const bool over = x > lambda32 * y;
          sp += x;
          sq += y;
          sp_over += over ? x : 0.f;
          sq_over += over ? y : 0.f;
        }
        s.p += sp;
        s.q += sq;
        s.p_over += sp_over;
        s.q_over += sq_over;
        continue;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double x = weight_floor(f[e], top_p, scale), y = weight_floor(g[e], top_q, scale);
        const bool over = x > rec.lambda * y;
        s.p += x;
        s.q += y;
        s.p_over += only(over, x);
        s.q_over += only(over, y);
      }
    }
    s.q = sum_of(s.q);
    s.q_over = sum_of(s.q_over);
  } else {
    Refused& refused = s_refused[wave];
    bool some = false;
    if (rec.mode == kWithout) {
      find_refused(p, rec, b, E * cbeg, E * cend, refused);
      wait_lds();
      some = refused.count != 0;
    }
    for (int c0 = cbeg; c0 < cend; c0 += 64, c += 64) {  // uniform
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = -INFINITY;
      if (c < cend) row.values(c, in, f);
      in = row.load(c + 64);
      if (some) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const double x = weight_floor(f[e], top_p, scale);
          s.p += x;
          s.p_over += is_refused(refused, E * c + e) ? 0.0 : x;
        }
      } else if (small(f, top_p32)) {  // uniform
        float sp = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) sp += fast_exp2((f[e] - top_p32) * scale_f);
        s.p += sp;
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) s.p += weight_floor(f[e], top_p, scale);
      }
    }
    if (!some) s.p_over = s.p;
  }
  s.p = sum_of(s.p);
  s.p_over = sum_of(s.p_over);
  if (lane == 0) p.sums[static_cast<int64_t>(b) * p.ranges + range] = s;
}

// ---------------------------------------------------------------- the next token

template <typename T>
__global__ __launch_bounds__(kThreads) void next_token_kernel(const VerifyParams p) {
  constexpr int E = Chunk<T>::kSize;
  __shared__ double s_lambda, s_left;
  __shared__ int s_range, s_mode;
  __shared__ double s_wave[kWaves];
  __shared__ u64 s_key[kWaves];
  __shared__ Refused s_refused;
  const int b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // the first wave's sums together with the record: a round trip less
  constexpr int kHeld = 2;  // all 128 that a row has in a batch of 32 sequences and more
  const Sums* sums = p.sums + static_cast<int64_t>(b) * p.ranges;
  Sums held[kHeld];
  if (wave == 0) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) held[k] = sums[min(lane + 64 * k, p.ranges - 1)];
  }
  const Record rec = p.records[b];
  if (rec.mode == kDone) return;
  int64_t* out = p.out + static_cast<int64_t>(b) * p.max_rows + rec.count;
  const Row<T> row(static_cast<const T*>(p.logits) + rec.row * p.row_stride, p.vocab);
  if (rec.mode == kUndefined) {  // the greedy token
    const u64 key = key_of(row, 64 * wave, kWaves, row.chunks());
    if (lane == 0) s_key[wave] = key;
    __syncthreads();
    const u64 best = best_of<16>(s_key[lane & (kWaves - 1)]);
    if (tid == 0) *out = token_of(best);
    return;
  }
  if (wave == 0) {
    Sums all{0, 0, 0, 0};
    auto add = [&](const Sums& x) {
      all = {all.p + x.p, all.q + x.q, all.p_over + x.p_over, all.q_over + x.q_over};
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (lane + 64 * k < p.ranges) add(held[k]);
    for (int r = lane + 64 * kHeld; r < p.ranges; r += 64) add(sums[r]);
    all = {sum_of(all.p), sum_of(all.q), sum_of(all.p_over), sum_of(all.q_over)};
    const double lambda = rec.mode == kRest ? all.p / all.q : 0.0;
    int mode = rec.mode;
    double whole = all.p_over - lambda * all.q_over;
    if (!(whole > kLeft * all.p)) {  // nothing is left: from p as it is
      mode = kAll;
      whole = all.p;
    }
    auto of_range = [&](const Sums& x) {
      const double w = mode == kAll ? x.p : x.p_over - lambda * x.q_over;
      return w > kNothing ? w : 0.0;
    };
    double border, before, left;
    int found, last;
    auto take = [&](int r0, const Sums& x) {
      const double mine = r0 + lane < p.ranges ? of_range(x) : 0.0;
      const double upto = before + scan_f64(mine);
      const u64 past = __ballot(mine > 0 && upto > border), some = __ballot(mine > 0);
      if (past) {
        const int at = __builtin_ctzll(past);
        found = r0 + at;
        left = border - lane_of(upto - mine, at);
      } else if (some) {
        last = r0 + 63 - __builtin_clzll(some);
      }
      before = lane_of(upto, 63);
    };
    for (;;) {  // uniform
      border = rec.u * whole;
      before = 0;
      found = last = -1;
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (found < 0 && 64 * k < p.ranges) take(64 * k, held[k]);
      for (int r0 = 64 * kHeld; r0 < p.ranges && found < 0; r0 += 64) take(r0, sums[min(r0 + lane, p.ranges - 1)]);
      if (found >= 0 || last >= 0 || mode == kAll) break;
      mode = kAll;  // the ranges have too little each
      whole = all.p;
    }
    if (lane == 0) {
      s_lambda = lambda;
      s_mode = mode;
      s_range = found < 0 ? max(last, 0) : found;
      s_left = found < 0 ? INFINITY : left;
    }
  }
  __syncthreads();
  const int mode = s_mode, range = s_range;
  const double lambda = s_lambda, left = s_left;
  const int cbeg = range * p.range_chunks, cend = min(cbeg + p.range_chunks, row.chunks());
  if (mode == kWithout) {
    if (wave == 0) find_refused(p, rec, b, E * cbeg, E * cend, s_refused);
    __syncthreads();
  }
  // the range again, a chunk per thread
  double w[E], mine = 0;
  const int c = cbeg + tid;
  u32 end = 0;  // behind the last value with a weight in p
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = 0;
  if (c < cend) {
    const double scale = rec.scale;
    float f[E];
    row.values(c, row.load(c), f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = weight(f[e], rec.top_p, scale);
      if (mode == kWithout && is_refused(s_refused, E * c + e)) w[e] = 0;
      if (w[e] > 0) end = E * c + e + 1;
    }
    if (mode == kRest) {
      const Row<T> row_q(static_cast<const T*>(p.draft) + rec.row * p.draft_stride, p.vocab);
      float g[E];
      row_q.values(c, row_q.load(c), g);
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = fmax(w[e] - lambda * weight(g[e], rec.top_q, scale), 0.0);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) mine += w[e];
  }
  const double upto = scan_f64(mine);
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  double before = 0;
  for (int k = 0; k < wave; ++k) before += s_wave[k];
  // the first value whose running sum is past the border, or the last that has a weight, or, where the range's sum
  // was a rounding of nothing, the last that has one in p: as keys
  double run = before + upto - mine;
  u64 key = end;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (!(w[e] > 0)) continue;
    run += w[e];
    const u32 v = E * c + e;
    const u64 k = run > left ? 2ull << 32 | (0xffffffffu - v) : 1ull << 32 | (v + 1);
    key = k > key ? k : key;
  }
  key = best_of(key);
  if (lane == 0) s_key[wave] = key;
  __syncthreads();
  const u64 best = best_of<16>(s_key[lane & (kWaves - 1)]);
  if (tid == 0) *out = best >> 33 ? token_of(best) : static_cast<int64_t>(static_cast<u32>(best)) - 1;
}

// ---------------------------------------------------------------- sizes

// Segments of a row: some 4096 workgroups for the rows of a pass, or their next power of two below.
int segments_of(int64_t rows) {
  int segments = 1;
  while (segments < kMaxSegments && 2 * segments * rows <= 4096) segments *= 2;
  return segments;
}
// Chunks of a range, whole 64s: a batch has no more than 4096 ranges, which fill the GPU once, unless rows would have fewer
// than kLeastRanges, and a row no more than kMostRanges.
int range_chunks_of(int64_t num_seqs, int64_t chunks) {
  const int64_t per_row = std::max<int64_t>(kLeastRanges, std::min<int64_t>(kMostRanges, 4096 / std::max<int64_t>(num_seqs, 1)));
  const int64_t per = (chunks + per_row - 1) / per_row;
  return static_cast<int>(std::min<int64_t>(kMaxRange, (per + 63) / 64 * 64));
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

struct Layout {
  int64_t stats, drafts, list, counts, records, sums, bytes;
};
Layout layout_of(int64_t num_seqs, int64_t max_rows, int64_t vocab) {
  Layout l{};
  // of every row one segment, or up to 16 in batches that have no more than 4096 of them
  const int64_t lists = std::max(num_seqs, std::min<int64_t>(num_seqs * kMaxSegments, 4096));
  l.drafts = round16(2 * max_rows * lists * sizeof(float4));
  l.list = l.drafts + round16(2 * num_seqs * max_rows * sizeof(uint4));
  l.counts = l.list + round16(2 * num_seqs * max_rows * sizeof(u32));
  l.records = l.counts + round16(kMaxPasses * sizeof(u32));
  l.sums = l.records + round16(num_seqs * sizeof(Record));
  // ranges of all rows, by the type with the most chunks; as range_chunks_of() has them, and growing with both arguments
  const int64_t chunks = (vocab + 3) / 4;
  const int64_t wanted = std::max(std::min<int64_t>(num_seqs * kMostRanges, 4096), num_seqs * kLeastRanges);
  const int64_t ranges = std::max(std::min(wanted, num_seqs * ((chunks + 63) / 64)), num_seqs * ((chunks + kMaxRange - 1) / kMaxRange));
  l.bytes = l.sums + ranges * sizeof(Sums);
  return l;
}

template <typename T>
int launch(const char* fn, VerifyParams p, hipStream_t s) {
  const LaunchOrder order;
  // All rows in one pass; or, in a large batch, row 0 first, then those 1 and 2 steps behind it that sequences get to,
  // then 3 to 6, .. and in the last pass the rest.  About half of what is left is expected to be got to each time; the
  // first cut pays earlier where drafts were chosen, of which fewer stay (8 trees of 60 rows, 139 MB: 35 us with one,
  // 45 without; 64 sampled chains of 5, 166 MB: 70 and 66), one more each 200 MB.
  const int per_row = p.draft ? 2 : 1;
  const int64_t rows = std::max<int64_t>(static_cast<int64_t>(p.total) * per_row, p.num_seqs);
  int64_t bytes = rows * p.vocab * static_cast<int64_t>(sizeof(T));
  const bool one = bytes < kOnePass / (p.draft ? 1 : 2) || p.max_rows == 1;
  p.segments = segments_of(one ? rows : p.num_seqs * per_row);
  hipLaunchKernelGGL(row_stats_kernel<T>, dim3(p.segments, (one ? p.max_rows : 1) * per_row + 1, p.num_seqs), dim3(kRowThreads),
                     0, s, p);
  for (int from = 1, to, pass = 0; !one && from < p.max_rows; from = to, ++pass) {
    bytes /= 2;
    to = bytes < kOnePass ? kMaxRows : 2 * from + 1;
    hipLaunchKernelGGL(list_rows_kernel, dim3(p.num_seqs), dim3(64), 0, s, p, from, to, pass);
    hipLaunchKernelGGL(listed_stats_kernel<T>, dim3(4096), dim3(kRowThreads), 0, s, p, pass);
  }
  const dim3 sums((p.ranges + kSumWaves - 1) / kSumWaves, p.num_seqs);
  if (p.num_seqs >= kKnown) {
    hipLaunchKernelGGL(last_row_kernel, dim3(p.num_seqs), dim3(64), 0, s, p);
    hipLaunchKernelGGL((range_sums_kernel<T, true>), sums, dim3(kSumThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((range_sums_kernel<T, false>), sums, dim3(kSumThreads), 0, s, p);
  }
  hipLaunchKernelGGL(next_token_kernel<T>, dim3(p.num_seqs), dim3(kThreads), 0, s, p);
  return launch_status(fn);
}

}  // namespace
}  // namespace kvp

using namespace kvp;

extern "C" size_t kvp_verify_workspace_bytes(int32_t max_num_seqs, int32_t max_seqlen_q, int32_t vocab) {
  if (max_num_seqs <= 0 || max_num_seqs > 65535 || max_seqlen_q <= 0 || max_seqlen_q > kMaxRows || vocab <= 0 ||
      vocab > 1 << 30)
    return 0;
  return static_cast<size_t>(layout_of(max_num_seqs, max_seqlen_q, vocab).bytes);
}

extern "C" int kvp_verify_drafts(const void* logits, int32_t logits_fp32, int64_t row_stride, int32_t total_q,
                                 int32_t vocab, const void* draft_logits, int64_t draft_row_stride,
                                 const int64_t* tokens, const float* uniforms, const float* temperatures,
                                 const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t max_seqlen_q,
                                 const int64_t* tree_mask, int32_t* accepted, int32_t* path, int64_t* out_tokens,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  static const char fn[] = "kvp_verify_drafts";
  clear_error();
  if (num_seqs < 0 || total_q < 0 || vocab < 1)
    return fail(KVP_EINVAL, "%s: num_seqs=%d total_q=%d vocab=%d", fn, num_seqs, total_q, vocab);
  if (num_seqs > 65535 || max_seqlen_q < 1 || max_seqlen_q > kMaxRows || vocab > 1 << 30)
    return fail(KVP_EUNSUPPORTED, "%s: num_seqs=%d max_seqlen_q=%d vocab=%d (supported: up to 65535, 1 to %d, up to 2^30)",
                fn, num_seqs, max_seqlen_q, vocab, kMaxRows);
  if (draft_logits && tree_mask)
    return fail(KVP_EUNSUPPORTED, "%s: draft_logits go with a chain, not with a tree_mask", fn);
  if (num_seqs == 0) return KVP_OK;
  if (!cu_seqlens_q || !accepted || !path || !out_tokens || !temperatures ||
      (total_q > 0 && (!logits || !tokens || !uniforms)))
    return fail(KVP_EINVAL, "%s: null pointer", fn);
  const int per16 = logits_fp32 ? 4 : 8;
  if (total_q > 0 && (!aligned16(logits) || row_stride % per16 || row_stride < vocab))
    return fail(KVP_EINVAL, "%s: logits must be 16-byte aligned with a row stride >= vocab that is a multiple of "
                "16 bytes", fn);
  if (draft_logits && (!aligned16(draft_logits) || draft_row_stride % per16 || draft_row_stride < vocab))
    return fail(KVP_EINVAL, "%s: draft_logits must be 16-byte aligned with a row stride >= vocab that is a multiple of "
                "16 bytes", fn);
  auto off = [](const void* ptr, unsigned by) { return (reinterpret_cast<uintptr_t>(ptr) & (by - 1)) != 0; };
  if (off(tokens, 8) || off(uniforms, 4) || off(temperatures, 4) || off(cu_seqlens_q, 4) || off(tree_mask, 8) ||
      off(accepted, 4) || off(path, 4) || off(out_tokens, 8))
    return fail(KVP_EINVAL, "%s: misaligned inputs or outputs", fn);
  const size_t need = kvp_verify_workspace_bytes(num_seqs, max_seqlen_q, vocab);
  if (!workspace || workspace_bytes < need)
    return fail(KVP_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, need);
  if (!aligned16(workspace)) return fail(KVP_EINVAL, "%s: workspace must be 16-byte aligned", fn);
  // the kernels that write a sequence's results still read these, or run beside others that do
  const int64_t seqs = num_seqs, value = logits_fp32 ? 4 : 2;
  const struct { const void* at; int64_t bytes; } results[] = {
      {accepted, 4 * seqs}, {path, 4 * seqs * max_seqlen_q}, {out_tokens, 8 * seqs * max_seqlen_q}};
  for (const auto& r : results) {
    bool shared = overlap(r.at, r.bytes, tokens, 8 * static_cast<int64_t>(total_q)) ||
                  overlap(r.at, r.bytes, temperatures, 4 * seqs) || overlap(r.at, r.bytes, cu_seqlens_q, 4 * (seqs + 1)) ||
                  (total_q > 0 && overlap(r.at, r.bytes, logits, total_q, value * row_stride, value * vocab)) ||
                  (draft_logits && overlap(r.at, r.bytes, draft_logits, total_q, value * draft_row_stride, value * vocab));
    for (const auto& x : results) shared = shared || (&x != &r && overlap(r.at, r.bytes, x.at, x.bytes));
    if (shared) return fail(KVP_EINVAL, "%s: the results must not share memory with the inputs or each other", fn);
  }
  const Layout at = layout_of(num_seqs, max_seqlen_q, vocab);
  char* ws = static_cast<char*>(workspace);
  VerifyParams p{};
  p.logits = logits;
  p.draft = draft_logits;
  p.row_stride = row_stride;
  p.draft_stride = draft_row_stride;
  p.vocab = vocab;
  p.total = total_q;
  p.num_seqs = num_seqs;
  p.max_rows = max_seqlen_q;
  p.tokens = tokens;
  p.uniforms = uniforms;
  p.temps = temperatures;
  p.cu = cu_seqlens_q;
  p.masks = tree_mask;
  p.accepted = accepted;
  p.path = path;
  p.out = out_tokens;
  const int chunks = (vocab + per16 - 1) / per16;
  p.range_chunks = range_chunks_of(num_seqs, chunks);
  p.ranges = (chunks + p.range_chunks - 1) / p.range_chunks;
  p.stats = reinterpret_cast<float4*>(ws + at.stats);
  p.drafts = reinterpret_cast<uint4*>(ws + at.drafts);
  p.list = reinterpret_cast<u32*>(ws + at.list);
  p.counts = reinterpret_cast<u32*>(ws + at.counts);
  p.records = reinterpret_cast<Record*>(ws + at.records);
  p.sums = reinterpret_cast<Sums*>(ws + at.sums);
  const auto s = static_cast<hipStream_t>(stream);
  return logits_fp32 ? launch<float>(fn, p, s) : launch<uint16_t>(fn, p, s);
}
