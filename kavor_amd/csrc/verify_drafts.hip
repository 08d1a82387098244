// Drafted tokens kept or refused by the target's probabilities and given random numbers, and the token that
// follows the last one kept (kvp_verify_drafts).
//
// With p = softmax(z / T) of a row of logits and q the draft's distribution, a draft x that was sampled from
// q is kept where u q(x) < p(x); behind a refused one the next token follows max(p - q, 0).  A draft that was
// chosen (no q) is kept where u (1 - what its refused siblings have of p) < p(x); behind refused ones the next
// token follows p without them.  Either way a token of the output is distributed as p.
//
// What a row decides about its drafts is independent of what other rows decide, so all of it is computed at
// once, a row of a sequence per lane: a row is kept where it and all that its mask sees have won, which is
// one test of 64-bit words.
//
// The next token is the least index whose running sum of weights passes u times their sum.  A vocabulary's
// borders lie down to 1e-9 of the sum apart, closer than 32-bit sums tell, so the weights of the one row that
// a sequence ends at are computed and added in 64 bits, in ranges; the range that holds the border is taken
// again value by value.  All other rows need their maximum and sum in 32 bits only.
#include <math.h>

#include <algorithm>

#include "paged.h"

namespace kvp {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxRows = 64;  // rows of a sequence, as in kvp_tree_attention: one per lane
constexpr int kMaxSegments = 16;
constexpr int kRangeChunks = 512;  // chunks of a range, at most: one per thread where it is taken again
constexpr float kReach = 16.f;     // binary orders that a value may lie above the reference
constexpr float kHuge = 3.4028234e38f;

// What a sequence has left to draw.
enum Mode : int32_t { kDone = 0, kAll = 1, kRest = 2, kWithout = 3, kUndefined = 4 };

struct Record {   // of a sequence
  int32_t row;    // of logits
  int32_t mode;
  double scale;   // log2(e) / T
  double top_p, top_q;  // the rows' maxima
  double lambda;  // sum of exp(p's logits) over that of q's, in 32 bits
  u64 gone;       // kWithout: the sequence's rows whose tokens are refused
};

struct Sums {  // of a range, relative to the maxima: of p's and q's weights, and of those where p's is larger
  double p, q, p_over, q_over;  // kWithout: p_over is p's without the refused tokens
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
  float4* stats;    // [sequence][row][p, q][segment]: maximum, sum, index of the maximum
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

// A row's chunk c; values behind the row's end are -inf, weights of 0.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int c, int vocab, float (&f)[Chunk<T>::kSize]) {
  constexpr int E = Chunk<T>::kSize;
  if (E * (c + 1) <= vocab) {
    Chunk<T>::widen(*reinterpret_cast<const uint4*>(row + static_cast<int64_t>(E) * c), f);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = E * c + e < vocab ? Chunk<T>::one(row[E * c + e]) : -INFINITY;
  }
}

__device__ __forceinline__ float clamped(float m) { return fminf(fmaxf(m, -kHuge), kHuge); }

// log2(e) / T, 0 for a temperature that asks for the greedy token (0, negative, NaN).  Not below 1e-30: -inf
// stays a weight of 0 at any temperature.
__device__ __forceinline__ double scale_of(float temp) {
  return temp > 0.f ? fmax(1.4426950408889634 / static_cast<double>(temp), 1e-30) : 0.0;
}

// 2^t for t <= 0, to 1e-14 of it: the Taylor series of e^x over |x| <= ln(2) / 2, its exponent added.  0 below 2^-1000.
__device__ __forceinline__ double exp2_64(double t) {
  const double k = rint(t), x = (t - k) * 0.6931471805599453;
  double y = 1.0 / 39916800;
  y = fma(y, x, 1.0 / 3628800);
  y = fma(y, x, 1.0 / 362880);
  y = fma(y, x, 1.0 / 40320);
  y = fma(y, x, 1.0 / 5040);
  y = fma(y, x, 1.0 / 720);
  y = fma(y, x, 1.0 / 120);
  y = fma(y, x, 1.0 / 24);
  y = fma(y, x, 1.0 / 6);
  y = fma(y, x, 0.5);
  y = fma(y, x, 1.0);
  y = fma(y, x, 1.0);
  const int shift = static_cast<int>(fmax(k, -1001.0));
  const double r = __longlong_as_double(__double_as_longlong(y) + (static_cast<long long>(shift) << 52));
  return k < -1000.0 ? 0.0 : r;
}
__device__ __forceinline__ double weight(float x, double top, double scale) {
  return exp2_64((static_cast<double>(x) - top) * scale);
}

// Order of the greedy token: NaN above all, the lower index first among equals.
__device__ __forceinline__ u64 greedy_key(float x, u32 index) {
  const u32 b = __float_as_uint(x + 0.f);
  const u32 o = x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
  return static_cast<u64>(o) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ u64 shfl_key(u64 k, int from) {
  return static_cast<u64>(__shfl(static_cast<u32>(k >> 32), from)) << 32 | __shfl(static_cast<u32>(k), from);
}
__device__ __forceinline__ u64 wave_max_key(u64 k) {
#pragma unroll
  for (int s = 32; s; s >>= 1) {
    const u64 o = shfl_key(k, (threadIdx.x & 63) ^ s);
    k = o > k ? o : k;
  }
  return k;
}
__device__ __forceinline__ double shfl_f64(double x, int from) {
  return __longlong_as_double(static_cast<long long>(shfl_key(static_cast<u64>(__double_as_longlong(x)), from)));
}
// x of one lane, the same for all.
__device__ __forceinline__ double lane_f64(double x, int lane) {
  const long long v = __double_as_longlong(x);
  const u32 lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return __longlong_as_double(static_cast<long long>(static_cast<u64>(hi) << 32 | lo));
}
__device__ __forceinline__ double wave_sum_f64(double x) {
#pragma unroll
  for (int s = 32; s; s >>= 1) x += shfl_f64(x, (threadIdx.x & 63) ^ s);
  return x;
}
// Sum of x over the lanes up to this one.
__device__ __forceinline__ double wave_scan_f64(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const double o = shfl_f64(x, max(lane - s, 0));
    x += lane >= s ? o : 0.0;
  }
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int s = 32; s; s >>= 1) x = fmaxf(x, __shfl_xor(x, s));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int s = 32; s; s >>= 1) x += __shfl_xor(x, s);
  return x;
}

// ---------------------------------------------------------------- maximum and sum of every row

// A segment of a row per workgroup: maximum m and sum of 2^((x - m) scale), or the greedy key.
template <typename T>
__global__ __launch_bounds__(kThreads) void row_stats_kernel(const VerifyParams p) {
  constexpr int E = Chunk<T>::kSize;
  __shared__ float s_max[kWaves], s_sum[kWaves];
  __shared__ u64 s_key[kWaves];
  const int seg = static_cast<int>(blockIdx.x), i = blockIdx.y >> (p.draft ? 1 : 0), b = blockIdx.z;
  const bool of_draft = p.draft && (blockIdx.y & 1);
  const int q0 = p.cu[b], n = p.cu[b + 1] - q0;
  if (n > p.max_rows || q0 < 0 || q0 + n > p.total || i >= n - (of_draft ? 1 : 0)) return;
  const float temp = p.temps[b];
  const double scale64 = scale_of(temp);
  if (of_draft && scale64 == 0) return;
  const T* row = of_draft ? static_cast<const T*>(p.draft) + (q0 + i) * p.draft_stride
                          : static_cast<const T*>(p.logits) + (q0 + i) * p.row_stride;
  const int chunks = (p.vocab + E - 1) / E, per = (chunks + p.segments - 1) / p.segments;
  const int cbeg = min(seg * per, chunks), cend = min(cbeg + per, chunks);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = -INFINITY, s = 0.f;
  u64 key = 0;
  if (scale64 == 0) {
    for (int c = cbeg + threadIdx.x; c < cend; c += kThreads) {
      float f[E];
      load_chunk(row, c, p.vocab, f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const u64 k = greedy_key(f[e], E * c + e);
        if (E * c + e < p.vocab && k > key) key = k;
      }
    }
    key = wave_max_key(key);
    if (lane == 0) s_key[wave] = key;
  } else {
    const float scale = fminf(static_cast<float>(scale64), 3e38f);
    float ref = -kHuge;
    for (int c0 = cbeg + (wave << 6); c0 < cend; c0 += kThreads) {  // uniform in a wave
      const int c = c0 + lane;
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = -INFINITY;
      if (c < cend) load_chunk(row, c, p.vocab, f);
      float most = f[0];
#pragma unroll
      for (int e = 1; e < E; ++e) most = fmaxf(most, f[e]);
      if (__any((most - ref) * scale > kReach)) {
        const float to = clamped(wave_max(most));
        s *= fast_exp2((ref - to) * scale);
        ref = to;
      }
      m = fmaxf(m, most);
#pragma unroll
      for (int e = 0; e < E; ++e) s += fast_exp2((f[e] - ref) * scale);
    }
    m = wave_max(m);
    s = wave_sum(s) * fast_exp2((ref - clamped(m)) * scale);
    if (lane == 0) {
      s_max[wave] = m;
      s_sum[wave] = s;
    }
  }
  __syncthreads();
  if (threadIdx.x) return;
  float4& out = p.stats[(((static_cast<int64_t>(b) * p.max_rows + i) << 1) + of_draft) * p.segments + seg];
  if (scale64 == 0) {
    for (int w = 1; w < kWaves; ++w) key = s_key[w] > key ? s_key[w] : key;
    out = make_float4(__uint_as_float(static_cast<u32>(key)), __uint_as_float(static_cast<u32>(key >> 32)), 0.f, 0.f);
    return;
  }
  const float scale = fminf(static_cast<float>(scale64), 3e38f);
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_max[w]);
  float sum = 0.f;
  for (int w = 0; w < kWaves; ++w) sum += s_sum[w] * fast_exp2((clamped(s_max[w]) - clamped(m)) * scale);
  out = make_float4(m, sum, 0.f, 0.f);
}

struct RowStats {
  double top, sum;
  bool ok;  // the softmax exists: no NaN, no +inf, not -inf alone
};
__device__ __forceinline__ RowStats join(const float4* seg, int segments, double scale) {
  float m = -INFINITY;
  for (int k = 0; k < segments; ++k) m = fmaxf(m, seg[k].x);
  const float top = clamped(m), sc = fminf(static_cast<float>(scale), 3e38f);
  double s = 0;
  for (int k = 0; k < segments; ++k) s += static_cast<double>(seg[k].y) * fast_exp2((clamped(seg[k].x) - top) * sc);
  return {top, s, s > 0 && s < 1e300 && fabsf(m) <= kHuge};
}

// ---------------------------------------------------------------- drafts kept

// A wave per sequence, a row per lane.
template <typename T>
__global__ __launch_bounds__(64) void keep_kernel(const VerifyParams p) {
  const int b = blockIdx.x, i = threadIdx.x;
  const int q0 = p.cu[b], n = p.cu[b + 1] - q0;
  int32_t* path = p.path + static_cast<int64_t>(b) * p.max_rows;
  int64_t* out = p.out + static_cast<int64_t>(b) * p.max_rows;
  Record& rec = p.records[b];
  if (n <= 0 || n > p.max_rows || q0 < 0 || q0 + n > p.total) {
    if (i < p.max_rows) {
      path[i] = -1;
      out[i] = -1;
    }
    if (i == 0) {
      p.accepted[b] = 0;
      rec.mode = kDone;
    }
    return;
  }
  const bool real = i < n;
  const double scale = scale_of(p.temps[b]);
  const int64_t token = real ? p.tokens[q0 + i] : -1;
  const double u = real ? p.uniforms[q0 + i] : 0.0;
  const u64 below = (1ull << i) - 1;
  const u64 sees = real ? (p.masks ? static_cast<u64>(p.masks[q0 + i]) & below : below) : 0;
  const int parent = sees ? 63 - __builtin_clzll(sees) : -1;
  // the row's own statistics, then those of the parent
  const float4* stats = p.stats + ((static_cast<int64_t>(b) * p.max_rows + min(i, n - 1)) << 1) * p.segments;
  bool test = false, fresh = true;
  RowStats mine{0, 0, false}, mine_q{0, 0, false};
  u64 best = 0, siblings = 0;
  double px = 0;
  const int up = max(parent, 0);
  const bool inside = token >= 0 && token < p.vocab && parent >= 0;
  if (scale == 0) {
    for (int k = 0; k < p.segments; ++k) {
      const u64 key = static_cast<u64>(__float_as_uint(stats[k].y)) << 32 | __float_as_uint(stats[k].x);
      best = key > best ? key : best;
    }
    const u32 first = 0xffffffffu - __shfl(static_cast<u32>(best), up);
    test = inside && token == first;
  } else {
    mine = join(stats, p.segments, scale);
    if (p.draft && i < n - 1) mine_q = join(stats + p.segments, p.segments, scale);
    const double top = shfl_f64(mine.top, up), sum = shfl_f64(mine.sum, up);
    const bool ok = __shfl(static_cast<int>(mine.ok), up);
    if (inside) px = weight(Chunk<T>::one(static_cast<const T*>(p.logits)[(q0 + up) * p.row_stride + token]), top, scale) / sum;
    if (p.draft) {
      const double top_q = shfl_f64(mine_q.top, up), sum_q = shfl_f64(mine_q.sum, up);
      const bool ok_q = __shfl(static_cast<int>(mine_q.ok), up);
      double qx = 0;
      if (inside) qx = weight(Chunk<T>::one(static_cast<const T*>(p.draft)[(q0 + up) * p.draft_stride + token]), top_q, scale) / sum_q;
      test = inside && ok && ok_q && u * qx < px;
    } else {
      test = inside && ok;
    }
  }
  if (p.masks) {  // siblings in turn
    double left = 1;
    const int token_lo = static_cast<int>(token), token_hi = static_cast<int>(token >> 32);
    for (int j = 1; j < n; ++j) {
      const int parent_j = __builtin_amdgcn_readlane(parent, j);
      const bool twin = __builtin_amdgcn_readlane(token_lo, j) == token_lo &&
                        __builtin_amdgcn_readlane(token_hi, j) == token_hi;
      const bool fresh_j = __builtin_amdgcn_readlane(static_cast<int>(fresh), j);
      const double pj = lane_f64(px, j);
      if (j < i && parent >= 0 && parent_j == parent) {
        siblings |= 1ull << j;
        if (twin) fresh = false;
        else if (fresh_j) left -= pj;
      }
    }
    if (scale != 0 && !p.draft) test = test && fresh && u * left < px;
  } else if (scale != 0 && !p.draft) {
    test = test && u < px;
  }
  const u64 tests = __ballot(test);
  const u64 wins = __ballot(test && (tests & siblings) == 0);
  const bool kept = (wins >> i & 1) && (sees & ~1ull & ~wins) == 0;
  const u64 keeps = __ballot(kept);
  const int count = __popcll(keeps), end = keeps ? 63 - __builtin_clzll(keeps) : 0;
  const u64 gone = __ballot(real && parent == end);
  if (kept) {
    const int at = __popcll(keeps & below);
    path[at] = i;
    out[at] = token;
  }
  if (i >= count && i < p.max_rows) path[i] = -1;
  if (i > count && i < p.max_rows) out[i] = -1;
  if (i == 0) p.accepted[b] = count;
  if (i != end) return;
  rec.row = q0 + end;
  rec.scale = scale;
  rec.top_p = mine.top;
  rec.top_q = mine_q.top;
  rec.lambda = mine.sum / mine_q.sum;
  rec.gone = gone;
  if (scale == 0) {
    out[count] = 0xffffffffu - static_cast<u32>(best);
    rec.mode = kDone;
  } else if (!mine.ok) {
    rec.mode = kUndefined;
  } else if (p.draft) {
    rec.mode = gone && mine_q.ok ? kRest : kAll;
  } else {
    rec.mode = gone ? kWithout : kAll;
  }
}

// ---------------------------------------------------------------- sums of the last row

// The refused tokens of a sequence that lie in chunks [cbeg, cend), up to 64 of them, in LDS.
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
__device__ __forceinline__ void find_refused(const VerifyParams& p, const Record& rec, int q0, int vbeg, int vend, Refused& r) {
  const int lane = threadIdx.x & 63;
  const int64_t t = rec.gone >> lane & 1 ? p.tokens[q0 + lane] : -1;
  const bool in = t >= vbeg && t < vend;
  const u64 which = __ballot(in);
  if (in) r.token[__popcll(which & ((1ull << lane) - 1))] = static_cast<int32_t>(t);
  if (lane == 0) r.count = __popcll(which);
}

// A range per wave.
template <typename T>
__global__ __launch_bounds__(kThreads) void range_sums_kernel(const VerifyParams p) {
  constexpr int E = Chunk<T>::kSize;
  __shared__ Refused s_refused[kWaves];
  const int b = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int range = blockIdx.x * kWaves + wave;
  const Record rec = p.records[b];
  if (rec.mode == kDone || rec.mode == kUndefined || range >= p.ranges) return;
  const int chunks = (p.vocab + E - 1) / E;
  const int cbeg = range * p.range_chunks, cend = min(cbeg + p.range_chunks, chunks);
  Refused& refused = s_refused[wave];
  if (rec.mode == kWithout) {
    find_refused(p, rec, p.cu[b], E * cbeg, E * cend, refused);
    wait_lds();
  }
  const T* row = static_cast<const T*>(p.logits) + rec.row * p.row_stride;
  const T* row_q = rec.mode == kRest ? static_cast<const T*>(p.draft) + rec.row * p.draft_stride : row;
  Sums s{0, 0, 0, 0};
  for (int c = cbeg + lane; c < cend; c += 64) {
    float f[E];
    load_chunk(row, c, p.vocab, f);
    if (rec.mode == kRest) {
      float g[E];
      load_chunk(row_q, c, p.vocab, g);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double x = weight(f[e], rec.top_p, rec.scale), y = weight(g[e], rec.top_q, rec.scale);
        const bool over = x > rec.lambda * y;
        s.p += x;
        s.q += y;
        s.p_over += over ? x : 0.0;
        s.q_over += over ? y : 0.0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double x = weight(f[e], rec.top_p, rec.scale);
        s.p += x;
        if (rec.mode == kWithout && refused.count) s.p_over += is_refused(refused, E * c + e) ? 0.0 : x;
        else s.p_over += x;
      }
    }
  }
  s.p = wave_sum_f64(s.p);
  s.q = wave_sum_f64(s.q);
  s.p_over = wave_sum_f64(s.p_over);
  s.q_over = wave_sum_f64(s.q_over);
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
  const Record rec = p.records[b];
  if (rec.mode == kDone) return;
  const int q0 = p.cu[b];
  int64_t* out = p.out + static_cast<int64_t>(b) * p.max_rows + p.accepted[b];
  const T* row = static_cast<const T*>(p.logits) + rec.row * p.row_stride;
  const int chunks = (p.vocab + E - 1) / E;
  if (rec.mode == kUndefined) {  // the greedy token
    u64 key = 0;
    for (int c = tid; c < chunks; c += kThreads) {
      float f[E];
      load_chunk(row, c, p.vocab, f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const u64 k = greedy_key(f[e], E * c + e);
        if (E * c + e < p.vocab && k > key) key = k;
      }
    }
    key = wave_max_key(key);
    if (lane == 0) s_key[wave] = key;
    __syncthreads();
    if (tid) return;
    for (int w = 1; w < kWaves; ++w) key = s_key[w] > key ? s_key[w] : key;
    *out = 0xffffffffu - static_cast<u32>(key);
    return;
  }
  const double u = p.uniforms[q0];
  if (wave == 0) {
    const Sums* sums = p.sums + static_cast<int64_t>(b) * p.ranges;
    double all_p = 0, all_q = 0, over_p = 0, over_q = 0;
    for (int r = lane; r < p.ranges; r += 64) {
      all_p += sums[r].p;
      all_q += sums[r].q;
      over_p += sums[r].p_over;
      over_q += sums[r].q_over;
    }
    all_p = wave_sum_f64(all_p);
    all_q = wave_sum_f64(all_q);
    over_p = wave_sum_f64(over_p);
    over_q = wave_sum_f64(over_q);
    const double lambda = rec.mode == kRest ? all_p / all_q : 0.0;
    int mode = rec.mode;
    double whole = mode == kRest ? over_p - lambda * over_q : over_p;
    if (!(whole > 0)) {  // nothing is left: from p as it is
      mode = kAll;
      whole = all_p;
    }
    auto of_range = [&](int r) {
      if (r >= p.ranges) return 0.0;
      const Sums s = sums[r];
      return mode == kAll ? s.p : mode == kRest ? fmax(s.p_over - lambda * s.q_over, 0.0) : s.p_over;
    };
    const double border = u * whole;
    double before = 0, left = border;
    int found = -1, last = 0;
    for (int r0 = 0; r0 < p.ranges && found < 0; r0 += 64) {
      const double mine = of_range(r0 + lane);
      const double upto = before + wave_scan_f64(mine);
      const u64 past = __ballot(mine > 0 && upto > border), some = __ballot(mine > 0);
      if (past) {
        const int at = __builtin_ctzll(past);
        found = r0 + at;
        left = border - shfl_f64(upto - mine, at);
      } else if (some) {
        last = r0 + 63 - __builtin_clzll(some);
      }
      before = shfl_f64(upto, 63);
    }
    if (lane == 0) {
      s_lambda = lambda;
      s_mode = mode;
      s_range = found < 0 ? last : found;
      s_left = found < 0 ? INFINITY : left;
    }
  }
  __syncthreads();
  const int mode = s_mode, range = s_range;
  const double lambda = s_lambda, left = s_left;
  const int cbeg = range * p.range_chunks, cend = min(cbeg + p.range_chunks, chunks);
  if (mode == kWithout && wave == 0) find_refused(p, rec, q0, E * cbeg, E * cend, s_refused);
  __syncthreads();
  // the range again, a chunk per thread
  double w[E], mine = 0;
  const int c = cbeg + tid;
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = 0;
  if (c < cend) {
    float f[E];
    load_chunk(row, c, p.vocab, f);
    if (mode == kRest) {
      float g[E];
      load_chunk(static_cast<const T*>(p.draft) + rec.row * p.draft_stride, c, p.vocab, g);
#pragma unroll
      for (int e = 0; e < E; ++e)
        w[e] = fmax(weight(f[e], rec.top_p, rec.scale) - lambda * weight(g[e], rec.top_q, rec.scale), 0.0);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        w[e] = weight(f[e], rec.top_p, rec.scale);
        if (mode == kWithout && is_refused(s_refused, E * c + e)) w[e] = 0;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) mine += w[e];
  }
  double upto = wave_scan_f64(mine);
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  double before = 0;
  for (int k = 0; k < wave; ++k) before += s_wave[k];
  // the first value whose running sum is past the border, or the last that has a weight: as keys, least index first
  double run = before + upto - mine;
  u64 key = tid == 0 ? E * cbeg + 1 : 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (!(w[e] > 0)) continue;
    run += w[e];
    const u32 v = E * c + e;
    const u64 k = run > left ? 1ull << 32 | (0xffffffffu - v) : v + 1;
    key = k > key ? k : key;
  }
  key = wave_max_key(key);
  if (lane == 0) s_key[wave] = key;
  __syncthreads();
  if (tid) return;
  for (int k = 1; k < kWaves; ++k) key = s_key[k] > key ? s_key[k] : key;
  *out = key >> 32 ? 0xffffffffu - static_cast<u32>(key) : static_cast<int64_t>(key) - 1;
}

// ---------------------------------------------------------------- sizes

int segments_of(int64_t rows) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxSegments, 512 / std::max<int64_t>(rows, 1))));
}
int range_chunks_of(int) { return kRangeChunks; }
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

struct Layout {
  int64_t stats, records, sums, bytes;
};
Layout layout_of(int64_t num_seqs, int64_t max_rows, int64_t vocab) {
  Layout l{};
  // the stats of every row in one segment, or of up to 512 segments and a row
  const int64_t rows = 2 * num_seqs * max_rows;
  l.records = round16(std::max(rows, std::min<int64_t>(rows * kMaxSegments, 1024)) * sizeof(float4));
  l.sums = l.records + round16(num_seqs * sizeof(Record));
  const int64_t ranges = ((vocab + 3) / 4 + 63) / 64;  // the most that any type and range length has
  l.bytes = l.sums + num_seqs * ranges * sizeof(Sums);
  return l;
}

template <typename T>
int launch(const char* fn, const VerifyParams& p, hipStream_t s) {
  const LaunchOrder order;
  const dim3 stats(p.segments, p.max_rows * (p.draft ? 2 : 1), p.num_seqs);
  hipLaunchKernelGGL(row_stats_kernel<T>, stats, dim3(kThreads), 0, s, p);
  hipLaunchKernelGGL(keep_kernel<T>, dim3(p.num_seqs), dim3(64), 0, s, p);
  hipLaunchKernelGGL(range_sums_kernel<T>, dim3((p.ranges + kWaves - 1) / kWaves, p.num_seqs), dim3(kThreads), 0, s, p);
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
  p.segments = segments_of(2ll * num_seqs * max_seqlen_q);
  p.range_chunks = range_chunks_of(num_seqs);
  const int chunks = (vocab + per16 - 1) / per16;
  p.ranges = (chunks + p.range_chunks - 1) / p.range_chunks;
  p.stats = reinterpret_cast<float4*>(ws + at.stats);
  p.records = reinterpret_cast<Record*>(ws + at.records);
  p.sums = reinterpret_cast<Sums*>(ws + at.sums);
  const auto s = static_cast<hipStream_t>(stream);
  return logits_fp32 ? launch<float>(fn, p, s) : launch<uint16_t>(fn, p, s);
}
