// Log probabilities of given tokens, the entropy of their distributions, and the most probable
// alternatives (kvp_token_logprobs), in one pass over the logits.
//
// With c = log2(e) and a reference R near the row's maximum,
//   s = sum_i 2^(c x_i - R),   w = sum_i 2^(c x_i - R) (c x_i - R)
// give   log p_t = ln 2 (c x_t - R - log2 s)   and   H = ln 2 (log2 s - w / s).  c x_i - R is one
// fma; R need not be the maximum (nor a multiple of c), so a wave takes the largest of its first
// values and changes R only where a value lies 16 binary orders above it.
//
// What bounds it: HBM, with the vector ALUs close behind: a bf16 value has to be widened, entered
// into a maximum, exponentiated (at less than the full rate) and summed twice.  4096 bf16 rows of
// 151936 take 211 us (5.9 TB/s, the ALUs 80% busy), with 64 alternatives 290; 256 fp32 rows of
// 151643 32 us (4.9 TB/s: finding the alternatives takes the last 5).
//
// Alternatives, without a comparison more per value: a thread keeps the largest of its own values,
// which it needs anyway, so the k-th largest of the threads' maxima is a lower bound of the row's k-th
// largest value, and the values that reach it lie with the few threads whose maxima do.  Only those
// threads' chunks are read again (about k of 512), and what reaches the bound is sorted by value and index.
//
// A NaN or an infinity among the logits makes what depends on the sum NaN, as log_softmax does;
// -inf is probability 0.  Beyond 1e38, where c x overflows and neighbouring values are 2^100
// apart, only values equal to the maximum count.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace kvp {
namespace {

typedef unsigned long long Key;  // (ordered value, ~index): larger is better; 0: none

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;  // a sorted list of alternatives, one per lane
constexpr int kMaxSegments = 16;
constexpr int kList = kWaves * 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kHuge = 1e38f;
constexpr float kReach = 16.f;  // how far above R a value may lie

struct LogprobParams {
  const void* logits;
  int64_t row_stride;  // elements
  int32_t vocab, top, segments;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  int64_t* rank;
  float* top_logprobs;  // [rows][top]
  int64_t* top_tokens;
  float4* states;  // split rows: [row][segment] (max, s, w, values above the token's)
  Key* lists;      // [row][segment][top]
};

template <typename T>
struct Chunk;  // 16 bytes of logits
template <>
struct Chunk<uint16_t> {
  static constexpr int kSize = 8;
  static constexpr int kLowest = 16;  // lowest bit of an ordered value that can be set
  static __device__ __forceinline__ float one(uint16_t x) { return __uint_as_float(static_cast<u32>(x) << 16); }
  static __device__ __forceinline__ void widen(uint4 w, float (&f)[8]) { unpack8(w, f); }
};
template <>
struct Chunk<float> {
  static constexpr int kSize = 4;
  static constexpr int kLowest = 0;
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ void widen(uint4 w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
  }
};

// Monotone map of the values to unsigned numbers; NaN counts as largest, -0 equals 0.
__device__ __forceinline__ u32 ordered(float x) {
  if (x != x) return 0xffffffffu;
  const u32 b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(Key k) {
  const u32 o = static_cast<u32>(k >> 32);
  return o == 0xffffffffu ? __builtin_nanf("") : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ Key key_of(float x, u32 index) {
  return static_cast<Key>(ordered(x)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ u32 index_of(Key k) { return 0xffffffffu - static_cast<u32>(k); }

__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp_f32<kDppQuadXor1>(x));
  x = fmaxf(x, dpp_f32<kDppQuadXor2>(x));
  x = fmaxf(x, dpp_f32<kDppRowHalfMirror>(x));
  x = fmaxf(x, dpp_f32<kDppRowMirror>(x));
  return xor32_max(xor16_max(x));
}
__device__ __forceinline__ float wave_sum(float x) { return xor32_sum(xor16_sum(row16_sum(x))); }

// x of lane ^ S, on the vector ALU (through LDS a sort of 64 keys waits 21 times for two round trips).
template <int S>
__device__ __forceinline__ u32 across(u32 x) {
  const int v = static_cast<int>(x), lane = threadIdx.x & 63;
  if constexpr (S == 1) return __builtin_amdgcn_update_dpp(0, v, kDppQuadXor1, 0xf, 0xf, false);
  if constexpr (S == 2) return __builtin_amdgcn_update_dpp(0, v, kDppQuadXor2, 0xf, 0xf, false);
  if constexpr (S == 4)  // groups 0 and 2 of four lanes from 4 up, 1 and 3 from 4 down
    return __builtin_amdgcn_update_dpp(__builtin_amdgcn_update_dpp(v, v, 0x104, 0xf, 0x5, false), v, 0x114, 0xf, 0xa, false);
  if constexpr (S == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false);  // row_ror:8
  if constexpr (S == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return lane & 32 ? r[0] : r[1];
}
template <int S>
__device__ __forceinline__ float across_f(float x) {
  return __uint_as_float(across<S>(__float_as_uint(x)));
}
// Lists of 64 keys, one per lane, largest first.
template <int S>
__device__ __forceinline__ Key exchange(Key k, bool keep_max) {
  const Key o = static_cast<Key>(across<S>(static_cast<u32>(k >> 32))) << 32 | across<S>(static_cast<u32>(k));
  return (k > o) == keep_max ? k : o;
}
// Bitonic stages of strides S, S / 2, .. 1, in falling order where `falls`.
template <int S>
__device__ __forceinline__ Key stages(Key k, bool falls) {
  k = exchange<S>(k, falls == ((threadIdx.x & S) == 0));
  if constexpr (S > 1) k = stages<S / 2>(k, falls);
  return k;
}
__device__ __forceinline__ Key sort64(Key k) {
  const int lane = threadIdx.x & 63;
  k = stages<1>(k, (lane & 2) == 0);
  k = stages<2>(k, (lane & 4) == 0);
  k = stages<4>(k, (lane & 8) == 0);
  k = stages<8>(k, (lane & 16) == 0);
  k = stages<16>(k, (lane & 32) == 0);
  return stages<32>(k, true);
}
__device__ __forceinline__ Key reversed64(Key k) {
  const int lane = threadIdx.x & 63;
  return static_cast<Key>(static_cast<u32>(__builtin_amdgcn_ds_bpermute(4 * (63 - lane), static_cast<int>(k >> 32)))) << 32 |
         static_cast<u32>(__builtin_amdgcn_ds_bpermute(4 * (63 - lane), static_cast<int>(k)));
}
// The 64 largest of a list and another one given in reverse order.
__device__ __forceinline__ Key merge64(Key k, Key reversed) { return stages<32>(k > reversed ? k : reversed, true); }
// The 64 largest of `count` keys in LDS, by one wave.
__device__ __forceinline__ Key best64(const Key* s_keys, int count) {
  const int lane = threadIdx.x & 63;
  Key list = 0;
#pragma unroll 1
  for (int i = 0; i < count; i += 64) {
    const int at = i + lane;
    const Key k = sort64(at < count ? s_keys[at] : 0);
    list = i == 0 ? k : merge64(list, reversed64(k));
  }
  return list;
}

// One row's share of the sums; m is the exact maximum.
struct State {
  float m, s, w;
  int above;  // values above the token's
};
// R of a maximum.  The product is rounded here: fused into a subtraction, a reference would differ
// from itself by that rounding.
__device__ __forceinline__ float reference(float m) {
#pragma clang fp contract(off)
  return fminf(fmaxf(m, -kHuge), kHuge) * kLog2e;
}
__device__ __forceinline__ void rebase(float& s, float& w, float from, float to) {
  const float d = from - to, a = fast_exp2(d);
  w = a * (a == 0.f ? s : fmaf(s, d, w));  // s d may overflow; a NaN stays one
  s = a * s;
}
// The sum of two states, each taken at its own reference(m).
__device__ __forceinline__ State join(State a, State b) {
  State r{fmaxf(a.m, b.m), 0.f, 0.f, a.above + b.above};
  if (fabsf(r.m) > kHuge) {
    r.s = (a.m == r.m || a.s != a.s ? a.s : 0.f) + (b.m == r.m || b.s != b.s ? b.s : 0.f);
  } else {
    const float to = reference(r.m);
    rebase(a.s, a.w, reference(a.m), to);
    rebase(b.s, b.w, reference(b.m), to);
    r.s = a.s + b.s;
    r.w = a.w + b.w;
  }
  return r;
}
// ln p of a value, given the row's state; no more than 0.
__device__ __forceinline__ float log_prob(float x, const State& st) {
  float lp;
  if (fabsf(st.m) > kHuge || fabsf(x) > kHuge) lp = st.m - st.m != 0.f ? __builtin_nanf("") : x - st.m - logf(st.s);
  else lp = kLn2 * (fmaf(x, kLog2e, -reference(st.m)) - log2f(st.s));
  return lp > 0.f ? 0.f : lp;
}
__device__ __forceinline__ float entropy_of(const State& st) {
  if (fabsf(st.m) > kHuge) return st.m - st.m != 0.f ? __builtin_nanf("") : logf(st.s);
  const float h = kLn2 * (log2f(st.s) - st.w / st.s);
  return h < 0.f ? 0.f : h;
}
__device__ __forceinline__ void finish_row(const LogprobParams& p, int r, const State& st, int64_t token, float x) {
  const bool ok = token >= 0 && token < p.vocab;
  p.logprobs[r] = ok ? log_prob(x, st) : __builtin_nanf("");
  p.entropy[r] = entropy_of(st);
  p.rank[r] = ok ? st.above + 1 : 0;
}
__device__ __forceinline__ void write_top(const LogprobParams& p, int r, const State& st, Key k) {
  const int lane = threadIdx.x & 63;
  if (lane >= p.top) return;
  const int64_t at = static_cast<int64_t>(r) * p.top + lane;
  p.top_logprobs[at] = log_prob(value_of(k), st);
  p.top_tokens[at] = index_of(k);
}

// A segment of a row per workgroup: chunks [cbeg, cend), the row's last one maybe not full.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const LogprobParams p) {
  constexpr int E = Chunk<T>::kSize;
  __shared__ Key s_keys[kList];
  __shared__ State s_state[kWaves];
  __shared__ u32 s_bound[kThreads], s_least;
  __shared__ uint16_t s_winner[kThreads];
  __shared__ int s_count[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = static_cast<int>(blockIdx.x) / p.segments, seg = static_cast<int>(blockIdx.x) - r * p.segments;
  const T* row = static_cast<const T*>(p.logits) + r * p.row_stride;
  const int chunks = (p.vocab + E - 1) / E, full = p.vocab / E;
  const int per = (chunks + p.segments - 1) / p.segments;
  const int cbeg = min(seg * per, chunks), cend = min(cbeg + per, chunks);
  // The chunk's values; those behind the row's end are -inf.
  auto values = [&](int c, uint4 w, float (&f)[E]) {
    if (c < full) {
      Chunk<T>::widen(w, f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = E * c + e < p.vocab ? Chunk<T>::one(row[E * c + e]) : -INFINITY;
    }
  };
  auto load = [&](int c) {  // a whole chunk of the row, whatever c
    return full > 0 ? load16_nt(row + E * static_cast<int64_t>(min(c, full - 1))) : make_uint4(0, 0, 0, 0);
  };

  // Batches of 32 values per thread, the next one in flight while one is taken; what is left of the
  // segment behind them chunk by chunk.
  constexpr int kBatch = 32 / E;
  const int whole = min(full, cend);  // chunks up to here are whole
  uint4 in[kBatch];
  auto load_batch = [&](int c0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) in[u] = load(c0 + u * kThreads + lane);
  };
  int c0 = cbeg + (wave << 6);
  load_batch(c0);  // before the token, whose logit is two round trips away
  const int64_t token = p.tokens[r];
  const float mine = token >= 0 && token < p.vocab ? Chunk<T>::one(row[token]) : __builtin_nanf("");

  float m = -INFINITY, s = 0.f, w = 0.f, R = 0.f;
  int above = 0;
  bool first = true;
  auto take = [&](auto count, const float* f) __attribute__((always_inline)) {  // the lane's values
    constexpr int N = decltype(count)::value;
    float most = max3(f[0], f[1], f[2]);
#pragma unroll
    for (int e = 3; e < N; e += 2) most = max3(most, f[e], f[min(e + 1, N - 1)]);
    if (first || __any(fmaf(most, kLog2e, -R) > kReach)) {  // uniform
      const float to = reference(wave_max(most));
      if (!first) rebase(s, w, R, to);
      R = to;
      first = false;
    }
    m = max3(m, most, most);
    if (__any(most > mine)) {  // of a likely token's row few batches have one
#pragma unroll
      for (int e = 0; e < N; ++e) above += __popcll(__ballot(f[e] > mine));
    }
    const float s0 = s, w0 = w;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float t = fmaf(f[e], kLog2e, -R), x = fast_exp2(t);
      s += x;
      w = fmaf(x, t, w);
    }
    if (__any(w != w)) {  // 0 times -inf (or a NaN): once more; 2^t is 0 long before t is -inf
      s = s0;
      w = w0;
      float again = R;
      asm volatile("" : "+v"(again));  // or the compiler makes one loop of the two and every batch pays for both
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float t = fmaf(f[e], kLog2e, -again), x = fast_exp2(t);
        s += x;
        w = fmaf(x, fmaxf(t, -1024.f), w);
      }
    }
  };
  constexpr int kStride = kThreads * kBatch, kSpan = kThreads * (kBatch - 1) + 64;
#pragma unroll 1
  for (; c0 + kSpan <= whole; c0 += kStride) {  // uniform
    float f[kBatch * E];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) Chunk<T>::widen(in[u], *reinterpret_cast<float(*)[E]>(f + u * E));
    if (c0 + kStride + kSpan <= whole) load_batch(c0 + kStride);
    take(std::integral_constant<int, kBatch * E>{}, f);
  }
#pragma unroll 1
  for (; c0 < cend; c0 += kThreads) {  // uniform
    const int c = c0 + lane;
    float f[E];
    if (c < cend) {
      values(c, load(c), f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = -INFINITY;
    }
    take(std::integral_constant<int, E>{}, f);
  }

  // ---- the workgroup's state
  const bool odd = s != s;  // the thread may have seen a NaN
  State st{wave_max(m), 0.f, 0.f, above};
  float ws = wave_sum(s), ww = wave_sum(w);
  if (fabsf(st.m) <= kHuge) rebase(ws, ww, R, reference(st.m));
  st.s = ws;
  st.w = ww;
  if (lane == 0) s_state[wave] = st;
  // ... and every thread's maximum, ordered, NaN above all
  u32 bound = ordered(m);
  if (p.top > 0) {
    if (odd) {
      for (int c = cbeg + tid; c < cend; c += kThreads) {
        float f[E];
        values(c, load(c), f);
#pragma unroll
        for (int e = 0; e < E; ++e) bound = max(bound, ordered(f[e]));
      }
    }
    s_bound[tid] = cbeg + tid < cend ? bound : 0;
  }
  if (tid == 0) s_count[0] = s_count[1] = 0;
  __syncthreads();
  float top_m = s_state[0].m;
#pragma unroll
  for (int i = 1; i < kWaves; ++i) top_m = fmaxf(top_m, s_state[i].m);
  if (fabsf(top_m) > kHuge && top_m - top_m == 0.f) {  // uniform: values equal to the maximum
    float equal = 0.f;
    for (int c = cbeg + tid; c < cend; c += kThreads) {
      float f[E];
      values(c, load(c), f);
#pragma unroll
      for (int e = 0; e < E; ++e) equal += f[e] != f[e] ? f[e] : (f[e] == top_m ? 1.f : 0.f);
    }
    equal = wave_sum(equal);
    __syncthreads();
    if (lane == 0) s_state[wave] = State{top_m, equal, 0.f, above};
    __syncthreads();
  }
  if (wave == 0) {
    st = s_state[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) st = join(st, s_state[i]);
  }

  // ---- alternatives
  Key list = 0;
  if (p.top > 0) {
    if (wave == 0) {  // the top-th largest of the maxima, bit by bit; 0 if there are fewer
      u32 mine8[kWaves], least = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) mine8[i] = s_bound[64 * i + lane];
#pragma unroll 1
      for (int bit = 31; bit >= Chunk<T>::kLowest; --bit) {
        const u32 with = least | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) reach += __popcll(__ballot(mine8[i] >= with));
        if (reach >= p.top) least = with;
      }
      if (lane == 0) s_least = least;
    }
    __syncthreads();
    const u32 least = s_least;
    // the threads whose maxima reach it
    const bool wins = s_bound[tid] >= max(least, 1u);
    if (wins) s_winner[atomicAdd(&s_count[0], 1)] = static_cast<uint16_t>(tid);
    __syncthreads();
    const int winners = s_count[0], rounds = (cend - cbeg + kThreads - 1) / kThreads, items = winners * rounds;
    // item i: chunk i / winners of winner i % winners
    auto chunk_of = [&](int i) {
      const int j = i / winners;
      return cbeg + s_winner[i - j * winners] + j * kThreads;
    };
    for (int i = tid; i < items; i += kThreads) {
      const int c = chunk_of(i);
      if (c >= cend) continue;
      float f[E];
      values(c, load(c), f);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (ordered(f[e]) >= least && E * c + e < p.vocab) {
          const int at = atomicAdd(&s_count[1], 1);
          if (at < kList) s_keys[at] = key_of(f[e], E * c + e);
        }
    }
    __syncthreads();
    int count = s_count[1];
    if (count > kList) {  // many equal values: every wave keeps the best of what it sees
      Key last = 0;       // its top-th best
#pragma unroll 1
      for (int i0 = wave << 6; i0 < items; i0 += kThreads) {
        const int i = i0 + lane, c = chunk_of(min(i, items - 1));
        float f[E];
        values(min(c, cend - 1), load(c), f);
#pragma unroll 1
        for (int e = 0; e < E; ++e) {
          float x = f[0];
#pragma unroll
          for (int j = 1; j < E; ++j) x = e == j ? f[j] : x;
          const Key k = i < items && c < cend && E * c + e < p.vocab ? key_of(x, E * c + e) : 0;
          if (!__any(k > last)) continue;
          list = merge64(list, reversed64(sort64(k)));
          last = __shfl(list, p.top - 1);
        }
      }
      s_keys[tid] = list;
      count = kList;
      __syncthreads();
    }
    if (wave == 0) list = best64(s_keys, count);
  }

  // ---- out, or to the merge
  if (p.segments == 1) {
    if (tid == 0) finish_row(p, r, st, token, mine);
    if (wave == 0) write_top(p, r, st, list);
  } else {
    if (tid == 0) p.states[blockIdx.x] = make_float4(st.m, st.s, st.w, __int_as_float(st.above));
    if (wave == 0 && lane < p.top) p.lists[static_cast<int64_t>(blockIdx.x) * p.top + lane] = list;
  }
}

// A split row's segments, one row per workgroup.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_merge_kernel(const LogprobParams p) {
  __shared__ Key s_keys[kList];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = static_cast<int>(blockIdx.x);
  // the segments' alternatives side by side, 64 to a wave and round
  const int keys = p.segments * p.top;
  const Key* lists = p.lists + static_cast<int64_t>(r) * keys;
  constexpr int kRounds = kMaxSegments * kMaxTop / kThreads;
  Key key[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) key[i] = tid + i * kThreads < keys ? lists[tid + i * kThreads] : 0;
  // every wave joins all segments' states, one per lane
  const float4 x = p.states[static_cast<int64_t>(r) * p.segments + min(lane, p.segments - 1)];
  State st = lane < p.segments ? State{x.x, x.y, x.z, __float_as_int(x.w)} : State{-INFINITY, 0.f, 0.f, 0};
  auto with = [&](auto stride) {
    constexpr int S = decltype(stride)::value;
    st = join(st, State{across_f<S>(st.m), across_f<S>(st.s), across_f<S>(st.w), static_cast<int>(across<S>(st.above))});
  };
  with(std::integral_constant<int, 1>{});
  with(std::integral_constant<int, 2>{});
  with(std::integral_constant<int, 4>{});
  with(std::integral_constant<int, 8>{});
  with(std::integral_constant<int, 16>{});
  with(std::integral_constant<int, 32>{});
  if (tid == 0) {
    const int64_t token = p.tokens[r];
    const T* row = static_cast<const T*>(p.logits) + r * p.row_stride;
    finish_row(p, r, st, token, token >= 0 && token < p.vocab ? Chunk<T>::one(row[token]) : 0.f);
  }
  if (p.top == 0) return;  // uniform
  Key list = 0;
#pragma unroll
  for (int i = 0; i < kRounds; ++i)
    if (64 * wave + i * kThreads < keys) list = i == 0 ? sort64(key[0]) : merge64(list, reversed64(sort64(key[i])));
  s_keys[tid] = list;
  __syncthreads();
  if (wave == 0) {
    const int waves = min(kWaves, (keys + 63) / 64);
#pragma unroll 1
    for (int i = 1; i < waves; ++i) list = merge64(list, s_keys[64 * i + 63 - lane]);
    write_top(p, r, st, list);
  }
}

// Segments of a row: no more workgroups than are resident at once (two per CU), since every segment
// pays for its alternatives anew and a second round of workgroups for a second time: 64 fp32 rows of
// 151936 take 20 us in 8 segments, 33 in 16.  From one row per CU on splitting is not worth its join
// (256 rows: 33 us whole, 39 in halves), and behind 16 segments only the join grows.
int segments_of(int32_t rows) { return rows >= 256 ? 1 : std::min(kMaxSegments, 512 / std::max(rows, 1)); }

template <typename T>
int launch(const char* fn, LogprobParams p, int rows, hipStream_t s) {
  const LaunchOrder order;
  hipLaunchKernelGGL(logprobs_kernel<T>, dim3(static_cast<unsigned>(rows) * p.segments), dim3(kThreads), 0, s, p);
  if (p.segments > 1)
    hipLaunchKernelGGL(logprobs_merge_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, s, p);
  return launch_status(fn);
}

}  // namespace
}  // namespace kvp

using namespace kvp;

extern "C" size_t kvp_token_logprobs_workspace_bytes(int32_t num_rows) {
  if (num_rows <= 0) return 0;
  const int s = segments_of(num_rows);
  return s == 1 ? 0 : static_cast<size_t>(num_rows) * s * (sizeof(float4) + kMaxTop * sizeof(Key));
}

extern "C" int kvp_token_logprobs(const void* logits, int32_t logits_fp32, int64_t row_stride, int32_t num_rows,
                                  int32_t vocab, const int64_t* tokens, int32_t top, float* logprobs, float* entropy,
                                  int64_t* rank, float* top_logprobs, int64_t* top_tokens, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  static const char fn[] = "kvp_token_logprobs";
  clear_error();
  if (num_rows < 0 || vocab < 1) return fail(KVP_EINVAL, "%s: num_rows=%d vocab=%d", fn, num_rows, vocab);
  if (top < 0 || top > kMaxTop || top > vocab)
    return fail(KVP_EUNSUPPORTED, "%s: top=%d (supported: 0 to %d, and no more than vocab)", fn, top, kMaxTop);
  if (num_rows == 0) return KVP_OK;
  if (!logits || !tokens || !logprobs || !entropy || !rank || (top > 0 && (!top_logprobs || !top_tokens)))
    return fail(KVP_EINVAL, "%s: null pointer", fn);
  auto off = [](const void* ptr, unsigned by) { return (reinterpret_cast<uintptr_t>(ptr) & (by - 1)) != 0; };
  if (!aligned16(logits) || row_stride % (logits_fp32 ? 4 : 8) || row_stride < vocab)
    return fail(KVP_EINVAL, "%s: logits must be 16-byte aligned with a row stride >= vocab that is a multiple of "
                "16 bytes", fn);
  if (off(tokens, 8) || off(logprobs, 4) || off(entropy, 4) || off(rank, 8) || off(top_logprobs, 4) ||
      off(top_tokens, 8))
    return fail(KVP_EINVAL, "%s: misaligned tokens or outputs", fn);
  if (num_rows > INT32_MAX / kMaxSegments) return fail(KVP_EINVAL, "%s: too many rows", fn);
  const int segments = segments_of(num_rows);
  const size_t need = kvp_token_logprobs_workspace_bytes(num_rows);
  if (segments > 1 && (!workspace || workspace_bytes < need))
    return fail(KVP_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, need);
  if (!aligned16(workspace)) return fail(KVP_EINVAL, "%s: workspace must be 16-byte aligned", fn);
  char* ws = static_cast<char*>(workspace);
  LogprobParams p{logits, row_stride, vocab, top, segments, tokens, logprobs, entropy, rank, top_logprobs, top_tokens,
                  reinterpret_cast<float4*>(ws),
                  reinterpret_cast<Key*>(ws + static_cast<size_t>(num_rows) * segments * sizeof(float4))};
  const auto s = static_cast<hipStream_t>(stream);
  return logits_fp32 ? launch<float>(fn, p, num_rows, s) : launch<uint16_t>(fn, p, num_rows, s);
}
