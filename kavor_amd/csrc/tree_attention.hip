// Attention of a few query tokens per sequence over its paged KV cache, in bf16 or quantised:
// the drafted tokens of a speculative step (kvp_tree_attention_*), and the one token of a decode
// step over the quantised cache (kvp_paged_decode_fp8).
//
// Sequence b has n_b query tokens (at most 64) and a cache of len_b tokens, the last n_b of which
// are the query tokens themselves.  With ctx_b = len_b - n_b, query i sees every token t < ctx_b
// and of the drafts those whose bit is set in its mask:
//   out[i, h] = softmax_t(scale * q[i, h] . K[t]) V[t]  over  t < ctx_b or bit (t - ctx_b) of mask_i
// A row that sees no token is zero.  In a quantised cache K[t] = 2^(ek_t) k_t and V[t] = 2^(ev_t) v_t
// with k_t, v_t in e4m3 and one exponent for each token and head.
//
// What bounds it: HBM while the rows that share a K/V head (n_b times G = Hq / Hkv) are few, since
// every K/V byte is read once for all of them: rows flops to a byte of bf16 cache, twice that
// quantised.
//
// Work decomposition: work is counted in steps, 8 KiB of K and as much of V (32 tokens of bf16, 64
// quantised), laid end to end over the sequences.  The rows of a kv head are cut into groups of
// 16 NT; a stream is one such group of one head.  A wave takes one stream over one contiguous
// range of the steps, all ranges equally long, and meets no barrier behind the prefix sums.
// Streams of one range are neighbouring waves.  A sequence that lies in one range gets its output
// from there; of the others every range leaves (max, sum, unnormalised sum of V) in 32 bits, which
// tree_merge_kernel joins.  Only the first and the last sequence of a range can be cut by it, so a
// range has two places for states whatever the batch: the first for a sequence that it takes up
// at its own start, the second for one that starts later and goes on behind it.
//
// Layouts are those of the decode kernel (lane l: n = l % 16, q4 = l / 16): S = K Q^T has tokens
// 4 q4 + j of every 16 in the lane and row n as its column, O^T = V^T P^T takes P from the same
// registers.  e4m3 is widened to bf16, exactly, on its way from LDS to the matrix cores, K with its
// scale (the lane's own token); V's scale goes into P, a multiplication by a power of two.  P is
// rounded to bf16 there: at most 2^-8 of each weight, of either sign, so below the rounding of the
// bf16 output where the values do not cancel; the sum of the weights is of the unrounded ones, and
// running maxima, sums and products stay in 32 bits.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.h"

namespace kvp {
namespace {

constexpr int kDim = 128;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 8192;         // bytes of K, or of V, of one step
constexpr int kMaxQ = 64;           // query tokens per sequence: the bits of a mask
constexpr int kMaxGroup = 16;       // query heads per kv head
constexpr int kSeqsPerLaunch = 2048;  // prefix sums in LDS; more sequences run as consecutive launches
constexpr int kMaxTokens = 1 << 24;   // per sequence: the steps of a launch fit 32 bits
constexpr int kHeaderInts = 16;
constexpr int64_t kHeaderBytes = ((kHeaderInts + kSeqsPerLaunch + 1) * 4 + 255) / 256 * 256;
constexpr int kMaxWorkgroups = 512;  // bounds the workspace, whatever the device

template <bool FP8>
struct Format {
  static constexpr int kRow = FP8 ? kDim : 2 * kDim;  // bytes of a token's row
  static constexpr int kStep = kTile / kRow;          // tokens per step
  static constexpr int kParts = kStep / 16;           // of 16 tokens
  static constexpr int kKOps = FP8 ? 10 : 8;          // vector memory operations of a K tile and both scales
  static constexpr int kVOps = 8;
};

struct TreeParams {
  const uint16_t* q;
  int64_t q_tok_stride, q_head_stride;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  int64_t blk_stride, slot_stride, head_stride;  // bytes
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  int64_t scale_blk_stride, scale_head_stride;
  int32_t num_cache_blocks, block_size, max_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu_q;  // NULL: one query token per sequence
  const int32_t* kv_lens;
  int32_t num_seqs, total_q, max_q;
  int32_t num_q_heads, num_kv_heads, group;
  const int64_t* mask;  // NULL: causal
  float scale_log2;
  uint16_t* out;
  int64_t o_tok_stride, o_head_stride;
  int32_t* header;  // [0] steps per range, [kHeaderInts ..] step prefix sums
  float* part_o;    // [range][2][kv head][max rows][128]
  float* part_ml;   // [range][2][kv head][max rows][2]
  int32_t streams, ranges, row_groups, max_rows;
  Divisor div_streams, div_row_groups, div_ranges, div_block, div_group;
};

// A sequence's query rows and cached tokens; kind says what there is to do.
enum SeqKind { kNone, kZeros, kNans, kWork };
struct SeqShape {
  int q0, n, len;
  SeqKind kind;
};
__device__ __forceinline__ SeqShape shape_of(const TreeParams& p, int q0, int q1, int len) {
  SeqShape s{q0, q1 - q0, len, kWork};
  if (q0 < 0 || q1 > p.total_q || q1 <= q0) s.kind = kNone;
  else if (len <= 0) s.kind = kZeros;  // a padding row of a captured graph
  else if (s.n > p.max_q || len < s.n || len > p.max_blocks * p.block_size) s.kind = kNans;
  return s;
}
__device__ __forceinline__ SeqShape load_shape(const TreeParams& p, int b) {
  return shape_of(p, p.cu_q ? load_uniform(p.cu_q, b) : b, p.cu_q ? load_uniform(p.cu_q, b + 1) : b + 1,
                  load_uniform(p.kv_lens, b));
}

// s_cum[b] = steps of sequences 0 .. b - 1, built by the whole workgroup.
template <int STEP>
__device__ __forceinline__ void build_prefix(const TreeParams& p, int* s_cum, int* s_part) {
  const int tid = threadIdx.x, B = p.num_seqs;
  const int per = (B + kThreads - 1) / kThreads;
  const int j0 = min(tid * per, B), j1 = min(j0 + per, B);
  int local = 0;
#pragma unroll 1
  for (int b = j0; b < j1; ++b) {
    const SeqShape s = shape_of(p, p.cu_q ? p.cu_q[b] : b, p.cu_q ? p.cu_q[b + 1] : b + 1, p.kv_lens[b]);
    const int steps = s.kind == kWork ? (s.len + STEP - 1) / STEP : 0;
    s_cum[b] = steps;
    local += steps;
  }
  const int wave = tid >> 6;
  const int incl = wave_incl_scan(local);
  if ((tid & 63) == 63) s_part[wave] = incl;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w)
    if (w < wave) before += s_part[w];
  int run = before + incl - local;
#pragma unroll 1
  for (int b = j0; b < j1; ++b) {
    const int steps = s_cum[b];
    s_cum[b] = run;
    run += steps;
  }
  if (tid == kThreads - 1) s_cum[B] = before + incl;
  __syncthreads();
}

// Rows of sequences that have nothing to attend to, or impossible lengths.
__device__ __forceinline__ void fill_rows(const TreeParams& p, const int* s_cum) {
#pragma unroll 1
  for (int b = blockIdx.x; b < p.num_seqs; b += gridDim.x) {
    if (s_cum[b + 1] != s_cum[b]) continue;
    const SeqShape s = load_shape(p, b);
    if (s.kind == kNone) continue;
    const u32 w = s.kind == kZeros ? 0u : 0x7fc07fc0u;
    const int chunks = s.n * p.num_q_heads * (kDim / 8);
#pragma unroll 1
    for (int i = threadIdx.x; i < chunks; i += kThreads) {
      const int row = i / (kDim / 8), tok = row / p.num_q_heads, h = row - tok * p.num_q_heads;
      *reinterpret_cast<uint4*>(p.out + (s.q0 + tok) * p.o_tok_stride + h * p.o_head_stride + i % (kDim / 8) * 8) =
          make_uint4(w, w, w, w);
    }
  }
}

// A wave's place in the steps of its range.
struct Cursor {
  int b, j, nsteps;   // sequence, step within it, its steps
  int q0, n, len;
  int lblk, blk, pf_blk;  // logical block, its id, and the id of the next one (-1: not loaded)
  int active;         // the sequence has rows in the wave's row group
  int bad;            // a needed block id was out of range
  int mark;           // vector memory operations issued up to the step's K tile
};
__device__ __forceinline__ void enter_block(const TreeParams& p, Cursor& c, int lblk, int blk) {
  const int bad = blk < 0 || blk >= p.num_cache_blocks;
  c.bad |= bad;
  c.blk = bad ? 0 : blk;
  c.lblk = lblk;
  c.pf_blk = (lblk + 1) * p.block_size < c.len ? load_uniform(p.block_tables + c.b * p.bt_stride, lblk + 1) : -1;
}
template <int STEP>
__device__ __forceinline__ void start_seq(const TreeParams& p, Cursor& c, int b, int j, int first_row) {
  const SeqShape s = load_shape(p, b);
  c.b = b;
  c.j = j;
  c.q0 = s.q0;
  c.n = s.n;
  c.len = s.len;
  c.nsteps = (s.len + STEP - 1) / STEP;
  c.active = s.n * p.group > first_row;
  c.bad = 0;
  const int lblk = div_by(j * STEP, p.div_block);
  enter_block(p, c, lblk, load_uniform(p.block_tables + b * p.bt_stride, lblk));
}

// The lane's part of a tile fill.  Instruction i fills rows R i .. R i + R - 1 of a tile (R = 4 rows
// of 256 bytes, 8 of 128): the lane writes row R i + r at physical chunk c, which holds logical
// chunk c ^ f(row) so that neither kind of read meets a bank twice: f = row % 16 for K and
// 2 (row % 8) for V in bf16, (row / 2) % 8 for both in e4m3 (two rows fill the banks once).
struct TileLane {
  int row_off;  // byte offset of row r
  int k_chunk[4], v_chunk[2];
};
template <bool FP8>
__device__ __forceinline__ TileLane tile_lane(const TreeParams& p, int lane) {
  TileLane t{};
  const int r = FP8 ? lane >> 3 : lane >> 4, c = FP8 ? lane & 7 : lane & 15;
  t.row_off = r * static_cast<int>(p.slot_stride);
#pragma unroll
  for (int i = 0; i < 4; ++i) t.k_chunk[i] = 16 * (FP8 ? c ^ (4 * (i & 1) + (r >> 1)) : c ^ (4 * i + r));
#pragma unroll
  for (int i = 0; i < 2; ++i) t.v_chunk[i] = FP8 ? t.k_chunk[i] : 16 * (c ^ (2 * ((4 * i + r) & 7)));
  return t;
}
typedef __attribute__((address_space(3))) void* LdsPtr;
// A tile from byte `base` of the cache: row r is token r, those past the last one repeat it.
template <bool FP8, bool V>
__device__ __forceinline__ void issue_tile(const TreeParams& p, const TileLane& t, int64_t base, int rows, char* tile) {
  constexpr int kPer = 1024 / Format<FP8>::kRow;  // rows per instruction
  const int stride = static_cast<int>(p.slot_stride);
  const BufferRsrc rsrc = buffer_rsrc((V ? p.v_cache : p.k_cache) + base,
                                      static_cast<uint32_t>((Format<FP8>::kStep - 1) * stride + Format<FP8>::kRow));
  const int last = (rows - 1) * stride;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    raw_buffer_load_lds(rsrc, (LdsPtr)(tile + 1024 * i), 16,
                        min(t.row_off + kPer * i * stride, last) + (V ? t.v_chunk[i & 1] : t.k_chunk[i & 3]), 0, 0, 0);
}
// The scales of a step's 64 tokens: K's bytes, then V's.
__device__ __forceinline__ void issue_scales(const TreeParams& p, int64_t base, int lane, char* to) {
  if (lane < 16) {
    raw_buffer_load_lds(buffer_rsrc(p.k_scale + base, 64), (LdsPtr)to, 4, 4 * lane, 0, 0, 0);
    raw_buffer_load_lds(buffer_rsrc(p.v_scale + base, 64), (LdsPtr)(to + 64), 4, 4 * lane, 0, 0, 0);
  }
}

// K of a step in e4m3: the lane's 16 bytes at a[i] of each 16 tokens, k[4 i + part].
__device__ __forceinline__ void read_k8_tile(u32 a0, u32 a1, u32x4_t (&k)[8]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:2048\n\t"
      "ds_read_b128 %2, %8 offset:4096\n\tds_read_b128 %3, %8 offset:6144\n\t"
      "ds_read_b128 %4, %9\n\tds_read_b128 %5, %9 offset:2048\n\t"
      "ds_read_b128 %6, %9 offset:4096\n\tds_read_b128 %7, %9 offset:6144\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4]), "=&v"(k[5]), "=&v"(k[6]), "=&v"(k[7])
      : "v"(a0), "v"(a1)
      : "memory");
}
// V of 32 tokens in e4m3, transposed: 8 bytes at a[i], i = 0..7.
__device__ __forceinline__ void read_v8_tile(const u32 (&a)[8], u32x2_t (&v)[8]) {
  asm volatile(
      "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %9\n\t"
      "ds_read_b64_tr_b8 %2, %10\n\tds_read_b64_tr_b8 %3, %11\n\t"
      "ds_read_b64_tr_b8 %4, %12\n\tds_read_b64_tr_b8 %5, %13\n\t"
      "ds_read_b64_tr_b8 %6, %14\n\tds_read_b64_tr_b8 %7, %15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
      : "memory");
}
// Exponent bytes of a step: K's of token 16 i + n at a + 16 i, V's of tokens 16 i + 4 q4 .. + 3 at b + 16 i.
__device__ __forceinline__ void read_scales(u32 a, u32 b, u32 (&k)[4], u32 (&v)[4]) {
  asm volatile(
      "ds_read_u8 %0, %8\n\tds_read_u8 %1, %8 offset:16\n\tds_read_u8 %2, %8 offset:32\n\tds_read_u8 %3, %8 offset:48\n\t"
      "ds_read_b32 %4, %9\n\tds_read_b32 %5, %9 offset:16\n\tds_read_b32 %6, %9 offset:32\n\tds_read_b32 %7, %9 offset:48\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(a), "v"(b)
      : "memory");
}
// Eight e4m3 values as bf16, times a power of two: exact.
__device__ __forceinline__ u32x4_t widen8(u32 lo, u32 hi, float scale) {
  return u32x4_t{__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
}

// Waits until at most `most` vector memory operations are in flight, rounded down to a count that
// the loop below has between a tile and its use.
template <int K, int V>
__device__ __forceinline__ void wait_tiles(int most) {
  if (most >= 2 * K + V) wait_vmem<2 * K + V>();
  else if (most >= K + 2 * V) wait_vmem<K + 2 * V>();
  else if (most >= K + V) wait_vmem<K + V>();
  else if (most >= K) wait_vmem<K>();
  else if (most >= V) wait_vmem<V>();
  else wait_vmem<0>();
}

template <bool FP8, int NT>
__global__ __launch_bounds__(kThreads) void tree_attention_kernel(const TreeParams p) {
  using F = Format<FP8>;
  constexpr int STEP = F::kStep, PARTS = F::kParts;
  __shared__ __attribute__((aligned(16))) char s_tile[kWaves][2][2 * kTile];
  __shared__ __attribute__((aligned(16))) char s_scale[FP8 ? kWaves : 1][2][128];
  __shared__ int s_cum[kSeqsPerLaunch + 1];
  __shared__ int s_part[kWaves];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, q4 = lane >> 4;

  build_prefix<STEP>(p, s_cum, s_part);
  fill_rows(p, s_cum);
  const int B = p.num_seqs;
  const int total = __builtin_amdgcn_readfirstlane(s_cum[B]);
  const int spr = max(1, div_by(total + p.ranges - 1, p.div_ranges));
  if (blockIdx.x == 0) {  // for the merge
    if (tid == 0) p.header[0] = spr;
    for (int b = tid; b <= B; b += kThreads) p.header[kHeaderInts + b] = s_cum[b];
  }
  const int unit = static_cast<int>(blockIdx.x) * kWaves + wave;
  const int range = div_by(unit, p.div_streams), stream = unit - range * p.streams;
  const int kvh = div_by(stream, p.div_row_groups), rg = stream - kvh * p.row_groups;
  const int S0 = range * spr, S1 = min(total, S0 + spr);
  if (range >= p.ranges || S0 >= S1) return;  // no barrier follows

  int lo = 0, hi = B;  // s_cum[lo] <= S0 < s_cum[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_cum[mid] <= S0) lo = mid;
    else hi = mid;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);

  const int first_row = rg * 16 * NT;
  const int64_t head_off = kvh * p.head_stride, scale_head = kvh * p.scale_head_stride;
  const TileLane ln = tile_lane<FP8>(p, lane);
  // LDS addresses of the lane's operands in a tile at address 0 (see the swizzles)
  u32 ka[4], va[8];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)
    ka[kk] = FP8 ? 128 * n + 16 * ((4 * (kk & 1) + q4) ^ (n >> 1)) : 256 * n + 16 * ((4 * kk + q4) ^ n);
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) {
    if (FP8) {
      const int e = n >> 1, row = 16 * (e >> 2) + 4 * q4 + (e & 3);
      va[mt] = kTile + 128 * row + 16 * (mt ^ ((row >> 1) & 7)) + 8 * (n & 1);
    } else {
      const int row = 4 * q4 + (n >> 2);
      va[mt] = kTile + 256 * row + 8 * (n & 3) + 32 * (mt ^ (row & 7));
    }
  }
  int tok[NT], head[NT];  // the token and query head of the lane's column in each 16 rows
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = first_row + 16 * nt + n;
    tok[nt] = div_by(row, p.div_group);
    head[nt] = kvh * p.group + row - tok[nt] * p.group;
  }

  u32x4_t qv[NT][4];
  uint64_t seen[NT];  // the drafts that the column's token sees
  float m[NT], l[NT];
  mfma_f32x4_t acc[NT][8];
  auto reset = [&] {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = kMaxFloor;
      l[nt] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) acc[nt][mt] = mfma_f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  };
  auto load_q = [&](const Cursor& c) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int i = min(tok[nt], c.n - 1);
      const uint16_t* src = p.q + (c.q0 + i) * p.q_tok_stride + head[nt] * p.q_head_stride;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        qv[nt][kk] = *reinterpret_cast<const u32x4_t*>(
            src + (FP8 ? 64 * (kk >> 1) + 16 * q4 + 8 * (kk & 1) : 32 * kk + 8 * q4));
      const uint64_t all = ~0ull >> (64 - c.n);
      const uint64_t bits = p.mask ? static_cast<uint64_t>(p.mask[c.q0 + i]) : ~0ull >> (63 - i);
      seen[nt] = bits & all;
    }
  };
  // The state of the wave's rows of a sequence: its output, or a partial state at `place`.
  auto emit = [&](const Cursor& c, bool whole, int place) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum = xor32_sum(xor16_sum(l[nt]));
      if (c.bad) sum = NAN;
      if (tok[nt] >= c.n) continue;
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t* out = p.out + (c.q0 + tok[nt]) * p.o_tok_stride + head[nt] * p.o_head_stride + 4 * q4;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          const mfma_f32x4_t o = acc[nt][mt] * inv;
          *reinterpret_cast<u32x2_t*>(out + 16 * mt) = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
        }
      } else {
        const int64_t at = (static_cast<int64_t>(place) * p.num_kv_heads + kvh) * p.max_rows + first_row + 16 * nt + n;
        float* part = p.part_o + at * kDim + 4 * q4;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) *reinterpret_cast<mfma_f32x4_t*>(part + 16 * mt) = acc[nt][mt];
        if (q4 == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m[nt], sum);
      }
    }
  };

  // The loop.  Iteration S computes step S and issues the tiles of step S + 2, each as soon as its
  // tile has been read; the first two only issue.  c[i]: the place of step S + i.
  Cursor c[3] = {};
  Cursor &c0 = c[0], &cn = c[2];
  int issued = 0;
  reset();
#pragma unroll 1
  for (int S = S0 - 2; S < S1; ++S) {
    const int buf = (S - S0) & 1;
    char* const tiles = s_tile[wave][buf];
    char* const scales = s_scale[FP8 ? wave : 0][buf];
    const u32 tile = lds_addr(tiles);
    const bool live = S >= S0 && c0.active, issue = S + 2 < S1;
    const bool starts = S == S0 || c0.j == 0;
    const int t0 = c0.j * STEP, ctx = c0.len - c0.n;
    const bool tail = t0 + STEP > ctx;  // the step holds drafts, or ends behind the last token
    mfma_f32x4_t s[NT][PARTS];
    u32 vexp[4] = {};
    if (live) {
      if (starts) load_q(c0);
      wait_tiles<F::kKOps, F::kVOps>(issued - c0.mark);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < PARTS; ++h) s[nt][h] = mfma_f32x4_t{0.f, 0.f, 0.f, 0.f};
      u32x4_t k[8];
      if constexpr (FP8) {
        u32 kexp[4];
        const u32 at = lds_addr(scales);
        read_scales(at + n, at + 64 + 4 * q4, kexp, vexp);
        read_k8_tile(tile + ka[0], tile + ka[1], k);
#pragma unroll
        for (int h = 0; h < PARTS; ++h) {
          const float scale = __uint_as_float(kexp[h] << 23);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const u32x4_t w = k[4 * (kk >> 1) + h];
            const u32x4_t a = widen8(w[2 * (kk & 1)], w[2 * (kk & 1) + 1], scale);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][h] = mfma16(a, qv[nt][kk], s[nt][h]);
          }
        }
      } else {
        const u32 at[4] = {tile + ka[0], tile + ka[1], tile + ka[2], tile + ka[3]};
        read_k_tile(at, k);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[nt][i & 1] = mfma16(k[i], qv[nt][i >> 1], s[nt][i & 1]);
      }
    }
    int64_t base = 0;
    int rows = 0;
    if (issue) {  // K has been read: its tile takes step S + 2
      const Cursor& prev = c[1];
      if (S + 2 == S0) {
        const int cum = __builtin_amdgcn_readfirstlane(s_cum[lo]);
        start_seq<STEP>(p, cn, lo, S0 - cum, first_row);
      } else if (prev.j + 1 == prev.nsteps) {
        int b = prev.b + 1;
        while (__builtin_amdgcn_readfirstlane(s_cum[b + 1]) == __builtin_amdgcn_readfirstlane(s_cum[b])) ++b;
        start_seq<STEP>(p, cn, b, 0, first_row);  // a step follows, so a sequence with steps does
      } else {
        cn = prev;
        cn.j = prev.j + 1;
      }
      if (cn.active) {
        const int at = cn.j * STEP, lblk = div_by(at, p.div_block);
        if (lblk != cn.lblk)
          enter_block(p, cn, lblk,
                      cn.pf_blk != -1 ? cn.pf_blk : load_uniform(p.block_tables + cn.b * p.bt_stride, lblk));
        const int off = at - lblk * p.block_size;
        rows = min(STEP, cn.len - at);
        base = cn.blk * p.blk_stride + off * p.slot_stride + head_off;
        issue_tile<FP8, false>(p, ln, base, rows, tiles);
        if (FP8) issue_scales(p, cn.blk * p.scale_blk_stride + scale_head + off, lane, scales);
        issued += F::kKOps;
        cn.mark = issued;
      }
    }
    if (live) {
      u32 pk[NT][2 * PARTS];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4 * PARTS], mx = kMaxFloor;
#pragma unroll
        for (int e = 0; e < 4 * PARTS; ++e) x[e] = s[nt][e >> 2][e & 3] * p.scale_log2;
        if (tail) {
#pragma unroll
          for (int e = 0; e < 4 * PARTS; ++e) {
            const int d = t0 + 16 * (e >> 2) + 4 * q4 + (e & 3) - ctx;  // the draft, or below 0
            if (!(d < 0 || (d < 64 && (seen[nt] >> (d & 63) & 1)))) x[e] = -INFINITY;
          }
        }
#pragma unroll
        for (int e = 0; e < 4 * PARTS; ++e) mx = fmaxf(mx, x[e]);
        mx = xor32_max(xor16_max(mx));
        const float m_new = fmaxf(m[nt], mx);
        const float alpha = fast_exp2(m[nt] - m_new);
        m[nt] = m_new;
        if (__any(alpha != 1.f)) {
          l[nt] *= alpha;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) acc[nt][mt] *= alpha;
        }
#pragma unroll
        for (int e = 0; e < 4 * PARTS; e += 2) {
          float w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            w[i] = fast_exp2(x[e + i] - m_new);
            l[nt] += w[i];
            if (FP8) w[i] = __builtin_amdgcn_ldexpf(w[i], static_cast<int>(vexp[e >> 2] >> (8 * ((e + i) & 3)) & 0xff) - 127);
          }
          pk[nt][e >> 1] = pack_bf16x2(w[0], w[1]);
        }
      }
      wait_tiles<F::kKOps, F::kVOps>(issued - c0.mark - F::kVOps);
#pragma unroll
      for (int kb = 0; kb < PARTS / 2; ++kb) {  // 32 tokens
        u32x4_t vt[8];
        if constexpr (FP8) {
          u32x2_t v8[8];
          const u32 at = tile + 4096 * kb;
          const u32 a[8] = {at + va[0], at + va[1], at + va[2], at + va[3],
                            at + va[4], at + va[5], at + va[6], at + va[7]};
          read_v8_tile(a, v8);
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) vt[mt] = widen8(v8[mt].x, v8[mt].y, 1.f);
        } else {
          u32x2_t vlo[8], vhi[8];
          const u32 a[8] = {tile + va[0], tile + va[1], tile + va[2], tile + va[3],
                            tile + va[4], tile + va[5], tile + va[6], tile + va[7]};
          read_v_tile(a, vlo, vhi);
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) vt[mt] = u32x4_t{vlo[mt].x, vlo[mt].y, vhi[mt].x, vhi[mt].y};
        }
        auto pf = [&](int nt) {
          return u32x4_t{pk[nt][4 * kb], pk[nt][4 * kb + 1], pk[nt][4 * kb + 2], pk[nt][4 * kb + 3]};
        };
        if (tail) {
          // A weight of 0 does not undo an infinity or NaN in V: tokens behind the last one are
          // cleared, and drafts that are not finite leave the product and are added one by one to
          // the rows that see them.
          const int at = t0 + 32 * kb + 4 * q4;  // element e of the lane is token at + e, or at + 12 + e for e >= 4
          u32x4_t live_w;
          u32 odd = 0;  // bit e: element e is a cached token that is not finite in some dim
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int t = at + 16 * (w >> 1) + 2 * (w & 1);
            live_w[w] = (t < c0.len ? 0xffffu : 0u) | (t + 1 < c0.len ? 0xffff0000u : 0u);
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
              const u32 x = vt[mt][w] & live_w[w];
              odd |= ((x & 0x7f80u) == 0x7f80u ? 1u : 0u) << (2 * w);
              odd |= ((x & 0x7f800000u) == 0x7f800000u ? 2u : 0u) << (2 * w);
            }
          }
          u32x4_t fine = live_w;
          if (__any(odd != 0)) {
#pragma unroll 1
            for (int i = 0; i < 32; ++i) {  // element e = i % 8 of the lanes of row group i / 8
              const int e = i & 7, g = i >> 3;
              if (!__any(q4 == g && (odd >> e & 1))) continue;
              const u32 mine = q4 == g ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
              u32x4_t only;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                only[w] = w == e >> 1 ? mine : 0u;
                fine[w] &= ~only[w];
              }
              const int d = t0 + 32 * kb + 16 * (e >> 2) + 4 * g + (e & 3) - ctx;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const bool sees = d < 0 || (seen[nt] >> (d & 63) & 1);
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) {
                  const mfma_f32x4_t with = mfma16(vt[mt] & only, pf(nt), acc[nt][mt]);
                  if (sees) acc[nt][mt] = with;
                }
              }
            }
          }
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) vt[mt] &= fine;
        }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][mt] = mfma16(vt[mt], pf(nt), acc[nt][mt]);
      }
    }
    if (issue && cn.active) {
      issue_tile<FP8, true>(p, ln, base, rows, tiles + kTile);
      issued += F::kVOps;
    }
    if (live && (c0.j + 1 == c0.nsteps || S + 1 == S1)) {
      const int from = S - c0.j, to = from + c0.nsteps;  // the sequence's steps
      emit(c0, from >= S0 && to <= S1, 2 * range + (from > S0 ? 1 : 0));
      reset();
    }
    c[0] = c[1];
    c[1] = c[2];
  }
}

// Joins the states of sequences that several ranges share: one wave for a query token and head.
// The wave's four 16-lane rows take the sequence's ranges round robin, 8 dims to a lane.
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(const TreeParams p) {
  const int row = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // token and q head
  const int b = blockIdx.y;
  const int cb = load_uniform(p.header, kHeaderInts + b), cb1 = load_uniform(p.header, kHeaderInts + b + 1);
  const int spr = load_uniform(p.header, 0);
  if (cb1 <= cb) return;  // no steps
  const int first = cb / spr, np = (cb1 - 1) / spr - first + 1;
  if (np <= 1) return;  // written already
  const SeqShape s = load_shape(p, b);
  if (row >= s.n * p.num_q_heads) return;
  const int tok = row / p.num_q_heads, h = row - tok * p.num_q_heads;
  const int kvh = div_by(h, p.div_group), g = h - kvh * p.group;
  const int r4 = (threadIdx.x >> 4) & 3, d = 8 * (threadIdx.x & 15);
  float m = kMaxFloor, l = 0.f, o[8] = {};
#pragma unroll 1
  for (int k = r4; k < np; k += 4) {
    const int place = 2 * (first + k) + (k == 0 && cb > first * spr ? 1 : 0);
    const int64_t at = (static_cast<int64_t>(place) * p.num_kv_heads + kvh) * p.max_rows + tok * p.group + g;
    const float2 st = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
    const float4 x = *reinterpret_cast<const float4*>(p.part_o + at * kDim + d);
    const float4 y = *reinterpret_cast<const float4*>(p.part_o + at * kDim + d + 4);
    const float m_new = fmaxf(m, st.x), alpha = fast_exp2(m - m_new), w = fast_exp2(st.x - m_new);
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    m = m_new;
    l = l * alpha + w * st.y;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = o[j] * alpha + w * v[j];
  }
  const float mm = xor32_max(xor16_max(m));
  const float w = fast_exp2(m - mm);
  const float sum = xor32_sum(xor16_sum(l * w));
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = xor32_sum(xor16_sum(o[j] * w)) * inv;
  if (r4 == 0) *reinterpret_cast<uint4*>(p.out + (s.q0 + tok) * p.o_tok_stride + h * p.o_head_stride + d) = pack8(o);
}

// Rows of a kv head are taken 16 at a time where they are no more, otherwise 32.
int row_tiles(int rows) { return rows <= 16 ? 1 : 2; }

// How a batch is cut: the same for the workspace's size and for the launch.
struct Plan {
  int nt, row_groups, streams, ranges;
  int64_t places() const { return 2ll * ranges; }
};
Plan plan_of(int64_t seqs, int max_q, int hq, int hkv, int64_t max_tokens_per_seq, int step, int workgroups) {
  Plan pl{};
  const int rows = max_q * (hq / hkv);
  pl.nt = row_tiles(rows);
  pl.row_groups = (rows + 16 * pl.nt - 1) / (16 * pl.nt);
  pl.streams = hkv * pl.row_groups;
  const int64_t steps = seqs * ((max_tokens_per_seq + step - 1) / step);
  pl.ranges = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(static_cast<int64_t>(workgroups) * kWaves / pl.streams, steps)));
  return pl;
}
int64_t workspace_of(const Plan& pl) {
  return kHeaderBytes + pl.places() * pl.streams * 16 * pl.nt * (kDim + 2) * 4;
}

// Workgroups of the kernel resident on the current device at once.
template <bool FP8, int NT>
int resident() {
  static std::atomic<int> cached[16];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 16) dev = 0;
  int v = cached[dev].load(std::memory_order_relaxed);
  if (v > 0) return v;
  int cus = 0, per_cu = 0;
  bool ok = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && cus > 0;
  if (!ok) cus = 256;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, tree_attention_kernel<FP8, NT>, kThreads, 0) != hipSuccess ||
      per_cu <= 0) {
    per_cu = 1;
    ok = false;
  }
  v = std::min(cus * per_cu, kMaxWorkgroups);
  if (ok) cached[dev].store(v, std::memory_order_relaxed);
  return v;
}

struct TreeArgs {
  bool fp8;
  const void* q;
  int64_t q_tok_stride, q_head_stride;
  const void* k_cache;
  const void* v_cache;
  int64_t blk_stride, slot_stride, head_stride;  // elements
  const void* k_scale;
  const void* v_scale;
  int64_t scale_blk_stride, scale_head_stride;
  int32_t num_cache_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  int32_t num_seqs, total_q, max_q, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks;
  const int64_t* mask;
  float softmax_scale;
  void* out;
  int64_t o_tok_stride, o_head_stride;
  void* workspace;
  size_t workspace_bytes;
};

int check_shape(const char* fn, int32_t max_q, int32_t hq, int32_t hkv, int32_t head_dim, int32_t block_size,
                int32_t max_blocks) {
  if (head_dim != kDim) return fail(KVP_EUNSUPPORTED, "%s: head_dim=%d (supported: 128)", fn, head_dim);
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0)
    return fail(KVP_EINVAL, "%s: num_q_heads=%d not a multiple of num_kv_heads=%d", fn, hq, hkv);
  if (hq / hkv > kMaxGroup)
    return fail(KVP_EUNSUPPORTED, "%s: GQA ratio %d (supported: up to %d)", fn, hq / hkv, kMaxGroup);
  if (hkv > 256) return fail(KVP_EUNSUPPORTED, "%s: num_kv_heads=%d (supported: up to 256)", fn, hkv);
  if (max_q < 1 || max_q > kMaxQ)
    return fail(KVP_EUNSUPPORTED, "%s: max_seqlen_q=%d (supported: 1 to %d)", fn, max_q, kMaxQ);
  if (block_size <= 0 || block_size % 64 != 0)
    return fail(KVP_EINVAL, "%s: block_size=%d must be a positive multiple of 64", fn, block_size);
  if (max_blocks <= 0) return fail(KVP_EINVAL, "%s: max_blocks_per_seq=%d", fn, max_blocks);
  if (static_cast<int64_t>(max_blocks) * block_size > kMaxTokens)
    return fail(KVP_EUNSUPPORTED, "%s: block tables of %d x %d tokens (supported: up to %d)", fn, max_blocks, block_size,
                kMaxTokens);
  return KVP_OK;
}

int check_args(const char* fn, const TreeArgs& a) {
  const int rc = check_shape(fn, a.max_q, a.num_q_heads, a.num_kv_heads, a.head_dim, a.block_size, a.max_blocks);
  if (rc != KVP_OK) return rc;
  if (a.num_seqs < 0 || a.total_q < 0 || a.num_cache_blocks <= 0)
    return fail(KVP_EINVAL, "%s: num_seqs=%d total_q=%d num_cache_blocks=%d", fn, a.num_seqs, a.total_q,
                a.num_cache_blocks);
  if (a.bt_stride < a.max_blocks)
    return fail(KVP_EINVAL, "%s: block_table_stride=%lld < max_blocks_per_seq=%d", fn,
                static_cast<long long>(a.bt_stride), a.max_blocks);
  if (a.num_seqs == 0 || a.total_q == 0) return KVP_OK;
  if (!a.q || !a.k_cache || !a.v_cache || !a.block_tables || !a.kv_lens || !a.out ||
      (a.fp8 && (!a.k_scale || !a.v_scale)))
    return fail(KVP_EINVAL, "%s: null pointer", fn);
  if (!aligned16(a.q) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.out))
    return fail(KVP_EINVAL, "%s: q, out and cache pointers must be 16-byte aligned", fn);
  auto off = [](const void* ptr, unsigned by) { return (reinterpret_cast<uintptr_t>(ptr) & (by - 1)) != 0; };
  if (off(a.block_tables, 4) || off(a.kv_lens, 4) || off(a.cu_q, 4) || off(a.mask, 8))
    return fail(KVP_EINVAL, "%s: misaligned block_tables / cache_seqlens / cu_seqlens_q / tree_mask", fn);
  const int64_t unit = a.fp8 ? 16 : 8;  // 16 bytes
  if (!mult8(a.q_tok_stride) || !mult8(a.q_head_stride) || !mult8(a.o_tok_stride) || !mult8(a.o_head_stride) ||
      a.blk_stride % unit || a.slot_stride % unit || a.head_stride % unit)
    return fail(KVP_EINVAL, "%s: q, out and cache strides must be multiples of 16 bytes", fn);
  const int64_t size = a.fp8 ? 1 : 2;
  if (a.slot_stride < 0) return fail(KVP_EINVAL, "%s: negative slot stride", fn);
  if (a.slot_stride * size > (1 << 24))
    return fail(KVP_EUNSUPPORTED, "%s: slot stride of %lld elements (a step is addressed in 32 bits)", fn,
                static_cast<long long>(a.slot_stride));
  if (a.fp8 && (off(a.k_scale, 4) || off(a.v_scale, 4) || a.scale_blk_stride % 4 || a.scale_head_stride % 4 ||
                a.scale_blk_stride < 0 || a.scale_head_stride < 0))
    return fail(KVP_EINVAL, "%s: scale pointers and strides must be multiples of 4 bytes", fn);
  return KVP_OK;
}

template <bool FP8, int NT>
int launch(const char* fn, const TreeArgs& a, hipStream_t stream) {
  const int most = std::min(a.num_seqs, kSeqsPerLaunch);
  const int64_t tokens = static_cast<int64_t>(a.max_blocks) * a.block_size;
  const Plan pl = plan_of(most, a.max_q, a.num_q_heads, a.num_kv_heads, tokens, Format<FP8>::kStep,
                          resident<FP8, NT>());
  const size_t need = static_cast<size_t>(workspace_of(pl));
  if (!a.workspace || a.workspace_bytes < need)
    return fail(KVP_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, a.workspace_bytes, need);
  const int64_t size = FP8 ? 1 : 2;
  TreeParams p{};
  p.q = static_cast<const uint16_t*>(a.q);
  p.q_tok_stride = a.q_tok_stride;
  p.q_head_stride = a.q_head_stride;
  p.k_cache = static_cast<const uint8_t*>(a.k_cache);
  p.v_cache = static_cast<const uint8_t*>(a.v_cache);
  p.blk_stride = a.blk_stride * size;
  p.slot_stride = a.slot_stride * size;
  p.head_stride = a.head_stride * size;
  p.k_scale = static_cast<const uint8_t*>(a.k_scale);
  p.v_scale = static_cast<const uint8_t*>(a.v_scale);
  p.scale_blk_stride = a.scale_blk_stride;
  p.scale_head_stride = a.scale_head_stride;
  p.num_cache_blocks = a.num_cache_blocks;
  p.block_size = a.block_size;
  p.max_blocks = a.max_blocks;
  p.bt_stride = a.bt_stride;
  p.max_q = a.max_q;
  p.num_q_heads = a.num_q_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.group = a.num_q_heads / a.num_kv_heads;
  p.mask = a.mask;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  p.o_tok_stride = a.o_tok_stride;
  p.o_head_stride = a.o_head_stride;
  p.streams = pl.streams;
  p.ranges = pl.ranges;
  p.row_groups = pl.row_groups;
  p.max_rows = pl.row_groups * 16 * pl.nt;
  p.div_streams = divisor(pl.streams);
  p.div_row_groups = divisor(pl.row_groups);
  p.div_ranges = divisor(pl.ranges);
  p.div_block = divisor(a.block_size);
  p.div_group = divisor(p.group);
  char* ws = static_cast<char*>(a.workspace);
  p.header = reinterpret_cast<int32_t*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + kHeaderBytes);
  p.part_ml = p.part_o + pl.places() * a.num_kv_heads * p.max_rows * kDim;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(pl.ranges) * pl.streams + kWaves - 1) / kWaves);
  for (int b0 = 0; b0 < a.num_seqs; b0 += kSeqsPerLaunch) {
    p.num_seqs = std::min(kSeqsPerLaunch, a.num_seqs - b0);
    p.block_tables = a.block_tables + b0 * a.bt_stride;
    p.kv_lens = a.kv_lens + b0;
    p.cu_q = a.cu_q ? a.cu_q + b0 : nullptr;
    const int64_t row0 = a.cu_q ? 0 : b0;  // without cu_q row b is sequence b's
    p.q = static_cast<const uint16_t*>(a.q) + row0 * a.q_tok_stride;
    p.out = static_cast<uint16_t*>(a.out) + row0 * a.o_tok_stride;
    p.total_q = a.cu_q ? a.total_q : p.num_seqs;
    hipLaunchKernelGGL((tree_attention_kernel<FP8, NT>), dim3(grid), dim3(kThreads), 0, stream, p);
    if (pl.ranges > 1)
      hipLaunchKernelGGL(tree_merge_kernel, dim3((a.max_q * a.num_q_heads + kWaves - 1) / kWaves, p.num_seqs),
                         dim3(kThreads), 0, stream, p);
    const int rc = launch_status(fn);
    if (rc != KVP_OK) return rc;
  }
  return KVP_OK;
}

int enqueue(const char* fn, const TreeArgs& a, void* stream) {
  const int rc = check_args(fn, a);
  if (rc != KVP_OK || a.num_seqs == 0 || a.total_q == 0) return rc;
  if (reinterpret_cast<uintptr_t>(a.workspace) & 255u)
    return fail(KVP_EINVAL, "%s: workspace must be 256-byte aligned", fn);
  const auto s = static_cast<hipStream_t>(stream);
  const bool one = row_tiles(a.max_q * (a.num_q_heads / a.num_kv_heads)) == 1;
  if (a.fp8) return one ? launch<true, 1>(fn, a, s) : launch<true, 2>(fn, a, s);
  return one ? launch<false, 1>(fn, a, s) : launch<false, 2>(fn, a, s);
}

}  // namespace
}  // namespace kvp

using namespace kvp;

extern "C" size_t kvp_tree_workspace_bytes(int32_t max_num_seqs, int32_t max_seqlen_q, int32_t num_q_heads,
                                           int32_t num_kv_heads, int32_t head_dim, int32_t max_blocks_per_seq,
                                           int32_t block_size) {
  if (max_num_seqs <= 0 ||
      check_shape("", max_seqlen_q, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq) != KVP_OK)
    return 0;
  // ranges x streams of any launch within these sizes, on any device; it grows with each of them
  Plan pl = plan_of(1, max_seqlen_q, num_q_heads, num_kv_heads, 1, 1, 0);
  const int64_t steps = static_cast<int64_t>(std::min(max_num_seqs, kSeqsPerLaunch)) *
                        ((static_cast<int64_t>(max_blocks_per_seq) * block_size + 31) / 32);
  pl.streams = static_cast<int>(std::min<int64_t>(std::max(kMaxWorkgroups * kWaves, pl.streams), steps * pl.streams));
  pl.ranges = 1;
  return static_cast<size_t>(workspace_of(pl));
}

extern "C" int kvp_paged_decode_fp8(const void* q, int64_t q_seq_stride, int64_t q_head_stride, const void* k_cache,
                                    const void* v_cache, int64_t cache_block_stride, int64_t cache_slot_stride,
                                    int64_t cache_head_stride, const void* k_scale, const void* v_scale,
                                    int64_t scale_block_stride, int64_t scale_head_stride, int32_t num_cache_blocks,
                                    const int32_t* block_tables, int64_t block_table_stride,
                                    const int32_t* context_lens, int32_t num_seqs, int32_t num_q_heads,
                                    int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                    int32_t max_blocks_per_seq, float softmax_scale, void* out, int64_t out_seq_stride,
                                    int64_t out_head_stride, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const TreeArgs a = {true, q, q_seq_stride, q_head_stride, k_cache, v_cache, cache_block_stride, cache_slot_stride,
                      cache_head_stride, k_scale, v_scale, scale_block_stride, scale_head_stride, num_cache_blocks,
                      block_tables, block_table_stride, nullptr, context_lens, num_seqs, num_seqs, 1, num_q_heads,
                      num_kv_heads, head_dim, block_size, max_blocks_per_seq, nullptr, softmax_scale, out,
                      out_seq_stride, out_head_stride, workspace, workspace_bytes};
  return enqueue("kvp_paged_decode_fp8", a, stream);
}

extern "C" int kvp_tree_attention(const void* q, int64_t q_tok_stride, int64_t q_head_stride, const void* k_cache,
                                  const void* v_cache, int64_t cache_block_stride, int64_t cache_slot_stride,
                                  int64_t cache_head_stride, const void* k_scale, const void* v_scale,
                                  int64_t scale_block_stride, int64_t scale_head_stride, int32_t num_cache_blocks,
                                  const int32_t* block_tables, int64_t block_table_stride,
                                  const int32_t* cu_seqlens_q, const int32_t* cache_seqlens, int32_t num_seqs,
                                  int32_t total_q, int32_t max_seqlen_q, const int64_t* tree_mask,
                                  int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                  int32_t max_blocks_per_seq, float softmax_scale, void* out, int64_t out_tok_stride,
                                  int64_t out_head_stride, void* workspace, size_t workspace_bytes, void* stream) {
  static const char fn[] = "kvp_tree_attention";
  clear_error();
  if ((k_scale == nullptr) != (v_scale == nullptr)) return fail(KVP_EINVAL, "%s: one of the scales is missing", fn);
  if (!cu_seqlens_q && num_seqs > 0) return fail(KVP_EINVAL, "%s: null cu_seqlens_q", fn);
  const TreeArgs a = {k_scale != nullptr, q, q_tok_stride, q_head_stride, k_cache, v_cache, cache_block_stride,
                      cache_slot_stride, cache_head_stride, k_scale, v_scale, scale_block_stride, scale_head_stride,
                      num_cache_blocks, block_tables, block_table_stride, cu_seqlens_q, cache_seqlens, num_seqs,
                      total_q, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                      tree_mask, softmax_scale, out, out_tok_stride, out_head_stride, workspace, workspace_bytes};
  return enqueue(fn, a, stream);
}
