// Attention of a few query tokens per sequence over its paged KV cache, in bf16 or quantised:
// the drafted tokens of a speculative step (kvp_tree_attention), and the one token of a decode
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
// Work decomposition: the tokens of all sequences are laid end to end in steps of 64 (32 for few rows
// on a bf16 cache) and cut into equally long ranges, whatever the lengths.  With up to 16 rows per
// kv head a wave takes one head over one range (tree_few_kernel); with more, a workgroup does, whose
// four waves share the tiles and take 32 rows each, and of more than 128 rows blocks of 128 run side
// by side (tree_many_kernel).  A sequence that lies in one range gets its output from
// there; of the others every range leaves (max, sum, unnormalised sum of V) in 32 bits, which
// tree_merge_kernel joins.  Only the first and the last sequence of a range can be cut by it, so a
// range has two places for states whatever the batch: the first for a sequence that it takes up at
// its own start, the second for one that starts later and goes on behind it.
//
// Layouts are those of the decode kernel (lane l: n = l % 16, q4 = l / 16): S = K Q^T has tokens
// 4 q4 + j of every 16 in the lane and row n as its column, O^T = V^T P^T takes P from the same
// registers.  e4m3 is widened to bf16, exactly, on its way from LDS to the matrix cores, K with its
// scale (the lane's own token), V's scale going into P.  Up to 16 rows, where the matrix cores wait for
// memory, P enters its product as two bf16 parts, off by 2^-15 of each weight (one part alone was no
// faster); beyond, where they bound it, P is rounded to bf16 as in the prefill: at most 2^-8 of each
// weight, of either sign, so below the rounding of the bf16 output where the values do not cancel.  The
// sum of the weights is of the unrounded ones, and running maxima, sums and products stay in 32 bits.
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
constexpr int kMaxFew = 1024, kMaxMany = 512;  // units at once at most: bounds the workspace, whatever the device

template <bool FP8>
struct Format {
  static constexpr int kRow = FP8 ? kDim : 2 * kDim;  // bytes of a token's row
  static constexpr int kStep = kTile / kRow;          // tokens per step
  static constexpr int kSubs = kStep / 32;            // products of 32 tokens each
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
  float* part_o;    // [range][2][kv head][rows][128]
  float* part_ml;   // [range][2][kv head][rows][2]
  int32_t ranges, streams, blocks, rows;  // streams: kv heads x blocks of rows; rows: of all blocks
  u32 q_flip;       // sign bits that turn a negative scale into a positive one
  Divisor div_streams, div_blocks, div_ranges, div_block, div_group;
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
    const int per = p.num_q_heads * (kDim / 8);  // 16-byte chunks of a row; a sequence's may pass 32 bits
    int tok = 0;
#pragma unroll 1
    for (int i = threadIdx.x;; i += kThreads) {
      while (i >= per) i -= per, ++tok;
      if (tok >= s.n) break;
      *reinterpret_cast<uint4*>(p.out + (s.q0 + tok) * p.o_tok_stride + i / (kDim / 8) * p.o_head_stride +
                                i % (kDim / 8) * 8) = make_uint4(w, w, w, w);
    }
  }
}

// A wave-uniform value in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return static_cast<int64_t>(uniform(static_cast<int>(x >> 32))) << 32 | static_cast<u32>(uniform(static_cast<int>(x)));
}

// The range of unit `unit` (stream fastest), or false if it has none.  One workgroup leaves what the
// merge needs.
struct Range {
  int index, S0, S1;  // steps
  int first;          // the sequence that holds step S0
  int kvh, block;
};
__device__ __forceinline__ bool find_range(const TreeParams& p, const int* s_cum, int unit, Range& r) {
  const int B = p.num_seqs, total = uniform(s_cum[B]);
  const int spr = max(1, div_by(total + p.ranges - 1, p.div_ranges));
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) p.header[0] = spr;
    for (int b = threadIdx.x; b <= B; b += kThreads) p.header[kHeaderInts + b] = s_cum[b];
  }
  r.index = div_by(unit, p.div_streams);
  const int stream = unit - r.index * p.streams;
  r.kvh = div_by(stream, p.div_blocks);
  r.block = stream - r.kvh * p.blocks;
  r.S0 = r.index * spr;
  r.S1 = min(total, r.S0 + spr);
  if (r.index >= p.ranges || r.S0 >= r.S1) return false;
  int lo = 0, hi = B;  // s_cum[lo] <= S0 < s_cum[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_cum[mid] <= r.S0) lo = mid;
    else hi = mid;
  }
  r.first = uniform(lo);
  return true;
}

// A place in the steps of a range.
struct Cursor {
  int b, j, nsteps;  // sequence, step within it, its steps
  int q0, n, len;
  int lblk, blk, pf_blk;  // logical block, its id, and the id of the next one (-1: not loaded)
  int bad;           // a needed block id was out of range
  int mark;          // vector memory operations issued up to the step's K tile
};
__device__ __forceinline__ int table_entry(const TreeParams& p, int b, int lblk) {
  return load_uniform(p.block_tables + b * p.bt_stride, lblk);
}
__device__ __forceinline__ void enter_block(const TreeParams& p, Cursor& c, int lblk, int blk) {
  const int bad = blk < 0 || blk >= p.num_cache_blocks;
  c.bad |= bad;
  c.blk = bad ? 0 : blk;
  c.lblk = lblk;
  c.pf_blk = (lblk + 1) * p.block_size < c.len ? table_entry(p, c.b, lblk + 1) : -1;
}
template <int STEP>
__device__ __forceinline__ void start_seq(const TreeParams& p, Cursor& c, int b, int j) {
  const SeqShape s = load_shape(p, b);
  c.b = b;
  c.j = j;
  c.q0 = s.q0;
  c.n = s.n;
  c.len = s.len;
  c.nsteps = (s.len + STEP - 1) / STEP;
  c.bad = 0;
  const int lblk = div_by(j * STEP, p.div_block);
  enter_block(p, c, lblk, table_entry(p, b, lblk));
}
// c: the step behind prev's, which there is.
template <int STEP>
__device__ __forceinline__ void next_step(const TreeParams& p, const int* s_cum, const Cursor& prev, Cursor& c) {
  if (prev.j + 1 < prev.nsteps) {
    c = prev;
    c.j = prev.j + 1;
    const int lblk = div_by(c.j * STEP, p.div_block);
    if (lblk != c.lblk) enter_block(p, c, lblk, c.pf_blk != -1 ? c.pf_blk : table_entry(p, c.b, lblk));
  } else {
    int b = prev.b + 1;
    while (uniform(s_cum[b + 1]) == uniform(s_cum[b])) ++b;
    start_seq<STEP>(p, c, b, 0);
  }
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
  for (int i = 0; i < 8; ++i)  // nontemporal: every row is read once
    raw_buffer_load_lds(rsrc, (LdsPtr)(tile + 1024 * i), 16,
                        min(t.row_off + kPer * i * stride, last) + (V ? t.v_chunk[i & 1] : t.k_chunk[i & 3]), 0, 0, 2);
}
// The scales of a step's 64 tokens: K's bytes, then V's.
__device__ __forceinline__ void issue_scales(const TreeParams& p, int64_t base, int lane, char* to) {
  if (lane < 16) {
    raw_buffer_load_lds(buffer_rsrc(p.k_scale + base, 64), (LdsPtr)to, 4, 4 * lane, 0, 0, 0);
    raw_buffer_load_lds(buffer_rsrc(p.v_scale + base, 64), (LdsPtr)(to + 64), 4, 4 * lane, 0, 0, 0);
  }
}

// K of a step in e4m3: the lane's 16 bytes at a0 and a1 of each 16 tokens, k[4 i + part].
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

// A weight times its token's V scale, byte `i` of `bytes`: exact down to 2^-126, and 0 stays 0 whatever the byte (those
// behind the last token can be anything).  Two instructions, one of which picks the byte; -127 is held in a vector
// register, since scalar ones are short (32 sequences of 8192, 8 drafts: 123 us against 129).
__device__ __forceinline__ float scale_weight(float w, u32 bytes, int i) {
  int less = -127;
  asm("" : "+v"(less));
  return __builtin_ldexpf(w, static_cast<int>(bytes >> (8 * i) & 0xffu) + less);
}

// Whether a row sees draft d (below 0: a token of the context), given the bits of its drafts.
__device__ __forceinline__ bool sees(uint64_t seen, int d) {
  return (d < 0) | ((d < kMaxQ) & static_cast<int>(seen >> (d & (kMaxQ - 1))));
}

// Weights of two tokens as bf16 parts that sum up to them, but for 2^-15 of each: `hi` is cut off just below the weight,
// so that the rest is above 0 even of a weight that bf16 holds (0 times an infinity of V would be NaN).
__device__ __forceinline__ void split_weights(float w0, float w1, u32& hi, u32& lo) {
  const u32 h0 = __builtin_elementwise_sub_sat(__float_as_uint(w0), 1u) & 0xffff0000u;
  const u32 h1 = __builtin_elementwise_sub_sat(__float_as_uint(w1), 1u) & 0xffff0000u;
  hi = h0 >> 16 | h1;
  lo = pack_bf16x2(w0 - __uint_as_float(h0), w1 - __uint_as_float(h1));
}
struct Split {
  u32x4_t hi, lo;
};
__device__ __forceinline__ mfma_f32x4_t mfma16_split(u32x4_t a, const Split& b, mfma_f32x4_t c) {
  return mfma16(a, b.lo, mfma16(a, b.hi, c));
}

// The 16 rows that a wave works on, and the online softmax over the tokens that they have met.
struct Rows {
  int row, tok, head;  // of the lane's column
  u32x4_t q[4];
  uint64_t seen;  // the drafts that the column's token sees
  float m, l;
  mfma_f32x4_t acc[8];  // dims 16 mt + 4 q4 + j

  __device__ __forceinline__ void place(const TreeParams& p, int kvh, int n) {
    row = n;
    tok = div_by(row, p.div_group);
    head = kvh * p.group + row - tok * p.group;
  }
  __device__ __forceinline__ void reset() {
    m = kMaxFloor;
    l = 0.f;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) acc[mt] = mfma_f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // WIDE: dims in the order of 16-byte reads of an e4m3 row.
  template <bool WIDE>
  __device__ __forceinline__ void load_q(const TreeParams& p, const Cursor& c, int q4) {
    const int i = min(tok, c.n - 1);
    const uint16_t* src = p.q + (c.q0 + i) * p.q_tok_stride + head * p.q_head_stride;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      q[kk] = *reinterpret_cast<const u32x4_t*>(
          src + (WIDE ? 64 * (kk >> 1) + 16 * q4 + 8 * (kk & 1) : 32 * kk + 8 * q4)) ^ p.q_flip;
    const uint64_t all = ~0ull >> (64 - c.n);
    const uint64_t bits = p.mask ? static_cast<uint64_t>(p.mask[c.q0 + i]) : ~0ull >> (63 - i);
    seen = bits & all;
    asm volatile("" : "+v"(seen));  // waited for here, not where its registers are next written
  }
  // Weights of 32 tokens from their scores s0 (tokens 4 q4 + j) and s1 (16 + 4 q4 + j), split as the second
  // product's operands; `draft` is the first token's draft, below 0 in the context.  The running maximum m
  // follows every score above it: weights are 1 at most, so sums stay within the number of tokens times the
  // largest V.  The loop waits for memory, and neither the multiplications of the sums nor the second part's
  // products cost time.
  // SCALED: each is multiplied by its V scale, the bytes of v0 and v1.
  template <bool SCALED>
  __device__ __forceinline__ Split weigh(mfma_f32x4_t s0, mfma_f32x4_t s1, u32 v0, u32 v1, float scale, bool tail,
                                         int draft, int q4) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < 4 ? s0[e] : s1[e - 4];
    if (tail) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = draft + 16 * (e >> 2) + 4 * q4 + (e & 3);
        x[e] = sees(seen, d) ? x[e] : -INFINITY;
      }
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
    mx = xor32_max(xor16_max(mx)) * scale;
    if (__any(mx > m)) {
      const float m_new = fmaxf(m, mx);
      const float alpha = fast_exp2(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) acc[mt] *= alpha;
    }
    Split pf;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float w0 = fast_exp2(fmaf(x[e], scale, -m)), w1 = fast_exp2(fmaf(x[e + 1], scale, -m));
      l += w0 + w1;
      if (SCALED) {
        w0 = scale_weight(w0, e < 4 ? v0 : v1, e & 3);
        w1 = scale_weight(w1, e < 4 ? v0 : v1, (e & 3) + 1);
      }
      u32 hi, lo;
      split_weights(w0, w1, hi, lo);
      pf.hi[e >> 1] = hi;
      pf.lo[e >> 1] = lo;
    }
    return pf;
  }
  // The tail's V: a weight of 0 does not undo an infinity or NaN, so tokens behind the last one (from
  // `left` on) are cleared, and drafts that are not finite leave the product and are added one by one
  // to the rows that see them.
  __device__ __forceinline__ void clean(u32x4_t (&vt)[8], const Split& pf, int draft, int left, int q4) {
    u32x4_t fine;
    u32 odd = 0;  // bit e: element e (token 4 q4 + e, or 12 + 4 q4 + e for e >= 4) is cached and not finite
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int t = 4 * q4 + 16 * (w >> 1) + 2 * (w & 1);
      fine[w] = (t < left ? 0xffffu : 0u) | (t + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        const u32 v = vt[mt][w] & fine[w];
        odd |= ((v & 0x7f80u) == 0x7f80u ? 1u : 0u) << (2 * w);
        odd |= ((v & 0x7f800000u) == 0x7f800000u ? 2u : 0u) << (2 * w);
      }
    }
    if (__any(odd != 0)) {
#pragma unroll 1
      for (int i = 0; i < 32; ++i) {  // element e = i % 8 of the lanes of group i / 8
        const int e = i & 7, g = i >> 3;
        if (!__any(q4 == g && (odd >> e & 1))) continue;
        const u32 half = q4 == g ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
        u32x4_t only;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          only[w] = w == e >> 1 ? half : 0u;
          fine[w] &= ~only[w];
        }
        const int d = draft + 16 * (e >> 2) + 4 * g + (e & 3);
        const bool mine = sees(seen, d);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          const mfma_f32x4_t with = mfma16_split(vt[mt] & only, pf, acc[mt]);
          if (mine) acc[mt] = with;
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) vt[mt] &= fine;
  }
  // The rows' output where a range held all of the sequence, otherwise a partial state at `place`.
  __device__ __forceinline__ void emit(const TreeParams& p, const Cursor& c, int kvh, bool whole, int place, int q4) {
    float sum = xor32_sum(xor16_sum(l));
    if (c.bad) sum = NAN;
    if (tok >= c.n) return;
    if (whole) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint16_t* out = p.out + (c.q0 + tok) * p.o_tok_stride + head * p.o_head_stride + 4 * q4;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        const mfma_f32x4_t o = acc[mt] * inv;
        *reinterpret_cast<u32x2_t*>(out + 16 * mt) = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
      }
    } else {
      const int64_t at = (static_cast<int64_t>(place) * p.num_kv_heads + kvh) * p.rows + row;
      float* part = p.part_o + at * kDim + 4 * q4;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) *reinterpret_cast<mfma_f32x4_t*>(part + 16 * mt) = acc[mt];
      if (q4 == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, sum);
    }
  }
};

// Up to 16 rows per kv head: a wave for itself, with the tiles of two steps in flight in its own LDS,
// so that no wave waits for another.  One query token and e4m3, 8 kv heads: 256 sequences of 100 to
// 2048 tokens take 95 us (6.0 TB/s), 128 of 1024 to 32768 643 us (6.9 TB/s; with loads that are not
// nontemporal 80 more), one of 611 7.5 us (a chain of dependent loads).  Four drafts of 32 sequences of
// 8192 at four query heads to a kv head: 162 us in bf16 (6.6 TB/s), 91 in e4m3 (6.0 TB/s).
template <bool FP8>
__global__ __launch_bounds__(kThreads) void tree_few_kernel(const TreeParams p) {
  using F = Format<FP8>;
  constexpr int STEP = F::kStep, SUBS = F::kSubs;
  __shared__ __attribute__((aligned(16))) char s_tile[kWaves][2][2 * kTile];
  __shared__ __attribute__((aligned(16))) char s_scale[FP8 ? kWaves : 1][2][128];
  __shared__ int s_cum[kSeqsPerLaunch + 1];
  __shared__ int s_part[kWaves];

  const int lane = threadIdx.x & 63, wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int n = lane & 15, q4 = lane >> 4;
  build_prefix<STEP>(p, s_cum, s_part);
  fill_rows(p, s_cum);
  Range r;
  if (!find_range(p, s_cum, static_cast<int>(blockIdx.x) * kWaves + wave, r)) return;  // no barrier follows

  const int64_t head_off = r.kvh * p.head_stride, scale_head = r.kvh * p.scale_head_stride;
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
  Rows rows;
  rows.place(p, r.kvh, n);
  rows.reset();

  // Iteration S computes step S and issues the tiles of step S + 2, each as soon as its tile has been
  // read; the first two only issue.  c[i]: the place of step S + i.
  Cursor c[3] = {};
  Cursor &c0 = c[0], &cn = c[2];
  int issued = 0;
#pragma unroll 1
  for (int S = r.S0 - 2; S < r.S1; ++S) {
    const int buf = (S - r.S0) & 1;
    char* const tiles = s_tile[wave][buf];
    char* const scales = s_scale[FP8 ? wave : 0][buf];
    const u32 tile = lds_addr(tiles);
    const bool live = S >= r.S0, issue = S + 2 < r.S1;
    const int t0 = c0.j * STEP, ctx = c0.len - c0.n;
    // ---- S = K Q^T of the step
    mfma_f32x4_t s[2 * SUBS];
    u32 vexp[2 * SUBS] = {};
    if (live) {
      if (S == r.S0 || c0.j == 0) rows.load_q<FP8>(p, c0, q4);
      wait_tiles<F::kKOps, F::kVOps>(issued - c0.mark);
#pragma unroll
      for (int h = 0; h < 2 * SUBS; ++h) s[h] = mfma_f32x4_t{0.f, 0.f, 0.f, 0.f};
      u32x4_t k[8];
      if constexpr (FP8) {
        u32 kexp[4];
        const u32 at = lds_addr(scales);
        read_scales(at + n, at + 64 + 4 * q4, kexp, vexp);
        read_k8_tile(tile + ka[0], tile + ka[1], k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const u32x4_t w = k[4 * (kk >> 1) + h];
            s[h] = mfma16(widen8(w[2 * (kk & 1)], w[2 * (kk & 1) + 1], __uint_as_float(kexp[h] << 23)), rows.q[kk], s[h]);
          }
      } else {
        const u32 at[4] = {tile + ka[0], tile + ka[1], tile + ka[2], tile + ka[3]};
        read_k_tile(at, k);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i & 1] = mfma16(k[i], rows.q[i >> 1], s[i & 1]);
      }
    }
    int64_t base = 0;
    int left = 0;
    if (issue) {  // K has been read: its tile takes step S + 2
      if (S + 2 == r.S0) start_seq<STEP>(p, cn, r.first, r.S0 - uniform(s_cum[r.first]));
      else next_step<STEP>(p, s_cum, c[1], cn);
      const int off = cn.j * STEP - cn.lblk * p.block_size;
      left = min(STEP, cn.len - cn.j * STEP);
      base = uniform(cn.blk * p.blk_stride + off * p.slot_stride + head_off);
      issue_tile<FP8, false>(p, ln, base, left, tiles);
      if (FP8) issue_scales(p, cn.blk * p.scale_blk_stride + scale_head + off, lane, scales);
      issued += F::kKOps;
      cn.mark = issued;
    }
    if (live) {
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {  // 32 tokens
        const int draft = t0 + 32 * sub - ctx;
        const bool tail = draft > -32;  // drafts among them, or the last token in front of them
        const Split pf = rows.template weigh<FP8>(s[2 * sub], s[2 * sub + 1], vexp[2 * sub], vexp[2 * sub + 1],
                                                  p.scale_log2, tail, draft, q4);
        // ---- O^T += V^T P^T
        if (sub == 0) wait_tiles<F::kKOps, F::kVOps>(issued - c0.mark - F::kVOps);
        u32x4_t vt[8];
        if constexpr (FP8) {
          u32x2_t v8[8];
          const u32 at = tile + 4096 * sub;
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
        if (tail) rows.clean(vt, pf, draft, c0.len - t0 - 32 * sub, q4);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) rows.acc[mt] = mfma16_split(vt[mt], pf, rows.acc[mt]);
      }
    }
    if (issue) {
      issue_tile<FP8, true>(p, ln, base, left, tiles + kTile);
      issued += F::kVOps;
    }
    if (live && (c0.j + 1 == c0.nsteps || S + 1 == r.S1)) {
      const int from = S - c0.j, to = from + c0.nsteps;  // the sequence's steps
      rows.emit(p, c0, r.kvh, from >= r.S0 && to <= r.S1, 2 * r.index + (from > r.S0 ? 1 : 0), q4);
      rows.reset();
    }
    c[0] = c[1];
    c[1] = c[2];
  }
}

// More rows: the four waves of a workgroup share tiles of 64 tokens, and a wave has 32 rows
// (v_mfma_f32_32x32x16_bf16; lane l: row l % 32, hf = l / 32).  KW = 1: wave w has rows 32 w .. of a block of
// 128.  KW = 2, up to 64 rows: waves w and w + 2 have rows 32 (w % 2) .. and 32 tokens of every step each; their
// states are joined through LDS where the sequence ends.
//
// Two workgroups on a CU: one computes while the other waits.  bf16: two tiles, the next one loaded while a tile
// is used.  e4m3: four, three of them being loaded, and every wave widens what it reads.
//
// Matrix and vector instructions take most of the time, and they add up: 64 tokens of a wave with 32 rows are 1024
// cycles of products and 281 vector instructions in bf16, 501 in e4m3 (whole launches, counted).  End to end they
// would fill 72% of the first call below and 82% of the last; what is left is a step's chain of LDS reads,
// products and softmax, which the other workgroup covers in part.  24 sequences of 1000 to 9000 tokens with 61 to 64
// drafts at 64 heads take 320 us (775 TFLOP/s); a call of 32 of 8192 with 8, 16 and 25 drafts at 32 heads in e4m3 121,
// 151 and 210 us (KW = 2, 2, 1), with tiles that are widened once for all waves through LDS 146, 168 and 235.
//
// Tile rows are 256 bytes, 16-byte chunk c of token r at chunk c ^ (r % 16) of K and c ^ 4 (r % 4) of V; in
// e4m3 128 bytes, c ^ ((r / 2) % 8) and c ^ ((r & 2) + (r & 8) / 2).  The lane
// gets the scores of tokens 8 (i / 4) + 4 hf + i % 4 of each 32, and of O^T dims 32 mb + 8 (j / 4) + 4 hf + j % 4.
constexpr int kManyStep = 64;
constexpr int kTileElems = kManyStep * kDim;
constexpr int kRawTiles = 4, kRawBytes = 2 * kTile + 2 * kManyStep;

// One or two blocks of 32 tokens (4096 bytes each) in e4m3: K from the lane's four addresses in the first, its
// exponent byte at `ka`, those of V's tokens 8 i + 0 .. 3 at `va` + 8 i.
template <int BLOCKS>
__device__ __forceinline__ void read_k8_blocks(const u32 (&at)[4], u32 ka, u32 va, u32x4_t (&k)[BLOCKS][4],
                                               u32 (&kexp)[BLOCKS], u32 (&vexp)[BLOCKS][4]) {
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
    asm volatile(
        "ds_read_u8 %4, %13\n\t"
        "ds_read_b128 %0, %9\n\tds_read_b128 %1, %10\n\tds_read_b128 %2, %11\n\tds_read_b128 %3, %12\n\t"
        "ds_read_b32 %5, %14\n\tds_read_b32 %6, %14 offset:8\n\tds_read_b32 %7, %14 offset:16\n\t"
        "ds_read_b32 %8, %14 offset:24\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[b][0]), "=&v"(k[b][1]), "=&v"(k[b][2]), "=&v"(k[b][3]), "=&v"(kexp[b]), "=&v"(vexp[b][0]),
          "=&v"(vexp[b][1]), "=&v"(vexp[b][2]), "=&v"(vexp[b][3])
        : "v"(at[0] + 4096 * b), "v"(at[1] + 4096 * b), "v"(at[2] + 4096 * b), "v"(at[3] + 4096 * b), "v"(ka + 32 * b),
          "v"(va + 32 * b)
        : "memory");
}
// V of 16 or 32 tokens in e4m3, transposed: 8 bytes at a[mb] + off, and 2048 further.
__device__ __forceinline__ void read_v8_16(const int (&a)[4], int off, u32x2_t (&v)[4]) {
  asm volatile(
      "ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %5\n\t"
      "ds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %7\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(a[0] + off), "v"(a[1] + off), "v"(a[2] + off), "v"(a[3] + off)
      : "memory");
}
__device__ __forceinline__ void read_v8_32(const int (&a)[4], int off, u32x2_t (&v)[2][4]) {
  asm volatile(
      "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %9\n\t"
      "ds_read_b64_tr_b8 %2, %10\n\tds_read_b64_tr_b8 %3, %11\n\t"
      "ds_read_b64_tr_b8 %4, %8 offset:2048\n\tds_read_b64_tr_b8 %5, %9 offset:2048\n\t"
      "ds_read_b64_tr_b8 %6, %10 offset:2048\n\tds_read_b64_tr_b8 %7, %11 offset:2048\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[1][2]),
        "=&v"(v[1][3])
      : "v"(a[0] + off), "v"(a[1] + off), "v"(a[2] + off), "v"(a[3] + off)
      : "memory");
}

// All waves' LDS accesses are done, but not their loads.
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <bool FP8, int KW>
__global__ __launch_bounds__(kThreads, 2) void tree_many_kernel(const TreeParams p) {
  constexpr int STEP = kManyStep, BLOCKS = 2 / KW;  // blocks of 32 tokens of a step that a wave takes
  // bf16: the compiler has to tell the tile that is read from the one that is loaded
  __shared__ __attribute__((aligned(16))) uint16_t s_k0[FP8 ? 8 : kTileElems];
  __shared__ __attribute__((aligned(16))) uint16_t s_v0[FP8 ? 8 : kTileElems];
  __shared__ __attribute__((aligned(16))) uint16_t s_k1[FP8 ? 8 : kTileElems];
  __shared__ __attribute__((aligned(16))) uint16_t s_v1[FP8 ? 8 : kTileElems];
  // e4m3: K, V, K's scales, V's scales
  __shared__ __attribute__((aligned(16))) char s_raw[FP8 ? kRawTiles : 1][FP8 ? kRawBytes : 16];
  __shared__ float2 s_ml[KW == 2 ? 2 : 1][64];
  __shared__ int s_cum[kSeqsPerLaunch + 1];
  __shared__ int s_part[kWaves];

  const int lane = threadIdx.x & 63, wave = uniform(static_cast<int>(threadIdx.x >> 6));
  build_prefix<STEP>(p, s_cum, s_part);
  fill_rows(p, s_cum);
  Range r;
  // Workgroups are dealt out over the 8 XCDs in turn: neighbouring units, which read the same tokens, go to
  // one XCD, whose L2 then reads them once.
  const int unit = static_cast<int>(blockIdx.x & 7) * static_cast<int>(gridDim.x >> 3) + static_cast<int>(blockIdx.x >> 3);
  if (!find_range(p, s_cum, unit, r)) return;  // the whole workgroup

  // ---- loads: the wave fills tokens 16 wave .. + 15, 4 (e4m3: 8) per instruction
  const int64_t head_off = r.kvh * p.head_stride, scale_head = r.kvh * p.scale_head_stride;
  const int stride = static_cast<int>(p.slot_stride);
  // What follows from the lane is derived anew in each step: held over the loop, it would take the registers
  // that the products need.
  auto fresh_lane = [&]() __attribute__((always_inline)) {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  constexpr int kFills = FP8 ? 2 : 4;               // instructions of a wave for K, and for V
  constexpr int kOps = 2 * kFills + (FP8 ? 2 : 0);  // and every wave loads the scales
  auto issue = [&](const Cursor& c, char* k_to, char* v_to, char* scale_to) __attribute__((always_inline)) {
    const int off = c.j * STEP - c.lblk * p.block_size, last = (min(STEP, c.len - c.j * STEP) - 1) * stride;
    const int64_t base = uniform(c.blk * p.blk_stride + off * p.slot_stride + head_off);
    const uint32_t bytes = static_cast<uint32_t>((STEP - 1) * stride + (FP8 ? kDim : 2 * kDim));
    const int ln = fresh_lane(), lr = FP8 ? ln >> 3 : ln >> 4, lc = FP8 ? ln & 7 : ln & 15;
    const int row_off = (16 * wave + lr) * stride;
    const int k_chunk = 16 * (FP8 ? lc ^ (lr >> 1) : lc ^ lr), v_chunk = 16 * (FP8 ? lc ^ (lr & 2) : lc ^ (4 * (lr & 3)));
    const BufferRsrc kr = buffer_rsrc(p.k_cache + base, bytes), vr = buffer_rsrc(p.v_cache + base, bytes);
    // Nontemporal where rows are read once: 32 sequences of 8192, 16 drafts at 32 heads in bf16 188 us against 212.
    // Blocks of 128 rows read them again (8 heads to a kv head: 394 us against 368).
    constexpr int kNt = KW == 2 ? 2 : 0;
    // row 16 wave + 4 i + lr (e4m3: 8 i): the part of i in the swizzle is 4 i chunks, but none in bf16's V
#pragma unroll
    for (int i = 0; i < kFills; ++i)
      raw_buffer_load_lds(kr, (LdsPtr)(k_to + 1024 * (kFills * wave + i)), 16,
                          min(row_off + (FP8 ? 8 : 4) * i * stride, last) + (k_chunk ^ (64 * i)), 0, 0, kNt);
#pragma unroll
    for (int i = 0; i < kFills; ++i)
      raw_buffer_load_lds(vr, (LdsPtr)(v_to + 1024 * (kFills * wave + i)), 16,
                          min(row_off + (FP8 ? 8 : 4) * i * stride, last) + (FP8 ? v_chunk ^ (64 * i) : v_chunk), 0, 0, kNt);
    if (FP8) issue_scales(p, uniform(c.blk * p.scale_blk_stride + scale_head + off), ln, scale_to);
  };
  // ---- the wave's rows
  const int kw = KW == 2 ? wave >> 1 : 0, rw = KW == 2 ? wave & 1 : wave;
  const int first_row = r.block * 128 + 32 * rw;
  auto token_of = [&](int row) __attribute__((always_inline)) { return div_by(row, p.div_group); };
  uint4 q[8];
  uint64_t seen = 0;  // the drafts that the row's token sees
  float m = kMaxFloor, l = 0.f;
  f32x16_t acc[4];
  bool fresh = true;  // no step of the sequence has been taken
  auto start = [&](const Cursor& c) __attribute__((always_inline)) {
    const int ln = fresh_lane(), row = first_row + (ln & 31), tok = token_of(row);
    const int i = min(tok, c.n - 1), head = r.kvh * p.group + row - tok * p.group;
    const uint16_t* src = p.q + (c.q0 + i) * p.q_tok_stride + head * p.q_head_stride + (FP8 ? 16 : 8) * (ln >> 5);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint4 x = *reinterpret_cast<const uint4*>(src + (FP8 ? 32 * (ks >> 1) + 8 * (ks & 1) : 16 * ks));
      q[ks] = make_uint4(x.x ^ p.q_flip, x.y ^ p.q_flip, x.z ^ p.q_flip, x.w ^ p.q_flip);
    }
    const uint64_t all = ~0ull >> (64 - c.n);
    seen = (p.mask ? static_cast<uint64_t>(p.mask[c.q0 + i]) : ~0ull >> (63 - i)) & all;
    asm volatile("" : "+v"(seen));  // waited for here, not in front of every product that reuses its registers
    m = kMaxFloor;
    l = 0.f;
    fresh = true;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[mb][j] = 0.f;
  };

  // The step's tiles: sk and sv, or in e4m3 at LDS address `raw`.
  auto compute = [&](const Cursor& c, const uint16_t* sk, const uint16_t* sv, u32 raw) __attribute__((always_inline)) {
    const int t0 = c.j * STEP + 32 * kw, left = c.len - t0;  // the wave's tokens
    if (left <= 0) return;
    const int ln = fresh_lane(), n = ln & 31, hf = ln >> 5;
    const int draft = t0 - (c.len - c.n);        // the first token's draft, below 0 in the context
    const bool tail = draft + 32 * BLOCKS > 0;  // drafts among the tokens, or the last one in front of them
    // ---- S = K Q^T
    f32x16_t sc[BLOCKS];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int mb = 0; mb < BLOCKS; ++mb)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[mb][j] = 0.f;
    u32 vexp[BLOCKS][4];  // V's scales of tokens 8 i + 4 hf + 0 .. 3, one a byte
    if constexpr (FP8) {
      u32x4_t k[BLOCKS][4];  // dims 32 i + 16 hf .. + 15
      u32 kexp[BLOCKS];
      const u32 row = raw + 128 * (32 * kw + n), f = (n >> 1) & 7;
      const u32 at[4] = {row + 16 * (hf ^ f), row + 16 * ((2 + hf) ^ f), row + 16 * ((4 + hf) ^ f), row + 16 * ((6 + hf) ^ f)};
      read_k8_blocks(at, raw + 2 * kTile + 32 * kw + n, raw + 2 * kTile + kManyStep + 32 * kw + 4 * hf, k, kexp, vexp);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int mb = 0; mb < BLOCKS; ++mb) {
          const u32x4_t w = k[mb][ks >> 1];
          sc[mb] = mfma32(__builtin_bit_cast(uint4, widen8(w[2 * (ks & 1)], w[2 * (ks & 1) + 1], __uint_as_float(kexp[mb] << 23))),
                          q[ks], sc[mb]);
        }
    } else {  // steps (16 dims, block), a ring of four fragments in flight ahead of the products
      auto frag = [&](int st) __attribute__((always_inline)) {
        const int ks = st / BLOCKS, mb = st % BLOCKS;
        return *reinterpret_cast<const uint4*>(sk + ((32 * (kw + mb) + n) * kDim + 8 * ((2 * ks + hf) ^ (n & 15))));
      };
      uint4 ka[4];
#pragma unroll
      for (int st = 0; st < 4; ++st) ka[st] = frag(st);
#pragma unroll
      for (int st = 0; st < 8 * BLOCKS; ++st) {
        sc[st % BLOCKS] = mfma32(ka[st & 3], q[st / BLOCKS], sc[st % BLOCKS]);
        if (st + 4 < 8 * BLOCKS) ka[st & 3] = frag(st + 4);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int st = 0; st < 8 * BLOCKS - 4; ++st) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    }
    __builtin_amdgcn_s_setprio(0);
    if (tail) {
#pragma unroll
      for (int mb = 0; mb < BLOCKS; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int d = draft + 32 * mb + 8 * (j >> 2) + 4 * hf + (j & 3);
          sc[mb][j] = sees(seen, d) ? sc[mb][j] : -INFINITY;
        }
    }
    // ---- weights.  A row's maximum is taken of the first step, and again only where the weights of a step sum up to
    // more than its tokens (equal scores can lie above their maximum by its rounding), so that no sum over a row's tokens
    // is larger than their number times the largest V, but for these 2%.
    auto step_max = [&]() __attribute__((always_inline)) {
      float mx = kMaxFloor;
#pragma unroll
      for (int mb = 0; mb < BLOCKS; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[mb][j]);
      return half_swap_max(mx) * p.scale_log2;
    };
    if (fresh) m = fmaxf(step_max(), kMaxFloor);
    fresh = false;
    float sum;
    u32 pk[BLOCKS][8];  // packed pairs
    auto weigh = [&]() __attribute__((always_inline)) {
      sum = 0.f;
#pragma unroll
      for (int mb = 0; mb < BLOCKS; ++mb)
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          float w0 = fast_exp2(fmaf(sc[mb][j], p.scale_log2, -m));
          float w1 = fast_exp2(fmaf(sc[mb][j + 1], p.scale_log2, -m));
          sum += w0 + w1;
          if (FP8) {
            w0 = scale_weight(w0, vexp[mb][j >> 2], j & 3);
            w1 = scale_weight(w1, vexp[mb][j >> 2], (j & 3) + 1);
          }
          pk[mb][j >> 1] = pack_bf16x2(w0, w1);
        }
      sum = half_swap_sum(sum);
    };
    weigh();
    if (__any(!(sum <= 32.5f * BLOCKS))) {  // rare
      const float m_new = fmaxf(m, step_max());
      const float alpha = fast_exp2(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[mb][j] *= alpha;
      weigh();
    }
    l += sum;
    // ---- O^T += V^T P^T, 16 tokens at a time
    auto pf = [&](int kk) __attribute__((always_inline)) {
      const u32* w = &pk[kk >> 1][4 * (kk & 1)];
      return make_uint4(w[0], w[1], w[2], w[3]);
    };
    // V^T operand (see lds_read_tr16's use in the prefill): the lane addresses token 4 hf + (l % 16) / 4 of 16 at
    // dims 16 ((l / 16) % 2) + 4 (l % 4) of 32, and gets dim l % 32 of tokens 4 hf + e.  e4m3: it addresses token
    // 8 (e / 4) + 4 hf + e % 4, e = (l % 16) / 2, at dims 16 ((l / 16) % 2) + 8 (l % 2), and gets all 8.
    const int tr_tok = FP8 ? 4 * hf + ((ln & 8) | ((ln & 7) >> 1)) : 4 * hf + ((ln & 15) >> 2);
    const int tr_chunk = 2 * ((ln >> 4) & 1) + ((ln & 3) >> 1), tr_sub = 4 * (ln & 1);
    int v_at[4];
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
      if (FP8) {
        v_at[mb] = static_cast<int>(raw) + kTile + 128 * (32 * kw + tr_tok) +
                   16 * ((2 * mb + ((ln >> 4) & 1)) ^ ((tr_tok & 2) | (tr_tok & 8) >> 1)) + 8 * (ln & 1);
        continue;
      }
      v_at[mb] = (32 * kw + tr_tok) * kDim + 8 * ((4 * mb + tr_chunk) ^ (4 * (tr_tok & 3))) + tr_sub;
      // The compiler is not to take the sum apart: behind several additions it no longer knows the array, and
      // would wait for the next tile in front of the read.
      asm volatile("" : "+v"(v_at[mb]));
    }
    auto read_v = [&](int kk, uint4 (&dst)[4]) __attribute__((always_inline)) {
      if constexpr (FP8) {
        u32x2_t v[4];
        read_v8_16(v_at, 2048 * kk, v);
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) dst[mb] = __builtin_bit_cast(uint4, widen8(v[mb].x, v[mb].y, 1.f));
        return;
      }
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) {
        const uint2 lo = lds_read_tr16(sv + (v_at[mb] + 16 * kk * kDim));
        const uint2 hi = lds_read_tr16(sv + (v_at[mb] + (16 * kk + 8) * kDim));
        dst[mb] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    };
    if (FP8 && !tail) {
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int h = 0; h < BLOCKS; ++h) {
        u32x2_t v[2][4];
        read_v8_32(v_at, 4096 * h, v);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int mb = 0; mb < 4; ++mb)
            acc[mb] = mfma32(__builtin_bit_cast(uint4, widen8(v[kk][mb].x, v[kk][mb].y, 1.f)), pf(2 * h + kk), acc[mb]);
      }
      __builtin_amdgcn_s_setprio(0);
    } else if (!tail) {
      __builtin_amdgcn_s_setprio(1);
      uint4 vf[2][4];
      read_v(0, vf[0]);
#pragma unroll
      for (int kk = 0; kk < 2 * BLOCKS; ++kk) {
        if (kk + 1 < 2 * BLOCKS) read_v(kk + 1, vf[(kk + 1) & 1]);
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) acc[mb] = mfma32(vf[kk & 1][mb], pf(kk), acc[mb]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
      for (int i = 0; i < 4 * (2 * BLOCKS - 1); ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
      __builtin_amdgcn_s_setprio(0);
    } else {
      // As in Rows::clean: tokens behind the last one are cleared, drafts that are not finite added apart.
      // Element e of the lane is token 4 hf + e, or 4 + 4 hf + e for e >= 4, of the 16.
#pragma unroll
      for (int kk = 0; kk < 2 * BLOCKS; ++kk) {
        if (16 * kk >= left) break;
        uint4 vr[4];
        read_v(kk, vr);
        u32x4_t vt[4], fine;
        u32 odd = 0;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) vt[mb] = __builtin_bit_cast(u32x4_t, vr[mb]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int t = 16 * kk + 4 * hf + 8 * (w >> 1) + 2 * (w & 1);
          fine[w] = (t < left ? 0xffffu : 0u) | (t + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
          for (int mb = 0; mb < 4; ++mb) {
            const u32 v = vt[mb][w] & fine[w];
            odd |= ((v & 0x7f80u) == 0x7f80u ? 1u : 0u) << (2 * w);
            odd |= ((v & 0x7f800000u) == 0x7f800000u ? 2u : 0u) << (2 * w);
          }
        }
        if (__any(odd != 0)) {
#pragma unroll 1
          for (int i = 0; i < 16; ++i) {  // element e = i % 8 of the lanes of half i / 8
            const int e = i & 7, g = i >> 3;
            if (!__any(hf == g && (odd >> e & 1))) continue;
            const u32 half = hf == g ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
            u32x4_t only;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              only[w] = w == e >> 1 ? half : 0u;
              fine[w] &= ~only[w];
            }
            const int d = draft + 16 * kk + 4 * g + (e & 3) + 8 * (e >> 2);
            const bool mine = sees(seen, d);
#pragma unroll
            for (int mb = 0; mb < 4; ++mb) {
              const f32x16_t with = mfma32(__builtin_bit_cast(uint4, vt[mb] & only), pf(kk), acc[mb]);
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[mb][j] = mine ? with[j] : acc[mb][j];
            }
          }
        }
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) acc[mb] = mfma32(__builtin_bit_cast(uint4, vt[mb] & fine), pf(kk), acc[mb]);
      }
    }
  };

  // The rows' output where the range held all of the sequence, otherwise a partial state at `place`.
  auto emit = [&](const Cursor& c, bool whole, int place) __attribute__((always_inline)) {
    const float sum = c.bad ? NAN : l;
    const int ln = fresh_lane(), hf = ln >> 5, row = first_row + (ln & 31), tok = token_of(row);
    const int head = r.kvh * p.group + row - tok * p.group;
    if (tok >= c.n) return;
    if (whole) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint16_t* out = p.out + (c.q0 + tok) * p.o_tok_stride + head * p.o_head_stride + 4 * hf;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *reinterpret_cast<u32x2_t*>(out + 32 * mb + 2 * j) =
              u32x2_t{pack_bf16x2(acc[mb][j] * inv, acc[mb][j + 1] * inv), pack_bf16x2(acc[mb][j + 2] * inv, acc[mb][j + 3] * inv)};
    } else {
      const int64_t at = (static_cast<int64_t>(place) * p.num_kv_heads + r.kvh) * p.rows + row;
      float* part = p.part_o + at * kDim + 4 * hf;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *reinterpret_cast<float4*>(part + 32 * mb + 2 * j) =
              make_float4(acc[mb][j], acc[mb][j + 1], acc[mb][j + 2], acc[mb][j + 3]);
      if (hf == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, sum);
    }
  };
  // KW = 2: wave w takes over the state of wave w + 2, by way of the step's tile (in e4m3 it is half as large).
  auto join = [&](uint16_t* sk, uint16_t* sv, u32 buf) __attribute__((always_inline)) {
    constexpr int kRounds = FP8 ? 2 : 1, MB = 4 / kRounds;
    float* const area = (FP8 ? reinterpret_cast<float*>(s_raw[FP8 ? buf : 0] + (FP8 ? kTile * rw : 0))
                             : reinterpret_cast<float*>(rw == 0 ? sk : sv)) + lane;
    float a = 0.f, w = 0.f;
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
      tile_barrier();  // the tile is done with
      if (kw == 1) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int j = 0; j < 16; ++j) area[64 * (16 * mb + j)] = acc[MB * round + mb][j];
        if (round == 0) s_ml[rw][lane] = make_float2(m, l);
      }
      tile_barrier();
      if (kw == 0) {
        if (round == 0) {
          const float2 o = s_ml[rw][lane];
          const float m_new = fmaxf(m, o.x);
          a = fast_exp2(m - m_new), w = fast_exp2(o.x - m_new);
          m = m_new;
          l = l * a + o.y * w;
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[MB * round + mb][j] = acc[MB * round + mb][j] * a + area[64 * (16 * mb + j)] * w;
      }
    }
  };

  // One step: its place c0, and those behind it (bf16 uses one).
  Cursor c0{}, c1{}, c2{}, c3{};
  auto take = [&](int S, uint16_t* sk, uint16_t* sv, u32 buf) __attribute__((always_inline)) {
    const bool active = c0.n * p.group > first_row;
    if (active && (S == r.S0 || c0.j == 0)) start(c0);
    if (active) compute(c0, sk, sv, lds_addr(s_raw[FP8 ? buf : 0]));
    if (c0.j + 1 == c0.nsteps || S + 1 == r.S1) {
      const int from = S - c0.j, to = from + c0.nsteps;  // the sequence's steps
      if (KW == 2) join(sk, sv, buf);
      if (active && kw == 0) emit(c0, from >= r.S0 && to <= r.S1, 2 * r.index + (from > r.S0 ? 1 : 0));
    }
  };
  start_seq<STEP>(p, c0, r.first, r.S0 - uniform(s_cum[r.first]));
  if constexpr (FP8) {
    auto issue_to = [&](const Cursor& c, int buf) __attribute__((always_inline)) {
      issue(c, s_raw[buf], s_raw[buf] + kTile, s_raw[buf] + 2 * kTile);
    };
    issue_to(c0, 0);
    if (r.S0 + 1 < r.S1) {
      next_step<STEP>(p, s_cum, c0, c1);
      issue_to(c1, FP8 ? 1 : 0);
    }
    if (r.S0 + 2 < r.S1) {
      next_step<STEP>(p, s_cum, c1, c2);
      issue_to(c2, FP8 ? 2 : 0);
    }
#pragma unroll 1
    for (int S = r.S0; S < r.S1; ++S) {
      const int buf = (S - r.S0) & (kRawTiles - 1);
      if (S + 3 < r.S1) next_step<STEP>(p, s_cum, c2, c3);
      if (S + 2 < r.S1) wait_vmem<2 * kOps>();  // later steps' loads stay in flight
      else if (S + 1 < r.S1) wait_vmem<kOps>();
      else wait_vmem<0>();
      tile_barrier();  // the other waves' part of the tile, and they are done with the one before
      if (S + 3 < r.S1) issue_to(c3, (buf + 3) & (kRawTiles - 1));
      take(S, s_k0, s_v0, buf);
      c0 = c1;
      c1 = c2;
      c2 = c3;
    }
  } else {
    issue(c0, reinterpret_cast<char*>(s_k0), reinterpret_cast<char*>(s_v0), nullptr);
    auto step = [&](int S, uint16_t* sk, uint16_t* sv, uint16_t* nk, uint16_t* nv) __attribute__((always_inline)) {
      const bool more = S + 1 < r.S1;
      if (more) next_step<STEP>(p, s_cum, c0, c1);
      wait_vmem<0>();   // the wave's part of the tile
      __syncthreads();  // the others', and they are done with the tile before.  (The compiler has to see a fence:
                        // it would wait for the next tile in front of the first read of this one.)
      if (more) issue(c1, reinterpret_cast<char*>(nk), reinterpret_cast<char*>(nv), nullptr);
      take(S, sk, sv, 0);
      c0 = c1;
    };
#pragma unroll 1
    for (int S = r.S0; S < r.S1; S += 2) {
      step(S, s_k0, s_v0, s_k1, s_v1);
      if (S + 1 < r.S1) step(S + 1, s_k1, s_v1, s_k0, s_v0);
    }
  }
}

// Joins the states of sequences that several ranges share, 8 dims to a lane, four ranges per round
// trip.  SPLIT: one wave for a query token and head, whose four 16-lane rows take the ranges round
// robin; otherwise each of them has a token and head of its own.
template <bool SPLIT>
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(const TreeParams p) {
  constexpr int SPAN = SPLIT ? 4 : 1;
  const int r4 = (threadIdx.x >> 4) & 3, d = 8 * (threadIdx.x & 15);
  const int wave = blockIdx.x * kWaves + uniform(static_cast<int>(threadIdx.x >> 6));
  const int row = SPLIT ? wave : 4 * wave + r4;  // token and q head
  const int b = blockIdx.y;
  const int cb = load_uniform(p.header, kHeaderInts + b), cb1 = load_uniform(p.header, kHeaderInts + b + 1);
  const int spr = load_uniform(p.header, 0);
  const SeqShape s = load_shape(p, b);
  if (cb1 <= cb || row >= s.n * p.num_q_heads) return;  // no steps, or rows
  const int first = cb / spr, np = (cb1 - 1) / spr - first + 1;
  if (np <= 1) return;  // written already
  const int tok = row / p.num_q_heads, h = row - tok * p.num_q_heads;
  const int kvh = div_by(h, p.div_group), r = tok * p.group + h - kvh * p.group;  // row of the kv head
  const int k_first = SPLIT ? r4 : 0;
  float m = kMaxFloor, l = 0.f, o[8] = {};
#pragma unroll 1
  for (int k0 = k_first; k0 - k_first < np; k0 += 4 * SPAN) {
    float2 st[4];
    float4 x[4], y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = min(k0 + SPAN * u, np - 1);
      const int place = 2 * (first + k) + (k == 0 && cb > first * spr ? 1 : 0);
      const int64_t at = (static_cast<int64_t>(place) * p.num_kv_heads + kvh) * p.rows + r;
      st[u] = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
      x[u] = *reinterpret_cast<const float4*>(p.part_o + at * kDim + d);
      y[u] = *reinterpret_cast<const float4*>(p.part_o + at * kDim + d + 4);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (k0 + SPAN * u >= np) break;
      const float m_new = fmaxf(m, st[u].x), alpha = fast_exp2(m - m_new), w = fast_exp2(st[u].x - m_new);
      const float v[8] = {x[u].x, x[u].y, x[u].z, x[u].w, y[u].x, y[u].y, y[u].z, y[u].w};
      m = m_new;
      l = l * alpha + w * st[u].y;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = o[j] * alpha + w * v[j];
    }
  }
  if constexpr (SPLIT) {
    const float mm = xor32_max(xor16_max(m));
    const float w = fast_exp2(m - mm);
    l = xor32_sum(xor16_sum(l * w));
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = xor32_sum(xor16_sum(o[j] * w));
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] *= inv;
  if (!SPLIT || r4 == 0) *reinterpret_cast<uint4*>(p.out + (s.q0 + tok) * p.o_tok_stride + h * p.o_head_stride + d) = pack8(o);
}

// How a batch is cut: by its rows per kv head, and into as many ranges as the GPU holds at once.
struct Plan {
  int waves;   // of 32 rows side by side; 0: tree_few_kernel
  int blocks;  // of rows
  int ranges, seqs;  // seqs: per launch
  int rows() const { return waves ? blocks * 32 * waves : 16; }
  int64_t bytes(int hkv) const { return kHeaderBytes + 2ll * ranges * hkv * rows() * (kDim + 2) * 4; }
};
void set_rows(Plan& pl, int rows) {
  pl.waves = rows <= 16 ? 0 : rows <= 64 ? 2 : 4;
  pl.blocks = pl.waves ? (rows + 32 * pl.waves - 1) / (32 * pl.waves) : 1;
}
// units: waves of tree_few_kernel, or workgroups of tree_many_kernel, that are resident at once.
void set_ranges(Plan& pl, int64_t seqs, int hkv, int64_t max_tokens, int step, int units) {
  const int64_t steps = (max_tokens + step - 1) / step;  // of a sequence
  pl.seqs = static_cast<int>(std::min<int64_t>(std::min<int64_t>(seqs, kSeqsPerLaunch), (1ll << 30) / steps));
  pl.ranges = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(units / (hkv * pl.blocks), pl.seqs * steps)));
}

// Workgroups of a kernel resident on the current device at once.
template <typename K>
int resident(K kernel, std::atomic<int> (&cached)[16]) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 16) dev = 0;
  int v = cached[dev].load(std::memory_order_relaxed);
  if (v > 0) return v;
  int cus = 0, per_cu = 0;
  bool ok = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && cus > 0;
  if (!ok) cus = 256;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, kThreads, 0) != hipSuccess || per_cu <= 0) {
    per_cu = 1;
    ok = false;
  }
  v = cus * per_cu;
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

template <bool FP8>
int launch(const char* fn, const TreeArgs& a, hipStream_t stream) {
  static std::atomic<int> cached[3][16];
  const int64_t tokens = static_cast<int64_t>(a.max_blocks) * a.block_size;
  Plan pl{};
  set_rows(pl, a.max_q * (a.num_q_heads / a.num_kv_heads));
  const int wgs = pl.waves == 0   ? resident(tree_few_kernel<FP8>, cached[0])
                  : pl.waves == 2 ? resident(tree_many_kernel<FP8, 2>, cached[1])
                                  : resident(tree_many_kernel<FP8, 1>, cached[2]);
  const int units = pl.waves == 0 ? std::min(wgs * kWaves, kMaxFew) : std::min(wgs, kMaxMany);
  set_ranges(pl, a.num_seqs, a.num_kv_heads, tokens, pl.waves ? kManyStep : Format<FP8>::kStep, units);
  const size_t need = static_cast<size_t>(pl.bytes(a.num_kv_heads));
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
  // The kernels hide a score as -inf and scale it afterwards, which asks for a positive scale: its sign goes into q,
  // and 0 counts as 2^-149, which moves no score that is finite in 32 bits by more than 2^-21.
  p.scale_log2 = fabsf(a.softmax_scale) * 1.4426950408889634f;
  if (p.scale_log2 == 0.f) p.scale_log2 = __FLT_DENORM_MIN__;
  p.q_flip = a.softmax_scale < 0.f ? 0x80008000u : 0u;
  p.o_tok_stride = a.o_tok_stride;
  p.o_head_stride = a.o_head_stride;
  p.ranges = pl.ranges;
  p.blocks = pl.blocks;
  p.streams = a.num_kv_heads * pl.blocks;
  p.rows = pl.rows();
  p.div_streams = divisor(p.streams);
  p.div_blocks = divisor(pl.blocks);
  p.div_ranges = divisor(pl.ranges);
  p.div_block = divisor(a.block_size);
  p.div_group = divisor(p.group);
  char* ws = static_cast<char*>(a.workspace);
  p.header = reinterpret_cast<int32_t*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + kHeaderBytes);
  p.part_ml = p.part_o + 2ll * pl.ranges * a.num_kv_heads * p.rows * kDim;
  const int n = pl.ranges * p.streams;
  const dim3 grid(static_cast<unsigned>(pl.waves ? (n + 7) / 8 * 8 : (n + kWaves - 1) / kWaves)), block(kThreads);
  const LaunchOrder order;
  for (int b0 = 0; b0 < a.num_seqs; b0 += pl.seqs) {
    p.num_seqs = std::min(pl.seqs, a.num_seqs - b0);
    p.block_tables = a.block_tables + b0 * a.bt_stride;
    p.kv_lens = a.kv_lens + b0;
    p.cu_q = a.cu_q ? a.cu_q + b0 : nullptr;
    const int64_t row0 = a.cu_q ? 0 : b0;  // without cu_q row b is sequence b's
    p.q = static_cast<const uint16_t*>(a.q) + row0 * a.q_tok_stride;
    p.out = static_cast<uint16_t*>(a.out) + row0 * a.o_tok_stride;
    p.total_q = a.cu_q ? a.total_q : p.num_seqs;
    if (pl.waves == 0) hipLaunchKernelGGL(tree_few_kernel<FP8>, grid, block, 0, stream, p);
    else if (pl.waves == 2) hipLaunchKernelGGL((tree_many_kernel<FP8, 2>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((tree_many_kernel<FP8, 1>), grid, block, 0, stream, p);
    if (pl.ranges > 1) {
      // A wave for every row while they fit the GPU at once (32 to a CU): rows are few then, and of many
      // ranges each.
      const int rows = a.max_q * a.num_q_heads;
      const bool split = static_cast<int64_t>(rows) * p.num_seqs <= 8192;
      const int per = split ? kWaves : 4 * kWaves;
      const dim3 rows_grid(static_cast<unsigned>((rows + per - 1) / per), static_cast<unsigned>(p.num_seqs));
      if (split) hipLaunchKernelGGL(tree_merge_kernel<true>, rows_grid, block, 0, stream, p);
      else hipLaunchKernelGGL(tree_merge_kernel<false>, rows_grid, block, 0, stream, p);
    }
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
  return a.fp8 ? launch<true>(fn, a, s) : launch<false>(fn, a, s);
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
  // The most that any launch within these sizes needs, on any device, be its rows few or many (fewer kv
  // heads have more rows each): a launch has as many (range, stream) pairs as units at most, or one range,
  // and no more than steps.
  const int64_t tokens = static_cast<int64_t>(max_blocks_per_seq) * block_size;
  int64_t most = 0;
  for (int hkv = 1; hkv <= num_kv_heads; ++hkv) {
    const int rows = max_seqlen_q * std::min(kMaxGroup, num_q_heads / hkv);
    for (const int some : {std::min(rows, 16), std::min(rows, 64), rows}) {
      Plan pl{};
      set_rows(pl, some);
      const int step = pl.waves ? kManyStep : Format<false>::kStep;
      const int64_t streams = hkv * pl.blocks, steps = max_num_seqs * ((tokens + step - 1) / step);
      const int64_t pairs = std::min(std::max<int64_t>(pl.waves ? kMaxMany : kMaxFew, streams), steps * streams);
      most = std::max(most, kHeaderBytes + 2 * pairs * (pl.waves ? 32 * pl.waves : 16) * (kDim + 2) * 4);
    }
  }
  return static_cast<size_t>(most);
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
