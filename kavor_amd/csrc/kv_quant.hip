// The quantised paged cache: keys and values in e4m3 with one power-of-two scale for each token
// and head, written as new tokens arrive (kvp_append_fp8) and read back in bf16
// (kvp_load_fp8).  kvp_paged_decode_fp8 and kvp_tree_attention read it as it is.
//
// A row x of head_dim values becomes  x_i = 2^e q_i  with q_i in e4m3 and e the least exponent
// that brings the largest finite magnitude to 448 = 1.75 * 2^8, the format's largest, or below.
// The scale is a power of two because the format floats: a finer scale would not make a value's
// rounding (half a step, 2^-4 relative) any smaller, while this one is exact to divide and to
// multiply by, so the rounding to e4m3 is the only one, and its biased exponent fits a byte:
// 129 bytes for a row of 128, against 256 in bf16.  An infinity becomes NaN (the format has none)
// and leaves the row's scale to the finite values.
//
// Both kernels are bound by HBM.  A wave takes 1024 / head_dim rows, 16 values to a lane, so a lane
// moves 32 bytes of bf16 and 16 of e4m3.  The rows of a wave are consecutive tokens of one head,
// whose scales are neighbours in a page.  16384 tokens of 8 heads of 128 are written in 21.5 us
// (101 MB, 4.7 TB/s), 32 sequences of 100 to 4096 read back in 84.6 us (413 MB, 4.9 TB/s); a plain
// copy reaches 5.1 TB/s.
#include <type_traits>

#include "paged.h"

namespace kvp {
namespace {

constexpr int kThreads = 256;
constexpr int kLane = 16;  // values of a row per lane

struct QuantParams {
  const uint16_t* x[2];  // key, value
  int64_t tok_stride[2], head_stride[2];
  uint8_t* cache[2];  // k, v: stride in bytes
  int64_t blk_stride, slot_stride, cache_head_stride;
  uint8_t* scale[2];
  int64_t scale_blk_stride, scale_head_stride;
  int64_t num_slots;
  const int32_t* slots;
  int32_t num_tokens, num_heads;
  Divisor div_block, div_heads;
  int32_t block_size;
};

// Largest finite magnitude, as bf16 bits, of a packed pair and `top`.
__device__ __forceinline__ u32 top_of(u32 w, u32 top) {
  const u32 lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  return max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
}
// x of the lanes of a 4-, 8- or 16-lane group, combined by maximum.
template <int LANES>
__device__ __forceinline__ u32 group_max(u32 x) {
  auto with = [&](auto ctrl) {
    x = max(x, static_cast<u32>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf,
                                                            false)));
  };
  with(std::integral_constant<int, kDppQuadXor1>{});
  with(std::integral_constant<int, kDppQuadXor2>{});
  if (LANES >= 8) with(std::integral_constant<int, kDppRowHalfMirror>{});
  if (LANES >= 16) with(std::integral_constant<int, kDppRowMirror>{});
  return x;
}
// Four values to e4m3 bytes, round to nearest even.
__device__ __forceinline__ u32 pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<u32>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
// An infinity as the NaN that it is stored as.
__device__ __forceinline__ float finite_or_nan(float x) { return __builtin_isinf(x) ? __builtin_nanf("") : x; }

template <int D>
__global__ __launch_bounds__(kThreads) void append_fp8_kernel(const QuantParams p) {
  constexpr int kRowLanes = D / kLane, kTokens = 64 / kRowLanes;  // tokens per wave
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6));
  const int group = div_by(wave, p.div_heads), h = wave - group * p.num_heads;
  const int t0 = group * kTokens + lane / kRowLanes, c = lane % kRowLanes;
  const int t = min(t0, p.num_tokens - 1);
  uint4 in[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t* src = p.x[i] + t * p.tok_stride[i] + h * p.head_stride[i] + kLane * c;
    in[i][0] = load16_nt(src);
    in[i][1] = load16_nt(src + 8);
  }
  const int slot = p.slots[t];
  if (t0 >= p.num_tokens || slot < 0 || slot >= p.num_slots) return;
  const int blk = div_by(slot, p.div_block), off = slot - blk * p.block_size;
  const int64_t at = blk * p.blk_stride + off * p.slot_stride + h * p.cache_head_stride + kLane * c;
  const int64_t scale_at = blk * p.scale_blk_stride + h * p.scale_head_stride + off;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32 w[8] = {in[i][0].x, in[i][0].y, in[i][0].z, in[i][0].w, in[i][1].x, in[i][1].y, in[i][1].z, in[i][1].w};
    u32 top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = top_of(w[j], top);
    top = group_max<kRowLanes>(top);
    // top = 1.f * 2^(E - 127): the exponent is E - 127 - 8, one more where 1.f is over 1.75
    const int byte = min(max(static_cast<int>(top >> 7) - 8 + ((top & 0x7f) > 0x60), 1), 254);
    const float inv = __uint_as_float(static_cast<u32>(254 - byte) << 23);
    float f[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[2 * j] = finite_or_nan(bf16_lo(w[j])) * inv;
      f[2 * j + 1] = finite_or_nan(bf16_hi(w[j])) * inv;
    }
    store16_nt(p.cache[i] + at,
               make_uint4(pack_e4m3(f[0], f[1], f[2], f[3]), pack_e4m3(f[4], f[5], f[6], f[7]),
                          pack_e4m3(f[8], f[9], f[10], f[11]), pack_e4m3(f[12], f[13], f[14], f[15])));
    if (c == 0) p.scale[i][scale_at] = static_cast<uint8_t>(byte);
  }
}

struct LoadParams {
  const uint8_t* cache[2];
  int64_t blk_stride, slot_stride, cache_head_stride;
  const uint8_t* scale[2];
  int64_t scale_blk_stride, scale_head_stride;
  int32_t num_cache_blocks, block_size, max_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu;
  int32_t num_seqs, total;
  int32_t num_heads;
  uint16_t* out[2];
  int64_t out_tok_stride[2], out_head_stride[2];
  Divisor div_block, div_heads;
};

// The e4m3 pair in the low (HIGH false) or high half of w, times the scale, as packed bf16: the
// product is a power of two times at most four significant bits, so nothing is rounded short of
// bf16's range.
template <bool HIGH>
__device__ __forceinline__ u32 widen_e4m3(u32 w, float scale) {
  return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}

// One head of 16384 / D tokens (64, 128 or 256 bytes of each) per workgroup.  Its first token's
// sequence is the number of cu[i] (i >= 1) up to it, counted by the workgroup in one round trip;
// the others lie a few sequences further.
template <int D>
__global__ __launch_bounds__(kThreads) void load_fp8_kernel(const LoadParams p) {
  constexpr int kRowLanes = D / kLane, kTokens = kThreads / kRowLanes;
  __shared__ int s_count[kThreads / 64];
  const int wg = static_cast<int>(blockIdx.x);
  const int tile = div_by(wg, p.div_heads), h = wg - tile * p.num_heads;
  const int tid = threadIdx.x;
  const int first = tile * kTokens;
  int count = 0;
  for (int i = tid + 1; i <= p.num_seqs; i += kThreads) count += p.cu[i] <= first;
  count = __builtin_amdgcn_readlane(wave_incl_scan(count), 63);
  if ((tid & 63) == 0) s_count[tid >> 6] = count;
  __syncthreads();
  int b = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) b += s_count[w];
  const int t = first + tid / kRowLanes, c = tid % kRowLanes;
  while (b < p.num_seqs && p.cu[b + 1] <= t) ++b;
  if (b >= p.num_seqs || t >= p.total) return;
  const int pos = t - p.cu[b];
  if (pos < 0) return;  // before the first sequence
  const int lblk = div_by(pos, p.div_block), off = pos - lblk * p.block_size;
  const int blk = lblk < p.max_blocks ? p.block_tables[b * p.bt_stride + lblk] : -1;
  const bool ok = blk >= 0 && blk < p.num_cache_blocks;
  const int64_t at = ok ? blk * p.blk_stride + off * p.slot_stride + h * p.cache_head_stride + kLane * c : 0;
  const int64_t scale_at = ok ? blk * p.scale_blk_stride + h * p.scale_head_stride + off : 0;
  uint4 in[2];
  float scale[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    in[i] = load16_nt(p.cache[i] + at);
    scale[i] = __uint_as_float(static_cast<u32>(p.scale[i][scale_at]) << 23);
    if (!ok) scale[i] = __builtin_nanf("");
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint16_t* out = p.out[i] + t * p.out_tok_stride[i] + h * p.out_head_stride[i] + kLane * c;
    const u32 nan = 0x7fc07fc0u;
    const uint4 w = in[i];
    uint4 lo = make_uint4(widen_e4m3<false>(w.x, scale[i]), widen_e4m3<true>(w.x, scale[i]),
                          widen_e4m3<false>(w.y, scale[i]), widen_e4m3<true>(w.y, scale[i]));
    uint4 hi = make_uint4(widen_e4m3<false>(w.z, scale[i]), widen_e4m3<true>(w.z, scale[i]),
                          widen_e4m3<false>(w.w, scale[i]), widen_e4m3<true>(w.w, scale[i]));
    if (!ok) lo = hi = make_uint4(nan, nan, nan, nan);
    store16_nt(out, lo);
    store16_nt(out + 8, hi);
  }
}

bool dim_ok(int32_t d) { return d == 64 || d == 128 || d == 256; }
bool mult16(int64_t stride) { return (stride & 15) == 0; }

// Checks of a quantised cache shared by both directions.
int check_cache(const char* fn, const void* k_cache, const void* v_cache, int64_t blk, int64_t slot, int64_t head,
                const void* k_scale, const void* v_scale, int64_t scale_blk, int64_t scale_head, int32_t num_heads,
                int32_t head_dim, int32_t block_size) {
  if (!dim_ok(head_dim)) return fail(KVP_EUNSUPPORTED, "%s: head_dim=%d (supported: 64, 128, 256)", fn, head_dim);
  if (num_heads <= 0 || block_size <= 0)
    return fail(KVP_EINVAL, "%s: num_kv_heads=%d block_size=%d", fn, num_heads, block_size);
  if (!k_cache || !v_cache || !k_scale || !v_scale) return fail(KVP_EINVAL, "%s: null pointer", fn);
  if (!aligned16(k_cache) || !aligned16(v_cache) || !mult16(blk) || !mult16(slot) || !mult16(head))
    return fail(KVP_EINVAL, "%s: cache pointers and strides must be multiples of 16 bytes", fn);
  if (scale_blk < 0 || scale_head < 0)
    return fail(KVP_EINVAL, "%s: scale strides must not be negative", fn);
  return KVP_OK;
}

}  // namespace
}  // namespace kvp

using namespace kvp;

extern "C" int kvp_append_fp8(const void* key, int64_t key_tok_stride, int64_t key_head_stride, const void* value,
                              int64_t value_tok_stride, int64_t value_head_stride, void* k_cache, void* v_cache,
                              int64_t cache_block_stride, int64_t cache_slot_stride, int64_t cache_head_stride,
                              void* k_scale, void* v_scale, int64_t scale_block_stride, int64_t scale_head_stride,
                              int64_t num_cache_slots, const int32_t* slot_mapping, int32_t num_tokens,
                              int32_t num_kv_heads, int32_t head_dim, int32_t block_size, void* stream) {
  static const char fn[] = "kvp_append_fp8";
  clear_error();
  if (num_tokens < 0 || num_cache_slots < 0)
    return fail(KVP_EINVAL, "%s: num_tokens=%d num_cache_slots=%lld", fn, num_tokens,
                static_cast<long long>(num_cache_slots));
  const int rc = check_cache(fn, k_cache, v_cache, cache_block_stride, cache_slot_stride, cache_head_stride, k_scale,
                             v_scale, scale_block_stride, scale_head_stride, num_kv_heads, head_dim, block_size);
  if (rc != KVP_OK) return rc;
  if (num_tokens == 0) return KVP_OK;
  if (!key || !value || !slot_mapping) return fail(KVP_EINVAL, "%s: null pointer", fn);
  if (!aligned16(key) || !aligned16(value) || (reinterpret_cast<uintptr_t>(slot_mapping) & 3u))
    return fail(KVP_EINVAL, "%s: misaligned key / value / slot_mapping", fn);
  if (!mult8(key_tok_stride) || !mult8(key_head_stride) || !mult8(value_tok_stride) || !mult8(value_head_stride))
    return fail(KVP_EINVAL, "%s: key and value strides must be multiples of 8 elements", fn);
  QuantParams p{};
  p.x[0] = static_cast<const uint16_t*>(key);
  p.x[1] = static_cast<const uint16_t*>(value);
  p.tok_stride[0] = key_tok_stride;
  p.tok_stride[1] = value_tok_stride;
  p.head_stride[0] = key_head_stride;
  p.head_stride[1] = value_head_stride;
  p.cache[0] = static_cast<uint8_t*>(k_cache);
  p.cache[1] = static_cast<uint8_t*>(v_cache);
  p.blk_stride = cache_block_stride;
  p.slot_stride = cache_slot_stride;
  p.cache_head_stride = cache_head_stride;
  p.scale[0] = static_cast<uint8_t*>(k_scale);
  p.scale[1] = static_cast<uint8_t*>(v_scale);
  p.scale_blk_stride = scale_block_stride;
  p.scale_head_stride = scale_head_stride;
  p.num_slots = num_cache_slots;
  p.slots = slot_mapping;
  p.num_tokens = num_tokens;
  p.num_heads = num_kv_heads;
  p.div_block = divisor(static_cast<uint32_t>(block_size));
  p.div_heads = divisor(static_cast<uint32_t>(num_kv_heads));
  p.block_size = block_size;
  const int tokens = 64 * kLane / head_dim;  // per wave
  const int64_t waves = (static_cast<int64_t>(num_tokens) + tokens - 1) / tokens * num_kv_heads;
  const int64_t grid = (waves + kThreads / 64 - 1) / (kThreads / 64);
  if (waves > INT32_MAX - 4) return fail(KVP_EINVAL, "%s: too many tokens", fn);
  const auto s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>(grid)), b(kThreads);
  if (head_dim == 64) hipLaunchKernelGGL(append_fp8_kernel<64>, g, b, 0, s, p);
  else if (head_dim == 128) hipLaunchKernelGGL(append_fp8_kernel<128>, g, b, 0, s, p);
  else hipLaunchKernelGGL(append_fp8_kernel<256>, g, b, 0, s, p);
  return launch_status(fn);
}

extern "C" int kvp_load_fp8(const void* k_cache, const void* v_cache, int64_t cache_block_stride,
                            int64_t cache_slot_stride, int64_t cache_head_stride, const void* k_scale,
                            const void* v_scale, int64_t scale_block_stride, int64_t scale_head_stride,
                            int32_t num_cache_blocks, const int32_t* block_tables, int64_t block_table_stride,
                            int32_t max_blocks_per_seq, const int32_t* cu_seqlens_k, int32_t num_seqs, int32_t total_k,
                            int32_t num_kv_heads, int32_t head_dim, int32_t block_size, void* k_out,
                            int64_t k_out_tok_stride, int64_t k_out_head_stride, void* v_out, int64_t v_out_tok_stride,
                            int64_t v_out_head_stride, void* stream) {
  static const char fn[] = "kvp_load_fp8";
  clear_error();
  if (num_seqs < 0 || total_k < 0 || num_cache_blocks <= 0 || max_blocks_per_seq <= 0)
    return fail(KVP_EINVAL, "%s: num_seqs=%d total_k=%d num_cache_blocks=%d max_blocks_per_seq=%d", fn, num_seqs,
                total_k, num_cache_blocks, max_blocks_per_seq);
  const int rc = check_cache(fn, k_cache, v_cache, cache_block_stride, cache_slot_stride, cache_head_stride, k_scale,
                             v_scale, scale_block_stride, scale_head_stride, num_kv_heads, head_dim, block_size);
  if (rc != KVP_OK) return rc;
  if (block_table_stride < max_blocks_per_seq)
    return fail(KVP_EINVAL, "%s: block_table_stride=%lld < max_blocks_per_seq=%d", fn,
                static_cast<long long>(block_table_stride), max_blocks_per_seq);
  if (num_seqs == 0 || total_k == 0) return KVP_OK;
  if (!block_tables || !cu_seqlens_k || !k_out || !v_out) return fail(KVP_EINVAL, "%s: null pointer", fn);
  if (!aligned16(k_out) || !aligned16(v_out) || (reinterpret_cast<uintptr_t>(block_tables) & 3u) ||
      (reinterpret_cast<uintptr_t>(cu_seqlens_k) & 3u))
    return fail(KVP_EINVAL, "%s: misaligned outputs / block_tables / cu_seqlens_k", fn);
  if (!mult8(k_out_tok_stride) || !mult8(k_out_head_stride) || !mult8(v_out_tok_stride) || !mult8(v_out_head_stride))
    return fail(KVP_EINVAL, "%s: output strides must be multiples of 8 elements", fn);
  LoadParams p{};
  p.cache[0] = static_cast<const uint8_t*>(k_cache);
  p.cache[1] = static_cast<const uint8_t*>(v_cache);
  p.blk_stride = cache_block_stride;
  p.slot_stride = cache_slot_stride;
  p.cache_head_stride = cache_head_stride;
  p.scale[0] = static_cast<const uint8_t*>(k_scale);
  p.scale[1] = static_cast<const uint8_t*>(v_scale);
  p.scale_blk_stride = scale_block_stride;
  p.scale_head_stride = scale_head_stride;
  p.num_cache_blocks = num_cache_blocks;
  p.block_size = block_size;
  p.max_blocks = max_blocks_per_seq;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.cu = cu_seqlens_k;
  p.num_seqs = num_seqs;
  p.total = total_k;
  p.num_heads = num_kv_heads;
  p.out[0] = static_cast<uint16_t*>(k_out);
  p.out[1] = static_cast<uint16_t*>(v_out);
  p.out_tok_stride[0] = k_out_tok_stride;
  p.out_tok_stride[1] = v_out_tok_stride;
  p.out_head_stride[0] = k_out_head_stride;
  p.out_head_stride[1] = v_out_head_stride;
  p.div_block = divisor(static_cast<uint32_t>(block_size));
  p.div_heads = divisor(static_cast<uint32_t>(num_kv_heads));
  const int tokens = kThreads * kLane / head_dim;  // per workgroup
  const int64_t grid = (static_cast<int64_t>(total_k) + tokens - 1) / tokens * num_kv_heads;
  if (grid > INT32_MAX) return fail(KVP_EINVAL, "%s: too many tokens", fn);
  const auto s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>(grid)), b(kThreads);
  if (head_dim == 64) hipLaunchKernelGGL(load_fp8_kernel<64>, g, b, 0, s, p);
  else if (head_dim == 128) hipLaunchKernelGGL(load_fp8_kernel<128>, g, b, 0, s, p);
  else hipLaunchKernelGGL(load_fp8_kernel<256>, g, b, 0, s, p);
  return launch_status(fn);
}
