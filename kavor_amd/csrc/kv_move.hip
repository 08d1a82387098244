// Keys and values moved inside a paged cache: the drafts that verification keeps, next to their context
// (kvp_keep_drafts), and whole pages (kvp_copy_pages).  Bytes are moved as they are, in every layer at once.
//
// Both are bound by HBM (each byte read and written once) or by the latency of a launch and two or three
// dependent loads.  Neither needs a temporary: a thread owns 16 bytes of every row (page) it moves and takes
// them in an order in which nothing is overwritten before it is read, so no thread waits for another.
// The drafts of 64 trees of 5 to 25 rows that stay, in 28 layers (41 MB): 17 us, 4.9 TB/s read and written; with nontemporal
// loads 24, as they were written and attended to just before.  A page of 1 MiB in 28 layers: 11.4 us, 5.1 TB/s; 96
// pages of 256 KiB from 32: 168 us, 5.6 TB/s; 300 of 129 KiB, half of which are also read: 407 us, 5.5 TB/s (cached
// loads: 429).
#include <algorithm>
#include <new>
#include <vector>

#include "paged.h"

namespace kvp {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRows = 64;  // rows of a sequence, as in kvp_tree_attention
constexpr int kBatch = 8;     // rows in flight per thread
constexpr int kMostGroups = 2048;  // workgroups from which one takes several layers

// ---------------------------------------------------------------- drafts kept

struct KeepParams {
  uint8_t* cache[2];  // k, v; strides in bytes
  int64_t layer_stride, blk_stride, slot_stride, head_stride;
  uint8_t* scale[2];  // or null
  int64_t scale_layer_stride, scale_blk_stride, scale_head_stride;
  int32_t layers, layers_per_wg, num_cache_blocks, block_size, max_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* path;
  int64_t path_stride;
  int32_t width;  // entries of a path
  const int32_t* accepted;
  const int32_t* cu;
  const int32_t* lens;
  int32_t* new_lens;
  int32_t heads, row_units, units;  // 16-byte units of a head's row; of K and V of a token, with the scale bytes behind
  int32_t parts;                    // workgroups over the units
  Divisor div_block, div_units;
};

__device__ __forceinline__ int64_t of_lane(int64_t x, int lane) {
  const uint64_t v = static_cast<uint64_t>(x);
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<u32>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
                              static_cast<u32>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)));
}

// Moves a unit of each row in `which`, a row's offsets per lane, in layers first .. last - 1.
template <typename V, typename Load, typename Store>
__device__ __forceinline__ void move_rows(unsigned long long which, int64_t src, int64_t dst, uint8_t* base, int first, int last,
                                          int64_t layer_stride, Load load, Store store) {
  unsigned long long rest = which;
  int layer = first;
#pragma unroll 1
  while (layer < last) {  // uniform, as all that follows but the data
    V v[kBatch];
    int64_t to[kBatch];
    int count = 0;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (layer >= last) continue;
      const int row = __builtin_ctzll(rest);
      v[j] = load(base + layer * layer_stride + of_lane(src, row));
      to[j] = layer * layer_stride + of_lane(dst, row);
      ++count;
      rest &= rest - 1;
      if (rest == 0) {
        rest = which;
        ++layer;
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (j < count) store(base + to[j], v[j]);
  }
}

// A sequence's tokens base + path[j] go to base + 1 + j.  A path rises, so path[j] > j and what is written
// was read before: in the batch of the same thread, or an earlier one.
__global__ __launch_bounds__(kThreads) void keep_drafts_kernel(const KeepParams p) {
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int n = p.cu[b + 1] - p.cu[b], len = p.lens[b], kept = p.accepted[b];
  const int entry = lane < p.width ? p.path[b * p.path_stride + lane] : 0;  // with the others: a round trip less
  const bool ok = n > 0 && n <= len && kept >= 0 && kept < n && kept <= p.width;
  if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) p.new_lens[b] = ok ? len - n + 1 + kept : len;
  if (!ok || kept == 0) return;  // uniform
  // every wave finds the moves, one per lane: up to the first entry that does not rise or has no page
  const int row = lane < kept ? entry : n;
  const int before = __shfl_up(row, 1);
  bool good = lane < kept && row < n && row > (lane == 0 ? 0 : before);
  const int from = len - n + row, to = len - n + 1 + lane;
  const int from_page = div_by(max(from, 0), p.div_block), to_page = div_by(max(to, 0), p.div_block);
  good = good && from_page < p.max_blocks;  // to <= from
  const int from_blk = good ? p.block_tables[b * p.bt_stride + from_page] : -1;
  const int to_blk = good ? p.block_tables[b * p.bt_stride + to_page] : -1;
  good = good && from_blk >= 0 && from_blk < p.num_cache_blocks && to_blk >= 0 && to_blk < p.num_cache_blocks;
  const unsigned long long bad = ~__ballot(good);
  const unsigned long long run = bad ? (1ull << __builtin_ctzll(bad)) - 1 : ~0ull;  // lanes before the first bad one
  const unsigned long long which = __ballot((run >> lane & 1) && from != to);        // what is in its place stays there
  if (which == 0) return;  // uniform
  const int from_off = from - from_page * p.block_size, to_off = to - to_page * p.block_size;
  const int unit = blockIdx.x * blockDim.x + threadIdx.x, per_side = p.heads * p.row_units;
  const int first = blockIdx.z * p.layers_per_wg, last = min(first + p.layers_per_wg, p.layers);
  // the whole wave goes both ways: the rows' offsets are its lanes'
  const bool of_rows = unit < 2 * per_side, of_scales = !of_rows && unit < p.units;
  if (__any(of_rows)) {
    const int64_t src = from_blk * p.blk_stride + from_off * p.slot_stride, dst = to_blk * p.blk_stride + to_off * p.slot_stride;
    const int side = unit >= per_side, in_side = of_rows ? unit - side * per_side : 0;
    const int h = div_by(in_side, p.div_units), c = in_side - h * p.row_units;
    move_rows<uint4>(which, src, dst, p.cache[side] + h * p.head_stride + 16 * c, first, last, p.layer_stride,
                     [&](const uint8_t* at) { return of_rows ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0); },
                     [&](uint8_t* at, uint4 v) { if (of_rows) store16_nt(at, v); });
  }
  if (__any(of_scales)) {  // a head's scales: one byte a token
    const int64_t src = from_blk * p.scale_blk_stride + from_off, dst = to_blk * p.scale_blk_stride + to_off;
    const int i = of_scales ? unit - 2 * per_side : 0, side = i >= p.heads, h = i - side * p.heads;
    move_rows<uint8_t>(which, src, dst, p.scale[side] + h * p.scale_head_stride, first, last, p.scale_layer_stride,
                       [&](const uint8_t* at) { return of_scales ? *at : uint8_t{0}; },
                       [&](uint8_t* at, uint8_t v) { if (of_scales) *at = v; });
  }
}

// ---------------------------------------------------------------- pages copied

constexpr int kMaxPairs = 384;  // of a launch: they travel in its arguments, so nothing is copied to the GPU before
constexpr int kHold = -1;       // as a destination: kept in a register; as a source: what was kept

struct PagePairs {
  int32_t src[kMaxPairs], dst[kMaxPairs];
  uint16_t begin[kMaxPairs + 1];  // of each strand's pairs
};
static_assert(sizeof(PagePairs) <= 3900, "kernel arguments have 4 KiB");

struct CopyParams {
  uint8_t* pages;
  int64_t layer_stride, page_stride;  // bytes
  int32_t columns;                    // 16-byte columns of a page
};

// One source and its destinations per strand; no destination is a source.
template <int C>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(const CopyParams p, const PagePairs pairs) {
  const int begin = pairs.begin[blockIdx.y], end = pairs.begin[blockIdx.y + 1];
  const int c0 = blockIdx.x * (kThreads * C) + threadIdx.x;
  uint8_t* layer = p.pages + blockIdx.z * p.layer_stride + 16 * static_cast<int64_t>(c0);
  const uint8_t* src = layer + pairs.src[begin] * p.page_stride;
  uint4 v[C];
#pragma unroll
  for (int j = 0; j < C; ++j)
    if (c0 + j * kThreads < p.columns) v[j] = load16_nt(src + 16 * j * kThreads);
  for (int i = begin; i < end; ++i) {
    uint8_t* dst = layer + pairs.dst[i] * p.page_stride;
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (c0 + j * kThreads < p.columns) store16_nt(dst + 16 * j * kThreads, v[j]);
  }
}

// A strand's pairs in order: no page is written before the last pair that reads it is past, or in its batch.
__global__ __launch_bounds__(kThreads) void copy_pages_ordered_kernel(const CopyParams p, const PagePairs pairs) {
  const int begin = pairs.begin[blockIdx.y], end = pairs.begin[blockIdx.y + 1];
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= p.columns) return;
  uint8_t* layer = p.pages + blockIdx.z * p.layer_stride + 16 * static_cast<int64_t>(c);
  uint4 held = make_uint4(0, 0, 0, 0);
  for (int i = begin; i < end; i += kBatch) {
    uint4 v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (i + j < end && pairs.src[i + j] != kHold) v[j] = load16_nt(layer + pairs.src[i + j] * p.page_stride);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (i + j >= end) continue;
      const int dst = pairs.dst[i + j];
      if (dst == kHold) held = v[j];
      else store16_nt(layer + dst * p.page_stride, pairs.src[i + j] == kHold ? held : v[j]);
    }
  }
}

// What a call's pairs come to.
struct Schedule {
  std::vector<std::pair<int32_t, int32_t>> apart;    // (source, destination) by source: no destination is a source
  std::vector<std::pair<int32_t, int32_t>> ordered;  // behind them: strands side by side
  std::vector<int32_t> begin;                        // of each strand, and the end
};

// Orders pairs so that all reads come before all writes.  A pair has to follow the pairs that read its
// destination; each of those precedes that one alone, so the pairs form trees, and cycles with trees on them.
// Pairs whose destination nobody reads come first, all at once.  The rest is taken tree by tree from the
// leaves, then the cycle that it may end in, with one page of it held back.
// Returns a page that is written twice, or -1.
int32_t schedule_pairs(const int32_t* src, const int32_t* dst, int n, Schedule& out) {
  std::vector<std::pair<int32_t, int32_t>> by_dst;  // (destination, pair)
  by_dst.reserve(n);
  for (int i = 0; i < n; ++i)
    if (src[i] != dst[i]) by_dst.emplace_back(dst[i], i);
    else by_dst.emplace_back(dst[i], -1);  // already there, but written once all the same
  std::sort(by_dst.begin(), by_dst.end());
  for (size_t k = 1; k < by_dst.size(); ++k)
    if (by_dst[k].first == by_dst[k - 1].first) return by_dst[k].first;
  auto writer = [&](int32_t page) {  // the pair that writes a page, or -1
    const auto it = std::lower_bound(by_dst.begin(), by_dst.end(), std::make_pair(page, INT32_MIN));
    return it != by_dst.end() && it->first == page ? it->second : -1;
  };
  std::vector<int32_t> next(n, -1), readers(n, 0), queue;
  for (int i = 0; i < n; ++i) {
    if (src[i] == dst[i]) continue;
    next[i] = writer(src[i]);
    if (next[i] >= 0) ++readers[next[i]];
  }
  for (int i = 0; i < n; ++i)
    if (src[i] != dst[i] && readers[i] == 0) {
      out.apart.emplace_back(src[i], dst[i]);
      queue.push_back(i);
    }
  std::sort(out.apart.begin(), out.apart.end());
  std::vector<char> done(n, 0);
  const size_t leaves = queue.size();
  for (size_t k = 0; k < queue.size(); ++k) {
    done[queue[k]] = 1;
    const int after = next[queue[k]];
    if (after >= 0 && --readers[after] == 0) queue.push_back(after);
  }
  // the strand of a pair: the last pair of its tree, or the least one of its cycle
  std::vector<int32_t> strand(n, -1);
  auto strand_of = [&](int i) {
    std::vector<int32_t> way;
    int at = i;
    while (strand[at] < 0) {
      if (!done[at]) {  // on a cycle
        int least = at;
        for (int k = next[at]; k != at; k = next[k]) least = std::min(least, k);
        strand[at] = least;
        for (int k = next[at]; k != at; k = next[k]) strand[k] = least;
        break;
      }
      way.push_back(at);
      if (next[at] < 0) {
        strand[at] = at;
        break;
      }
      at = next[at];
    }
    for (int k : way) strand[k] = strand[at];
    return strand[i];
  };
  std::vector<std::pair<int32_t, int32_t>> rest;  // (strand, place)
  for (size_t k = leaves; k < queue.size(); ++k) rest.emplace_back(strand_of(queue[k]), static_cast<int32_t>(k));
  for (int i = 0; i < n; ++i)
    if (src[i] != dst[i] && !done[i] && strand_of(i) == i) rest.emplace_back(i, INT32_MAX);  // a cycle, behind its trees
  std::sort(rest.begin(), rest.end());
  for (size_t k = 0; k < rest.size(); ++k) {
    if (k == 0 || rest[k].first != rest[k - 1].first) out.begin.push_back(static_cast<int32_t>(out.ordered.size()));
    if (rest[k].second != INT32_MAX) {
      const int i = queue[rest[k].second];
      out.ordered.emplace_back(src[i], dst[i]);
      continue;
    }
    // pages c0 -> c1 -> .. -> c0: back to front, with the last one held back.  A long one goes through c0
    // piece by piece, so that a launch can end behind any of them: each leaves there what the next one
    // starts with, more than a batch before it is read.
    const int start = rest[k].first;
    std::vector<int32_t> c;  // next[] leads against the copies
    for (int i = start;; i = next[i]) {
      c.push_back(dst[i]);
      if (next[i] == start) break;
    }
    std::reverse(c.begin() + 1, c.end());
    static_assert(kMaxPairs / 4 > kBatch, "the next piece reads c0 behind the batch that wrote it");
    const size_t pieces = (c.size() - 1 + kMaxPairs / 2 - 1) / (kMaxPairs / 2);
    for (size_t j0 = 0, at = 1; j0 < pieces; ++j0) {  // of about equal length
      const size_t end = 1 + (c.size() - 1) * (j0 + 1) / pieces;
      out.ordered.emplace_back(c[end - 1], kHold);
      for (size_t j = end - 1; j > at; --j) out.ordered.emplace_back(c[j - 1], c[j]);
      out.ordered.emplace_back(c[0], c[at]);
      out.ordered.emplace_back(kHold, c[0]);
      at = end;
    }
  }
  out.begin.push_back(static_cast<int32_t>(out.ordered.size()));
  return -1;
}

// Whether elements of these sizes and strides lie apart, each of `inner` bytes.
template <int N>
bool lie_apart(std::pair<int64_t, int64_t> (&dims)[N], int64_t inner) {  // (stride in bytes, size)
  std::sort(dims, dims + N);
  for (const auto& d : dims) {
    if (d.second <= 1) continue;
    if (d.first < inner) return false;
    inner += (d.second - 1) * d.first;
  }
  return true;
}

bool mult16(int64_t stride) { return (stride & 15) == 0; }
bool dim_ok(int32_t d) { return d == 64 || d == 128 || d == 256; }

}  // namespace
}  // namespace kvp

using namespace kvp;

extern "C" int kvp_keep_drafts(void* k_cache, void* v_cache, int64_t cache_layer_stride, int64_t cache_block_stride,
                               int64_t cache_slot_stride, int64_t cache_head_stride, void* k_scale, void* v_scale,
                               int64_t scale_layer_stride, int64_t scale_block_stride, int64_t scale_head_stride,
                               int32_t num_layers, int32_t num_cache_blocks, const int32_t* block_tables,
                               int64_t block_table_stride, const int32_t* path, int64_t path_stride, int32_t path_width,
                               const int32_t* accepted, const int32_t* cu_seqlens_q, const int32_t* cache_seqlens,
                               int32_t num_seqs, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                               int32_t max_blocks_per_seq, int32_t* new_seqlens, void* stream) {
  static const char fn[] = "kvp_keep_drafts";
  clear_error();
  if (!dim_ok(head_dim)) return fail(KVP_EUNSUPPORTED, "%s: head_dim=%d (supported: 64, 128, 256)", fn, head_dim);
  if (num_seqs < 0 || num_layers <= 0 || num_cache_blocks <= 0 || num_kv_heads <= 0 || block_size <= 0 ||
      max_blocks_per_seq <= 0)
    return fail(KVP_EINVAL, "%s: num_seqs=%d num_layers=%d num_cache_blocks=%d num_kv_heads=%d block_size=%d "
                "max_blocks_per_seq=%d", fn, num_seqs, num_layers, num_cache_blocks, num_kv_heads, block_size,
                max_blocks_per_seq);
  if (path_width < 0 || path_width > kMaxRows)
    return fail(KVP_EUNSUPPORTED, "%s: path_width=%d (supported: 0 to %d)", fn, path_width, kMaxRows);
  if (num_seqs > 65535 || num_kv_heads > 1 << 16)
    return fail(KVP_EUNSUPPORTED, "%s: num_seqs=%d num_kv_heads=%d (supported: up to 65535 and 65536)", fn, num_seqs,
                num_kv_heads);
  if (static_cast<int64_t>(max_blocks_per_seq) * block_size > INT32_MAX)
    return fail(KVP_EUNSUPPORTED, "%s: block tables of more than 2^31 tokens", fn);
  if (block_table_stride < max_blocks_per_seq || path_stride < path_width)
    return fail(KVP_EINVAL, "%s: rows of block_tables or path overlap", fn);
  if (!k_cache || !v_cache || (k_scale == nullptr) != (v_scale == nullptr))
    return fail(KVP_EINVAL, "%s: null pointer", fn);
  const int item = k_scale ? 1 : 2;
  if (!aligned16(k_cache) || !aligned16(v_cache) || !mult16(cache_layer_stride * item) ||
      !mult16(cache_block_stride * item) || !mult16(cache_slot_stride * item) || !mult16(cache_head_stride * item))
    return fail(KVP_EINVAL, "%s: cache pointers and strides must be multiples of 16 bytes", fn);
  std::pair<int64_t, int64_t> dims[4] = {{cache_layer_stride * item, num_layers},
                                         {cache_block_stride * item, num_cache_blocks},
                                         {cache_slot_stride * item, block_size},
                                         {cache_head_stride * item, num_kv_heads}};
  std::pair<int64_t, int64_t> scale_dims[3] = {{scale_layer_stride, num_layers},
                                               {scale_block_stride, num_cache_blocks},
                                               {scale_head_stride, num_kv_heads}};
  if (!lie_apart(dims, head_dim * item) || (k_scale && !lie_apart(scale_dims, block_size)))
    return fail(KVP_EINVAL, "%s: rows of the cache overlap", fn);
  if (num_seqs == 0) return KVP_OK;
  if (!block_tables || (!path && path_width > 0) || !accepted || !cu_seqlens_q || !cache_seqlens || !new_seqlens)
    return fail(KVP_EINVAL, "%s: null pointer", fn);
  auto off4 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 3u) != 0; };
  if (off4(block_tables) || off4(path) || off4(accepted) || off4(cu_seqlens_q) || off4(cache_seqlens) ||
      off4(new_seqlens))
    return fail(KVP_EINVAL, "%s: misaligned integers", fn);
  // a sequence's new length is written by one of its workgroups while the others read these
  const int64_t seqs = num_seqs, bytes = 4 * seqs;
  if (overlap(new_seqlens, bytes, cache_seqlens, bytes) || overlap(new_seqlens, bytes, accepted, bytes) ||
      overlap(new_seqlens, bytes, cu_seqlens_q, bytes + 4) ||
      overlap(new_seqlens, bytes, path, seqs, 4 * path_stride, 4 * path_width) ||
      overlap(new_seqlens, bytes, block_tables, seqs, 4 * block_table_stride, 4 * static_cast<int64_t>(max_blocks_per_seq)))
    return fail(KVP_EINVAL, "%s: new_seqlens overlaps an input", fn);
  // a row is moved by threads of its own for K and for V
  if (k_cache == v_cache || (k_scale && k_scale == v_scale))
    return fail(KVP_EINVAL, "%s: k_cache and v_cache, k_scale and v_scale must not be the same memory", fn);
  KeepParams p{};
  p.cache[0] = static_cast<uint8_t*>(k_cache);
  p.cache[1] = static_cast<uint8_t*>(v_cache);
  p.layer_stride = cache_layer_stride * item;
  p.blk_stride = cache_block_stride * item;
  p.slot_stride = cache_slot_stride * item;
  p.head_stride = cache_head_stride * item;
  p.scale[0] = static_cast<uint8_t*>(k_scale);
  p.scale[1] = static_cast<uint8_t*>(v_scale);
  p.scale_layer_stride = scale_layer_stride;
  p.scale_blk_stride = scale_block_stride;
  p.scale_head_stride = scale_head_stride;
  p.layers = num_layers;
  p.num_cache_blocks = num_cache_blocks;
  p.block_size = block_size;
  p.max_blocks = max_blocks_per_seq;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.path = path;
  p.path_stride = path_stride;
  p.width = path_width;
  p.accepted = accepted;
  p.cu = cu_seqlens_q;
  p.lens = cache_seqlens;
  p.new_lens = new_seqlens;
  p.heads = num_kv_heads;
  p.row_units = head_dim * item / 16;
  p.units = 2 * num_kv_heads * (p.row_units + (k_scale ? 1 : 0));
  p.div_block = divisor(static_cast<uint32_t>(block_size));
  p.div_units = divisor(static_cast<uint32_t>(p.row_units));
  // workgroups of as many waves as the units have, four at most
  const int threads = std::min(kThreads, (p.units + 63) / 64 * 64), parts = (p.units + threads - 1) / threads;
  const int64_t all = static_cast<int64_t>(parts) * num_seqs * num_layers;
  p.layers_per_wg = static_cast<int>(std::min<int64_t>(num_layers, std::max<int64_t>(1, all / kMostGroups)));
  const int z = (num_layers + p.layers_per_wg - 1) / p.layers_per_wg;
  if (z > 65535) return fail(KVP_EUNSUPPORTED, "%s: too many layers", fn);
  hipLaunchKernelGGL(keep_drafts_kernel, dim3(parts, num_seqs, z), dim3(threads), 0, static_cast<hipStream_t>(stream), p);
  return launch_status(fn);
}

extern "C" int kvp_copy_pages(void* pages, int64_t layer_stride, int64_t page_stride, int32_t num_layers,
                              int32_t num_pages, int64_t page_bytes, const int32_t* src, const int32_t* dst,
                              int32_t num_pairs, void* stream) {
  static const char fn[] = "kvp_copy_pages";
  clear_error();
  if (num_layers < 0 || num_pages < 0 || num_pairs < 0 || page_bytes < 0)
    return fail(KVP_EINVAL, "%s: num_layers=%d num_pages=%d page_bytes=%lld num_pairs=%d", fn, num_layers, num_pages,
                static_cast<long long>(page_bytes), num_pairs);
  if (num_pairs == 0 || num_layers == 0) return KVP_OK;
  if (!pages || !src || !dst) return fail(KVP_EINVAL, "%s: null pointer", fn);
  if (!aligned16(pages) || !mult16(layer_stride) || !mult16(page_stride) || !mult16(page_bytes))
    return fail(KVP_EINVAL, "%s: pages, strides and page_bytes must be multiples of 16 bytes", fn);
  if (num_layers > 65535 || page_bytes >= int64_t{1} << 34)
    return fail(KVP_EUNSUPPORTED, "%s: num_layers=%d page_bytes=%lld (supported: up to 65535, below 2^34)", fn,
                num_layers, static_cast<long long>(page_bytes));
  std::pair<int64_t, int64_t> dims[2] = {{layer_stride, num_layers}, {page_stride, num_pages}};
  if (!lie_apart(dims, page_bytes)) return fail(KVP_EINVAL, "%s: pages overlap", fn);
  for (int i = 0; i < num_pairs; ++i)
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
      return fail(KVP_EINVAL, "%s: pair %d copies page %d to %d of %d", fn, i, src[i], dst[i], num_pages);
  const CopyParams p{static_cast<uint8_t*>(pages), layer_stride, page_stride, static_cast<int32_t>(page_bytes / 16)};
  const auto s = static_cast<hipStream_t>(stream);
  Schedule plan;
  try {
    const int32_t twice = schedule_pairs(src, dst, num_pairs, plan);
    if (twice >= 0) return fail(KVP_EINVAL, "%s: page %d is written twice", fn, twice);
  } catch (const std::bad_alloc&) {
    return fail(KVP_EINVAL, "%s: out of host memory for %d pairs", fn, num_pairs);
  }
  if (p.columns == 0 || (plan.apart.empty() && plan.ordered.empty())) return KVP_OK;
  const LaunchOrder order;  // an ordered launch relies on those before it
  PagePairs pairs;
  int count = 0, strands = 0;
  auto launch = [&](auto kernel, int columns_per_wg) {
    if (count == 0) return;
    pairs.begin[strands] = static_cast<uint16_t>(count);
    hipLaunchKernelGGL(kernel, dim3((p.columns + columns_per_wg - 1) / columns_per_wg, strands, num_layers),
                       dim3(kThreads), 0, s, p, pairs);
    count = strands = 0;
  };
  auto add = [&](const std::pair<int32_t, int32_t>& pair) {
    pairs.src[count] = pair.first;
    pairs.dst[count++] = pair.second;
  };
  auto launch_apart = [&] {
    const int64_t threads = static_cast<int64_t>(p.columns) * num_layers * strands;
    if (threads >= 1 << 20) launch(copy_pages_kernel<4>, 4 * kThreads);
    else launch(copy_pages_kernel<1>, kThreads);
  };
  for (size_t i = 0; i < plan.apart.size(); ++i) {
    if (count == kMaxPairs) launch_apart();
    if (count == 0 || plan.apart[i].first != plan.apart[i - 1].first) pairs.begin[strands++] = static_cast<uint16_t>(count);
    add(plan.apart[i]);
  }
  launch_apart();
  for (size_t k = 0; k + 1 < plan.begin.size(); ++k) {
    int at = plan.begin[k];
    const int end = plan.begin[k + 1];
    if (count + end - at > kMaxPairs) launch(copy_pages_ordered_kernel, kThreads);
    while (at < end) {  // more than a launch holds: cut where nothing is held back
      int cut = std::min(end, at + kMaxPairs - count);
      for (int j = cut - 1; cut < end && j >= at && plan.ordered[j].first != kHold; --j)
        if (plan.ordered[j].second == kHold) cut = j;
      pairs.begin[strands++] = static_cast<uint16_t>(count);
      for (; at < cut; ++at) add(plan.ordered[at]);
      if (at < end) launch(copy_pages_ordered_kernel, kThreads);
    }
  }
  launch(copy_pages_ordered_kernel, kThreads);
  return launch_status(fn);
}
