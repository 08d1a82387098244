"""Drop-in attention boundary of the paged KV-cache path, backed by libkvpath.so.

Mirrors kavor/layers/attention/flash_attention_kvcache.py:
  store_kvcache(key, value, k_cache, v_cache, slot_mapping)      (:37-46)
  Attention(num_heads, head_dim, scale, num_kv_heads, num_kv_slots=1)
      .forward(q, k, v, slot=0)                                   (:49-84)
and replaces the two flash-attn calls it makes with
  paged_decode(...)    for flash_attn_with_kvcache(...)           (:80-83)
  varlen_prefill(...)  for flash_attn_varlen_func(...)            (:76-79)
which keep flash-attn's argument names and meaning.  Without a counterpart there, and in the
same manner:
  store_kvcache_fp8, load_kvcache_fp8   a quantised cache (e4m3, one power-of-two scale for
                                        each token and head) written, and read back in bf16
  paged_decode_fp8                      paged_decode over it
  tree_attention                        drafted tokens over a cache of either kind
Every function here only
validates layouts and forwards raw pointers and strides to the C ABI (include/kvpath.h)
on the current stream; nothing computes on the host and there is no fallback.
"""

from __future__ import annotations

from functools import lru_cache

import torch
from torch import nn

from kavor_amd._lib import check, lib
from kavor_amd.layers.workspace import Workspaces, retired
from kavor_amd.utils.context import get_context

__all__ = [
    "store_kvcache", "paged_decode", "paged_decode_fused", "varlen_prefill", "Attention",
    "reserve_decode_workspace", "decode_workspace_bytes",
    "reserve_prefill_workspace", "prefill_workspace_bytes",
    "flash_attn_with_kvcache", "flash_attn_varlen_func",
    "store_kvcache_fp8", "load_kvcache_fp8", "paged_decode_fp8", "tree_attention",
    "reserve_tree_workspace", "tree_workspace_bytes",
]


def _stream(t: torch.Tensor) -> int:
    """The current stream's handle (building a torch.cuda.Stream for it takes 3.5 us)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _require_cuda_bf16(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor, got device {t.device}")
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")


def _require_int32(name: str, t: torch.Tensor, device: torch.device) -> None:
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must live on {device}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


# ----------------------------------------------------------------------------- append

def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Writes key[i] / value[i] into slot slot_mapping[i] of k_cache / v_cache.

    Same contract and layout assertions as store_kvcache in
    kavor/layers/attention/flash_attention_kvcache.py:37-46: key/value are
    [N, num_kv_heads, head_dim] with contiguous heads (row strides may differ), the
    caches are [num_blocks, block_size, num_kv_heads, head_dim] views whose block
    stride may exceed block_size*num_kv_heads*head_dim (K/V interleaved pages), and
    slot -1 is skipped.  Bit-exact copy on the device.
    """
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    key_str, value_str, cache_str = key.stride(), value.stride(), k_cache.stride()
    assert key_str[-1] == 1 and value_str[-1] == 1
    assert key_str[1] == head_dim and value_str[1] == head_dim
    assert slot_mapping.numel() == N
    assert value.shape == key.shape
    assert k_cache.shape == v_cache.shape and cache_str == v_cache.stride()
    assert cache_str[1] == D
    assert k_cache.dim() == 4
    num_blocks, block_size, cache_heads, cache_dim = k_cache.shape
    assert (cache_heads, cache_dim) == (num_heads, head_dim)
    _require_cuda_bf16("key", key)
    _require_cuda_bf16("value", value)
    _require_cuda_bf16("k_cache", k_cache)
    _require_cuda_bf16("v_cache", v_cache)
    _require_int32("slot_mapping", slot_mapping, key.device)
    rc = lib().kvp_append_bf16(
        key.data_ptr(), key_str[0], key_str[1],
        value.data_ptr(), value_str[0], value_str[1],
        k_cache.data_ptr(), v_cache.data_ptr(),
        cache_str[0], cache_str[1], cache_str[2], num_blocks * block_size,
        slot_mapping.data_ptr(), N, num_heads, head_dim, block_size, _stream(key))
    check("kvp_append_bf16", rc)


# ----------------------------------------------------------------------------- decode

_decode_workspaces = Workspaces("paged-decode", "reserve_decode_workspace")
_workspaces = _decode_workspaces.default
_retired_workspaces = retired


@lru_cache(maxsize=1024)  # arithmetic on the sizes
def decode_workspace_bytes(max_num_seqs: int, num_q_heads: int, head_dim: int,
                           max_blocks_per_seq: int, block_size: int) -> int:
    return int(lib().kvp_decode_workspace_bytes(max_num_seqs, num_q_heads, head_dim,
                                                 max_blocks_per_seq, block_size))


def reserve_decode_workspace(max_num_seqs: int, num_q_heads: int, head_dim: int,
                             max_blocks_per_seq: int, block_size: int,
                             device: torch.device | str | int) -> torch.Tensor:
    """Allocates (or grows) the current stream's decode workspace on a device.  Call before graph
    capture with the largest batch a captured graph will use: the capture takes the buffer over,
    and eager calls, which need no reservation, go on in another.  It holds the states of
    one-step (32-token) ranges, four times as many as kvp_decode_workspace_bytes counts for the
    same block table: the one-launch step runs a small batch faster in them."""
    return _decode_workspaces.get(
        device, decode_workspace_bytes(max_num_seqs, num_q_heads, head_dim, 4 * max_blocks_per_seq, block_size),
        decode_workspace_bytes(max_num_seqs, num_q_heads, head_dim, max_blocks_per_seq, block_size))


def _decode_workspace(index, stream, num_seqs, num_q_heads, head_dim, max_blocks, block_size) -> torch.Tensor:
    nbytes = decode_workspace_bytes(num_seqs, num_q_heads, head_dim, 4 * max_blocks, block_size)
    ws = _decode_workspaces.ready(index, stream, nbytes)
    if ws is None:
        ws = reserve_decode_workspace(num_seqs, num_q_heads, head_dim, max_blocks, block_size, index)
    return ws


# ----------------------------------------------------------------------------- prefill workspace

_prefill_pool = Workspaces("prefill", "reserve_prefill_workspace")
_prefill_workspaces = _prefill_pool.default
_split_pool = Workspaces("split prefill", "reserve_prefill_workspace")


@lru_cache(maxsize=1024)
def prefill_workspace_bytes(num_seqs: int, max_seqlen_q: int, num_q_heads: int, num_kv_heads: int) -> int:
    return int(lib().kvp_prefill_workspace_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads))


@lru_cache(maxsize=1024)
def _prefill_split_bytes(num_seqs: int, max_seqlen_q: int, num_q_heads: int, num_kv_heads: int) -> int:
    nbytes = int(lib().kvp_prefill_split_workspace_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads))
    return -(-nbytes // (1 << 20)) << 20  # one size for all launches that can be split: their work lists are small


# Query tiles x kv heads of a launch that may be split, at most, and keys from which one may be.
_SPLIT_TILES, _SPLIT_MIN_KEYS = 512, 1024


def _may_split(num_seqs: int, max_seqlen_q: int, max_keys: int, num_q_heads: int, num_kv_heads: int) -> bool:
    """Whether the kernel may cut the keys of such a batch, given room for the partial states."""
    group = num_q_heads // num_kv_heads if num_kv_heads else 0
    if max_keys < _SPLIT_MIN_KEYS or group not in (1, 2, 4, 5, 8):
        return False
    return 0 < num_seqs * -(-max_seqlen_q // (128 // group)) * num_kv_heads <= _SPLIT_TILES


def _split_pays(num_seqs: int, total_q: int, max_seqlen_q: int, max_keys: int, num_q_heads: int,
                num_kv_heads: int) -> bool:
    """Whether cutting the keys of a batch that may be split is likely to gain, from what the host
    knows of its lengths.

    The plan kernel decides by the lengths themselves, but a split launch in which it cuts nothing
    costs 3 to 5 us over an uncut one (its plan, and a merge that finds no work): 4 prompts of
    1024 tokens (16q/8kv) 45.6 -> 48.7 us, 4 of 700 on 2048 cached 84.8 -> 88.2, 2 of 750 on
    15000 (32q/8kv) 408 -> 411.  So the plan's cost model runs here on an average tile first.  A
    batch of about equal new lengths is taken to have equal cached ones, a ragged batch to have
    0.6 of the longest on average; averages and thresholds are fitted over 900 shapes.  17 of them
    are slower than uncut, by 4 us each (174 where every batch that may be split takes the split
    launch); 50 of the 689 that would gain stay uncut, above all equal turns on very unequal
    histories (4 of 509 tokens on 0 to 16384: 425 us against 301)."""
    tok = 128 // (num_q_heads // num_kv_heads)
    slots = _SPLIT_TILES / num_kv_heads
    even = total_q >= 0.95 * num_seqs * max_seqlen_q
    longest = -(-max_keys // 64)  # all in key tiles
    own = max_seqlen_q / 64
    cached = max(0.0, longest - own)
    tiles = num_seqs * -(-max_seqlen_q // tok)
    if not even:
        tiles = min(tiles, total_q / tok + 0.5 * num_seqs)
        cached, own = 0.6 * cached, 0.7 * own
    mean = cached + own / 2
    arrive = num_seqs * (cached + own) * num_kv_heads / 300
    least = (1.0 if num_seqs == 1 else 0.95 if even else 0.9) * max(longest, arrive)
    for parts in (2, 3, 4, 6, 8, 12, 16):
        chunk = -(-longest // parts)
        if chunk < 8:
            break
        units = tiles * min(parts, mean / chunk + 0.5)
        busy = chunk if units <= slots else tiles * mean / slots + chunk / 2
        whole = tiles * min(1.0, max(0.0, chunk - cached) / own)
        if max(arrive, busy) + (units - whole) * num_kv_heads / 48 + 4 < least:
            return True
    return False


def reserve_prefill_workspace(num_seqs: int, max_seqlen_q: int, num_q_heads: int, num_kv_heads: int,
                              device: torch.device | str | int) -> torch.Tensor:
    """Allocates (or grows) the current stream's prefill workspaces on a device: the work list of a
    launch, which is returned, and the partial states of a batch whose keys are split
    (kvp_prefill_split_workspace_bytes, 69 MB).  A caller that captures prefill into a graph
    reserves the largest batch first: the capture takes the buffers over.  Eager calls need no
    reservation, and hold partial states only once a batch may be split."""
    _split_pool.get(device, _prefill_split_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads))
    return _work_list(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads, device)


@lru_cache(maxsize=1024)
def _work_list_bytes(num_seqs: int, max_seqlen_q: int, num_q_heads: int, num_kv_heads: int) -> int:
    nbytes = prefill_workspace_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads)
    return 1 << max(4095, nbytes - 1).bit_length()  # so that batches of growing size allocate few buffers


def _work_list(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads, device) -> torch.Tensor:
    return _prefill_pool.get(device, _work_list_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads),
                             prefill_workspace_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads))


@lru_cache(maxsize=4096)  # the layers of a step share one answer
def _split_room(num_seqs, total_q, max_seqlen_q, max_keys, num_q_heads, num_kv_heads) -> int:
    """Bytes of the workspace that a split launch of such a batch takes; 0 for an uncut one."""
    if _may_split(num_seqs, max_seqlen_q, max_keys, num_q_heads, num_kv_heads) and \
            _split_pays(num_seqs, total_q, max_seqlen_q, max_keys, num_q_heads, num_kv_heads):
        return _prefill_split_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads)
    return 0


def _prefill_workspace(index, stream, num_seqs, total_q, max_seqlen_q, max_keys, num_q_heads,
                       num_kv_heads) -> torch.Tensor:
    room = _split_room(num_seqs, total_q, max_seqlen_q, max_keys, num_q_heads, num_kv_heads)
    if room:
        ws = _split_pool.ready(index, stream, room)
        if ws is None:
            ws = _split_pool.get(index, room, optional=True)
        if ws is not None:  # inside a capture without it the launch is not split
            return ws
    ws = _prefill_pool.ready(index, stream, _work_list_bytes(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads))
    return ws if ws is not None else _work_list(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads, index)


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 cache_seqlens: torch.Tensor, block_table: torch.Tensor, softmax_scale: float,
                 causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """Paged decode attention, one query token per sequence.

    Argument meaning follows flash_attn_with_kvcache as called at
    kavor/layers/attention/flash_attention_kvcache.py:81-83: q is [B, 1, Hq, D] (or
    [B, Hq, D]), the caches are [num_blocks, block_size, Hkv, D], cache_seqlens int32 [B]
    counts the cached tokens including the one just appended, block_table int32
    [B, max_blocks] (entries past ceil(len/block_size) are never read).  Returns
    [B, 1, Hq, D] (or [B, Hq, D]) in bf16.  `causal` is accepted for signature
    compatibility; with one query token it changes nothing.
    """
    del causal
    if q.dim() == 4 and q.shape[1] == 1:
        q3, four_d = q[:, 0], True
    elif q.dim() == 3:
        q3, four_d = q, False
    else:
        raise ValueError(f"paged_decode takes one query token per sequence, got q of shape {tuple(q.shape)}")
    B, Hq, D = q3.shape
    _require_cuda_bf16("q", q3)
    _require_cuda_bf16("k_cache", k_cache)
    _require_cuda_bf16("v_cache", v_cache)
    cache_str, q_str = k_cache.stride(), q3.stride()
    if k_cache.shape != v_cache.shape or cache_str != v_cache.stride():
        raise ValueError("k_cache and v_cache must share shape and strides")
    num_blocks, block_size, Hkv, Dk = k_cache.shape
    if Dk != D or cache_str[3] != 1 or q_str[2] != 1:
        raise ValueError("head_dim mismatch or non-contiguous head_dim")
    _require_int32("cache_seqlens", cache_seqlens, q3.device)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise ValueError("block_table must be an int32 [B, max_blocks] tensor with contiguous rows")
    if cache_seqlens.numel() < B or block_table.shape[0] < B:
        raise ValueError("cache_seqlens / block_table have fewer rows than q")
    if out is None:
        out3 = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=q3.device)
        out = out3.unsqueeze(1) if four_d else out3
    else:
        out3 = out[:, 0] if out.dim() == 4 else out
        if out3.shape != (B, Hq, D) or out3.dtype != torch.bfloat16 or out3.stride(2) != 1:
            raise ValueError("out must be bf16 [B, 1, Hq, D] or [B, Hq, D] with contiguous head_dim")
    max_blocks = block_table.shape[1]
    stream = _stream(q3)
    ws = _decode_workspace(q3.get_device(), stream, B, Hq, D, max_blocks, block_size)
    rc = lib().kvp_paged_decode_bf16(
        q3.data_ptr(), q_str[0], q_str[1],
        k_cache.data_ptr(), v_cache.data_ptr(),
        cache_str[0], cache_str[1], cache_str[2], num_blocks,
        block_table.data_ptr(), block_table.stride(0),
        cache_seqlens.data_ptr(), B, Hq, Hkv, D, block_size, max_blocks,
        float(softmax_scale),
        out3.data_ptr(), out3.stride(0), out3.stride(1),
        ws.data_ptr(), ws.numel(), stream)
    check("kvp_paged_decode_bf16", rc)
    return out


def paged_decode_fused(qkv: torch.Tensor, cos_sin: torch.Tensor,
                       q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, eps: float,
                       num_q_heads: int, num_kv_heads: int, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, slot_mapping: torch.Tensor, cache_seqlens: torch.Tensor,
                       block_table: torch.Tensor, softmax_scale: float,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """A Qwen3 decode step of one attention layer in one launch: q/k RMSNorm + RoPE of
    each sequence's new token from its qkv row, the append of its k / v at slot_mapping,
    and paged decode attention over cache_seqlens tokens (the last one being the new
    token).  Returns [B, Hq, 128] bf16.  The token's position is cache_seqlens - 1 and
    slot_mapping must hold the slot of that position, as the engine's decode metadata
    has them."""
    B = qkv.shape[0]
    D = k_cache.shape[-1]
    for name, t in (("qkv", qkv), ("k_cache", k_cache), ("v_cache", v_cache)):
        _require_cuda_bf16(name, t)
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] != (num_q_heads + 2 * num_kv_heads) * D:
        raise ValueError("qkv must be [B, (Hq + 2 Hkv) * head_dim] with contiguous rows")
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("k_cache and v_cache must share shape and strides")
    num_blocks, block_size, Hkv, _ = k_cache.shape
    if Hkv != num_kv_heads:
        raise ValueError("cache heads do not match num_kv_heads")
    for name, t in (("slot_mapping", slot_mapping), ("cache_seqlens", cache_seqlens)):
        _require_int32(name, t, qkv.device)
        if t.numel() < B:
            raise ValueError(f"{name} has fewer rows than qkv")
    if cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.shape[1] != D:
        raise ValueError("cos_sin must be a contiguous fp32 [max_position, head_dim] table")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise ValueError("block_table must be an int32 [B, max_blocks] tensor with contiguous rows")
    if out is None:
        out = torch.empty(B, num_q_heads, D, dtype=torch.bfloat16, device=qkv.device)
    max_blocks = block_table.shape[1]
    stream = _stream(qkv)
    ws = _decode_workspace(qkv.get_device(), stream, B, num_q_heads, D, max_blocks, block_size)
    rc = lib().kvp_paged_decode_fused_bf16(
        qkv.data_ptr(), qkv.stride(0), cos_sin.data_ptr(), cos_sin.shape[0],
        q_norm_weight.data_ptr(), k_norm_weight.data_ptr(), float(eps),
        k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
        num_blocks, slot_mapping.data_ptr(), block_table.data_ptr(), block_table.stride(0),
        cache_seqlens.data_ptr(), B, num_q_heads, num_kv_heads, D, block_size, max_blocks,
        float(softmax_scale), out.data_ptr(), out.stride(0), out.stride(1),
        ws.data_ptr(), ws.numel(), stream)
    check("kvp_paged_decode_fused_bf16", rc)
    return out


# ----------------------------------------------------------------------------- prefill

def varlen_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, max_seqlen_q: int,
                   cu_seqlens_q: torch.Tensor, max_seqlen_k: int, cu_seqlens_k: torch.Tensor,
                   softmax_scale: float, causal: bool = True,
                   block_table: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Packed variable-length attention over dense or paged K/V (bf16 MFMA).

    Argument meaning follows flash_attn_varlen_func as called at
    kavor/layers/attention/flash_attention_kvcache.py:76-79: q is [Tq, Hq, D]; with
    block_table None, k / v are [Tk, Hkv, D] rows addressed through cu_seqlens_k; with
    a block_table they are the paged caches [num_blocks, block_size, Hkv, D].  The
    causal mask is bottom-right aligned.  Returns [Tq, Hq, D] bf16.  The kernel reads lengths
    on the device; max_seqlen_k (0 or no int: unknown) only helps to choose the launch.
    """
    Tq, Hq, D = q.shape
    _require_cuda_bf16("q", q)
    _require_cuda_bf16("k", k)
    _require_cuda_bf16("v", v)
    _require_int32("cu_seqlens_q", cu_seqlens_q, q.device)
    _require_int32("cu_seqlens_k", cu_seqlens_k, q.device)
    num_seqs = cu_seqlens_q.numel() - 1
    if cu_seqlens_k.numel() != num_seqs + 1:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must have the same length")
    if q.stride(2) != 1 or k.stride(-1) != 1 or v.stride(-1) != 1:
        raise ValueError("head_dim must be contiguous in q, k and v")
    if out is None:
        out = torch.empty(Tq, Hq, D, dtype=torch.bfloat16, device=q.device)
    if block_table is None:
        if k.dim() != 3 or v.shape != k.shape:
            raise ValueError("dense k / v must be [Tk, Hkv, D] of equal shape")
        Hkv = k.shape[1]
        kstr = (0, k.stride(0), k.stride(1))
        vstr = (0, v.stride(0), v.stride(1))
        bt_ptr, bt_stride, num_blocks, block_size, max_blocks = 0, 0, 0, 0, 0
    else:
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("paged k / v must be [num_blocks, block_size, Hkv, D] of equal shape")
        if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
            raise ValueError("block_table must be an int32 [B, max_blocks] tensor with contiguous rows")
        if block_table.shape[0] < num_seqs:
            raise ValueError("block_table has fewer rows than sequences")
        num_blocks, block_size, Hkv = k.shape[0], k.shape[1], k.shape[2]
        kstr = (k.stride(0), k.stride(1), k.stride(2))
        vstr = (v.stride(0), v.stride(1), v.stride(2))
        bt_ptr, bt_stride, max_blocks = block_table.data_ptr(), block_table.stride(0), block_table.shape[1]
    if k.shape[-1] != D:
        raise ValueError("head_dim mismatch between q and k")
    ws, stream = None, _stream(q)
    if num_seqs:
        max_keys = max_blocks * block_size if block_table is not None else int(max_seqlen_q)
        if isinstance(max_seqlen_k, int) and 0 < max_seqlen_k < max_keys:
            max_keys = max_seqlen_k
        ws = _prefill_workspace(q.get_device(), stream, num_seqs, Tq, int(max_seqlen_q), max_keys if causal else 0, Hq,
                                Hkv)
    rc = lib().kvp_varlen_prefill_bf16(
        q.data_ptr(), q.stride(0), q.stride(1),
        k.data_ptr(), *kstr,
        v.data_ptr(), *vstr,
        bt_ptr, bt_stride, num_blocks, block_size, max_blocks,
        cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), num_seqs, int(max_seqlen_q),
        Hq, Hkv, D, float(softmax_scale), 1 if causal else 0,
        out.data_ptr(), out.stride(0), out.stride(1),
        ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0, stream)
    check("kvp_varlen_prefill_bf16", rc)
    return out


# flash-attn spellings, so call sites written against flash_attn keep working.
flash_attn_with_kvcache = paged_decode
flash_attn_varlen_func = varlen_prefill


# ----------------------------------------------------------------------------- quantised cache

def _launch(fn: str, index: int, *args) -> None:
    """Calls a library function whose tensors are on device `index`, with that device current."""
    if torch._C._cuda_getDevice() == index:
        rc = getattr(lib(), fn)(*args)
    else:
        with torch.cuda.device(index):
            rc = getattr(lib(), fn)(*args)
    check(fn, rc)


_FP8 = torch.float8_e4m3fn


# Checks of small calls cost as much as their kernels: what is right passes in one expression, and only
# what is not is looked at again for its message.

def _is(t: torch.Tensor, dtype: torch.dtype, index: int, dim: int) -> bool:
    """Whether t has these, with a contiguous last dimension."""
    return t.dtype is dtype and t.get_device() == index and t.dim() == dim and (t.stride(-1) == 1 or t.shape[-1] <= 1)


def _refuse(name: str, t: torch.Tensor, dtype: torch.dtype, dim: int, device: torch.device) -> None:
    raise ValueError(f"{name} must be a {dim}-d {dtype} tensor on {device} whose last dimension is contiguous, got "
                     f"{t.dim()}-d {t.dtype} on {t.device} with strides {tuple(t.stride())}")


def _require(name: str, t: torch.Tensor, dtype: torch.dtype, like: torch.Tensor, dim: int) -> None:
    if not _is(t, dtype, like.get_device(), dim):
        _refuse(name, t, dtype, dim, like.device)


def _paired(k: torch.Tensor, v: torch.Tensor, k_name: str, dtype: torch.dtype, like: torch.Tensor, dim: int):
    """Shape and strides of a K tensor that its V tensor shares."""
    shape, strides = k.shape, k.stride()
    index = like.get_device()
    if not (_is(k, dtype, index, dim) and _is(v, dtype, index, dim) and shape == v.shape and strides == v.stride()):
        v_name = k_name.replace("k", "v", 1)
        _require(k_name, k, dtype, like, dim)
        _require(v_name, v, dtype, like, dim)
        raise ValueError(f"{k_name} and {v_name} must share shape and strides")
    return shape, strides


def _quantised(k_cache, v_cache, k_scale, v_scale, like: torch.Tensor):
    """The shape of a quantised cache, and its pointers and strides as the library takes them."""
    shape, cs = _paired(k_cache, v_cache, "k_cache", _FP8, like, 4)
    scales, ss = _paired(k_scale, v_scale, "k_scale", torch.uint8, like, 3)
    if scales != (shape[0], shape[2], shape[1]):
        raise ValueError(f"the scales must be [num_blocks, num_kv_heads, block_size] = "
                         f"{(shape[0], shape[2], shape[1])}, got {tuple(scales)}")
    return shape, (k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2],
                   k_scale.data_ptr(), v_scale.data_ptr(), ss[0], ss[1])


def _ints(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if not (t.dtype is torch.int32 and t.get_device() == like.get_device() and t.is_contiguous()):
        _require_int32(name, t, like.device)


def _table(block_table: torch.Tensor, rows: int, like: torch.Tensor):
    if not _is(block_table, torch.int32, like.get_device(), 2):
        _refuse("block_table", block_table, torch.int32, 2, like.device)
    n, width = block_table.shape
    if n < rows:
        raise ValueError("block_table has fewer rows than sequences")
    # a single row may have any stride; the library refuses rows that overlap
    return block_table.data_ptr(), block_table.stride(0) if n > 1 else width, width


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """store_kvcache into a quantised cache: key[i] / value[i] ([N, num_kv_heads, head_dim] bf16) go to
    slot slot_mapping[i], each head's row divided by the least power of two that brings it within
    e4m3's range and rounded to nearest even.

    The caches are [num_blocks, block_size, num_kv_heads, head_dim] in float8_e4m3fn, the scales
    [num_blocks, num_kv_heads, block_size] in uint8; byte e stands for 2^(e - 127), and value q of
    its row for 2^(e - 127) q.  Slots outside the cache, -1 among them, are skipped; a slot that
    several tokens name is left with bytes of one and perhaps the scale of another.  An infinity is
    stored as NaN."""
    index = key.get_device()
    if not (index >= 0 and _is(key, torch.bfloat16, index, 3) and _is(value, torch.bfloat16, index, 3)):
        _require_cuda_bf16("key", key)
        _require("key", key, torch.bfloat16, key, 3)
        _require("value", value, torch.bfloat16, key, 3)
    (num_blocks, block_size, heads, dim), cache = _quantised(k_cache, v_cache, k_scale, v_scale, key)
    shape, ks, vs = key.shape, key.stride(), value.stride()
    N = shape[0]
    if value.shape != shape:
        raise ValueError("key and value must share their shape")
    if shape[1] != heads or shape[2] != dim:
        raise ValueError(f"key and value must be [N, {heads}, {dim}] as the caches, got {tuple(shape)}")
    _ints("slot_mapping", slot_mapping, key)
    if slot_mapping.numel() != N:
        raise ValueError("slot_mapping must have one entry per token")
    _launch("kvp_append_fp8", index, key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1], *cache,
            num_blocks * block_size, slot_mapping.data_ptr(), N, heads, dim, block_size,
            torch._C._cuda_getCurrentRawStream(index))


def load_kvcache_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                     block_table: torch.Tensor, cu_seqlens_k: torch.Tensor, total_k: int,
                     out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Reads the sequences of a quantised cache (see store_kvcache_fp8) back as packed bf16 k and v
    [total_k, num_kv_heads, head_dim], which varlen_prefill takes as dense k / v: token j of
    sequence b is row cu_seqlens_k[b] + j.  total_k is the host's copy of cu_seqlens_k[-1]; rows
    of `out` that no sequence has are left as they were.  Tokens of invalid blocks are NaN."""
    if not k_cache.is_cuda:
        raise ValueError(f"k_cache must be a CUDA (HIP) tensor, got device {k_cache.device}")
    (num_blocks, block_size, heads, dim), cache = _quantised(k_cache, v_cache, k_scale, v_scale, k_cache)
    _ints("cu_seqlens_k", cu_seqlens_k, k_cache)
    num_seqs, total_k = cu_seqlens_k.numel() - 1, int(total_k)
    if num_seqs < 0 or total_k < 0:
        raise ValueError("cu_seqlens_k must have an entry more than sequences, and total_k not be negative")
    bt, bt_stride, width = _table(block_table, num_seqs, k_cache)
    if out is None:
        out = tuple(torch.empty((total_k, heads, dim), dtype=torch.bfloat16, device=k_cache.device) for _ in range(2))
    k, v = out
    for name, t in (("out[0]", k), ("out[1]", v)):
        _require(name, t, torch.bfloat16, k_cache, 3)
        if t.shape[0] < total_k or t.shape[1:] != (heads, dim):
            raise ValueError(f"{name} must be [{total_k} or more, {heads}, {dim}], got {tuple(t.shape)}")
    _launch("kvp_load_fp8", k_cache.get_device(),
            *cache, num_blocks, bt, bt_stride, width, cu_seqlens_k.data_ptr(), num_seqs, total_k, heads, dim,
            block_size, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            _stream(k_cache))
    return k, v


# ----------------------------------------------------------------------------- drafted tokens

_tree_pool = Workspaces("tree attention", "reserve_tree_workspace")


@lru_cache(maxsize=1024)
def tree_workspace_bytes(max_num_seqs: int, max_seqlen_q: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                         max_blocks_per_seq: int, block_size: int) -> int:
    return int(lib().kvp_tree_workspace_bytes(max_num_seqs, max_seqlen_q, num_q_heads, num_kv_heads, head_dim,
                                              max_blocks_per_seq, block_size))


def reserve_tree_workspace(max_num_seqs: int, max_seqlen_q: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                           max_blocks_per_seq: int, block_size: int,
                           device: torch.device | str | int) -> torch.Tensor:
    """Allocates (or grows) the current stream's workspace of tree_attention and, with max_seqlen_q 1,
    paged_decode_fp8.  Call before graph capture with the largest sizes that a captured graph will
    use: the capture takes the buffer over.  Eager calls need no reservation."""
    return _tree_pool.get(device, tree_workspace_bytes(max_num_seqs, max_seqlen_q, num_q_heads, num_kv_heads,
                                                       head_dim, max_blocks_per_seq, block_size))


def _tree_workspace(index, stream, *sizes) -> torch.Tensor:
    ws = _tree_pool.ready(index, stream, tree_workspace_bytes(*sizes))
    return ws if ws is not None else reserve_tree_workspace(*sizes, index)


def _paged_shape(q, k_cache, v_cache, k_scale, v_scale):
    """Sizes of q [N, Hq, D] over a cache of either kind, and the cache's pointers and strides."""
    if not (q.is_cuda and q.dtype is torch.bfloat16):
        _require_cuda_bf16("q", q)
    if k_scale is None:
        shape, cs = _paired(k_cache, v_cache, "k_cache", torch.bfloat16, q, 4)
        cache = (k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2], 0, 0, 0, 0)
    else:
        shape, cache = _quantised(k_cache, v_cache, k_scale, v_scale, q)
    if q.shape[2] != shape[3] or q.stride(2) != 1:
        raise ValueError("head_dim mismatch or non-contiguous head_dim")
    return shape, cache


def _like(q: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    """A bf16 output of q's shape, given or new."""
    if out is None:
        return q.new_empty(q.shape)
    if out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != q.device or out.stride(2) != 1:
        raise ValueError("out must be a bf16 tensor of q's shape on its device with contiguous head_dim")
    return out


def paged_decode_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                     softmax_scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode over a quantised cache (see store_kvcache_fp8): q [B, Hq, D] (or [B, 1, Hq, D]) in
    bf16, one query token per sequence, at any GQA ratio up to 16."""
    if q.dim() == 4 and q.shape[1] == 1:
        if out is not None and out.dim() != 4:
            raise ValueError("out must have q's shape")
        return paged_decode_fp8(q[:, 0], k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table,
                                softmax_scale, None if out is None else out[:, 0]).unsqueeze(1)
    if q.dim() != 3:
        raise ValueError(f"paged_decode_fp8 takes one query token per sequence, got q of shape {tuple(q.shape)}")
    (num_blocks, block_size, Hkv, D), cache = _paged_shape(q, k_cache, v_cache, k_scale, v_scale)
    B, Hq, _ = q.shape
    _ints("cache_seqlens", cache_seqlens, q)
    if cache_seqlens.numel() < B:
        raise ValueError("cache_seqlens has fewer rows than q")
    bt, bt_stride, width = _table(block_table, B, q)
    out, index, stream = _like(q, out), q.get_device(), _stream(q)
    ws = _tree_workspace(index, stream, B, 1, Hq, Hkv, D, width, block_size)
    qs, os = q.stride(), out.stride()
    _launch("kvp_paged_decode_fp8", index, q.data_ptr(), qs[0], qs[1], *cache, num_blocks, bt, bt_stride,
            cache_seqlens.data_ptr(), B, Hq, Hkv, D, block_size, width, softmax_scale, out.data_ptr(), os[0], os[1],
            ws.data_ptr(), ws.numel(), stream)
    return out


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cu_seqlens_q: torch.Tensor,
                   max_seqlen_q: int, cache_seqlens: torch.Tensor, block_table: torch.Tensor, softmax_scale: float,
                   tree_mask: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted tokens over a paged cache that holds them behind their contexts.

    q is [T, Hq, D] bf16; sequence b has rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 of it, at most
    max_seqlen_q <= 64, and cache_seqlens[b] cached tokens, these drafts (appended before) being
    the last.  A row sees every token before its sequence's drafts, and draft j where bit j of
    its int64 tree_mask entry is set; without a tree_mask the drafts are a chain (draft j for
    j <= its own).  Rows that see nothing are zeros, and what a masked token holds reaches no row.
    The caches are bf16 as paged_decode's or, with k_scale and v_scale, quantised as
    paged_decode_fp8's; any GQA ratio up to 16.  Rows of q that no sequence has are left as they
    were in `out`."""
    if q.dim() != 3:
        raise ValueError(f"q must be [T, num_q_heads, head_dim], got shape {tuple(q.shape)}")
    if (k_scale is None) != (v_scale is None):
        raise ValueError("k_scale and v_scale go together")
    (num_blocks, block_size, Hkv, D), cache = _paged_shape(q, k_cache, v_cache, k_scale, v_scale)
    T, Hq, _ = q.shape
    _ints("cu_seqlens_q", cu_seqlens_q, q)
    _ints("cache_seqlens", cache_seqlens, q)
    B, max_seqlen_q = cu_seqlens_q.numel() - 1, int(max_seqlen_q)
    if B < 0 or cache_seqlens.numel() < B:
        raise ValueError("cu_seqlens_q must have an entry more than sequences, and cache_seqlens one for each")
    index = q.get_device()
    if tree_mask is not None and not (tree_mask.dtype is torch.int64 and tree_mask.get_device() == index
                                      and tree_mask.is_contiguous() and tree_mask.numel() == T):
        raise ValueError("tree_mask must be a contiguous int64 tensor on q's device with one entry per row of q")
    bt, bt_stride, width = _table(block_table, B, q)
    out, stream = _like(q, out), _stream(q)
    if B == 0 or T == 0:
        return out
    ws = _tree_workspace(index, stream, B, max_seqlen_q, Hq, Hkv, D, width, block_size)
    qs, os = q.stride(), out.stride()
    _launch("kvp_tree_attention", index, q.data_ptr(), qs[0], qs[1], *cache, num_blocks, bt, bt_stride,
            cu_seqlens_q.data_ptr(), cache_seqlens.data_ptr(), B, T, max_seqlen_q,
            tree_mask.data_ptr() if tree_mask is not None else 0, Hq, Hkv, D, block_size, width,
            softmax_scale, out.data_ptr(), os[0], os[1], ws.data_ptr(), ws.numel(), stream)
    return out


# ----------------------------------------------------------------------------- module

class Attention(nn.Module):
    """Paged-KV attention layer; same constructor, attributes and forward as
    kavor/layers/attention/flash_attention_kvcache.py:49-84.

    k_cache / v_cache are lists with one entry per KV slot (num_kv_slots); a page pool
    binds them by duck typing (kavor/engine/cache_pool.py:98-101, 311-322).  forward
    appends k / v when a cache is bound, then runs varlen prefill (paged when the
    context carries block tables) or paged decode, reading the global Context.
    """

    def __init__(self, num_heads, head_dim, scale, num_kv_heads, num_kv_slots: int = 1):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.num_kv_slots = num_kv_slots
        self.k_cache = [torch.tensor([]) for _ in range(num_kv_slots)]
        self.v_cache = [torch.tensor([]) for _ in range(num_kv_slots)]

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot: int = 0):
        context = get_context()
        k_cache, v_cache = self.k_cache[slot], self.v_cache[slot]
        if k_cache.numel() and v_cache.numel():
            store_kvcache(k, v, k_cache, v_cache, context.slot_mapping)
        if context.is_prefill:
            if context.block_tables is not None:  # prefix cache: attend over the pages
                k, v = k_cache, v_cache
            return self._prefill(q, k, v, context)
        return self._decode(q, k_cache, v_cache, context)

    def forward_cached(self, q: torch.Tensor, slot: int = 0):
        """Attention over the pages when the caller has already appended this step's k / v
        (the fused q/k-norm + RoPE + append kernel).  Prefill then always reads the pages,
        so the context must carry block tables."""
        context = get_context()
        k_cache, v_cache = self.k_cache[slot], self.v_cache[slot]
        if context.is_prefill:
            if context.block_tables is None:
                raise ValueError("forward_cached prefill reads the pages: the context needs block tables")
            return self._prefill(q, k_cache, v_cache, context)
        return self._decode(q, k_cache, v_cache, context)

    def _prefill(self, q, k, v, context):
        return varlen_prefill(q, k, v, max_seqlen_q=context.max_seqlen_q,
                              cu_seqlens_q=context.cu_seqlens_q,
                              max_seqlen_k=context.max_seqlen_k,
                              cu_seqlens_k=context.cu_seqlens_k,
                              softmax_scale=self.scale, causal=True,
                              block_table=context.block_tables)

    def _decode(self, q, k_cache, v_cache, context):
        return paged_decode(q.unsqueeze(1), k_cache, v_cache,
                            cache_seqlens=context.context_lens,
                            block_table=context.block_tables,
                            softmax_scale=self.scale, causal=True)
