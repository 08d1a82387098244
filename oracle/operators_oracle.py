"""64-bit restatements, on the CPU, of the operators that have no counterpart in the reference: the
quantised cache, attention of drafted tokens, and token log probabilities.

e4m3 comes from its definition (sign, 4 exponent bits with bias 7, 3 mantissa bits, one NaN code and
no infinity), not from a library's conversion.
"""

from __future__ import annotations

import math

import numpy as np
import torch


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes."""
    out = np.empty(256)
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[code] = math.nan if code & 127 == 127 else -v if code & 128 else v
    return out


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Codes of |x| <= 448 by the nearest value, ties to the even code; NaN and infinities: 127."""
    values = e4m3_values()[:127]
    mag = np.where(np.isfinite(x), np.abs(x), 0.0)
    assert mag.size == 0 or mag.max() <= 448
    hi = np.clip(np.searchsorted(values, mag), 1, 126)
    lo = hi - 1
    below, above = mag - values[lo], values[hi] - mag
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(x), code + 128, code)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def quantise_rows(x: torch.Tensor) -> tuple[np.ndarray, np.ndarray]:
    """Codes of the rows (last dimension) of x and their exponent bytes."""
    x = x.double().numpy()
    finite = np.where(np.isfinite(x), np.abs(x), 0.0)
    top = finite.max(-1, initial=0.0)
    byte = np.ones(top.shape, dtype=np.int64)
    while (low := top > 448 * 2.0 ** (byte - 127)).any():
        byte = byte + low
    with np.errstate(invalid="ignore"):
        return to_e4m3(x * 2.0 ** (127 - byte)[..., None]), byte.astype(np.uint8)


def dequantise(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """[num_blocks, block_size, heads, D] in 64 bits of a quantised cache (bytes or float8) and its
    [num_blocks, heads, block_size] exponent bytes."""
    values = torch.from_numpy(e4m3_values())[codes.contiguous().view(torch.uint8).long()]
    return values * torch.exp2(scale.double() - 127).transpose(1, 2)[..., None]


def gather(cache: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    """The first n tokens of the pages that a sequence's table lists."""
    pages = table[: -(-n // cache.shape[1])].long()
    return cache[pages].flatten(0, 1)[:n]


def tree_attention(q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, scale, tree_mask=None):
    """(out, spread) [T, Hq, D] in 64 bits over caches of plain values: out as the operator defines it,
    NaN rows of no sequence, and spread = sum_t p_t |v_t|, which bounds what rounding the weights
    can change."""
    T, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    spread = torch.zeros(T, Hq, D, dtype=torch.float64)
    for b in range(len(cache_seqlens)):
        q0, q1, n = int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1]), int(cache_seqlens[b])
        if n <= 0:
            out[q0:q1] = 0
            continue
        ctx = n - (q1 - q0)
        k, v = (gather(c, block_table[b], n).double() for c in (k_cache, v_cache))
        for i in range(q1 - q0):
            bits = int(tree_mask[q0 + i]) if tree_mask is not None else (2 << i) - 1
            sees = [t for t in range(n) if t < ctx or bits >> (t - ctx) & 1]
            if not sees:
                out[q0 + i] = 0
                continue
            for h in range(Hq):
                kh, vh = k[sees, h * Hkv // Hq], v[sees, h * Hkv // Hq]
                p = torch.softmax(kh @ q[q0 + i, h].double() * scale, 0)
                out[q0 + i, h] = p @ vh
                spread[q0 + i, h] = p @ vh.abs()
    return out, spread


def token_logprobs(logits, tokens, top):
    """(logprobs, entropy, rank, top_logprobs, top_tokens) in 64 bits."""
    x = logits.double()
    logp = torch.log_softmax(x, -1)
    entropy = -torch.where(logp == -math.inf, 0.0, logp.exp() * logp).sum(-1)
    mine = x.gather(1, tokens[:, None])
    order = torch.where(x.isnan(), math.inf, x)
    first = x.isnan().double()  # NaN before an infinity
    ids = torch.argsort(order, dim=-1, descending=True, stable=True)
    ids = ids.gather(1, torch.argsort(first.gather(1, ids), dim=-1, descending=True, stable=True))[:, :top]
    return logp.gather(1, tokens[:, None])[:, 0], entropy, (x > mine).sum(-1) + 1, logp.gather(1, ids), ids
