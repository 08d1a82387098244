"""64-bit restatements, on the CPU, of the end of a step with drafted tokens: which drafts stay, the token that
follows them, and where their keys and values go.  Sequence by sequence, row by row, as the operators define them.
"""

from __future__ import annotations

import math

import torch


def softmax(row: torch.Tensor, temp: float) -> torch.Tensor | None:
    """softmax(row / temp) in 64 bits, or None where there is none."""
    x = row.double()
    top = x.max() if not x.isnan().any() else torch.tensor(math.nan)
    if not math.isfinite(float(top)):
        return None
    z = (x - top) / max(temp, 1e-45)
    w = torch.exp(torch.where(x == -math.inf, -math.inf, torch.where(x == top, 0.0, z)))
    return w / w.sum()


def greedy(row: torch.Tensor) -> int:
    """Index of the largest logit, NaN above all, the lowest one among equals."""
    x = row.double()
    if x.isnan().any():
        return int(x.isnan().nonzero()[0, 0])
    return int((x == x.max()).nonzero()[0, 0])


def draw(weights: torch.Tensor, u: float) -> int:
    """The least index whose running sum of weights exceeds u times their sum."""
    sums = torch.cumsum(weights, 0)
    past = ((sums > u * sums[-1]) & (weights > 0)).nonzero()
    return int(past[0, 0]) if len(past) else int((weights > 0).nonzero()[-1, 0])


def verify_drafts(logits, tokens, uniforms, temperatures, cu_seqlens_q, max_seqlen_q, tree_mask=None, draft_logits=None):
    """(accepted, path, out_tokens), and how near they come to be others: the least distance of the two sides of a
    decision, of the larger one, and that of a drawn number from a border, of the sum."""
    T, vocab = logits.shape
    B = len(cu_seqlens_q) - 1
    accepted = torch.zeros(B, dtype=torch.int32)
    path = torch.full((B, max_seqlen_q), -1, dtype=torch.int32)
    out = torch.full((B, max_seqlen_q), -1, dtype=torch.int64)
    decided = drawn = math.inf
    for b in range(B):
        q0, n = int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1] - cu_seqlens_q[b])
        if not (0 < n <= max_seqlen_q and q0 >= 0 and q0 + n <= T):
            continue
        temp = float(temperatures[b])
        parent = [-1] * n
        for i in range(1, n):
            seen = [j for j in range(i) if tree_mask is None or int(tree_mask[q0 + i]) >> j & 1]
            parent[i] = max(seen, default=-1)
        node, rows, toks = 0, [], []
        while True:
            row, children = logits[q0 + node], [i for i in range(1, n) if parent[i] == node]
            p = softmax(row, temp) if temp > 0 else None
            left, found, q = None if p is None else p.clone(), None, None
            for i in children:
                x, u = int(tokens[q0 + i]), float(uniforms[q0 + i])
                inside = 0 <= x < vocab
                if not temp > 0:
                    ok = x == greedy(row)
                elif p is None:
                    ok = False
                elif draft_logits is not None:
                    q = softmax(draft_logits[q0 + node], temp)
                    a, c = (u * float(q[x]), float(p[x])) if inside and q is not None else (1.0, 0.0)
                    ok = a < c
                    decided = min(decided, abs(a - c) / max(a, c, 1e-300))
                else:
                    a, c = (u * float(left.sum()), float(left[x])) if inside else (1.0, 0.0)
                    ok = a < c
                    decided = min(decided, abs(a - c) / max(a, c, 1e-300))
                if ok:
                    found = i
                    break
                if p is not None and draft_logits is None and inside:
                    left[x] = 0
            if found is None:
                break
            node = found
            rows.append(found)
            toks.append(int(tokens[q0 + found]))
        if p is None:
            last = greedy(row)
        else:
            if draft_logits is not None and q is not None and 0 <= int(tokens[q0 + children[0]]) < vocab:
                left = (p - q).clamp(min=0)
            if not left.sum() > 2.0 ** -46:
                left = p
            u = float(uniforms[q0])
            last = draw(left, u)
            sums = torch.cumsum(left, 0) / left.sum()
            drawn = min(drawn, float((sums - u).abs().min())) if u > 0 else drawn
        accepted[b] = len(rows)
        path[b, :len(rows)] = torch.tensor(rows, dtype=torch.int32)
        out[b, :len(rows) + 1] = torch.tensor(toks + [last])
    return accepted, path, out, decided, drawn


def keep_drafts(caches, path, accepted, cu_seqlens_q, cache_seqlens, block_table):
    """The sequences' new lengths; moves rows of the caches, [layers, num_blocks, block_size, ...] of anything, in place."""
    lens = cache_seqlens.clone()[:len(cu_seqlens_q) - 1]
    pages, block = caches[0].shape[1], caches[0].shape[2]
    for b in range(len(lens)):
        n, length, kept = int(cu_seqlens_q[b + 1] - cu_seqlens_q[b]), int(cache_seqlens[b]), int(accepted[b])
        if n <= 0 or n > length or not 0 <= kept <= min(n - 1, path.shape[1]):
            continue
        lens[b] = length - n + 1 + kept

        def place(pos):
            page = pos // block
            block_id = int(block_table[b, page]) if page < block_table.shape[1] else -1
            return (block_id, pos % block) if 0 <= block_id < pages else None
        before, moves = 0, []
        for j in range(kept):
            row = int(path[b, j])
            if not before < row < n:
                break
            src, dst = place(length - n + row), place(length - n + 1 + j)
            if src is None or dst is None:
                break
            moves.append((src, dst))
            before = row
        for c in caches:
            rows = [c[:, src[0], src[1]].clone() for src, _ in moves]
            for row, (_, dst) in zip(rows, moves):
                c[:, dst[0], dst[1]] = row
    return lens
