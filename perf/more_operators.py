"""The operators that end a step with drafted tokens, and those that move pages, as the programs that
serve a model call them, each beside its plain form.

  verify  drafted tokens kept or refused by the target's probabilities and given random numbers, and
          the token that follows the last one kept: chains that a draft model sampled (its logits are
          an input) and trees of chosen tokens (a bit mask says which drafts of its sequence a token sees)
  keep    the keys and values of the drafts that are kept moved next to their context, in every layer
  copy    whole pages copied in every layer, as if all were read before any is written: forks of a
          sequence, and pages that change places

Lengths are evenly spaced over the stated range, so that the work of a case does not depend on the
seed; their order, the page ids and all values come from the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

D = 128
BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn
TYPES = {"bf16": BF16, "fp32": torch.float32, "fp8": FP8}


# ----------------------------------------------------------------------------- the cases

def _verify(name, form, seqs, rows_min, rows_max, vocab, dtype, greedy=0.0, pad=0):
    return dict(name=name, kind="verify", form=form, seqs=seqs, rows_min=rows_min, rows_max=rows_max, vocab=vocab,
                dtype=dtype, greedy=greedy, pad=pad)


def _keep(name, cache, layers, kv_heads, block, seqs, rows_min, rows_max):
    return dict(name=name, kind="keep", cache=cache, layers=layers, kv_heads=kv_heads, block=block, seqs=seqs,
                rows_min=rows_min, rows_max=rows_max)


def _copy(name, layers, page_bytes, pairs, fan, moved=0.0):
    return dict(name=name, kind="copy", layers=layers, page_bytes=page_bytes, pairs=pairs, fan=fan, moved=moved)


def _page_bytes(cache, kv_heads, block):
    return 2 * block * kv_heads * (2 * D if cache == "bf16" else D + 1)


def listed():
    return [
        # one user, four tokens of a draft model: latency only
        _verify("verify_one", "chain", 1, 5, 5, 151936, "bf16"),
        # one user, a small tree of a draft head's best tokens
        _verify("verify_one_tree", "tree", 1, 12, 12, 151936, "bf16"),
        # a full batch with a draft model, some greedy requests and a padded graph's idle rows
        _verify("verify_batch", "chain", 256, 5, 5, 151936, "bf16", 0.125, 16),
        # ragged trees over logits in 32 bits, a vocabulary that no vector width divides
        _verify("verify_trees", "tree", 48, 5, 25, 151643, "fp32", 0.25),
        # the widest trees
        _verify("verify_wide", "tree", 24, 61, 64, 151936, "bf16"),
        # one user's accepted drafts
        _keep("keep_one", "bf16", 28, 8, 256, 1, 12, 12),
        # a batch of ragged trees
        _keep("keep_batch", "bf16", 28, 8, 256, 64, 5, 25),
        # a full batch over quantised pages
        _keep("keep_quantised", "fp8", 28, 8, 64, 256, 4, 12),
        # one sequence forked: the page that its last tokens share with no full one
        _copy("copy_fork", 28, _page_bytes("bf16", 8, 256), 1, 1),
        # parallel samples of a batch of prompts: each last page copied for three more sequences
        _copy("copy_samples", 28, _page_bytes("bf16", 8, 64), 96, 3),
        # a pool of quantised pages brought into another order
        _copy("copy_reorder", 28, _page_bytes("fp8", 8, 64), 300, 1, 0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "verify", "verify", "keep", "keep", "copy", "copy"])
    if kind == "verify":
        form = rng.choice(["chain", "tree"])
        rows_max = _log_int(rng, 1, 64 if form == "tree" else 16)
        rows_min = rng.randint(1, rows_max)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        room = 2400 // ((2 if form == "chain" else 1) * (2 if dtype == "fp32" else 1))
        seqs = max(1, min(_log_int(rng, 1, 256), room // rows_max))
        case = _verify("", form, seqs, rows_min, rows_max, rng.choice([151936, 151643, 32000, 1013]), dtype,
                       rng.choice([0.0, 0.0, 0.3, 1.0]), rng.choice([0, 0, seqs // 5]))
    elif kind == "keep":
        cache, kv_heads, block = rng.choice(["bf16", "fp8"]), rng.choice([8, 8, 4, 2, 1]), rng.choice([256, 64])
        layers = _log_int(rng, 1, 36)
        rows_max = _log_int(rng, 1, 64)
        room = (2 << 30) // (layers * _page_bytes(cache, kv_heads, block))
        seqs = max(1, min(_log_int(rng, 1, 256), room // 2 - 8))
        case = _keep("", cache, layers, kv_heads, block, seqs, rng.randint(1, rows_max), rows_max)
    else:
        page = _page_bytes(rng.choice(["bf16", "fp8"]), rng.choice([8, 4, 2]), rng.choice([256, 64]))
        layers = _log_int(rng, 1, 36)
        pairs = max(1, min(_log_int(rng, 1, 600), (1 << 30) // (layers * page)))
        case = _copy("", layers, page, pairs, rng.choice([1, 1, 2, 5]), rng.choice([0.0, 0.0, 0.5, 1.0]))
    del case["name"]
    return case


def _spaced(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [(lo + hi) // 2]


def _kept(rows):
    """Drafts kept of a sequence of `rows` rows (the first of which is no draft): a fixed share."""
    return max(0, rows - 2) * 2 // 5 + (1 if rows > 2 else 0)


# ----------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ends(lens):
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    return _ints(ends)


def _tree(rng, rows):
    """Parents and bit masks of a tree of `rows` rows: each sees its parent, what its parent sees, and itself."""
    parents, masks, wide = [-1], [1], rng.choice([1, 2, 3])
    for i in range(1, rows):
        parents.append(max(0, (i - 1) // wide - rng.randint(0, 1)))
        masks.append(masks[parents[i]] | 1 << i)
    return parents, [m - (1 << 64) if m >> 63 else m for m in masks]


def _rows(g, rows, vocab, dtype, near=None):
    """Logits of a trained model's shape, six rows of seven peaked; or others `near` given ones."""
    out = torch.empty(rows, -(-vocab // 8) * 8, device="cuda", dtype=dtype)[:, :vocab]
    for at in range(0, rows, 256):
        n = min(256, rows - at)
        flat = torch.randn(n, vocab, generator=g, device="cuda")
        if near is not None:
            out[at:at + n] = (near[at:at + n].float() + 0.6 * flat).to(dtype)
            continue
        peaked = torch.rand(n, 1, generator=g, device="cuda") < 6 / 7
        flat *= torch.where(peaked, 1.6, 0.64)
        tops = torch.randint(0, vocab // 40, (n, 40), generator=g, device="cuda")
        tops += torch.arange(40, device="cuda") * (vocab // 40)
        lift = 24.0 * torch.rand(n, 40, generator=g, device="cuda") + 8.0
        flat.scatter_(1, tops, torch.where(peaked, lift, flat.gather(1, tops)))
        out[at:at + n] = flat.to(dtype)
    return out


def _verify_inputs(case, seed):
    g, rng = _gen(seed), random.Random(seed)
    lens = _spaced(case["rows_min"], case["rows_max"], case["seqs"])
    rng.shuffle(lens)
    T, V, chain = sum(lens), case["vocab"], case["form"] == "chain"
    lens += [0] * case["pad"]
    B = len(lens)
    temps = [rng.uniform(0.6, 1.0) for _ in lens]
    for b in rng.sample(range(case["seqs"]), round(case["greedy"] * case["seqs"])):
        temps[b] = 0.0
    x = {"lens": lens, "max_q": case["rows_max"], "cu": _ends(lens),
         "temps": torch.tensor(temps, dtype=torch.float32, device="cuda"), "mask": None, "draft": None}
    x["logits"] = _rows(g, T, V, TYPES[case["dtype"]])
    x["uniforms"] = torch.rand(T, generator=g, device="cuda")
    if chain:
        parents = [p for n in lens for p in range(-1, n - 1)]
        x["draft"] = _rows(g, T, V, TYPES[case["dtype"]], near=x["logits"])
    else:
        trees = [_tree(rng, n) for n in lens if n]
        parents = [p for t in trees for p in t[0]]
        x["mask"] = torch.tensor([m for t in trees for m in t[1]], device="cuda")
    first = [at for at, n in zip(x["cu"].tolist(), lens) for _ in range(n)]
    above = torch.tensor([f + max(p, 0) for f, p in zip(first, parents)], device="cuda")
    nth = [sum(f == first[j] and p == parents[j] for j in range(max(f, i - 6), i))
           for i, (f, p) in enumerate(zip(first, parents))]
    tokens = torch.empty(T, dtype=torch.long, device="cuda")
    heat = torch.repeat_interleave(x["temps"], torch.tensor(lens, device="cuda"))
    for at in range(0, T, 256):  # a sample of the draft model's distribution, or its best tokens in turn
        up = above[at:at + 256]
        if chain:
            u = torch.rand(up.numel(), V, generator=g, device="cuda").clamp_(min=1e-20, max=1 - 1e-7)
            noise = -torch.log(-torch.log(u))
            tokens[at:at + 256] = (x["draft"][up].float() + noise * heat[at:at + 256, None]).argmax(-1)
        else:
            guess = x["logits"][up].float()
            guess += 0.5 * torch.randn(guess.shape, generator=g, device="cuda")
            best = torch.topk(guess, 7, dim=-1).indices
            tokens[at:at + 256] = best.gather(1, torch.tensor(nth[at:at + 256], device="cuda")[:, None])[:, 0]
    x["tokens"] = tokens
    return x


def _caches(g, case, pages):
    """A pool of bytes [layers, pages, page], and (k, v, k_scale, v_scale) views of it: K and V of a block side
    by side, then their scales where they are quantised."""
    L, H, block = case["layers"], case["kv_heads"], case["block"]
    size = _page_bytes(case["cache"], H, block)
    pool = torch.randint(0, 126, (L, pages, size), generator=g, device="cuda", dtype=torch.uint8)  # no NaN codes
    if case["cache"] == "bf16":
        flat, half = pool.view(BF16), block * H * D
        strides = (pages * size // 2, size // 2, H * D, D, 1)
        k, v = (flat.as_strided((L, pages, block, H, D), strides, i * half) for i in range(2))
        return pool, k, v, None, None
    flat, half = pool.view(FP8), block * H * D
    k, v = (flat.as_strided((L, pages, block, H, D), (pages * size, size, H * D, D, 1), i * half) for i in range(2))
    ks, vs = (pool.as_strided((L, pages, H, block), (pages * size, size, block, 1), 2 * half + i * block * H)
              for i in range(2))
    return pool, k, v, ks, vs


def _keep_inputs(case, seed):
    g, rng = _gen(seed), random.Random(seed)
    lens, block = _spaced(case["rows_min"], case["rows_max"], case["seqs"]), case["block"]
    rng.shuffle(lens)
    width = 3
    ctx = [rng.randint(1, width * block - max(lens)) + n for n in lens]
    # only the pages that hold drafts are this case's own; those of the contexts are shared
    pages = 2 * len(lens) + 8
    ids = list(range(pages))
    rng.shuffle(ids)
    rest, tables = ids[8:], []
    for n, c in zip(lens, ctx):
        table = [ids[j % 8] for j in range(width)]
        for j in range((c - n) // block, (c - 1) // block + 1):
            table[j] = rest.pop()
        tables.append(table)
    paths = [sorted(rng.sample(range(2, n), _kept(n))) if n > 2 else [] for n in lens]
    max_q = case["rows_max"]
    x = {"cu": _ends(lens), "ctx": _ints(ctx), "bt": _ints(tables), "accepted": _ints([len(p) for p in paths]),
         "path": _ints([p + [-1] * (max_q - len(p)) for p in paths]), "max_q": max_q}
    x["pool"], x["k"], x["v"], x["ks"], x["vs"] = _caches(g, case, pages)
    return x


def _copy_inputs(case, seed):
    """Pairs with `fan` copies of each source; a share `moved` of the pages written are sources as well."""
    g, rng = _gen(seed), random.Random(seed)
    n = case["pairs"]
    sources = -(-n // case["fan"])
    both = min(round(case["moved"] * n), sources, n)
    total = sources + n - both + 4
    ids = list(range(total))
    rng.shuffle(ids)
    src = [ids[i // case["fan"]] for i in range(n)]
    dst = ids[sources - both:sources - both + n]
    rng.shuffle(dst)
    pool = torch.randint(0, 256, (case["layers"], total, case["page_bytes"]), generator=g, device="cuda",
                         dtype=torch.uint8)
    return {"pool": pool, "src": src, "dst": dst}


@torch.inference_mode()
def prepare(case, seed):
    make = {"verify": _verify_inputs, "keep": _keep_inputs, "copy": _copy_inputs}[case["kind"]]
    return {"kind": case["kind"], **make(case, seed)}


# ----------------------------------------------------------------------------- plain forms

def _weights(x, temps):
    """exp of the rows of logits over a temperature, less their maximum, in 64 bits."""
    z = x.double() / temps[:, None]
    return torch.exp(z - z.amax(-1, keepdim=True))


def _plain_verify(s):
    """Row 0 of a sequence is its last token, the others are drafts; all rows of all sequences at once.

    In 64 bits: the token that a random number picks is a border of sums over the vocabulary."""
    n, V, N = s["cu"].diff()[:, None], s["logits"].shape[1], s["max_q"]
    i = torch.arange(N, device="cuda")
    real = i < n
    row = torch.where(real, s["cu"][:-1, None] + i, 0).long()
    mask = (2 << i) - 1 if s["mask"] is None else s["mask"][row]
    sees = (mask.expand(real.shape)[..., None] >> i & 1 == 1) & real[..., None]  # [B, row, row]
    before = sees & (i < i[:, None])
    parent = torch.where(before, i, -1).amax(-1)
    up = torch.where(real & (parent >= 0), row.gather(1, parent.clamp(min=0)), 0)
    token = s["tokens"][row]
    greedy = ~(s["temps"] > 0)
    heat = torch.where(greedy, 1.0, s["temps"]).double()
    heat_row = torch.ones(s["logits"].shape[0], dtype=torch.float64, device="cuda")
    heat_row[row[real]] = heat[:, None].expand(real.shape)[real]
    w = _weights(s["logits"], heat_row)
    z = w.sum(-1)
    p = w.view(-1)[up * V + token] / z[up]
    u = s["uniforms"][row].double()
    if s["draft"] is None:
        sibling = (parent[:, :, None] == parent[:, None]) & (i < i[:, None]) & real[:, None]  # [B, row, earlier row]
        twin = sibling & (token[:, :, None] == token[:, None])
        fresh = ~twin.any(-1)
        left = 1 - (torch.where(sibling & fresh[:, None], p[:, None], 0.0)).sum(-1)
        passes = (u * left < p) & fresh
    else:
        y = _weights(s["draft"], heat_row)
        zy = y.sum(-1)
        passes = u * (y.view(-1)[up * V + token] / zy[up]) < p
        sibling = torch.zeros_like(sees)
    first = torch.where(s["logits"] == s["logits"].amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1)
    passes = torch.where(greedy[:, None], token == first[up], passes) & real & (parent >= 0)
    if s["draft"] is None:
        passes &= ~(sibling & passes[:, None]).any(-1)
    kept = passes & ~(before & ~passes[:, None])[..., 1:].any(-1)  # all that the row sees behind row 0
    accepted = kept.sum(-1)
    end = torch.where(kept, i, 0).amax(-1)
    at = row.gather(1, end[:, None])[:, 0]
    weight = w[at]
    gone = real & (parent == end[:, None])  # the drafts refused behind the last one kept
    if s["draft"] is None:
        b, j = gone.nonzero(as_tuple=True)
        weight[b, token[b, j]] = 0
    else:
        rest = (weight / z[at][:, None] - y[at] / zy[at][:, None]).clamp(min=0)
        weight = torch.where(gone.any(-1, keepdim=True) & (rest.sum(-1, keepdim=True) > 0), rest, weight)
    sums = weight.cumsum(-1)
    border = s["uniforms"][row[:, 0]].double() * sums[:, -1]
    pick = (sums <= border[:, None]).sum(-1)
    last = torch.where(weight > 0, torch.arange(V, device="cuda"), 0).amax(-1)
    pick = torch.where(greedy, first[at], torch.minimum(pick, last))
    order = torch.where(kept, i, N).sort(-1).values
    path = torch.where(i < accepted[:, None], order, -1)
    tokens = torch.where(i < accepted[:, None], token.gather(1, path.clamp(min=0)), -1)
    tokens = torch.where((i == accepted[:, None]) & (n > 0), pick[:, None], tokens)
    return accepted.int(), path.int(), tokens


def _plain_keep(s):
    block, n = s["k"].shape[2], s["cu"].diff()
    j = torch.arange(s["max_q"], device="cuda")
    real = (j < s["accepted"][:, None]).nonzero(as_tuple=True)
    seq, to = real[0], real[1] + 1
    start = (s["ctx"] - n)[seq]
    src, dst = start + s["path"][real], start + to
    page = lambda pos: s["bt"][seq, pos // block].long()  # noqa: E731
    at, off, at2, off2 = page(src), src % block, page(dst), dst % block
    k, v = (c if c.dtype == BF16 else c.view(torch.uint8) for c in (s["k"], s["v"]))
    k[:, at2, off2], v[:, at2, off2] = k[:, at, off], v[:, at, off]
    if s["ks"] is not None:
        ks, vs = s["ks"].transpose(2, 3), s["vs"].transpose(2, 3)
        ks[:, at2, off2], vs[:, at2, off2] = ks[:, at, off], vs[:, at, off]
    return s["pool"], s["ctx"] - (n - 1 - s["accepted"])


def _plain_copy(s):
    src, dst = (torch.tensor(x, device="cuda") for x in (s["src"], s["dst"]))
    s["pool"][:, dst] = s["pool"][:, src]
    return s["pool"]


# ----------------------------------------------------------------------------- run

def _own(s):
    from kavor_amd.layers import attention, fused

    if s["kind"] == "verify":
        return fused.verify_drafts(s["logits"], s["tokens"], s["uniforms"], s["temps"], s["cu"], s["max_q"],
                                   tree_mask=s["mask"], draft_logits=s["draft"])
    if s["kind"] == "keep":
        lens = attention.keep_drafts(s["k"], s["v"], s["path"], s["accepted"], s["cu"], s["ctx"], s["bt"],
                                     k_scale=s["ks"], v_scale=s["vs"])
        return s["pool"], lens
    attention.copy_pages(s["pool"], s["src"], s["dst"])
    return s["pool"]


@torch.inference_mode()
def run(state):
    if own:
        return _own(state)
    return {"verify": _plain_verify, "keep": _plain_keep, "copy": _plain_copy}[state["kind"]](state)


def work(case):
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pairs"] * case["page_bytes"], "flops": 0}
    lens = _spaced(case["rows_min"], case["rows_max"], case["seqs"])
    if case["kind"] == "keep":
        row = 2 * case["layers"] * case["kv_heads"] * (2 * D if case["cache"] == "bf16" else D + 1)
        return {"bytes": 2 * row * sum(_kept(n) for n in lens) + 4 * len(lens) * (case["rows_max"] + 7), "flops": 0}
    # the rows that a sequence gets to, on average over the inputs above: those behind a refused draft decide nothing
    pass_on = 0.75 if case["form"] == "chain" else 0.5
    rows = sum(sum(pass_on ** i for i in range(n)) for n in lens)
    rows += sum(sum(pass_on ** i for i in range(n - 1)) for n in lens) if case["form"] == "chain" else 0
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": int(rows * case["vocab"] * size) + sum(lens) * 20 + len(lens) * (12 + 12 * case["rows_max"]),
            "flops": int(rows * case["vocab"] * 3)}


# ----------------------------------------------------------------------------- 64-bit results

def _softmax64(x, temp):
    z = x.double()
    return torch.softmax(z / temp, -1)


def _draw64(p, u):
    """The least index whose running sum passes u of the whole."""
    sums = torch.cumsum(p, 0)
    past = (sums > u * sums[-1]).nonzero()
    return int(past[0, 0]) if len(past) else int((p > 0).nonzero()[-1, 0])


@torch.inference_mode()
def exact(case, seed):
    if case["kind"] != "verify":
        return None  # nothing is computed
    x = _verify_inputs(case, seed)
    tokens, us, temps = x["tokens"].tolist(), x["uniforms"].tolist(), x["temps"].tolist()
    masks = x["mask"].tolist() if x["mask"] is not None else None
    accepted, paths, outs, base = [], [], [], 0
    for b, n in enumerate(x["lens"]):
        path, out, node = [], [], 0
        while n:
            z, rest = x["logits"][base + node], None
            if not temps[b] > 0:
                best = int((z == z.max()).nonzero()[0, 0])
            else:
                rest = _softmax64(z, temps[b])
            if masks is None:
                children = [node + 1] if node + 1 < n else []
            else:
                children = [i for i in range(node + 1, n)
                            if max(j for j in range(i) if masks[base + i] >> j & 1) == node]
            found = None
            for i in children:
                t = tokens[base + i]
                if rest is None:
                    ok = t == best
                elif masks is None:
                    q = _softmax64(x["draft"][base + node], temps[b])
                    ok = us[base + i] * float(q[t]) < float(rest[t])
                    if not ok:
                        rest = (rest - q).clamp(min=0)
                else:
                    ok = us[base + i] * float(rest.sum()) < float(rest[t])
                    if not ok:
                        rest[t] = 0
                if ok:
                    found = i
                    break
            if found is None:
                out.append(best if rest is None else _draw64(rest, us[base]))
                break
            path.append(found)
            out.append(tokens[base + found])
            node = found
        accepted.append(len(path))
        paths.append(path + [-1] * (x["max_q"] - len(path)))
        outs.append(out + [-1] * (x["max_q"] - len(out)))
        base += n
    return _ints(accepted), _ints(paths), torch.tensor(outs, device="cuda")
