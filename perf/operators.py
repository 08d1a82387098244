"""The operators of a quantised paged cache, of drafted tokens and of token log probabilities, as
the programs that serve a model call them, each beside its plain form.

  store     keys and values of new tokens quantised to e4m3 as they enter the pages: one
            power-of-two scale for each token and head, held as an exponent byte
  load      the pages of a batch read back, packed and in bf16, for a prefill over them
  decode    one query token per sequence over the quantised pages
  tree      the drafted tokens of a batch over pages that hold them behind their contexts; a
            bit mask says which drafts of its sequence a token sees
  logprobs  log probability and rank of given tokens, the entropy of their distributions and
            the most probable alternatives

Lengths are evenly spaced over the stated range, so that the work of a case does not depend on
the seed; their order, the page ids and all values come from the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

D = 128
BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn
SCALE = D ** -0.5
SPARE = 8  # pages of the pool that no sequence has


# ----------------------------------------------------------------------------- the cases

def _store(name, tokens, kv_heads, block=256, pad=0):
    return dict(name=name, kind="store", tokens=tokens, kv_heads=kv_heads, block=block, pad=pad)


def _load(name, seqs, kv_heads, ctx_min, ctx_max, block=256):
    return dict(name=name, kind="load", seqs=seqs, kv_heads=kv_heads, ctx_min=ctx_min, ctx_max=ctx_max, block=block)


def _decode(name, seqs, q_heads, kv_heads, ctx_min, ctx_max, block=256):
    return dict(name=name, kind="decode", seqs=seqs, q_heads=q_heads, kv_heads=kv_heads, ctx_min=ctx_min,
                ctx_max=ctx_max, block=block)


def _tree(name, cache, seqs, q_heads, kv_heads, ctx_min, ctx_max, draft_min, draft_max, block=256):
    return dict(name=name, kind="tree", cache=cache, seqs=seqs, q_heads=q_heads, kv_heads=kv_heads, ctx_min=ctx_min,
                ctx_max=ctx_max, draft_min=draft_min, draft_max=draft_max, block=block)


def _logprobs(name, rows, vocab, dtype, top, peaked=0.5):
    return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top, peaked=peaked)


def listed():
    return [
        # the new tokens of a full decode batch entering one layer's pages, with a padded graph's idle rows
        _store("store_step", 256, 8, pad=16),
        # a full prefill budget
        _store("store_prefill", 16384, 8),
        # prompts that share cached prefixes: the history that their prefill reads
        _load("load_prefix", 32, 8, 100, 4096),
        # one user generating: latency only
        _decode("decode_one", 1, 16, 8, 611, 611),
        # the engine's full batch
        _decode("decode_batch", 256, 16, 8, 100, 2048),
        # long contexts, four query heads per kv head
        _decode("decode_long", 128, 32, 8, 1024, 32768),
        # one user's short tree of drafts behind a chat's history
        _tree("tree_one", "bf16", 1, 16, 8, 2500, 2500, 12, 12),
        # a batch of ragged trees over quantised pages
        _tree("tree_batch", "fp8", 32, 32, 8, 600, 4096, 5, 25),
        # wide trees of a 64-head model: what the matrix cores have to compute
        _tree("tree_wide", "bf16", 24, 64, 8, 1000, 9000, 61, 64),
        # a few streaming users who ask for alternatives
        _logprobs("logprobs_few", 7, 151936, "bf16", 20),
        # a full decode batch in 32 bits, a vocabulary that no vector width divides
        _logprobs("logprobs_step", 256, 151643, "fp32", 5),
        # scoring a long prompt, every position
        _logprobs("logprobs_prompt", 4096, 151936, "bf16", 5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "load", "decode", "decode", "tree", "tree", "tree", "logprobs", "logprobs"])
    q_heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (40, 8), (64, 8), (8, 8), (32, 4), (28, 4), (6, 2)])
    block = rng.choice([256, 256, 64])
    ctx_max = _log_int(rng, 20, 32768)
    ctx_min = max(1, int(ctx_max * rng.uniform(0.03, 1.0)))
    seqs = max(1, min(_log_int(rng, 1, 256), 1_000_000 // ctx_max))
    if kind == "store":
        tokens = _log_int(rng, 1, 16384)
        case = _store("", tokens, kv_heads, block, rng.choice([0, 0, tokens // 9]))
    elif kind == "load":
        case = _load("", max(1, min(seqs, 200_000 // ctx_max)), kv_heads, ctx_min, ctx_max, block)
    elif kind == "decode":
        case = _decode("", seqs, q_heads, kv_heads, ctx_min, ctx_max, block)
    elif kind == "tree":
        draft_max = _log_int(rng, 1, 64)
        draft_min = rng.randint(1, draft_max)
        seqs = max(1, min(seqs, 96, 8_000_000 // (ctx_max * draft_max)))
        case = _tree("", rng.choice(["bf16", "fp8"]), seqs, q_heads, kv_heads, ctx_min, ctx_max, draft_min, draft_max,
                     block)
    else:
        vocab = rng.choice([151936, 151643, 32000, 1013])
        case = _logprobs("", _log_int(rng, 1, 2048), vocab, rng.choice(["bf16", "bf16", "fp32"]),
                         rng.choice([0, 1, 5, 20, 64]), rng.choice([0.0, 0.5, 1.0]))
    del case["name"]
    return case


def _spaced(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [(lo + hi) // 2]


def _drafts(case):
    """Drafted tokens of each sequence; the i-th context has the i-th of them."""
    n = _spaced(case["draft_min"], case["draft_max"], case["seqs"])
    random.Random(len(n)).shuffle(n)
    return n


# ----------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.empty(*shape, dtype=BF16, device="cuda").normal_(generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(rng, lens, block):
    """The pages of a pool and each sequence's table of them, in no order."""
    need = [-(-n // block) for n in lens]
    ids = list(range(sum(need) + SPARE))
    rng.shuffle(ids)
    tables, at = [], 0
    for n in need:
        tables.append(ids[at:at + n])
        at += n
    width = max(1, max(need))
    return len(ids), tables, _ints([t + [-1] * (width - len(t)) for t in tables])


def _two_to(byte):
    """The power of two, in 32 bits, that an exponent byte from 1 to 254 stands for."""
    return (byte.int() << 23).view(torch.float32)


def _pages_bf16(g, pages, block, heads):
    """(k, v) views [pages, block, heads, D] of one pool; K and V of a block side by side."""
    half = block * heads * D
    pool = _randn(g, pages, 2 * half)
    shape, strides = (pages, block, heads, D), (2 * half, heads * D, D, 1)
    return pool.as_strided(shape, strides, 0), pool.as_strided(shape, strides, half)


def _pages_fp8(g, pages, block, heads):
    """(k, v, k_scale, v_scale) views of one pool of bytes: K, V, then their scales, of one block.
    The values are those of a unit normal; scales of neighbouring tokens differ."""
    half, side = block * heads * D, block * heads
    pool = torch.empty(pages, 2 * (half + side), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (2 * half))
    for at in range(0, pages, step):
        part = pool[at:at + step]
        n = part.shape[0]
        expo = torch.randint(118, 122, (n, 2, heads, block), generator=g, device="cuda", dtype=torch.uint8)
        x = torch.empty(n, 2, block, heads, D, device="cuda").normal_(generator=g)
        x /= _two_to(expo).transpose(2, 3)[..., None]
        part[:, :2 * half] = x.clamp_(-448, 448).to(FP8).view(torch.uint8).view(n, -1)
        part[:, 2 * half:] = expo.view(n, -1)
    values, strides = pool.view(FP8), (pool.shape[1], heads * D, D, 1)
    k, v = (values.as_strided((pages, block, heads, D), strides, i * half) for i in range(2))
    strides = (pool.shape[1], block, 1)
    ks, vs = (pool.as_strided((pages, heads, block), strides, 2 * half + i * side) for i in range(2))
    return k, v, ks, vs


def _store_inputs(case, seed):
    g, rng = _gen(seed), random.Random(seed)
    T, heads, block = case["tokens"], case["kv_heads"], case["block"]
    pages, tables, _ = _tables(rng, [T], block)
    slots = [tables[0][i // block] * block + i % block for i in range(T)]
    for i in rng.sample(range(T), case["pad"]):
        slots[i] = -1
    x = {"slots": _ints(slots), "key": _randn(g, T, heads, D)}
    x["key"] *= torch.exp2(torch.randint(-3, 4, (T, heads, 1), generator=g, device="cuda").float()).to(BF16)
    rows = _randn(g, T, 4 * heads * D)  # the qkv projection's rows: v is a view of them
    x["value"] = rows[:, 3 * heads * D:].view(T, heads, D)
    x["k"], x["v"], x["ks"], x["vs"] = _pages_fp8(g, pages, block, heads)
    return x


def _lens(case, seed):
    """Cached tokens of each sequence (its drafts among them), and its drafts, in an order of the seed."""
    lens = _spaced(case["ctx_min"], case["ctx_max"], case["seqs"])
    drafts = _drafts(case) if case["kind"] == "tree" else [0] * len(lens)
    both = [(n + d, d) for n, d in zip(lens, drafts)]
    random.Random(seed).shuffle(both)
    return both


def _ancestors(rng, n):
    """Bit masks of n drafts that form a tree: each sees its parent, what its parent sees, and itself."""
    masks = []
    for i in range(n):
        parent = rng.randint(max(-1, i - 6), i - 1)
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _paged_inputs(case, seed):
    g, rng = _gen(seed), random.Random(seed + 1)
    both = _lens(case, seed)
    lens, drafts = [n for n, _ in both], [d for _, d in both]
    pages, x = None, {"lens": lens, "drafts": drafts, "ctx": _ints(lens), "max_k": max(lens)}
    pages, x["tables"], x["bt"] = _tables(rng, lens, case["block"])
    if case.get("cache") == "bf16":
        x["k"], x["v"] = _pages_bf16(g, pages, case["block"], case["kv_heads"])
        x["ks"] = x["vs"] = None
    else:
        x["k"], x["v"], x["ks"], x["vs"] = _pages_fp8(g, pages, case["block"], case["kv_heads"])
    if case["kind"] == "decode":
        x["q"] = _randn(g, len(lens), case["q_heads"], D)
    elif case["kind"] == "tree":
        x["q"] = _randn(g, sum(drafts), case["q_heads"], D)
        x["cu_q"] = _ints([sum(drafts[:i]) for i in range(len(drafts) + 1)])
        x["max_q"] = max(drafts)
        x["mask"] = torch.tensor([m for d in drafts for m in _ancestors(rng, d)], device="cuda")
    else:
        x["cu_k"] = _ints([sum(lens[:i]) for i in range(len(lens) + 1)])
        x["total"] = sum(lens)
    return x


def _logprobs_inputs(case, seed):
    """Logits of which the last `peaked` of an order of the seed have a trained model's shape."""
    g, rng = _gen(seed), random.Random(seed)
    R, V, dtype = case["rows"], case["vocab"], torch.float32 if case["dtype"] == "fp32" else BF16
    logits = torch.empty(R, -(-V // 8) * 8, device="cuda", dtype=dtype)[:, :V]
    width = torch.full((R, 1), 0.64, device="cuda")
    peaked = torch.tensor(sorted(rng.sample(range(R), round(case["peaked"] * R))), dtype=torch.long, device="cuda")
    width[peaked] = 2.2
    for at in range(0, R, 512):
        flat = torch.randn(min(512, R - at), V, generator=g, device="cuda")
        logits[at:at + 512] = (flat * width[at:at + 512]).to(dtype)
    tops = torch.randint(0, V // 40, (R, 40), generator=g, device="cuda")  # one of each fortieth: no index twice
    tops += torch.arange(40, device="cuda") * (V // 40)
    lift = 9.0 * torch.rand(R, 40, generator=g, device="cuda") + 8.0
    logits[peaked[:, None], tops[peaked]] = lift[peaked].to(dtype)
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda")
    tokens = torch.where(torch.rand(R, generator=g, device="cuda") < 0.5, tokens, tops[:, 0])
    return {"logits": logits, "tokens": tokens, "top": case["top"]}


@torch.inference_mode()
def prepare(case, seed):
    make = {"store": _store_inputs, "logprobs": _logprobs_inputs}.get(case["kind"], _paged_inputs)
    return {"kind": case["kind"], **make(case, seed)}


# ----------------------------------------------------------------------------- plain forms

def _quantise(x):
    """e4m3 values of x [T, H, D] and the exponent bytes [T, H] of their scales: the least power of
    two that brings a row's largest magnitude to 448 = 1.75 * 2^8 or below."""
    m, e = torch.frexp(x.float().abs().amax(-1))
    byte = (e - 9 + (m > 0.875) + 127).clamp(1, 254)
    byte = torch.where(m == 0, 1, byte)
    return (x.float() / _two_to(byte)[..., None]).to(FP8), byte.to(torch.uint8)


def _plain_store(s):
    block = s["k"].shape[1]
    keep = s["slots"] >= 0
    slots = s["slots"][keep].long()
    at, off = slots // block, slots % block
    for x, cache, scale in ((s["key"], s["k"], s["ks"]), (s["value"], s["v"], s["vs"])):
        q, byte = _quantise(x[keep])
        cache.view(torch.uint8)[at, off] = q.view(torch.uint8)
        scale[at, :, off] = byte
    return s["k"], s["v"], s["ks"], s["vs"]


def _padded(s, cache, scale):
    """[B, H, L, D] in 32 bits of the tokens of every sequence, padded to the longest."""
    block = cache.shape[1]
    t = torch.arange(s["max_k"], device="cuda")
    page, off = s["bt"].long().clamp(min=0)[:, t // block], (t % block).expand(len(s["lens"]), -1)
    if scale is None:
        return cache[page, off].transpose(1, 2).float().contiguous()
    rows = cache.view(torch.uint8)[page, off].view(FP8).transpose(1, 2).float().contiguous()
    return rows.mul_(_two_to(scale.transpose(1, 2)[page, off].transpose(1, 2))[..., None])


def _plain_load(s):
    real = torch.arange(s["max_k"], device="cuda") < s["ctx"][:, None]
    return tuple(_padded(s, s[c], s[c + "s"]).transpose(1, 2)[real].to(BF16) for c in ("k", "v"))


def _plain_attend(s, q, seen):
    """q [B, n, Hq, D] over the sequences' tokens; seen [B, n, L] says which tokens a query sees."""
    B, n, hq, _ = q.shape
    hkv = s["k"].shape[2]
    q = q.float().view(B, n, hkv, hq // hkv, D).transpose(1, 2).reshape(B, hkv, -1, D)
    score = torch.matmul(q, _padded(s, s["k"], s["ks"]).transpose(2, 3).contiguous()) * SCALE
    score = score.view(B, hkv, n, hq // hkv, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, hkv, n * (hq // hkv), -1)
    o = torch.matmul(p, _padded(s, s["v"], s["vs"])).view(B, hkv, n, hq // hkv, D)
    return o.transpose(1, 2).reshape(B, n, hq, D).to(BF16)


def _plain_decode(s):
    seen = torch.arange(s["max_k"], device="cuda") < s["ctx"][:, None, None]
    return _plain_attend(s, s["q"][:, None], seen)[:, 0]


def _plain_tree(s):
    n = s["cu_q"].diff()[:, None]
    i = torch.arange(s["max_q"], device="cuda")
    real = i < n
    row = torch.where(real, s["cu_q"][:-1, None] + i, 0)
    draft = torch.arange(s["max_k"], device="cuda") - (s["ctx"][:, None] - n)  # of each token; below 0: the context
    bit = s["mask"][row][:, :, None] >> draft.clamp(0, 63)[:, None, :] & 1
    seen = torch.where(draft[:, None] < 0, True, (bit == 1) & (draft < n)[:, None])
    return _plain_attend(s, s["q"][row], seen)[real]


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["top"]
    m = x.amax(-1, keepdim=True)
    logp = x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
    entropy = -(torch.exp(logp) * logp).sum(-1)
    mine = torch.gather(x, 1, s["tokens"][:, None])
    rank = (x > mine).sum(-1) + 1
    bits = x.view(torch.int32) if x.is_contiguous() else x.contiguous().view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32  # ties: the lowest index first
    order |= torch.arange(x.shape[1] - 1, -1, -1, device="cuda")
    ids = x.shape[1] - 1 - (torch.topk(order, top, dim=-1).values & 0xffffffff)
    return torch.gather(logp, 1, s["tokens"][:, None])[:, 0], entropy, rank, torch.gather(logp, 1, ids), ids


# ----------------------------------------------------------------------------- run

def _own(s):
    from kavor_amd.layers import attention, fused

    if s["kind"] == "store":
        attention.store_kvcache_fp8(s["key"], s["value"], s["k"], s["v"], s["ks"], s["vs"], s["slots"])
        return s["k"], s["v"], s["ks"], s["vs"]
    if s["kind"] == "load":
        return attention.load_kvcache_fp8(s["k"], s["v"], s["ks"], s["vs"], s["bt"], s["cu_k"], s["total"])
    if s["kind"] == "decode":
        return attention.paged_decode_fp8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["ctx"], s["bt"], SCALE)
    if s["kind"] == "tree":
        return attention.tree_attention(s["q"], s["k"], s["v"], s["cu_q"], s["max_q"], s["ctx"], s["bt"], SCALE,
                                        tree_mask=s["mask"], k_scale=s["ks"], v_scale=s["vs"])
    return fused.token_logprobs(s["logits"], s["tokens"], s["top"])


@torch.inference_mode()
def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "load": _plain_load, "decode": _plain_decode, "tree": _plain_tree,
            "logprobs": _plain_logprobs}[state["kind"]](state)


def work(case):
    kind, heads = case["kind"], case.get("kv_heads")
    if kind == "store":
        live = case["tokens"] - case["pad"]
        return {"bytes": live * 2 * heads * (2 * D + D + 1) + 4 * case["tokens"], "flops": live * 2 * heads * 3 * D}
    if kind == "logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 8 + 16 + 12 * case["top"]),
                "flops": case["rows"] * case["vocab"] * 6}
    both = _lens(case, 0)
    tokens = sum(n for n, _ in both)
    tables = 4 * sum(2 - (-n // case["block"]) for n, _ in both)
    row = 2 * heads * (2 * D if case.get("cache") == "bf16" else D + 1)
    if kind == "load":
        return {"bytes": tokens * (row + 2 * heads * 2 * D) + tables, "flops": tokens * 2 * heads * D}
    queries = sum(d for _, d in both) if kind == "tree" else len(both)
    pairs = sum(n * d for n, d in both) if kind == "tree" else tokens
    return {"bytes": tokens * row + tables + queries * (2 * case["q_heads"] * D * 2 + 8),
            "flops": 4 * case["q_heads"] * D * pairs}


# ----------------------------------------------------------------------------- 64-bit results

def _values64(x, page, name):
    """[tokens, H, D] in 64 bits of the listed pages."""
    c = x[name][page]
    if x[name + "s"] is None:
        return c.double().flatten(0, 1)
    scale = torch.exp2(x[name + "s"][page].double() - 127).transpose(1, 2)
    return (c.double() * scale[..., None]).flatten(0, 1)


def _store64(case, seed):
    x = _store_inputs(case, seed)
    keep = x["slots"] >= 0
    page, off = x["slots"][keep].long() // case["block"], x["slots"][keep].long() % case["block"]
    values, scales = [], []
    for new, name in ((x["key"], "k"), (x["value"], "v")):
        new, whole, scale = new[keep].double(), x[name].double(), x[name + "s"].clone()
        # bf16 values are 2^-8 apart, relative: the logarithms' own rounding decides nothing
        e = torch.ceil(torch.log2(new.abs().amax(-1) / 448) - 1e-9).clamp(-126, 127)
        y = new * torch.exp2(-e)[..., None]
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)) + 1e-9) - 3)
        whole[page, off] = torch.round(y / step) * step
        scale[page, :, off] = (e + 127).to(torch.uint8)
        values.append(whole)
        scales.append(scale)
    return *values, *scales


def _attend64(case, x):
    hq, hkv = case["q_heads"], case["kv_heads"]
    out, at = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, d) in enumerate(zip(x["lens"], x["drafts"])):
        page = torch.tensor(x["tables"][b], device="cuda")
        k, v = _values64(x, page, "k")[:n], _values64(x, page, "v")[:n]
        rows = d or 1
        hidden = torch.zeros(rows, n, dtype=torch.bool, device="cuda")
        for i in range(d):
            m = int(x["mask"][at + i])
            hidden[i, n - d:] = torch.tensor([not m >> j & 1 for j in range(d)], device="cuda")
        for h in range(hq):
            kh, vh = k[:, h * hkv // hq], v[:, h * hkv // hq]
            s = torch.mm(x["q"][at:at + rows, h].double(), kh.t().contiguous()) * SCALE
            out[at:at + rows, h] = torch.mm(torch.softmax(s.masked_fill_(hidden, -math.inf), -1), vh.contiguous())
        at += rows
    return out


def _logprobs64(case, seed):
    x = _logprobs_inputs(case, seed)
    outs = []
    for at in range(0, case["rows"], 256):
        z, tok = x["logits"][at:at + 256].double(), x["tokens"][at:at + 256, None]
        logp = torch.log_softmax(z, -1)
        order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        h = -torch.where(logp > -745, logp.exp() * logp, 0).sum(-1)
        outs.append((logp.gather(1, tok)[:, 0], h, (z > z.gather(1, tok)).sum(-1) + 1, logp.gather(1, order), order))
    return tuple(torch.cat(o) for o in zip(*outs))


@torch.inference_mode()
def exact(case, seed):
    if case["kind"] == "store":
        return _store64(case, seed)
    if case["kind"] == "logprobs":
        return _logprobs64(case, seed)
    x = _paged_inputs(case, seed)
    if case["kind"] == "load":
        pages = [torch.tensor(t, device="cuda") for t in x["tables"]]
        return tuple(torch.cat([_values64(x, p, c)[:n] for p, n in zip(pages, x["lens"])]) for c in ("k", "v"))
    return _attend64(case, x)
