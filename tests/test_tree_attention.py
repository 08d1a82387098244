"""Attention of drafted tokens over a paged cache (bf16 and quantised) and decode over the quantised
cache, against the 64-bit oracle, and what is refused.

Tolerance: the output is rounded to bf16 once (2^-8 of it) and every softmax weight once on its way
to the second product (2^-8 of the weight, so 2^-8 sum p |v| in all).  Scores of q.k in 32 bits are off
by less than 2^-24 * 128 * |q||k| scale, some 2^-13 here, which moves a weight by that much of itself.
"""

import math
import random

import pytest
import torch

from kavor_amd import _lib
from kavor_amd.layers import attention
from oracle import operators_oracle as oracle
from tests.helpers import bits_equal, gen, interleaved_pool, randn_bf16, random_block_tables
from tests.test_kv_quant import pool_views, quantised_pool

D = 128
SCALE = D ** -0.5


def signed(bits):
    return bits - (1 << 64) if bits >> 63 else bits


def tree_masks(drafts, rng):
    out = []
    for n in drafts:
        mine = []
        for i in range(n):
            parent = rng.randint(-1, i - 1)
            mine.append((mine[parent] if parent >= 0 else 0) | 1 << i)
        out += mine
    return torch.tensor([signed(m) for m in out], dtype=torch.int64)


class Batch:
    """Drafts behind contexts in a paged cache of one kind, on the CPU and on the GPU."""

    def __init__(self, contexts, drafts, hq, hkv, block, quantised, seed=0, device="cuda", width=None):
        g = gen(seed)
        self.drafts, self.quantised, self.block = drafts, quantised, block
        self.lens = [c + n for c, n in zip(contexts, drafts)]
        blocks = sum(-(-n // block) for n in self.lens) + 2
        self.bt = random_block_tables(self.lens, block, blocks, g, width=width)
        if quantised:
            self.pool = quantised_pool(blocks, block, hkv, D, g)
            # codes of magnitudes around 1 at scales around 1
            values = self.pool[:, :2 * block * hkv * D]
            values.copy_(randn_bf16(values.shape, g, 8.0).float().to(torch.float8_e4m3fn).view(torch.uint8))
            self.pool[:, 2 * block * hkv * D:] = torch.randint(
                122, 126, (blocks, 2 * block * hkv), generator=g, dtype=torch.uint8)
            views = pool_views(self.pool, block, hkv, D)
            self.plain = tuple(oracle.dequantise(c, s) for c, s in zip(views[:2], views[2:]))
            self.dev = pool_views(self.pool.to(device), block, hkv, D)
        else:
            _, k, v = interleaved_pool(blocks, block, hkv, D, g)
            self.plain, self.dev = (k, v), (k.to(device), v.to(device), None, None)
        self.q = randn_bf16((sum(drafts), hq, D), g)
        self.cu = torch.tensor([sum(drafts[:i]) for i in range(len(drafts) + 1)], dtype=torch.int32)
        self.ctx = torch.tensor(self.lens, dtype=torch.int32)
        self.mask = tree_masks(drafts, random.Random(seed))
        self.device = device

    def run(self, mask="own", out=None, q=None, max_q=None):
        mask = self.mask if isinstance(mask, str) else mask
        k, v, ks, vs = self.dev
        return attention.tree_attention(
            (self.q if q is None else q).to(self.device), k, v, self.cu.to(self.device), max_q or max(self.drafts),
            self.ctx.to(self.device), self.bt.to(self.device), SCALE,
            tree_mask=None if mask is None else mask.to(self.device), k_scale=ks, v_scale=vs, out=out)

    def check(self, got, mask="own"):
        mask = self.mask if isinstance(mask, str) else mask
        want, spread = oracle.tree_attention(self.q, *self.plain, self.cu, self.ctx, self.bt, SCALE, mask)
        close(got, want, spread)


def close(got, want, spread):
    got = got.cpu().double()
    bound = want.abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -12) + 1e-30
    off = ((got - want).abs() / bound).nan_to_num(math.inf)
    assert off.max() <= 1, f"{off.max():.2f} of the bound at {(off == off.max()).nonzero()[0].tolist()}"


CASES = [
    # contexts, drafts, Hq, Hkv, block
    ([0], [1], 2, 1, 64),
    ([0, 0, 3], [1, 7, 2], 8, 8, 64),
    ([31, 32, 33, 63, 64, 65], [1, 2, 3, 1, 1, 2], 16, 8, 64),
    ([130, 5, 70], [12, 64, 33], 4, 2, 128),
    ([100, 257], [16, 17], 6, 2, 64),
    ([700], [5], 7, 1, 256),
    ([90, 1], [4, 4], 32, 2, 64),
    ([200], [64], 8, 1, 64),
    ([40, 300, 2], [9, 3, 20], 10, 2, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"ctx{c[0]}n{c[1]}h{c[2]}x{c[3]}")
def test_trees_match_the_oracle(cuda_device, case, quantised):
    x = Batch(*case, quantised)
    x.check(x.run())
    x.check(x.run(mask=None), mask=None)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_sequences_cut_over_many_ranges(cuda_device, quantised):
    """Few long sequences: ranges begin and end inside them, and hold several short ones whole."""
    x = Batch([3000, 1, 40, 2000, 7, 0, 500], [3, 1, 2, 5, 1, 4, 2], 4, 2, 64, quantised)
    x.check(x.run())


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_more_sequences_than_one_launch_takes(cuda_device, quantised):
    rng = random.Random(3)
    n = 2100
    x = Batch([rng.randint(0, 70) for _ in range(n)], [rng.randint(1, 2) for _ in range(n)], 2, 1, 64, quantised)
    x.check(x.run())


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_masks_hide_rows_and_whole_rows_see_nothing(cuda_device, quantised):
    x = Batch([0, 0, 70], [6, 3, 4], 4, 2, 64, quantised)
    mask = x.mask.clone()
    mask[0] = 0                       # no context and no draft: a row of zeros
    mask[2] = signed(~0 & (1 << 64) - 1)  # bits beyond the drafts are ignored
    mask[3] = 1 << 5                  # a later draft, and not itself
    mask[7] = 0
    mask[9] = 0                       # the context alone
    got = x.run(mask=mask)
    assert (got[0] == 0).all() and (got[7] == 0).all()
    x.check(got, mask=mask)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("what", [math.inf, math.nan])
def test_what_masked_tokens_hold_reaches_no_row(cuda_device, what, quantised):
    """Drafts 1, 2 and 4 of sequence 0 and the slots behind the last tokens hold infinities or NaN in K
    and V: rows that do not see them are as if the slots held zeros; rows that do are not finite."""
    x = Batch([66, 3], [6, 2], 6, 2, 64, quantised)
    clean = Batch([66, 3], [6, 2], 6, 2, 64, quantised)
    k, v, ks, vs = x.dev
    ck, cv, _, _ = clean.dev
    bt = x.bt

    def put(caches, b, t, head, dim, value):
        for c in caches:
            if quantised:  # e4m3 has NaN alone
                c.view(torch.uint8)[int(bt[b, t // 64]), t % 64, head, dim] = 127 if value else 0
            else:
                c[int(bt[b, t // 64]), t % 64, head, dim] = value
    for b, t, head, dim in ((0, 67, 0, 5), (0, 68, 1, 127), (0, 70, 0, 64), (0, 70, 1, 64)):
        put((k, v), b, t, head, dim, what)
        put((ck, cv), b, t, head, dim, 0.0)
    for b, t in ((0, 72), (1, 5), (0, 80), (1, 63)):  # behind the last tokens
        for head in range(2):
            put((k, v), b, t, head, 9, what)
            put((ck, cv), b, t, head, 9, 0.0)
    mask = torch.tensor([1, 1, 0b1000, 0b1001, 0b10000, 0b100011, 1, 3], dtype=torch.int64)
    got, want = x.run(mask=mask), clean.run(mask=mask)
    hit = torch.zeros(8, 6, dtype=torch.bool)
    hit[4] = True                 # sees draft 4, bad in both kv heads
    hit[5, :3] = True             # sees draft 1, bad in kv head 0
    assert torch.equal((~got.isfinite()).any(-1).cpu(), hit)
    keep = ~hit.to(cuda_device)
    assert bits_equal(got[keep], want[keep])


@pytest.mark.gpu
def test_an_infinity_that_rows_see_stays_one(cuda_device):
    x = Batch([5], [3], 2, 1, 64, False)
    k, v, _, _ = x.dev
    page = int(x.bt[0, 0])
    v[page, 2, 0, 7], v[page, 6, 0, 9] = math.inf, -math.inf  # a context token, and draft 1
    got = x.run(mask=torch.tensor([1, 2, 4]))
    assert (got[:, :, 7] == math.inf).all()
    assert (got[1, :, 9] == -math.inf).all() and got[[0, 2], :, 9].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_impossible_sequences_and_padding(cuda_device, quantised):
    """NaN for lengths that cannot be and for pages that are not there, zeros for padding rows, rows
    of no sequence left alone, and the others as ever."""
    x = Batch([10, 100, 20, 30, 64, 5, 9], [2, 3, 2, 1, 5, 2, 1], 4, 2, 64, quantised, width=2)
    want = x.run(max_q=5)
    x.ctx[1] = 2             # fewer tokens than drafts
    x.ctx[2] = 0             # padding
    x.ctx[3] = 129           # beyond the table
    x.bt[4, 1] = 10_000      # no such page
    x.ctx[6] = -5
    out = torch.full((16 + 4, 4, D), 7.0, dtype=torch.bfloat16, device=cuda_device)
    q = torch.cat((x.q, x.q[:4]))
    got = x.run(mask=torch.cat((x.mask, x.mask[:4])), out=out, q=q, max_q=5)
    assert (got[16:] == 7).all()
    rows = [(0, 2), (2, 5), (5, 7), (7, 8), (8, 13), (13, 15), (15, 16)]
    for b, (i, j) in enumerate(rows):
        if b in (1, 3, 4):
            assert got[i:j].isnan().all(), b
        elif b in (2, 6):
            assert (got[i:j] == 0).all(), b
        else:
            assert bits_equal(got[i:j], want[i:j]), b
    y = Batch([10, 20], [2, 3], 4, 2, 64, quantised)
    got = y.run(max_q=2)     # three drafts where two were said
    assert got[2:].isnan().all() and bits_equal(got[:2], y.run()[:2])
    y.cu = torch.tensor([0, 2, 9], dtype=torch.int32)  # rows that q does not have
    out = torch.full((5, 4, D), 7.0, dtype=torch.bfloat16, device=cuda_device)
    got = y.run(out=out)
    assert (got[2:] == 7).all() and not (got[:2] == 7).any()


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_strides_of_every_tensor(cuda_device, quantised):
    """q and out as slices of wider rows with heads in front, caches with heads outside slots."""
    x = Batch([70, 3], [4, 2], 4, 2, 64, quantised)
    want = x.run()
    wide = torch.zeros(4, 6, 2 * D, dtype=torch.bfloat16, device=cuda_device)
    q = wide[:, :, D:].transpose(0, 1)
    q.copy_(x.q)
    out = torch.zeros(6, 4, 3 * D, dtype=torch.bfloat16, device=cuda_device)[:, :, 8:8 + D]
    k, v, ks, vs = x.dev

    def moved(c):  # [blocks, heads, block, D] in memory, in the middle of a larger page
        n, block, heads, _ = c.shape
        room = torch.zeros(n, heads + 1, block, D + 32, dtype=torch.uint8 if quantised else c.dtype, device=c.device)
        room = room.view(c.dtype)[:, 1:, :, 16:16 + D].transpose(1, 2)
        (room.view(torch.uint8) if quantised else room).copy_(c.view(torch.uint8) if quantised else c)
        return room

    if quantised:
        wider = [torch.zeros(s.shape[0], s.shape[1], s.shape[2] + 4, dtype=torch.uint8, device=s.device)[:, :, 4:]
                 for s in (ks, vs)]
        for a, b in zip(wider, (ks, vs)):
            a.copy_(b)
        ks, vs = wider
    got = attention.tree_attention(q, moved(k), moved(v), x.cu.cuda(), 4, x.ctx.cuda(), x.bt.cuda(), SCALE,
                                   tree_mask=x.mask.cuda(), k_scale=ks, v_scale=vs, out=out)
    assert got.data_ptr() == out.data_ptr() and bits_equal(got, want)


@pytest.mark.gpu
def test_scores_far_apart(cuda_device):
    """One key dominates by hundreds of binary orders, early or late: the running maximum has to hold."""
    x = Batch([400], [3], 2, 1, 64, False)
    k = x.plain[0]
    for t, size in ((3, 40.0), (390, 60.0)):
        k[int(x.bt[0, t // 64]), t % 64, 0] = (size * x.q[0, 0].float() / x.q[0, 0].float().norm()).bfloat16()
    x.dev = (k.to(cuda_device), x.dev[1], None, None)
    x.check(x.run())


def decode(x, **over):
    k, v, ks, vs = x.dev
    a = dict(q=x.q.to(x.device), k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, cache_seqlens=x.ctx.to(x.device),
             block_table=x.bt.to(x.device), softmax_scale=SCALE)
    a.update(over)
    return attention.paged_decode_fp8(**a)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(16, 8), (8, 8), (32, 8), (40, 8), (64, 8), (14, 2), (3, 1), (16, 1), (9, 9)])
def test_decode_matches_the_oracle(cuda_device, hq, hkv):
    lens = [1, 63, 64, 65, 128, 200, 611]
    x = Batch([n - 1 for n in lens], [1] * len(lens), hq, hkv, 64, True, seed=hq)
    x.check(decode(x), mask=None)


@pytest.mark.gpu
def test_decode_of_padding_and_bad_rows(cuda_device):
    x = Batch([70, 5, 9, 80], [1] * 4, 16, 8, 64, True)
    want = decode(x)
    x.ctx[1], x.ctx[2], x.bt[3, 0] = 0, 1000, -1
    got = decode(x)
    assert bits_equal(got[0], want[0])
    assert (got[1] == 0).all() and got[2].isnan().all() and got[3].isnan().all()
    q4 = x.q.to(cuda_device).unsqueeze(1)
    out = torch.empty_like(q4)
    assert decode(x, q=q4, out=out).shape == q4.shape and bits_equal(out[0, 0], want[0])


@pytest.mark.gpu
def test_decode_is_tree_attention_of_one_draft(cuda_device):
    x = Batch([200, 3, 64], [1] * 3, 16, 8, 64, True)
    assert bits_equal(decode(x), x.run(mask=None))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_captured_replays_follow_their_inputs(cuda_device, quantised):
    """A graph of a batch replayed with other lengths, masks and queries, eager calls of other sizes and
    on another stream between the replays: every replay has the eager result's bits."""
    x = Batch([500, 90, 3], [4, 2, 7], 16, 8, 64, quantised, width=12)
    k, v, ks, vs = x.dev
    q, cu, ctx, bt, mask = (t.to(cuda_device) for t in (x.q, x.cu, x.ctx, x.bt, x.mask))
    out = torch.empty_like(q)

    def step(o=None):
        return attention.tree_attention(q, k, v, cu, 7, ctx, bt, SCALE, tree_mask=mask, k_scale=ks, v_scale=vs, out=o)

    attention.reserve_tree_workspace(3, 7, 16, 8, D, 12, 64, cuda_device)
    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    side = torch.cuda.Stream()
    g = gen(1)
    for i in range(4):
        q.copy_(randn_bf16(q.shape, g))
        ctx.copy_(torch.tensor([[504, 92, 10], [33, 0, 8], [504, 2, 7], [100, 60, 10]][i], dtype=torch.int32))
        if i == 2:
            mask.fill_(-1)
        other = Batch([20 * i], [3], 16, 8, 64, quantised)
        with torch.cuda.stream(side):
            other.run()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert bits_equal(out, step()), i
    assert not bits_equal(out, torch.zeros_like(out))


def _tree(**over):
    a = dict(q=16, qs=2048, qh=128, kc=16, vc=16, bstr=1 << 18, sstr=1024, hstr=128, ks=16, vs=16, sbs=2048, shs=256,
             nblk=64, bt=16, bts=16, cu=16, ctx=16, b=4, total=20, maxq=8, mask=16, hq=16, hkv=8, d=128, bs=256,
             maxb=16, scale=0.088, out=16, os=2048, oh=128, ws=256, wsb=1 << 30, stream=None)
    a.update(over)
    return _lib.lib().kvp_tree_attention(*a.values())


def _decode(**over):
    a = dict(q=16, qs=2048, qh=128, kc=16, vc=16, bstr=1 << 18, sstr=1024, hstr=128, ks=16, vs=16, sbs=2048, shs=256,
             nblk=64, bt=16, bts=16, ctx=16, b=4, hq=16, hkv=8, d=128, bs=256, maxb=16, scale=0.088, out=16, os=2048,
             oh=128, ws=256, wsb=1 << 30, stream=None)
    a.update(over)
    return _lib.lib().kvp_paged_decode_fp8(*a.values())


def test_bad_arguments_are_refused_on_the_host():
    E, U = _lib.KVP_EINVAL, _lib.KVP_EUNSUPPORTED
    assert _tree(b=0) == _lib.KVP_OK and _tree(total=0) == _lib.KVP_OK and _decode(b=0) == _lib.KVP_OK
    for call in (_tree, _decode):
        for over in (dict(d=64), dict(hq=17 * 8), dict(maxb=1 << 17, bts=1 << 17), dict(sstr=1 << 25),
                     dict(hq=514, hkv=257)):
            assert call(**over) == U, over
        for over in (dict(hq=12), dict(bs=100), dict(bts=8), dict(q=8), dict(q=0), dict(kc=0), dict(vc=8), dict(bt=0),
                     dict(ctx=0), dict(ctx=2), dict(out=0), dict(out=8), dict(qs=2044), dict(oh=4), dict(sstr=1032),
                     dict(hstr=8), dict(bstr=4), dict(sbs=2), dict(shs=255), dict(vs=18), dict(sbs=-4), dict(ws=32),
                     dict(b=-1), dict(nblk=0), dict(maxb=0), dict(sstr=-16)):
            assert call(**over) == E, over
    for over in (dict(maxq=0), dict(maxq=65)):
        assert _tree(**over) == U, over
    for over in (dict(cu=0), dict(mask=20), dict(ks=0), dict(vs=0), dict(total=-1), dict(cu=18)):
        assert _tree(**over) == E, over
    assert b"cu_seqlens_q" in _lib.lib().kvp_last_error()
    assert _decode(ks=0) == E


def test_workspace_sizes_grow_with_every_argument():
    base = [3, 5, 16, 8, 128, 4, 64]
    size = attention.tree_workspace_bytes(*base)
    assert size > 0
    for i, values in ((0, (4, 100, 5000)), (1, (6, 17, 33, 64)), (5, (5, 64, 4000)), (6, (128, 256))):
        last = size
        for value in values:
            now = attention.tree_workspace_bytes(*[value if j == i else x for j, x in enumerate(base)])
            assert now >= last
            last = now
    for bad in ([0] + base[1:], base[:1] + [65] + base[2:], base[:4] + [64] + base[5:]):
        assert _lib.lib().kvp_tree_workspace_bytes(*bad) == 0


def test_wrappers_refuse_cpu_tensors():
    x = Batch([3], [2], 2, 1, 64, True, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        x.run()
    with pytest.raises(ValueError, match="CUDA"):
        decode(x)


@pytest.mark.gpu
def test_wrappers_check_types_shapes_and_devices(cuda_device):
    x = Batch([3], [2], 2, 1, 64, True)
    k, v, ks, vs = x.dev
    good = dict(q=x.q.cuda(), k_cache=k, v_cache=v, cu_seqlens_q=x.cu.cuda(), max_seqlen_q=2, cache_seqlens=x.ctx.cuda(),
                block_table=x.bt.cuda(), softmax_scale=SCALE, tree_mask=x.mask.cuda(), k_scale=ks, v_scale=vs)
    attention.tree_attention(**good)
    for bad in (dict(q=good["q"][0]), dict(q=good["q"][:, :, :64]), dict(k_scale=None), dict(k_scale=None, v_scale=None),
                dict(tree_mask=good["tree_mask"].int()), dict(tree_mask=good["tree_mask"][:1]),
                dict(tree_mask=x.mask), dict(cu_seqlens_q=x.cu), dict(cu_seqlens_q=good["cu_seqlens_q"].long()),
                dict(cache_seqlens=good["cache_seqlens"][:0]), dict(block_table=x.bt),
                dict(block_table=good["block_table"][:0]), dict(out=good["q"].float()), dict(out=good["q"][:1]),
                dict(v_cache=v[:1]), dict(k_cache=k.view(torch.uint8)), dict(k_scale=ks[:, :, :32], v_scale=vs[:, :, :32])):
        with pytest.raises(ValueError):
            attention.tree_attention(**{**good, **bad})
    for bad in (dict(max_seqlen_q=0), dict(max_seqlen_q=65)):
        with pytest.raises((_lib.KVPathError, ValueError, RuntimeError)):
            attention.tree_attention(**{**good, **bad})
    y = Batch([3, 4], [1, 1], 2, 1, 64, True)
    for bad in (dict(q=y.q.cuda()[None]), dict(cache_seqlens=y.ctx.cuda()[:1]), dict(block_table=y.bt.cuda()[:1]),
                dict(k_scale=None), dict(cache_seqlens=y.ctx), dict(out=y.q.cuda().float())):
        with pytest.raises((ValueError, AttributeError)):
            decode(y, **bad)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_many_rows_of_sequences_that_ranges_cut(cuda_device, quantised):
    """More rows than are joined a wave each: 24 sequences of up to 12 drafts at 32 heads."""
    rng = random.Random(9)
    x = Batch([rng.randint(0, 400) for _ in range(23)] + [1500], [rng.randint(1, 12) for _ in range(23)] + [12], 32, 8, 64,
              quantised)
    x.check(x.run())


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("case", [
    ([5, 70], [2, 3], 256, 256, 64), ([300, 10], [64, 40], 16, 1, 64), ([0, 1000], [64, 64], 32, 2, 128),
    ([200, 77], [22, 30], 9, 3, 64), ([5000, 10, 20], [20, 1, 3], 8, 2, 64)], ids=lambda c: f"n{c[1]}h{c[2]}x{c[3]}")
def test_the_ends_of_the_limits(cuda_device, case, quantised):
    """256 kv heads, 1024 rows of one kv head in blocks, three query heads to one, a long sequence among short ones."""
    x = Batch(*case, quantised)
    x.check(x.run())


@pytest.mark.gpu
def test_weights_times_the_largest_scale_stay_finite(cuda_device):
    """Rows of zeros at the largest scale, 2^120: the scale goes into the weights, and an infinite product
    of the two would make NaN of the zeros."""
    for drafts in (1, 30):
        x = Batch([200], [drafts], 2, 1, 64, True)
        k, v, ks, vs = x.dev
        vs.fill_(247)
        v.view(torch.uint8).zero_()
        got = x.run().cpu()
        assert torch.equal(got, torch.zeros_like(got))


@pytest.mark.gpu
def test_block_tables_whose_rows_overlap_are_refused(cuda_device):
    """An expanded table is one row in memory: with another stride the rows behind it would be read from
    beyond its end."""
    x = Batch([100, 90], [2, 3], 4, 2, 64, True)
    k, v, ks, vs = x.dev
    q, cu, ctx, bt = (t.to(cuda_device) for t in (x.q, x.cu, x.ctx, x.bt))
    shared = bt[:1].expand(2, -1)
    with pytest.raises((ValueError, _lib.KVPathError)):
        attention.tree_attention(q, k, v, cu, 3, ctx, shared, SCALE, k_scale=ks, v_scale=vs)
    with pytest.raises((ValueError, _lib.KVPathError)):
        attention.paged_decode_fp8(q[:2], k, v, ks, vs, ctx, shared, SCALE)
    with pytest.raises((ValueError, _lib.KVPathError)):
        attention.load_kvcache_fp8(k, v, ks, vs, shared, cu, 5)
    one = torch.empty_strided((1, bt.shape[1]), (1, 1), dtype=torch.int32, device=cuda_device).copy_(bt[:1])
    attention.load_kvcache_fp8(k, v, ks, vs, one, cu[:2], 2)
