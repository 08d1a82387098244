"""The quantised cache, its decode, drafted tokens and their log probabilities as a serving loop uses
them together: prompts are stored quantised, a token is decoded, drafts are stored behind it and
verified in one pass, the next prompt chunk reads its history back.  Eager and captured.

Every stage is held to the 64-bit oracle over the bytes that the cache really has, within the
tolerances of the operators' own tests; the prompt chunk over read-back K/V is held to what tree
attention defines for a chain of drafts, since both see the same tokens.
"""

import random

import pytest
import torch

from kavor_amd.layers import attention, fused
from oracle import operators_oracle as oracle
from tests.helpers import bits_equal, gen, randn_bf16, random_block_tables
from tests.test_kv_quant import pool_views, quantised_pool
from tests.test_token_logprobs import check as check_logprobs
from tests.test_tree_attention import close, tree_masks

H, HKV, D, BLOCK, VOCAB = 8, 2, 128, 64, 1013
SCALE = D ** -0.5
PROMPTS, DRAFTS = [70, 128, 1], [5, 1, 9]


class Loop:
    def __init__(self, device):
        g = gen(11)
        lens = [p + 1 + d for p, d in zip(PROMPTS, DRAFTS)]
        self.bt = random_block_tables(lens, BLOCK, 10, g)
        self.pool = quantised_pool(10, BLOCK, HKV, D, g).to(device)
        self.cache = pool_views(self.pool, BLOCK, HKV, D)
        table = self.bt.clone()

        def slots(first, count):  # per sequence
            return torch.tensor([int(table[b, t // BLOCK]) * BLOCK + t % BLOCK
                                 for b in range(3) for t in range(first[b], first[b] + count[b])], dtype=torch.int32)

        def ends(lengths):
            return torch.tensor([sum(lengths[:i]) for i in range(4)], dtype=torch.int32)

        after = [p + 1 for p in PROMPTS]
        self.host = dict(
            slots_prompt=slots([0] * 3, PROMPTS), slots_token=slots(PROMPTS, [1] * 3), slots_drafts=slots(after, DRAFTS),
            ctx_token=torch.tensor(after, dtype=torch.int32), ctx_drafts=torch.tensor(lens, dtype=torch.int32),
            cu_drafts=ends(DRAFTS), cu_all=ends(lens), mask=tree_masks(DRAFTS, random.Random(5)), bt=table,
            ids=torch.randint(0, VOCAB, (sum(DRAFTS),), generator=g))
        self.dev = {name: x.to(device) for name, x in self.host.items()}
        self.total = sum(lens)
        self.weight = torch.randn(H * D, VOCAB, generator=g).to(device)
        self.inputs = {name: torch.empty(n, heads, D, dtype=torch.bfloat16, device=device) for name, n, heads in (
            ("k_prompt", sum(PROMPTS), HKV), ("v_prompt", sum(PROMPTS), HKV), ("q_token", 3, H), ("k_token", 3, HKV),
            ("v_token", 3, HKV), ("q_drafts", sum(DRAFTS), H), ("k_drafts", sum(DRAFTS), HKV),
            ("v_drafts", sum(DRAFTS), HKV))}

    def fill(self, seed):
        g = gen(seed)
        for x in self.inputs.values():
            x.copy_(randn_bf16(x.shape, g))

    def step(self):
        i, d = self.inputs, self.dev
        k, v, ks, vs = self.cache
        for part in ("prompt", "token"):
            attention.store_kvcache_fp8(i["k_" + part], i["v_" + part], k, v, ks, vs, d["slots_" + part])
        token = attention.paged_decode_fp8(i["q_token"], k, v, ks, vs, d["ctx_token"], d["bt"], SCALE)
        attention.store_kvcache_fp8(i["k_drafts"], i["v_drafts"], k, v, ks, vs, d["slots_drafts"])
        drafts = attention.tree_attention(i["q_drafts"], k, v, d["cu_drafts"], max(DRAFTS), d["ctx_drafts"], d["bt"], SCALE,
                                          tree_mask=d["mask"], k_scale=ks, v_scale=vs)
        logits = torch.mm(drafts.view(-1, H * D).float(), self.weight)[:, :VOCAB]
        wide = torch.full((logits.shape[0], VOCAB + 3), -1.0, device=logits.device)
        wide[:, :VOCAB] = logits  # rows at a stride of 16 bytes
        scores = fused.token_logprobs(wide[:, :VOCAB], d["ids"], 4)
        history = attention.load_kvcache_fp8(k, v, ks, vs, d["bt"], d["cu_all"], self.total)
        chunk = attention.varlen_prefill(i["q_drafts"], *history, max(DRAFTS), d["cu_drafts"], 138, d["cu_all"], SCALE)
        return token, drafts, logits, scores, chunk

    def check(self, got):
        token, drafts, logits, scores, chunk = got
        h = self.host
        plain = tuple(oracle.dequantise(c.cpu(), s.cpu()) for c, s in zip(self.cache[:2], self.cache[2:]))
        q = self.inputs["q_token"].cpu()
        close(token, *oracle.tree_attention(q, *plain, torch.arange(4, dtype=torch.int32), h["ctx_token"], h["bt"], SCALE))
        q = self.inputs["q_drafts"].cpu()
        where = (h["cu_drafts"], h["ctx_drafts"], h["bt"], SCALE)
        close(drafts, *oracle.tree_attention(q, *plain, *where, h["mask"]))
        close(chunk, *oracle.tree_attention(q, *plain, *where))
        check_logprobs(scores, logits.cpu(), h["ids"], 4)


@pytest.mark.gpu
def test_the_steps_of_a_serving_loop(cuda_device):
    loop = Loop(cuda_device)
    side = torch.cuda.Stream()
    for seed in range(2):
        loop.fill(seed)
        loop.check(loop.step())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            again = loop.step()
        side.synchronize()
        loop.check(again)


@pytest.mark.gpu
def test_the_loop_captured_into_a_graph(cuda_device):
    loop = Loop(cuda_device)
    loop.fill(0)
    attention.reserve_tree_workspace(3, max(DRAFTS), H, HKV, D, loop.bt.shape[1], BLOCK, cuda_device)
    attention.reserve_prefill_workspace(3, max(DRAFTS), H, HKV, cuda_device)
    fused.reserve_logprobs_workspace(cuda_device)
    loop.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = loop.step()
    for seed in (3, 4, 5):
        loop.fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        loop.check(got)
        eager = loop.step()
        torch.cuda.synchronize()
        assert all(bits_equal(a, b) for a, b in zip(got[:2], eager[:2]))


def far_apart(x: torch.Tensor, stride: int) -> torch.Tensor:
    """x with its first dimension at another stride, on the GPU."""
    room = torch.empty((x.shape[0] - 1) * stride + x[0].numel(), dtype=x.dtype, device="cuda")
    y = room.as_strided(x.shape, (stride,) + x.stride()[1:])
    return y.copy_(x) if x.dtype != torch.float8_e4m3fn else (y.view(torch.uint8).copy_(x.view(torch.uint8)), y)[1]


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_device):
    """Pages and rows of logits more than 2^32 bytes from the first one: the same bits as close together."""
    g = gen(2)
    pool = quantised_pool(3, BLOCK, HKV, D, g).to(cuda_device)
    near = tuple(t.contiguous() for t in pool_views(pool, BLOCK, HKV, D))
    far = tuple(far_apart(t, (5 << 29) + 64) for t in near)
    bt = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=cuda_device)
    cu, ctx = (torch.tensor(t, dtype=torch.int32, device=cuda_device) for t in ([0, 5], [170]))
    slots = torch.tensor([2 * BLOCK + 3, BLOCK + 9], dtype=torch.int32, device=cuda_device)
    new = randn_bf16((2, HKV, D), g).to(cuda_device)
    for hq in (H, 16 * HKV):  # few rows per kv head, and many
        q = randn_bf16((5, hq, D), g).to(cuda_device)
        got = []
        for k, v, ks, vs in (near, far):
            attention.store_kvcache_fp8(new, new, k, v, ks, vs, slots)
            read = attention.load_kvcache_fp8(k, v, ks, vs, bt, torch.tensor([0, 170], dtype=torch.int32, device="cuda"), 170)
            got.append((*read, attention.paged_decode_fp8(q[:1], k, v, ks, vs, ctx, bt, SCALE),
                        attention.tree_attention(q, k, v, cu, 5, ctx, bt, SCALE, k_scale=ks, v_scale=vs)))
        assert all(bits_equal(a, b) for a, b in zip(*got))
        wide = [attention.load_kvcache_fp8(*near, torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"),
                                           torch.tensor([0, 3 * BLOCK], dtype=torch.int32, device="cuda"), 3 * BLOCK)][0]
        k, v = (t.view(3, BLOCK, HKV, D) for t in wide)
        a = attention.tree_attention(q, k, v, cu, 5, ctx, bt, SCALE)
        b = attention.tree_attention(q, far_apart(k, (5 << 28) + 64), far_apart(v, (5 << 28) + 64), cu, 5, ctx, bt, SCALE)
        assert bits_equal(a, b)
    logits = torch.randn(3, VOCAB + 3, generator=g).to(cuda_device)
    ids = torch.tensor([1, 2, 3], device=cuda_device)
    for a, b in zip(fused.token_logprobs(logits, ids, 4), fused.token_logprobs(far_apart(logits, 3 << 28), ids, 4)):
        assert torch.equal(a, b)
