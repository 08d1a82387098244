"""A step with drafted tokens as a serving loop runs it: the drafts' keys and values stored in every layer, attended to under
their tree, verified, those that stay moved next to their context, and the next token decoded over the result; then
a fork of the sequences on copied pages.  Eager and captured, over bf16 and quantised pages.

Verification is held to the 64-bit oracle over the logits that it really had, the caches byte for byte to the oracle's moves, and
the decode to the oracle over them within the tolerances of its own tests.
"""

import random

import pytest
import torch

from kavor_amd.layers import attention, fused
from oracle import drafts_oracle, operators_oracle
from tests.helpers import bits_equal, gen, randn_bf16
from tests.test_kept_drafts import oracle_caches, pool_of, views
from tests.test_tree_attention import close
from tests.test_verify_drafts import reach, same, trees

L, H, HKV, D, BLOCK, PAGES, VOCAB = 3, 8, 2, 128, 64, 14, 1013
SCALE = D ** -0.5
CONTEXTS, ROWS = [70, 124, 3, 60], [5, 9, 1, 12]


class Loop:
    def __init__(self, device, quantised, chain):
        g, rng = gen(3), random.Random(3)
        self.quantised = quantised
        pool = pool_of(L, PAGES, BLOCK, HKV, D, quantised, g)
        for c in views(pool, BLOCK, HKV, D, quantised):
            if c is not None:
                c.copy_(torch.randint(118, 122, c.shape, generator=g, dtype=torch.uint8) if c.dtype == torch.uint8
                        else torch.randn(c.shape, generator=g).to(c.dtype))
        self.pool = pool.to(device)
        self.cache = views(self.pool, BLOCK, HKV, D, quantised)
        lens = [c + r for c, r in zip(CONTEXTS, ROWS)]
        ids = torch.randperm(PAGES - 4, generator=g).tolist()
        need = [-(-n // BLOCK) for n in lens]
        tables = [[ids.pop() for _ in range(n)] for n in need]
        bt = torch.tensor([t + [-1] * (max(need) - len(t)) for t in tables], dtype=torch.int32)
        slots = [t[p // BLOCK] * BLOCK + p % BLOCK for t, c, n in zip(tables, CONTEXTS, lens) for p in range(c, n)]
        masks, _ = trees(ROWS, rng)
        self.host = dict(bt=bt, cu=torch.tensor([sum(ROWS[:i]) for i in range(5)], dtype=torch.int32),
                         ctx=torch.tensor(lens, dtype=torch.int32), slots=torch.tensor(slots, dtype=torch.int32),
                         temps=torch.tensor([0.7, 0.0, 1.0, 0.9]))
        if not chain:
            self.host["mask"] = masks
        self.dev = {k: t.to(device) for k, t in self.host.items()}
        self.weight = (torch.randn(H * D, VOCAB, generator=g) / 8).to(device)
        T = sum(ROWS)
        self.inputs = dict(k=torch.empty(L, T, HKV, D), v=torch.empty(L, T, HKV, D), q=torch.empty(L, T, H, D),
                           q_next=torch.empty(L, 4, H, D), draft=torch.empty(T, VOCAB + 3))
        self.inputs = {n: t.to(device, torch.float32 if n == "draft" else torch.bfloat16) for n, t in self.inputs.items()}
        self.inputs["tokens"] = torch.zeros(T, dtype=torch.int64, device=device)
        self.inputs["uniforms"] = torch.zeros(T, device=device)
        self.chain = chain

    def fill(self, seed):
        g, i = gen(seed), self.inputs
        for name in ("k", "v", "q", "q_next"):
            i[name].copy_(randn_bf16(i[name].shape, g, 2.0))
        logits = self.attend()[0].cpu()  # the drafts are good guesses: a model's that is near the target
        near = logits + 0.3 * torch.randn(logits.shape, generator=g)
        i["draft"].fill_(-1.0)
        i["draft"][:, :VOCAB] = near.to(i["draft"].device)
        first = [q for q, n in zip(self.host["cu"].tolist(), ROWS) for _ in range(n)]
        tokens = []
        for r in range(len(first)):
            below = (1 << (r - first[r])) - 1
            seen = (int(self.host["mask"][r]) & below) if not self.chain else below
            up = first[r] + max(seen.bit_length() - 1, 0)
            tokens.append(int(near[up].topk(3).indices[int(torch.randint(0, 3, (1,), generator=g))]) if not self.chain
                          else int(torch.multinomial(torch.softmax(near[up] / 0.8, 0), 1, generator=g)))
        i["tokens"].copy_(torch.tensor(tokens))
        i["uniforms"].copy_(torch.rand(len(tokens), generator=g))

    def attend(self):
        """The drafts into the pages of every layer, and the last layer's logits."""
        i, d = self.inputs, self.dev
        k, v, ks, vs = self.cache
        for layer in range(L):
            if self.quantised:
                attention.store_kvcache_fp8(i["k"][layer], i["v"][layer], k[layer], v[layer], ks[layer], vs[layer], d["slots"])
            else:
                attention.store_kvcache(i["k"][layer], i["v"][layer], k[layer], v[layer], d["slots"])
            o = attention.tree_attention(i["q"][layer], k[layer], v[layer], d["cu"], max(ROWS), d["ctx"], d["bt"], SCALE,
                                         tree_mask=d.get("mask"), k_scale=None if ks is None else ks[layer],
                                         v_scale=None if vs is None else vs[layer])
        logits = torch.mm(o.view(-1, H * D).float(), self.weight)
        wide = torch.full((logits.shape[0], VOCAB + 3), -1.0, device=logits.device)
        wide[:, :VOCAB] = logits
        return wide[:, :VOCAB], o

    def decode(self, lens, bt):
        k, v, ks, vs = self.cache
        q = self.inputs["q_next"]
        if self.quantised:
            return [attention.paged_decode_fp8(q[n], k[n], v[n], ks[n], vs[n], lens, bt, SCALE) for n in range(L)]
        return [attention.paged_decode(q[n], k[n], v[n], lens, bt, SCALE) for n in range(L)]

    def step(self):
        i, d = self.inputs, self.dev
        logits, _ = self.attend()
        got = fused.verify_drafts(logits, i["tokens"], i["uniforms"], d["temps"], d["cu"], max(ROWS), tree_mask=d.get("mask"),
                                  draft_logits=i["draft"][:, :VOCAB] if self.chain else None)
        before = self.pool.clone()
        k, v, ks, vs = self.cache
        lens = attention.keep_drafts(k, v, got[1], got[0], d["cu"], d["ctx"], d["bt"], ks, vs)
        return logits, got, before, lens, self.decode(lens, d["bt"])

    def check(self, results):
        logits, got, before, lens, outs = results
        h, i = self.host, {n: t.cpu() for n, t in self.inputs.items()}
        *want, decided, drawn = drafts_oracle.verify_drafts(
            logits.cpu(), i["tokens"], i["uniforms"], h["temps"], h["cu"], max(ROWS), h.get("mask"),
            i["draft"][:, :VOCAB] if self.chain else None)
        apart, off = reach(VOCAB)
        assert decided > apart and drawn > off
        same(got, want)
        moved = before.cpu()
        new = drafts_oracle.keep_drafts(oracle_caches(*views(moved, BLOCK, HKV, D, self.quantised)), want[1], want[0], h["cu"],
                                        h["ctx"], h["bt"])
        assert torch.equal(lens.cpu(), new) and torch.equal(self.pool.cpu(), moved)
        k, v, ks, vs = views(moved, BLOCK, HKV, D, self.quantised)
        for n, o in enumerate(outs):
            plain = (k[n].double(), v[n].double()) if ks is None else \
                tuple(operators_oracle.dequantise(c[n], s[n]) for c, s in ((k, ks), (v, vs)))
            close(o, *operators_oracle.tree_attention(i["q_next"][n], *plain, torch.arange(5, dtype=torch.int32), new, h["bt"], SCALE))
        return want[0]


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("chain", [False, True])
def test_steps_and_a_fork(cuda_device, quantised, chain):
    loop = Loop(cuda_device, quantised, chain)
    kept = 0
    for seed in range(3):
        loop.fill(seed)
        results = loop.step()
        kept += int(loop.check(results).sum())
    assert kept > 0
    # every sequence once more, on its own copy of the page that holds its last token
    lens, bt = results[3].tolist(), loop.host["bt"].clone()
    src = [int(bt[b, (n - 1) // BLOCK]) for b, n in enumerate(lens)]
    dst = list(range(PAGES - 4, PAGES))
    for b, n in enumerate(lens):
        bt[b, (n - 1) // BLOCK] = dst[b]
    attention.copy_pages(loop.pool, src, dst)
    fork = loop.decode(results[3], bt.to(cuda_device))
    assert all(bits_equal(a, b) for a, b in zip(fork, results[4]))
    assert torch.equal(loop.pool[:, src], loop.pool[:, dst])


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("chain", [False, True])
def test_the_step_captured_into_a_graph(cuda_device, quantised, chain):
    loop = Loop(cuda_device, quantised, chain)
    loop.fill(0)
    width = loop.host["bt"].shape[1]
    attention.reserve_tree_workspace(4, max(ROWS), H, HKV, D, width, BLOCK, cuda_device)
    attention.reserve_decode_workspace(4, H, D, width, BLOCK, cuda_device)
    fused.reserve_verify_workspace(4, max(ROWS), VOCAB, cuda_device)
    loop.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = loop.step()
    for seed in (4, 5, 6):
        loop.fill(seed)
        start = loop.pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        loop.check(got)
        end = loop.pool.clone()
        loop.pool.copy_(start)
        eager = loop.step()
        torch.cuda.synchronize()
        assert torch.equal(loop.pool, end) and all(torch.equal(a, b) for a, b in zip(eager[1], got[1]))
        assert all(bits_equal(a, b) for a, b in zip(eager[4], got[4]))
