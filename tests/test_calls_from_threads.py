"""Two threads that call on the same stream at once share its workspaces: every result has the bits of a call alone."""

import threading

import pytest
import torch

from kavor_amd.layers import attention, fused
from tests.helpers import gen
from tests.test_tree_attention import SCALE, Batch, decode


def calls(kind, i, device):
    """A call of its own for thread i."""
    if kind == "logprobs":
        x = (torch.randn(3 + 5 * i, 30_000, generator=gen(i)) * 3).bfloat16().to(device)
        return lambda: fused.token_logprobs(x, torch.arange(len(x), device=device), 5)[3]
    if kind == "argmax":
        x = torch.randn(3 + 5 * i, 60_000, generator=gen(i)).bfloat16().to(device)
        return lambda: fused.greedy_argmax(x)
    if kind == "prefill":
        x = Batch([0] * (2 + i), [30 + 30 * i] * (2 + i), 4, 2, 64, False, seed=i) if i else \
            Batch([0], [40], 8, 2, 64, False)
        k, v, _, _ = x.dev
        args = [t.to(device) for t in (x.q, x.cu, x.cu, x.bt)]
        return lambda: attention.varlen_prefill(args[0], k, v, max(x.drafts), args[1], max(x.drafts), args[2], SCALE,
                                                block_table=args[3])
    if kind == "tree":
        x = Batch([3000 - 2000 * i, 70], [12, 3 + i], 16, 8 >> i, 64, bool(i), seed=i)
        k, v, ks, vs = x.dev
        args = [t.to(device) for t in (x.q, x.cu, x.ctx, x.bt, x.mask)]
        return lambda: attention.tree_attention(args[0], k, v, args[1], 12, args[2], args[3], SCALE, args[4], ks, vs)
    x = Batch([2500 - 2000 * i, 70, 5][:3 - i], [1] * (3 - i), 16, 8 >> i, 64, kind == "decode_fp8", seed=i)
    q, ctx, bt = (t.to(device) for t in (x.q, x.ctx, x.bt))
    if kind == "decode_fp8":
        return lambda: decode(x, q=q, cache_seqlens=ctx, block_table=bt)
    return lambda: attention.paged_decode(q.unsqueeze(1), *x.dev[:2], cache_seqlens=ctx, block_table=bt, softmax_scale=SCALE)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["tree", "decode_fp8", "logprobs", "decode", "prefill", "argmax"])
def test_results_do_not_depend_on_another_threads_calls(cuda_device, kind):
    mine = [calls(kind, i, cuda_device) for i in range(2)]
    want = [call() for call in mine]
    torch.cuda.synchronize()
    got, errors = [[], []], []
    start = threading.Barrier(2)

    def work(i):
        try:
            start.wait()
            for _ in range(150):
                got[i].append(mine[i]())
        except Exception as e:  # reported by the test itself
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(2):
        same = torch.stack([(a.view(torch.uint8) == want[i].view(torch.uint8)).all() for a in got[i]])
        assert same.all(), f"{int((~same).sum())} of 150 calls of thread {i} differ"
