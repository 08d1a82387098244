"""The size of tree attention's workspace: a reservation for the largest sizes covers every smaller call."""

import itertools

import pytest
import torch

from kavor_amd import _lib
from kavor_amd.layers import attention
from tests.test_tree_attention import Batch


def size(*args):
    return _lib.lib().kvp_tree_workspace_bytes(*args)


@pytest.mark.parametrize("name,index,values", [
    ("num_seqs", 0, (1, 3, 64, 5000)), ("max_seqlen_q", 1, (1, 5, 16, 17, 64)), ("num_q_heads", 2, (16, 32, 64, 128)),
    ("num_kv_heads", 3, (1, 2, 4, 8, 16, 256)), ("table width", 5, (1, 4, 64)), ("block_size", 6, (64, 128, 256))])
def test_it_falls_with_no_argument_that_grows(name, index, values):
    others = [(1, 64), (1, 5, 16, 64), (16, 64, 256), (1, 2, 8, 16, 256), (128,), (4, 64), (64, 256)]
    for args in itertools.product(*[[None] if i == index else o for i, o in enumerate(others)]):
        sizes = [size(*[v if a is None else a for a in args]) for v in values]
        sizes = [s for s in sizes if s]  # 0: a GQA ratio that is not supported
        assert sizes == sorted(sizes), (args, sizes)


def test_sizes_are_those_of_the_header():
    for seqs, max_q, hq, hkv in itertools.product((1, 256, 3000), (1, 4, 16, 64), (16, 64), (1, 4, 8, 16)):
        if (n := size(seqs, max_q, hq, hkv, 128, 64, 256)) == 0:
            continue
        rows = max_q * min(16, hq)
        assert n <= (17_100_000 if rows <= 16 else 34_100_000 if rows <= 64 else 68_200_000), (seqs, max_q, hq, hkv)


@pytest.mark.gpu
def test_a_reservation_for_more_heads_serves_a_capture_with_fewer(cuda_device):
    """The draft model of a pair, with fewer kv heads and so more rows for each of them, captured after a
    reservation for the larger one."""
    x = Batch([700, 3], [16, 5], 16, 1, 64, False, width=4096)
    q, cu, ctx, bt, mask = (t.to(cuda_device) for t in (x.q, x.cu, x.ctx, x.bt, x.mask))
    k, v = x.dev[:2]
    need = attention.tree_workspace_bytes(2, 16, 16, 8, 128, 4096, 64)
    room = torch.empty(need, dtype=torch.uint8, device=cuda_device)
    out = torch.empty_like(q)
    rc = _lib.lib().kvp_tree_attention(
        q.data_ptr(), *q.stride()[:2], k.data_ptr(), v.data_ptr(), *k.stride()[:3], 0, 0, 0, 0, k.shape[0], bt.data_ptr(), 4096,
        cu.data_ptr(), ctx.data_ptr(), 2, q.shape[0], 16, mask.data_ptr(), 16, 1, 128, 64, 4096, 128 ** -0.5,
        out.data_ptr(), *out.stride()[:2], room.data_ptr(), need, torch._C._cuda_getCurrentRawStream(0))
    assert rc == _lib.KVP_OK, _lib.lib().kvp_last_error()
    x.check(out)
