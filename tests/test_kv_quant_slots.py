"""Slots that several tokens name in one call of the quantised append."""

import pytest
import torch

from kavor_amd.layers import attention
from oracle import operators_oracle as oracle
from tests.helpers import gen, randn_bf16
from tests.test_kv_quant import pool_views, quantised_pool


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,dim", [(40, 2, 128), (300, 8, 64), (7, 1, 256)])
def test_every_part_of_a_shared_slot_is_some_tokens(cuda_device, tokens, heads, dim):
    g, block = gen(tokens), 64
    key = randn_bf16((tokens, heads, dim), g) * torch.exp2(torch.randint(-9, 9, (tokens, 1, 1), generator=g)).bfloat16()
    value = randn_bf16((tokens, heads, dim), g)
    slots = torch.zeros(tokens, dtype=torch.int32)  # a padded graph's rows
    slots[tokens // 2] = 100                        # and one real one
    pool = quantised_pool(3, block, heads, dim, g)
    before = pool.clone()
    dev = pool.to(cuda_device)
    views = pool_views(dev, block, heads, dim)
    attention.store_kvcache_fp8(key.to(cuda_device), value.to(cuda_device), *views, slots.to(cuda_device))
    got = pool_views(dev.cpu(), block, heads, dim)
    shared = [t for t in range(tokens) if t != tokens // 2]
    for x, cache, scale in ((key, got[0], got[2]), (value, got[1], got[3])):
        codes, byte = (torch.from_numpy(a) for a in oracle.quantise_rows(x))
        rows = cache.view(torch.uint8)
        assert torch.equal(rows[1, 100 - block], codes[tokens // 2]) and torch.equal(scale[1, :, 100 - block], byte[tokens // 2])
        parts = rows[0, 0].view(heads, dim // 16, 16)
        assert (codes[shared].view(-1, heads, dim // 16, 16) == parts).all(-1).any(0).all()
        assert (byte[shared] == scale[0, :, 0]).any(0).all()
    want = pool_views(before, block, heads, dim)
    for a, b in zip(got, want):  # everything else as it was
        a, b = (t.contiguous().view(torch.uint8).clone() for t in (a, b))
        for t in (a, b):
            if t.dim() == 4:
                t[0, 0] = t[1, 100 - block] = 0
            else:
                t[0, :, 0] = t[1, :, 100 - block] = 0
        assert torch.equal(a, b)
