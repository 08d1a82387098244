"""Softmax scales of zero and below, in every kernel of tree attention and of the quantised decode,
against the 64-bit oracle within the tolerance of tests/test_tree_attention.py."""

import pytest

from kavor_amd.layers import attention
from oracle import operators_oracle as oracle
from tests.test_tree_attention import SCALE, Batch, close

# contexts, drafts, Hq, Hkv, block: up to 16 rows of a kv head, 17 to 64, and more, which three kernels take
ROWS = {"few": ([70, 3, 200], [3, 5, 1], 6, 2, 64), "some": ([70, 3, 200], [9, 5, 20], 6, 2, 64),
        "many": ([70, 3, 200], [40, 5, 64], 6, 2, 64)}


def run(x, scale, mask):
    k, v, ks, vs = x.dev
    return attention.tree_attention(x.q.cuda(), k, v, x.cu.cuda(), max(x.drafts), x.ctx.cuda(), x.bt.cuda(), scale,
                                    tree_mask=None if mask is None else mask.cuda(), k_scale=ks, v_scale=vs)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-42, 1e-60, -1e-60, -SCALE])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("rows", ROWS)
def test_scales_of_zero_and_below(cuda_device, rows, quantised, scale):
    """At 0 (and what 32 bits round to it) every token that a row sees has the same weight, and hidden ones none;
    below 0 the farthest key has the largest."""
    x = Batch(*ROWS[rows], quantised)
    for mask in (x.mask, None):
        close(run(x, scale, mask), *oracle.tree_attention(x.q, *x.plain, x.cu, x.ctx, x.bt, scale, mask))
    mask = x.mask.clone()
    mask[:2] = 0  # the context alone
    close(run(x, scale, mask), *oracle.tree_attention(x.q, *x.plain, x.cu, x.ctx, x.bt, scale, mask))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1e-60, -SCALE])
def test_decode_at_scales_of_zero_and_below(cuda_device, scale):
    lens = [1, 63, 64, 65, 200]
    x = Batch([n - 1 for n in lens], [1] * len(lens), 16, 8, 64, True)
    k, v, ks, vs = x.dev
    got = attention.paged_decode_fp8(x.q.cuda(), k, v, ks, vs, x.ctx.cuda(), x.bt.cuda(), scale)
    close(got, *oracle.tree_attention(x.q, *x.plain, x.cu, x.ctx, x.bt, scale))
