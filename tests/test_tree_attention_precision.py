"""Up to 16 rows of a kv head the softmax weights enter the second product in two bf16 parts (paged_decode: three):
decode over the quantised cache and small trees over both kinds, where the values of V cancel.

Tolerance: the output is rounded to bf16 once (2^-8 of it).  A weight's first part leaves less than 2^-7 of it, of
which the second part keeps all but 2^-8: 2^-15.  Scores of q.k are off by less than 2^-24 * 128 * |q||k| scale,
some 2^-13 here, which moves a weight by that much of itself.  Together 2^-12 sum p |v|; weights of a single bf16
would be off by up to 2^-8 sum p |v|.
"""

import math

import pytest
import torch

from oracle import operators_oracle as oracle
from tests.test_tree_attention import SCALE, Batch, decode


def close(got, want, spread):
    bound = want.abs() * 2.0 ** -8 + spread * 2.0 ** -12 + 1e-30
    off = ((got.cpu().double() - want).abs() / bound).nan_to_num(math.inf)
    assert off.max() <= 1, f"{off.max():.2f} of the bound at {(off == off.max()).nonzero()[0].tolist()}"


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(16, 8), (64, 8), (8, 8), (14, 2), (16, 1)])
def test_decode_weights_have_16_bits(cuda_device, hq, hkv):
    lens = [2, 3, 4, 5, 6, 7, 8, 40, 70, 300]
    x = Batch([n - 1 for n in lens], [1] * len(lens), hq, hkv, 64, True, seed=hq)
    close(decode(x), *oracle.tree_attention(x.q, *x.plain, x.cu, x.ctx, x.bt, SCALE))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("drafts,hq,hkv", [([1, 2, 5, 8, 3], 4, 2), ([4, 1, 2, 3], 8, 2), ([16, 7, 9], 3, 3), ([1, 1, 1], 16, 1)])
def test_tree_weights_have_16_bits(cuda_device, drafts, hq, hkv, quantised):
    x = Batch([3, 1, 0, 66, 200][:len(drafts)], drafts, hq, hkv, 64, quantised, seed=hq)
    close(x.run(), *oracle.tree_attention(x.q, *x.plain, x.cu, x.ctx, x.bt, SCALE, x.mask))


@pytest.mark.gpu
def test_an_infinity_with_an_exact_weight_stays_one(cuda_device):
    """A weight that one bf16 holds exactly leaves a second part too, or it would be 0 times infinity: equal scores,
    weights of exactly 1 on the way."""
    x = Batch([37, 2], [3, 1], 2, 1, 64, False)
    x.q.zero_()
    k, v, _, _ = x.dev
    page = int(x.bt[0, 0])
    v[page, 2, 0, 7], v[page, 33, 0, 7], v[page, 38, 0, 9] = math.inf, math.inf, -math.inf
    got = x.run(mask=torch.tensor([1, 2, 4, 1]))
    assert (got[:3, :, 7] == math.inf).all()
    assert (got[1, :, 9] == -math.inf).all() and got[[0, 2], :, 9].isfinite().all()
    assert got[3].isfinite().all()
