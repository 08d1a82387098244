"""Magnitudes at the ends of the cache's range: weights and running sums of every kernel of tree
attention and of the quantised decode, against the 64-bit oracle within the tolerance of
tests/test_tree_attention.py.

256 kv heads leave a range of tokens to few workgroups, so that each takes several steps in a row.
"""

import pytest
import torch

from oracle import operators_oracle as oracle
from tests.test_tree_attention import SCALE, Batch, close

HKV = 256
# contexts, drafts, Hq, Hkv, block: up to 16 rows of a kv head, 17 to 64, and more, which three kernels take
ROWS = {"few": ([600, 70], [3, 5], 256, HKV, 64), "some": ([600, 70], [20, 33], 256, HKV, 64),
        "many": ([600, 70], [40, 64], 512, HKV, 64)}
HEADS = [0, 1, HKV - 1]  # the kv heads that the oracle looks at


def slopes(rows, quantised, orders, value_exponent):
    """A batch whose scores rise by `orders` binary orders (or fall) with every 64 tokens, alike for every row, with V
    positive and around 2^value_exponent."""
    x = Batch(*ROWS[rows], quantised)
    x.q.zero_()
    x.q[:, :, 0] = abs(orders) / (SCALE * 1.4426950408889634)  # rounded to bf16: the oracle takes it as it is
    level = torch.zeros(x.plain[0].shape[:2])
    for b, n in enumerate(x.lens):
        for t in range(n):
            level[int(x.bt[b, t // 64]), t % 64] = t // 64 if orders > 0 else 11 - t // 64
    if quantised:
        k, v, ks, vs = x.dev
        k.view(torch.uint8)[..., 0] = level.to(torch.float8_e4m3fn).view(torch.uint8).cuda()[..., None]  # exact
        v.view(torch.uint8).bitwise_and_(127)
        ks.fill_(127)
        vs.fill_(124 + value_exponent)  # the codes are around 8
    else:
        k, v = x.plain
        k[..., 0] = level[..., None]
        v.abs_().mul_(2.0 ** value_exponent)
        x.dev = (k.cuda(), v.cuda(), None, None)
    return x


def check(x, got):
    k, v, ks, vs = x.dev
    plain = [oracle.dequantise(c.cpu(), s.cpu()) for c, s in ((k, ks), (v, vs))] if x.quantised else x.plain
    g = x.q.shape[1] // HKV
    heads = [h * g + i for h in HEADS for i in range(g)]
    close(got[:, heads], *oracle.tree_attention(x.q[:, heads], *(c[:, :, HEADS] for c in plain), x.cu, x.ctx, x.bt, SCALE))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("rows", ROWS)
def test_large_values_do_not_overflow_the_sums(cuda_device, rows, quantised):
    """Weights up to 1 sum up to 64 (1 + 1/8 + 1/64 ..) = 73 here, which times V of some 2^120 fits 32 bits.  A
    maximum that stays behind the scores makes the weights, and with them the sums, larger than that."""
    x = slopes(rows, quantised, 3, 120)
    got = x.run(mask=None)
    assert got.isfinite().all()
    check(x, got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_a_weight_of_zero_takes_no_part_whatever_its_scale(cuda_device, rows):
    """All tokens but the first 64 lie 200 binary orders and more below these and hold V of 2^121 at most, whose sums
    fit 32 bits; what they add, less than 700 * 2^-200 * 2^121, is nothing beside values around 2^-6."""
    x = slopes(rows, True, -200, -6)
    vs = x.dev[3]
    for b, n in enumerate(x.lens):
        for page in x.bt[b, 1:-(-n // 64)].tolist():
            vs[page] = 243
    check(x, x.run(mask=None))
