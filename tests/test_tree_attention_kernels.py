"""What tests/test_tree_attention.py asks of one kernel, asked of all three (up to 16 rows of a kv head, 17 to 64,
and more) and both cache kinds: hidden values, and maxima far apart."""

import math
import random

import pytest
import torch

from kavor_amd.layers import attention
from tests.test_tree_attention import SCALE, Batch, signed
from tests.test_tree_attention_reach import HKV, ROWS, check
from tests.helpers import bits_equal

HIDDEN = {  # contexts, drafts, Hq, Hkv, block: drafts on both sides of a step's end
    "few": ([55, 3, 118], [16, 2, 9], 2, 2, 64), "few, 2 heads": ([59, 30], [8, 5], 4, 2, 64),
    "some": ([55, 3, 90], [40, 2, 33], 2, 2, 64), "some, 3 heads": ([61, 100], [20, 9], 6, 2, 64),
    "many": ([55, 3, 20], [50, 2, 64], 4, 2, 64), "many, 16 heads": ([60, 7], [12, 9], 32, 2, 64)}


def hidden_batches(case, what, quantised, seed):
    """A batch with `what` in K and V of some drafts, and in all that lies behind the last tokens, the same one with
    zeros there, masks, and [T, Hkv] of the rows that see a bad draft."""
    x, clean = (Batch(*case, quantised, seed=seed) for _ in range(2))
    rng, hkv = random.Random(seed), case[3]
    mask = torch.tensor([signed(rng.getrandbits(64)) for _ in x.mask])
    hit = torch.zeros(len(mask), hkv, dtype=torch.bool)

    def put(batch, part, page, slot, head, dim, value):
        c = batch.dev[part]
        if quantised:  # e4m3 has NaN alone
            c.view(torch.uint8)[page, slot, head, dim] = 127 if value else 0
        else:
            c[page, slot, head, dim] = value

    for b, n in enumerate(x.lens):
        ctx, q0 = n - x.drafts[b], int(x.cu[b])
        for j in rng.sample(range(x.drafts[b]), (x.drafts[b] + 1) // 2):
            t, head, part = ctx + j, rng.randrange(hkv), rng.randrange(2)
            where = (part, int(x.bt[b, t // 64]), t % 64, head, rng.randrange(128))
            put(x, *where, what)
            put(clean, *where, 0.0)
            for i in range(x.drafts[b]):
                hit[q0 + i, head] |= bool(int(mask[q0 + i]) >> j & 1)
        page, end = int(x.bt[b, (n - 1) // 64]), (n - 1) % 64 + 1
        for part in (0, 1):
            put(x, part, page, slice(end, 64), slice(None), slice(None), what)
            put(clean, part, page, slice(end, 64), slice(None), slice(None), 0.0)
            if quantised:
                x.dev[2 + part][page, :, end:] = 255
                clean.dev[2 + part][page, :, end:] = 127
    return x, clean, mask, hit


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("what", [math.inf, math.nan])
@pytest.mark.parametrize("case", HIDDEN)
def test_what_hidden_tokens_hold_reaches_no_row(cuda_device, case, what, quantised):
    for seed in range(4):
        x, clean, mask, hit = hidden_batches(HIDDEN[case], what, quantised, seed)
        got, want = x.run(mask=mask).cpu(), clean.run(mask=mask).cpu()
        rows = hit.repeat_interleave(got.shape[1] // hit.shape[1], 1)
        assert bits_equal(got[~rows], want[~rows])
        assert got[~rows].isfinite().all()
        if math.isnan(what) or quantised:  # an infinity in K may also be a weight of 0
            assert (~got[rows].isfinite()).any(-1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("unit", [1.25, 40.0])
@pytest.mark.parametrize("rows", ROWS)
def test_maxima_that_lie_apart(cuda_device, rows, unit, quantised):
    """The scores of each 32 tokens lie 0 to 16 units of binary orders up, in no order, and down for every other
    query: the maximum is taken again within a workgroup's steps, and those that are joined lie far apart."""
    x = Batch(*ROWS[rows], quantised, seed=3)
    rng = random.Random(8)
    x.q.mul_(0.25)
    x.q[::2, :, 0] = unit / (SCALE * 1.4426950408889634)
    x.q[1::2, :, 0] = -unit / (SCALE * 1.4426950408889634)
    level = torch.zeros(x.plain[0].shape[:2])
    for b, n in enumerate(x.lens):
        levels = [rng.randint(0, 16) for _ in range(n // 32 + 1)]
        for t in range(n):
            level[int(x.bt[b, t // 64]), t % 64] = levels[t // 32]
    if quantised:
        k, _, ks, _ = x.dev
        k.view(torch.uint8)[..., 0] = level.to(torch.float8_e4m3fn).view(torch.uint8).cuda()[..., None]  # exact
        ks.fill_(127)
    else:
        x.plain[0][..., 0] = level[..., None]
        x.dev = (x.plain[0].cuda(), x.dev[1], None, None)
    assert x.plain[0].shape[2] == HKV
    check(x, x.run(mask=None))


@pytest.mark.gpu
def test_nan_rows_beyond_32_bit_counts(cuda_device):
    """One sequence of 40000 rows of 4096 heads, where two were said: 2^31.3 chunks of 16 bytes become NaN (all in the
    place of one row, whose stride is 0)."""
    T, hq = 40_000, 4096
    k, v = (torch.zeros(1, 64, 256, 128, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    out = torch.zeros(1, hq, 128, dtype=torch.bfloat16, device=cuda_device)
    cu, ctx = (torch.tensor(t, dtype=torch.int32, device=cuda_device) for t in ([0, T], [64]))
    attention.tree_attention(out.expand(T, -1, -1), k, v, cu, 2, ctx, torch.zeros(1, 1, dtype=torch.int32, device=cuda_device),
                             SCALE, out=out.expand(T, -1, -1))
    assert out.isnan().all()
