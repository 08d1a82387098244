"""The quantised cache: append and read back against the 64-bit oracle, and what is refused."""

import math

import numpy as np
import pytest
import torch

from kavor_amd import _lib
from kavor_amd.layers import attention
from oracle import operators_oracle as oracle
from tests.helpers import gen, randn_bf16, random_block_tables

FP8 = torch.float8_e4m3fn


def quantised_pool(num_blocks, block, heads, dim, g, spread=6):
    """One pool of bytes with K, V and their scales side by side in each page, as CPU views; finite values."""
    half, side = block * heads * dim, block * heads
    pool = torch.randint(0, 256, (num_blocks, 2 * (half + side)), generator=g, dtype=torch.uint8)
    values = pool[:, :2 * half]
    values[(values & 127) == 127] -= 1  # no NaN
    pool[:, 2 * half:] = torch.randint(116, 116 + spread, (num_blocks, 2 * side), generator=g, dtype=torch.uint8)
    return pool


def pool_views(pool, block, heads, dim):
    half, side, width = block * heads * dim, block * heads, pool.shape[1]
    f8 = pool.view(FP8)
    k, v = (f8.as_strided((pool.shape[0], block, heads, dim), (width, heads * dim, dim, 1), i * half) for i in (0, 1))
    ks, vs = (pool.as_strided((pool.shape[0], heads, block), (width, block, 1), 2 * half + i * side) for i in (0, 1))
    return k, v, ks, vs


def same_values(got: torch.Tensor, codes: np.ndarray):
    got = got.view(torch.uint8).cpu().numpy()
    nan = (codes & 127) == 127
    return np.array_equal(np.where(nan, 127, codes), np.where((got & 127) == 127, 127, got))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,dim,block,strided", [
    (1, 8, 128, 256, True), (1, 1, 64, 64, False), (7, 3, 128, 64, True), (33, 2, 256, 16, False),
    (300, 8, 128, 256, True), (1025, 5, 64, 48, True)])
def test_append_rounds_every_row_as_defined(cuda_device, tokens, heads, dim, block, strided):
    g = gen(tokens + heads)
    blocks = -(-tokens // block) + 3
    pool = quantised_pool(blocks, block, heads, dim, g)
    key = randn_bf16((tokens, heads, dim), g) * torch.exp2(torch.randint(-40, 40, (tokens, heads, 1), generator=g)).bfloat16()
    rows = randn_bf16((tokens, (heads + 2) * dim + 8), g)
    value = rows[:, 8:8 + heads * dim].view(tokens, heads, dim) if strided else randn_bf16((tokens, heads, dim), g)
    # rows at the edges: nothing, one value, infinities and NaN, the smallest and the largest magnitudes
    key[0, 0] = 0.0
    value[0, 0, 1:] = 0.0
    if tokens > 6:
        key[1, 0, 3], key[1, 0, 5], key[1, 1, 2] = math.inf, -math.inf, math.nan
        value[2] = math.inf
        key[3] *= 1e-38
        key[4, 0] = torch.finfo(torch.bfloat16).max
        value[5, 0, :4] = torch.tensor([448.0, 449.0, 1.0, -0.0])
        value[6, 0] = 2.0 ** -133
    slots = torch.randperm(blocks * block, generator=g)[:tokens].to(torch.int32)
    if tokens > 6:
        slots[[0, tokens - 1]] = torch.tensor([-1, blocks * block], dtype=torch.int32)
    want = pool.clone()
    wk, wv, wks, wvs = pool_views(want, block, heads, dim)
    for x, c, s in ((key, wk, wks), (value, wv, wvs)):
        codes, byte = oracle.quantise_rows(x)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < blocks * block:
                c.view(torch.uint8)[slot // block, slot % block] = torch.from_numpy(codes[t])
                s[slot // block, :, slot % block] = torch.from_numpy(byte[t])
    dev = pool.to(cuda_device)
    dk, dv, dks, dvs = pool_views(dev, block, heads, dim)
    dkey, dvalue = key.to(cuda_device), rows.to(cuda_device)[:, 8:8 + heads * dim].view(tokens, heads, dim) if strided \
        else value.to(cuda_device)
    if strided:
        dvalue.copy_(value)
    attention.store_kvcache_fp8(dkey, dvalue, dk, dv, dks, dvs, slots.to(cuda_device))
    torch.cuda.synchronize()
    side = 2 * block * heads
    assert torch.equal(dev.cpu()[:, -side:], want[:, -side:])  # scales, untouched ones too
    assert same_values(dev[:, :-side].contiguous(), want[:, :-side].numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,dim,block", [
    ([1], 8, 128, 256), ([0, 5, 0, 0, 64, 1, 0], 3, 128, 64), ([300, 40, 700], 8, 128, 256), ([129, 31], 2, 64, 48),
    ([17] * 300, 1, 256, 16)])
def test_load_gives_the_exact_values(cuda_device, lens, heads, dim, block):
    g = gen(len(lens))
    blocks = sum(-(-n // block) for n in lens) + 2
    pool = quantised_pool(blocks, block, heads, dim, g, spread=100)
    bt = random_block_tables(lens, block, blocks, g)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    views = pool_views(pool, block, heads, dim)
    dviews = pool_views(pool.to(cuda_device), block, heads, dim)
    total = sum(lens)
    out = tuple(torch.full((total + 5, heads, dim), 7.0, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    attention.load_kvcache_fp8(*dviews, bt.to(cuda_device), cu.to(cuda_device), total, out=out)
    fresh = attention.load_kvcache_fp8(*dviews, bt.to(cuda_device), cu.to(cuda_device), total)
    for got, again, cache, scale in zip(out, fresh, views[:2], views[2:]):
        plain = oracle.dequantise(cache, scale)
        want = torch.cat([oracle.gather(plain, t, n) for t, n in zip(bt, lens)])
        assert torch.equal(got[:total].cpu().double(), want)
        assert torch.equal(again, got[:total])
        assert (got[total:] == 7).all()  # rows behind the last sequence


@pytest.mark.gpu
def test_load_marks_tokens_without_a_page(cuda_device):
    g = gen(5)
    pool = quantised_pool(4, 64, 2, 128, g)
    views = pool_views(pool.to(cuda_device), 64, 2, 128)
    bt = torch.tensor([[1, 9], [-1, 2]], dtype=torch.int32, device=cuda_device)
    cu = torch.tensor([0, 200, 328], dtype=torch.int32, device=cuda_device)
    k, v = attention.load_kvcache_fp8(*views, bt, cu, 328)
    bad = torch.zeros(328, dtype=torch.bool)
    bad[64:264] = True  # page 9 and what lies behind the table; page -1
    for x in (k, v):
        assert torch.equal(x.isnan().flatten(1).all(1).cpu(), bad)
        assert torch.equal(x.isnan().flatten(1).any(1).cpu(), bad)


@pytest.mark.gpu
def test_append_then_load_is_within_half_a_step(cuda_device):
    """|x - load(store(x))| <= 2^-4 |x| for values within 2^14 of the row's largest."""
    g = gen(9)
    T, H, D, block = 200, 4, 128, 64
    key, value = randn_bf16((T, H, D), g), randn_bf16((T, H, D), g, 1e-3)
    views = pool_views(quantised_pool(6, block, H, D, g).to(cuda_device), block, H, D)
    bt = torch.tensor([[3, 0, 5, 1]], dtype=torch.int32)
    slots = torch.tensor([int(bt[0, t // block]) * block + t % block for t in range(T)], dtype=torch.int32)
    attention.store_kvcache_fp8(key.to(cuda_device), value.to(cuda_device), *views, slots.to(cuda_device))
    cu = torch.tensor([0, T], dtype=torch.int32, device=cuda_device)
    back = attention.load_kvcache_fp8(*views, bt.to(cuda_device), cu, T)
    for x, y in zip((key, value), back):
        x, y = x.double(), y.cpu().double()
        top = x.abs().amax(-1, keepdim=True)
        assert ((x - y).abs() <= 2.0 ** -4 * x.abs() + top * 2.0 ** -18).all()


def _append(**over):
    a = dict(key=16, kts=1024, khs=128, value=16, vts=4096, vhs=128, kc=16, vc=16, bstr=1 << 18, sstr=1024, hstr=128,
             ks=16, vs=16, sbs=2048, shs=256, nslots=1 << 12, slots=16, n=4, hkv=8, d=128, bs=256, stream=None)
    a.update(over)
    return _lib.lib().kvp_append_fp8(*a.values())


def _load(**over):
    a = dict(kc=16, vc=16, bstr=1 << 18, sstr=1024, hstr=128, ks=16, vs=16, sbs=2048, shs=256, nblk=16, bt=16, bts=4,
             maxb=4, cu=16, b=2, total=100, hkv=8, d=128, bs=256, k=16, kts=1024, khs=128, v=16, vts=1024, vhs=128,
             stream=None)
    a.update(over)
    return _lib.lib().kvp_load_fp8(*a.values())


def test_bad_arguments_are_refused_on_the_host():
    E, U = _lib.KVP_EINVAL, _lib.KVP_EUNSUPPORTED
    assert _append(n=0) == _lib.KVP_OK
    assert _load(b=0) == _lib.KVP_OK and _load(total=0) == _lib.KVP_OK
    for call in (_append, _load):
        assert call(d=96) == U
        assert b"head_dim=96" in _lib.lib().kvp_last_error()
        for over in (dict(kc=8), dict(vc=0), dict(ks=0), dict(vs=0), dict(sstr=1000), dict(bstr=8), dict(hstr=120),
                     dict(hkv=0), dict(bs=0), dict(sbs=-1), dict(kts=1020)):
            assert call(**over) == E, over
    for over in (dict(n=-1), dict(key=0), dict(value=8), dict(slots=0), dict(slots=2), dict(nslots=-1)):
        assert _append(**over) == E, over
    for over in (dict(b=-1), dict(total=-1), dict(nblk=0), dict(maxb=0), dict(bts=3), dict(cu=0), dict(k=0), dict(v=4),
                 dict(bt=2)):
        assert _load(**over) == E, over


def test_wrappers_refuse_what_does_not_fit():
    pool = quantised_pool(2, 64, 2, 128, gen(0))
    views = pool_views(pool, 64, 2, 128)
    x, slots = torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        attention.store_kvcache_fp8(x, x, *views, slots)
    with pytest.raises(ValueError, match="CUDA"):
        attention.load_kvcache_fp8(*views, slots.view(1, 3), slots, 3)


@pytest.mark.gpu
def test_wrappers_check_types_shapes_and_devices(cuda_device):
    pool = quantised_pool(2, 64, 2, 128, gen(0)).to(cuda_device)
    k, v, ks, vs = pool_views(pool, 64, 2, 128)
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=cuda_device)
    slots = torch.full((3,), -1, dtype=torch.int32, device=cuda_device)
    attention.store_kvcache_fp8(x, x, k, v, ks, vs, slots)
    for bad in ((x.float(), x, k, v, ks, vs, slots), (x, x[:2], k, v, ks, vs, slots),
                (x, x, k.view(torch.uint8), v, ks, vs, slots), (x, x, k, v, ks.transpose(1, 2), vs, slots),
                (x, x, k, v, ks, vs[:1], slots), (x, x, k[:1], v, ks, vs, slots), (x, x.cpu(), k, v, ks, vs, slots),
                (x, x, k, v, ks, vs, slots.long()), (x, x, k, v, ks, vs, slots[:2]), (x, x, k, v, ks, vs, slots.cpu()),
                (x[:, :1], x[:, :1], k, v, ks, vs, slots)):
        with pytest.raises(ValueError):
            attention.store_kvcache_fp8(*bad)
    bt, cu = torch.zeros(1, 2, dtype=torch.int32, device=cuda_device), torch.tensor([0, 9], dtype=torch.int32,
                                                                                    device=cuda_device)
    for bad in ((k, v, ks, vs, bt.long(), cu, 9), (k, v, ks, vs, bt, cu.long(), 9), (k, v, ks, vs, bt[:0], cu, 9),
                (k, v, ks, vs, bt, cu, -1), (k, v, ks, vs, bt.cpu(), cu, 9)):
        with pytest.raises(ValueError):
            attention.load_kvcache_fp8(*bad)
    with pytest.raises(ValueError):
        attention.load_kvcache_fp8(k, v, ks, vs, bt, cu, 9, out=(x, x))
