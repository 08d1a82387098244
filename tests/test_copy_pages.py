"""Whole pages copied as if all were read before any is written: every byte against indexing on the CPU."""

import random

import pytest
import torch

from kavor_amd import _lib
from kavor_amd.engine.cache_pool import CachePool
from kavor_amd.layers import attention
from tests.helpers import gen


def pool_of(layers, pages, size, seed=0):
    return torch.randint(0, 256, (layers, pages, size), generator=gen(seed), dtype=torch.uint8)


def check(pool, src, dst):
    want, got = pool.clone(), pool.cuda()
    want[:, dst] = pool[:, src]
    attention.copy_pages(got, src, dst)
    assert torch.equal(got.cpu(), want)


def cycle(ids):
    """Every page to the place of the next one."""
    return ids, ids[1:] + ids[:1]


@pytest.mark.gpu
@pytest.mark.parametrize("layers,pages,size", [(1, 2, 16), (1, 40, 4112), (3, 40, 64), (28, 40, 2 * 64 * 129), (2, 40, 65536)])
def test_pages_that_stay_apart(cuda_device, layers, pages, size):
    pool = pool_of(layers, pages, size)
    check(pool, [0], [1])
    check(pool, [], [])
    if pages > 2:
        check(pool, [5, 5, 5, 9, 9], [0, 1, 39, 20, 21])      # forks
        check(pool, list(range(20)), list(range(39, 19, -1)))
        check(pool, [7, 3, 7], [7, 3, 8])                    # to themselves


@pytest.mark.gpu
@pytest.mark.parametrize("size", [16, 4112, 66048])
def test_pages_that_change_places(cuda_device, size):
    pool = pool_of(2, 30, size, 1)
    check(pool, [1, 2], [2, 1])
    check(pool, list(range(29)), list(range(1, 30)))           # one long shift
    check(pool, list(range(1, 30)), list(range(29)))
    for n in (3, 7, 8, 9, 10, 30):
        check(pool, *cycle(random.Random(n).sample(range(30), n)))
    a, b = cycle([3, 4, 5]), cycle([10, 11])
    check(pool, a[0] + b[0] + [4, 10, 20, 0], a[1] + b[1] + [20, 21, 22, 23])  # with branches out of the cycles


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(30))
def test_any_pairs(cuda_device, seed):
    rng = random.Random(seed)
    pages = rng.choice([5, 40, 1000])
    pool = pool_of(rng.choice([1, 3]), pages, rng.choice([16, 272, 4096]), seed)
    n = rng.randint(1, pages)
    dst = rng.sample(range(pages), n)
    src = [rng.randrange(pages) for _ in dst] if seed % 3 else rng.sample(range(pages), n)
    check(pool, src, dst)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [193, 194, 200, 384, 385, 386, 400, 767, 1500])
def test_cycles_and_shifts_longer_than_a_launch(cuda_device, n):
    pool = pool_of(2, n + 5, 32, n)
    ids = random.Random(n).sample(range(n + 5), n)
    check(pool, *cycle(ids))
    check(pool, ids[:-1], ids[1:])
    check(pool, [ids[0]] * (n - 1), ids[1:])                   # one page to all


@pytest.mark.gpu
def test_types_and_layouts(cuda_device):
    whole = torch.randint(-1000, 1000, (4, 12, 80), generator=gen(3), dtype=torch.int16)
    for view in (lambda t: t, lambda t: t.transpose(0, 1), lambda t: t[:, :, :64], lambda t: t[::2, ::3], lambda t: t[1:, 2:, 8:]):
        want, got = whole.clone(), whole.cuda()
        w, pages = view(want), view(got)
        src, dst = [0, 1, 2], [2, 0, 3]
        w[:, dst] = w[:, src].clone()
        attention.copy_pages(pages, src, dst)
        assert torch.equal(got.cpu(), want)
    for dtype in (torch.bfloat16, torch.float32, torch.float8_e4m3fn):
        got = whole.cuda().view(torch.uint8).view(4, 12, 160).view(dtype)
        attention.copy_pages(got, [3, 4], [4, 3])
        assert torch.equal(got.view(torch.uint8)[:, [3, 4]].cpu(), whole.view(torch.uint8)[:, [4, 3]])


@pytest.mark.gpu
def test_pages_far_apart(cuda_device):
    step = (5 << 30) + 16
    room = torch.empty(2 * step + 4096, dtype=torch.uint8, device="cuda")
    pages = room.as_strided((2, 2, 4096), (2 * 4096, step, 1))
    want = pool_of(2, 2, 4096, 9)
    pages.copy_(want)
    attention.copy_pages(pages, [0, 1], [1, 0])
    assert torch.equal(pages.cpu(), want.flip(1))


@pytest.mark.gpu
def test_streams_and_a_captured_copy(cuda_device):
    pool = pool_of(3, 20, 8192, 4)
    got, side = pool.cuda(), torch.cuda.Stream()
    src, dst = cycle(list(range(12)))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        attention.copy_pages(got, src, dst)
    side.synchronize()
    want = pool.clone()
    want[:, dst] = pool[:, src]
    assert torch.equal(got.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.copy_pages(got, src, dst)
    for _ in range(3):
        graph.replay()
        want[:, dst] = want[:, src].clone()
        torch.cuda.synchronize()
        assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
def test_the_page_pool_copies_as_indexing_does(cuda_device):
    """Negative ids count from the end; of two pairs for one page the last one counts."""
    pool = CachePool.__new__(CachePool)
    pool.num_kv_heads, pool.head_dim, pool.block_size, pool.dtype = 2, 128, 64, torch.bfloat16
    host = pool_of(2, 9, pool.page_bytes, 5)
    for src, dst in (([3], [4]), ([0, 1, -1], [1, 0, 3]), ([1, 2], [5, 5]), ([2, 3], [-4, 5])):
        pool.pools = host.cuda()
        pool.copy_blocks(src, dst)
        want = host.clone()
        for s, d in zip(src, dst):
            want[:, d] = host[:, s]
        assert torch.equal(pool.pools.cpu(), want)
    with pytest.raises(_lib.KVPathError, match="pair 0"):
        pool.copy_blocks([9], [0])


def test_refusals_on_the_host():
    import ctypes

    lib = _lib.lib()

    def call(src=(0,), dst=(1,), **over):
        ids = [(ctypes.c_int32 * max(1, len(x)))(*x) for x in (src, dst)]
        args = dict(pages=16, ls=1 << 20, ps=4096, layers=2, pages_n=8, size=4096, s=ctypes.addressof(ids[0]),
                    d=ctypes.addressof(ids[1]), n=len(src), stream=None)
        return lib.kvp_copy_pages(*dict(args, **over).values())

    assert call((), ()) == _lib.KVP_OK
    assert call((2, 3), (2, 3)) == _lib.KVP_OK                 # nothing to do
    assert call(layers=0) == _lib.KVP_OK and call(size=0) == _lib.KVP_OK
    for bad in (dict(n=-1), dict(layers=-1), dict(pages_n=-1), dict(size=-16), dict(pages=None), dict(pages=8), dict(s=None),
                dict(d=None), dict(ls=(1 << 20) + 8), dict(ps=4104), dict(size=4088), dict(ps=4080), dict(ls=4096),
                dict(ls=0), dict(pages_n=1)):
        assert call(**bad) == _lib.KVP_EINVAL, bad
    for src, dst in (((8,), (0,)), ((0,), (8,)), ((-1,), (0,)), ((0,), (-1,)), ((0, 1), (5, 5)), ((5, 1), (5, 5))):
        assert call(src, dst) == _lib.KVP_EINVAL, (src, dst)
    assert b"written twice" in lib.kvp_last_error()
    assert call(layers=65536) == _lib.KVP_EUNSUPPORTED and call(size=1 << 34, ps=1 << 34) == _lib.KVP_EUNSUPPORTED


def test_refusals_of_the_python_layer():
    with pytest.raises(ValueError, match="CUDA"):
        attention.copy_pages(torch.zeros(1, 2, 16), [0], [1])


@pytest.mark.gpu
def test_refusals_of_wrong_arguments(cuda_device):
    pool = torch.zeros(2, 4, 64, dtype=torch.uint8, device="cuda")
    for pages, src, dst in ((pool[0], [0], [1]), (pool.transpose(1, 2), [0], [1]), (pool, [0, 1], [1]), (pool, [0.5], [1]),
                            (pool, [1 << 40], [1]), (pool, ["0"], [1])):
        with pytest.raises(ValueError):
            attention.copy_pages(pages, src, dst)
    for pages, src, dst in ((pool, [0], [4]), (pool, [0, 1], [2, 2]), (pool[:, :, :40], [0], [1]), (pool[:1].expand(3, -1, -1), [0], [1])):
        with pytest.raises(_lib.KVPathError):
            attention.copy_pages(pages, src, dst)


def test_page_ids_that_are_no_list():
    """Bytes are not page ids: four of them were taken as one id, and their count as four."""
    assert list(attention._page_ids([3, 1], (4, 5))) == [3, 1, 4, 5]
    for ids in (b"\0\0\0\0", bytearray(4), "0", None, [0.5], [1 << 40], ["0"], 7):
        for src, dst in ((ids, [1]), ([1], ids), (ids, ids)):
            with pytest.raises(ValueError):
                attention._page_ids(src, dst)
    with pytest.raises(ValueError, match="length"):
        attention._page_ids([0, 1], [1])
