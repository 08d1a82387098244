"""Drafts that stay, moved next to their context: the same bytes as the oracle's moves, and nothing else touched."""

import random

import pytest
import torch

from kavor_amd import _lib
from kavor_amd.layers import attention
from oracle import drafts_oracle as oracle
from tests.helpers import gen

FP8 = torch.float8_e4m3fn


def pool_of(layers, pages, block, heads, dim, quantised, g):
    """Bytes [layers, pages, page] with K, V and their scales side by side, on the CPU; whole 16 bytes a page."""
    size = 2 * block * heads * (dim + 1 if quantised else 2 * dim)
    return torch.randint(0, 256, (layers, pages, -(-size // 16) * 16), generator=g, dtype=torch.uint8)


def views(pool, block, heads, dim, quantised):
    """(k, v, k_scale, v_scale) of a pool: five-dimensional views."""
    L, pages, size = pool.shape
    half = block * heads * dim
    flat = pool.view(FP8 if quantised else torch.bfloat16)
    page = size if quantised else size // 2
    k, v = (flat.as_strided((L, pages, block, heads, dim), (pages * page, page, heads * dim, dim, 1), i * half) for i in (0, 1))
    if not quantised:
        return k, v, None, None
    ks, vs = (pool.as_strided((L, pages, heads, block), (pages * size, size, block, 1), 2 * half + i * block * heads)
              for i in (0, 1))
    return k, v, ks, vs


def integers(t):
    return t.view(torch.uint8) if t.dtype == FP8 else t.view(torch.int16)


def oracle_caches(k, v, ks, vs):
    """What the oracle moves: everything with a token dimension after the pages."""
    got = [integers(k), integers(v)]
    return got if ks is None else got + [ks.transpose(2, 3), vs.transpose(2, 3)]


class Step:
    def __init__(self, lens, rows, block, pages, g, rng, kept=None, width=None):
        """Sequences of `lens` cached tokens whose last `rows` are drafts (and the row before them)."""
        need = [-(-n // block) for n in lens]
        ids = torch.randperm(pages, generator=g)
        self.bt = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.bt[b, :n] = ids[at:at + n].int()
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
        width = max(rows + [1]) if width is None else width
        self.path = torch.full((len(lens), width), -1, dtype=torch.int32)
        self.accepted = torch.zeros(len(lens), dtype=torch.int32)
        for b, n in enumerate(rows):
            k = rng.randint(0, max(0, n - 1)) if kept is None else min(kept, max(0, n - 1))
            self.accepted[b] = k
            self.path[b, :k] = torch.tensor(sorted(rng.sample(range(1, n), k)) if k else [], dtype=torch.int32)

    def args(self, device="cpu"):
        return [t.to(device) for t in (self.path, self.accepted, self.cu, self.lens, self.bt)]


def check(pool, step, block, heads, dim, quantised):
    want, got = pool.clone(), pool.cuda()
    lens = oracle.keep_drafts(oracle_caches(*views(want, block, heads, dim, quantised)), *step.args())
    k, v, ks, vs = views(got, block, heads, dim, quantised)
    new = attention.keep_drafts(k, v, *step.args("cuda"), k_scale=ks, v_scale=vs)
    assert new.dtype == torch.int32 and torch.equal(new.cpu(), lens)
    assert torch.equal(got.cpu(), want)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("layers,heads,dim,block", [(1, 1, 64, 16), (3, 2, 128, 64), (2, 8, 128, 256), (5, 3, 256, 7), (28, 1, 64, 64)])
@pytest.mark.parametrize("lens,rows", [
    ([1], [1]), ([5], [5]), ([70, 3, 200], [2, 3, 12]), ([64, 65, 128, 1], [9, 9, 64, 1]), ([130] * 6, [64, 1, 33, 17, 8, 25])])
def test_rows_go_where_the_oracle_puts_them(cuda_device, quantised, layers, heads, dim, block, lens, rows):
    g, rng = gen(sum(lens) + block), random.Random(sum(rows))
    pages = sum(-(-n // block) for n in lens) + 2
    pool = pool_of(layers, pages, block, heads, dim, quantised, g)
    check(pool, Step(lens, rows, block, pages, g, rng), block, heads, dim, quantised)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("seqs,kept", [(300, None), (90, 3)])
def test_many_sequences(cuda_device, quantised, seqs, kept):
    g, rng = gen(seqs), random.Random(seqs)
    rows = [rng.randint(0, 12) for _ in range(seqs)]
    lens = [rng.randint(max(n, 1), 130) for n in rows]
    pool = pool_of(4, seqs * 3 + 1, 64, 2, 128, quantised, g)
    check(pool, Step(lens, rows, 64, seqs * 3 + 1, g, rng, kept), 64, 2, 128, quantised)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_paths_and_sequences_that_are_wrong(cuda_device, quantised):
    """Each ends its own moves, or is left alone; no byte elsewhere changes."""
    g, rng = gen(1), random.Random(1)
    step = Step([100] * 14, [10] * 14, 64, 40, g, rng, kept=4)
    step.path[:, :4] = torch.tensor([2, 4, 7, 9], dtype=torch.int32)
    step.path[0, 2] = 4                       # does not rise
    step.path[1, 1] = 10                      # behind the rows
    step.path[2, 0] = 0                       # row 0 stays where it is
    step.path[3, 3] = -5
    step.path[4, 1] = 2 ** 31 - 1
    step.accepted[5] = 10                     # as many as rows
    step.accepted[6] = -1
    step.accepted[7] = 2 ** 31 - 1
    step.lens[8] = 9                          # fewer tokens than rows
    step.lens[9] = 0
    step.lens[10] = 2 ** 31 - 1               # beyond the table
    step.bt[11, 1] = 40                       # no such page
    step.bt[12, 1] = -1
    step.lens[13] = 70                        # rows on both sides of a page's end
    pool = pool_of(2, 40, 64, 1, 128, quantised, g)
    check(pool, step, 64, 1, 128, quantised)
    step.cu[5:] += 3                          # a sequence of 13 rows; one of 7 that has 9 tokens
    step.cu[9:] -= 6
    check(pool, step, 64, 1, 128, quantised)


@pytest.mark.gpu
def test_a_path_wider_than_needed_and_one_that_is_too_narrow(cuda_device):
    g, rng = gen(3), random.Random(3)
    pool = pool_of(2, 12, 64, 2, 128, False, g)
    check(pool, Step([90, 80], [6, 9], 64, 12, g, rng, kept=5, width=64), 64, 2, 128, False)
    step = Step([90, 80], [6, 9], 64, 12, g, rng, kept=3, width=9)
    step.path = step.path[:, :2].contiguous()
    assert torch.equal(check(pool, step, 64, 2, 128, False), pool)  # three kept, two entries: left alone
    step.accepted[:] = 0
    step.path = step.path[:, :0].contiguous()
    check(pool, step, 64, 2, 128, False)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True])
def test_layouts(cuda_device, quantised):
    """One layer without its dimension; heads before tokens; layers inside the page; padded path rows."""
    g, rng = gen(5), random.Random(5)
    block, heads, dim, pages = 64, 3, 128, 9
    step = Step([70, 120, 9], [9, 12, 4], block, pages, g, rng)
    pool = pool_of(1, pages, block, heads, dim, quantised, g)
    want, got = pool.clone(), pool.cuda()
    oracle.keep_drafts(oracle_caches(*views(want, block, heads, dim, quantised)), *step.args())
    k, v, ks, vs = (t if t is None else t[0] for t in views(got, block, heads, dim, quantised))
    args = step.args("cuda")
    wide = torch.full((3, 30), 5, dtype=torch.int32, device="cuda")
    wide[:, :args[0].shape[1]] = args[0]
    attention.keep_drafts(k, v, wide[:, :args[0].shape[1]], *args[1:], k_scale=ks, v_scale=vs)
    assert torch.equal(got.cpu(), want)

    def scattered(order, sizes):  # a tensor [layers, pages, block, heads, ...] laid out in another order
        t = torch.randint(0, 100, [sizes[i] for i in order], generator=g, dtype=torch.uint8)
        return t.permute([order.index(i) for i in range(len(order))])
    for order in ((0, 1, 3, 2, 4), (1, 0, 2, 3, 4), (3, 1, 0, 2, 4)):
        sizes = (4, pages, block, heads, dim * (1 if quantised else 2))
        kb, vb = (scattered(order, sizes) for _ in range(2))
        scales = [scattered((1, 0, 2, 3), (4, pages, heads, block)) for _ in range(2)] if quantised else [None, None]
        dtype = FP8 if quantised else torch.bfloat16
        dev = [t if t is None else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda").copy_(t)
               for t in (kb, vb, *scales)]
        new = attention.keep_drafts(dev[0].view(dtype), dev[1].view(dtype), *args, k_scale=dev[2], v_scale=dev[3])
        host = [kb, vb] + ([s.transpose(2, 3) for s in scales] if quantised else [])
        assert torch.equal(new.cpu(), oracle.keep_drafts(host, *step.args()))
        assert all(torch.equal(d.cpu(), t) for d, t in zip(dev, (kb, vb, *scales)) if t is not None)


@pytest.mark.gpu
def test_pages_far_apart(cuda_device):
    """Pages and layers more than 2^32 bytes from the first one."""
    g, rng = gen(6), random.Random(6)
    step = Step([100], [20], 64, 2, g, rng, kept=9)
    shape, row = (2, 2, 64, 1, 128), 64 * 128
    near = torch.randint(0, 1000, shape, generator=g, dtype=torch.int16)
    strides = (4 * row, (5 << 28) + 64, 128, 128, 1)
    room = [torch.empty(4 * row + (5 << 28) + 64 + row, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    far = [r.as_strided(shape, strides) for r in room]
    for t in far:
        t.view(torch.int16).copy_(near)
    attention.keep_drafts(*far, *step.args("cuda"))
    want = near.clone()
    oracle.keep_drafts([want], *step.args())
    assert all(torch.equal(t.view(torch.int16).cpu(), want) for t in far)


@pytest.mark.gpu
def test_replayed_with_other_paths(cuda_device):
    g, rng = gen(7), random.Random(7)
    steps = [Step([90, 64, 30], [12, 9, 3], 64, 8, g, rng, width=12) for _ in range(3)]
    for s in steps:
        s.bt = steps[0].bt
    pool = pool_of(3, 8, 64, 2, 128, True, g)
    got, want = pool.cuda(), pool.clone()
    args = steps[0].args("cuda")
    caches = views(got, 64, 2, 128, True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = attention.keep_drafts(caches[0], caches[1], *args, k_scale=caches[2], v_scale=caches[3])
    for s in steps[1:] + steps:
        for a, b in zip(args, s.args()):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        lens = oracle.keep_drafts(oracle_caches(*views(want, 64, 2, 128, True)), *s.args())
        assert torch.equal(new.cpu(), lens) and torch.equal(got.cpu(), want)


def test_refusals_on_the_host():
    lib = _lib.lib()
    args = dict(k=16, v=16, ls=1 << 20, bs=16384, ss=128, hs=64, ksc=None, vsc=None, sls=0, sbs=0, shs=0, layers=2, pages=8,
                bt=16, bts=4, path=16, ps=8, width=8, accepted=16, cu=16, lens=16, seqs=2, heads=2, d=64, block=64, maxb=4,
                new=16, stream=None)

    def call(**over):
        return lib.kvp_keep_drafts(*dict(args, **over).values())

    assert call(seqs=0) == _lib.KVP_OK
    scales = dict(ksc=16, vsc=16, sls=1 << 20, sbs=128, shs=64)
    assert call(seqs=0, **scales) == _lib.KVP_OK
    for bad in (dict(seqs=-1), dict(layers=0), dict(pages=0), dict(heads=0), dict(block=0), dict(maxb=0), dict(bts=3), dict(ps=7),
                dict(k=None), dict(v=None), dict(ksc=16), dict(k=24), dict(ss=124), dict(ls=0), dict(ls=16384 * 7), dict(hs=56),
                dict(bs=8192 - 64), dict(bt=None), dict(path=None), dict(accepted=None), dict(cu=None), dict(lens=None),
                dict(new=None), dict(bt=18), dict(new=18), dict(scales, sls=0), dict(scales, shs=63), dict(scales, sbs=64)):
        assert call(**bad) == _lib.KVP_EINVAL, bad
    for bad in (dict(d=32), dict(d=96), dict(width=65, ps=65), dict(seqs=65536), dict(maxb=1 << 26, bts=1 << 26)):
        assert call(**bad) == _lib.KVP_EUNSUPPORTED, bad
    assert b"kvp_keep_drafts" in lib.kvp_last_error()


def test_refusals_of_the_python_layer():
    x = torch.zeros(1, 2, 64, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        attention.keep_drafts(x, x, i.view(1, 2), i[:1], i, i[:1], i.view(1, 2))


@pytest.mark.gpu
def test_refusals_of_wrong_tensors(cuda_device):
    g, rng = gen(1), random.Random(1)
    path, accepted, cu, lens, bt = Step([9, 9], [4, 4], 64, 4, g, rng).args("cuda")
    k, v, ks, vs = views(pool_of(2, 4, 64, 1, 64, True, g).cuda(), 64, 1, 64, True)
    good = dict(k_cache=k, v_cache=v, path=path, accepted=accepted, cu_seqlens_q=cu, cache_seqlens=lens, block_table=bt,
                k_scale=ks, v_scale=vs)
    attention.keep_drafts(**good)
    for name, value in (("k_cache", k.view(torch.uint8)), ("k_cache", k[0, 0]), ("v_cache", v[:1]), ("k_scale", None),
                        ("k_scale", ks[:, :, :, :32]), ("path", path.long()), ("path", path[0]), ("path", path.cpu()),
                        ("path", path[:1]), ("accepted", accepted[:1]), ("accepted", accepted.long()), ("cu_seqlens_q", cu[:0]),
                        ("cache_seqlens", lens[:1]), ("block_table", bt[:1]), ("block_table", bt.long())):
        with pytest.raises(ValueError):
            attention.keep_drafts(**{**good, name: value})
    with pytest.raises(_lib.KVPathError, match="overlap"):
        attention.keep_drafts(**{**good, "k_cache": k[:1].expand(2, -1, -1, -1, -1), "v_cache": v[:1].expand(2, -1, -1, -1, -1)})


def test_new_lengths_in_an_inputs_place_are_refused():
    """Workgroups of one sequence read its length and its path while another of them writes the new length."""
    lib = _lib.lib()
    at = dict(bt=1 << 12, path=2 << 12, accepted=3 << 12, cu=4 << 12, lens=5 << 12, new=6 << 12)
    sizes = dict(bt=4 * (2 * 7 + 4), path=4 * (2 * 9 + 8), accepted=12, cu=16, lens=12, new=12)  # three sequences

    def call(**over):
        p = dict(at, **over)
        return lib.kvp_keep_drafts(16, 16, 1 << 20, 16384, 128, 64, None, None, 0, 0, 0, 2, 8, p["bt"], 7, p["path"], 9, 8,
                                   p["accepted"], p["cu"], p["lens"], 3, 2, 64, 64, 4, p["new"], None)

    for name in ("bt", "path", "accepted", "cu", "lens"):
        for new in (at[name], at[name] + sizes[name] - 4, at[name] - sizes["new"] + 4):
            assert call(new=new) == _lib.KVP_EINVAL, (name, new)
            assert b"new_seqlens" in lib.kvp_last_error()


@pytest.mark.gpu
def test_new_lengths_between_an_inputs_rows(cuda_device):
    """What lies between rows of the tables is no part of them."""
    g, rng = gen(8), random.Random(8)
    step = Step([90, 70], [6, 9], 64, 8, g, rng, kept=3)
    pool = pool_of(2, 8, 64, 2, 128, False, g)
    want, got = pool.clone(), pool.cuda()
    lens = oracle.keep_drafts(oracle_caches(*views(want, 64, 2, 128, False)), *step.args())
    path, accepted, cu, old, bt = step.args("cuda")
    room = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
    room[:, :bt.shape[1]] = bt
    k, v, _, _ = views(got, 64, 2, 128, False)
    s = k.stride()
    rc = _lib.lib().kvp_keep_drafts(
        k.data_ptr(), v.data_ptr(), s[0], s[1], s[2], s[3], None, None, 0, 0, 0, 2, 8, room.data_ptr(), 8, path.data_ptr(),
        path.stride(0), path.shape[1], accepted.data_ptr(), cu.data_ptr(), old.data_ptr(), 2, 2, 128, 64, bt.shape[1],
        room.data_ptr() + 4 * 5, torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.KVP_OK
    assert torch.equal(room[0, 5:7].cpu(), lens) and torch.equal(got.cpu(), want)


def test_keys_and_values_in_one_place_are_refused():
    """Two threads would move each row, one of them perhaps after the other has written over it."""
    lib = _lib.lib()

    def call(k, v, ks=None, vs=None):
        return lib.kvp_keep_drafts(k, v, 1 << 20, 16384, 128, 64, ks, vs, 1 << 20, 128, 64, 2, 8, 1 << 12, 4, 2 << 12, 8, 8,
                                   3 << 12, 4 << 12, 5 << 12, 3, 2, 64, 64, 4, 6 << 12, None)

    assert call(1 << 24, 1 << 24) == _lib.KVP_EINVAL and b"k_cache" in lib.kvp_last_error()
    assert call(1 << 24, 1 << 25, 1 << 26, 1 << 26) == _lib.KVP_EINVAL and b"k_scale" in lib.kvp_last_error()
