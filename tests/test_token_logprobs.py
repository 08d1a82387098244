"""Log probabilities, entropy, rank and alternatives of given tokens against the 64-bit oracle.

Tolerance: of 2^t with t = c x - R the fma rounds t to 2^-24 of itself, the exponential is off by
2^-23, and a thread adds at most vocab / 512 + 8 values one after the other before a tree of ten
additions.  So s is off by at most (vocab / 512 + 20 + |t|) 2^-24 of itself, with |t| <= 40 wherever
2^t matters, and w by as much of sum 2^t |t|.  A log probability adds the rounding of c x - R, of the
logarithm and of the product: 4 * 2^-24 of each.
"""

import math

import pytest
import torch

from kavor_amd import _lib
from kavor_amd.layers import fused
from oracle import operators_oracle as oracle
from tests.helpers import gen

STEP = 2.0 ** -24


def check(got, logits, tokens, top):
    logp, entropy, rank, top_logp, ids = (t.cpu() for t in got)
    want = oracle.token_logprobs(logits, tokens, top)
    sums = (logits.shape[1] / 512 + 60) * STEP
    for x, y in ((logp, want[0]), (top_logp, want[3])):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.isinf(), y.isinf())
        fine = y.isfinite()
        assert ((x.double() - y).abs() <= sums + 12 * STEP * y.abs())[fine].all()
    assert torch.equal(entropy.isnan(), want[1].isnan())
    fine = want[1].isfinite()
    assert ((entropy.double() - want[1]).abs() <= sums * (2 + want[1].abs() * 2))[fine].all()
    assert torch.equal(rank, want[2])
    assert torch.equal(ids, want[4])


def run(logits, tokens, top):
    """On the GPU, rows padded to a multiple of 8 whose padding is not to be read."""
    n, vocab = logits.shape
    room = torch.full((n, -(-vocab // 8) * 8 + 8), math.nan, dtype=logits.dtype, device="cuda")
    room[:, :vocab] = logits.cuda()
    return fused.token_logprobs(room[:, :vocab], tokens.cuda(), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (2, 3, 3), (3, 7, 0), (1, 8, 8), (5, 100, 64), (1, 513, 20), (4, 1013, 64), (40, 4096, 5),
    (600, 257, 3), (513, 5000, 64), (1, 151936, 20), (7, 151643, 64), (33, 32003, 1)])
def test_rows_match_the_oracle(cuda_device, dtype, rows, vocab, top):
    g = gen(rows + vocab)
    logits = (torch.randn(rows, vocab, generator=g) * torch.linspace(0.3, 6, rows)[:, None]).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    tokens[0] = int(logits[0].float().argmax())
    tokens[-1] = vocab - 1
    check(run(logits, tokens, top), logits, tokens, top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 700])
@pytest.mark.parametrize("vocab", [300, 40_000])
def test_equal_values_go_to_the_lowest_index(cuda_device, rows, vocab):
    """A handful of levels, so that hundreds of values tie with the last alternative; and all equal."""
    g = gen(vocab)
    logits = torch.randint(0, 6, (rows, vocab), generator=g).bfloat16()
    logits[0] = 2.5
    logits[1, ::2], logits[1, 1::2] = -0.0, 0.0
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    for top in (1, 20, 64):
        check(run(logits, tokens, top), logits, tokens, top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [12, 600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows_infinities_and_nan(cuda_device, rows, dtype):
    vocab, g = 9001, gen(4)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.randn(rows, vocab, generator=g).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    x[0, 100:] = -math.inf
    x[1] = -math.inf
    x[2, 1:] = -math.inf
    x[3, 4000] = math.nan
    x[4, [77, 5000]] = math.inf
    x[5] = low                          # all masked with the type's lowest value
    x[6, 20:] = low
    x[7, :300] = high
    x[8] = math.nan
    x[9, 8500], x[9, 3] = math.nan, math.inf
    x[10] = -math.inf
    x[10, 8990] = low
    x[11, 0], x[11, 8000] = 2e38, 3e38
    tokens[0], tokens[2], tokens[6], tokens[7], tokens[10], tokens[11] = 200, 0, 30, 5, 8990, 8000
    check(run(x, tokens, 30), x, tokens, 30)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["up", "down", "steps"])
def test_values_that_climb_along_the_row(cuda_device, order):
    """The reference of the sums has to follow maxima that come late, by hundreds at a time."""
    vocab = 20_000
    x = torch.arange(vocab, dtype=torch.float32) / 20
    if order == "down":
        x = x.flip(0)
    elif order == "steps":
        x = (x // 100) * 300 - 700
    x = torch.stack((x, x - 500, x * 30))
    tokens = torch.tensor([vocab - 1, 0, vocab // 2])
    check(run(x, tokens, 10), x, tokens, 10)


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary(cuda_device):
    x = torch.randn(4, 1000, generator=gen(2)).bfloat16()
    logp, entropy, rank, _, _ = run(x, torch.tensor([-1, 1000, 5, 1 << 40]), 0)
    assert logp.isnan().tolist() == [True, True, False, True] and rank[[0, 1, 3]].tolist() == [0, 0, 0]
    assert entropy.isfinite().all()


@pytest.mark.gpu
def test_captured_replays_follow_their_inputs(cuda_device):
    logits = torch.empty(6, 30_000, dtype=torch.bfloat16, device=cuda_device)
    tokens = torch.zeros(6, dtype=torch.int64, device=cuda_device)
    fused.reserve_logprobs_workspace(cuda_device)
    logits.normal_()
    fused.token_logprobs(logits, tokens, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused.token_logprobs(logits, tokens, 5)
    side = torch.cuda.Stream()
    for i in range(3):
        logits.normal_()
        tokens.fill_(17 * i)
        with torch.cuda.stream(side):
            fused.token_logprobs(torch.zeros(3, 64, device=cuda_device), tokens[:3], 2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, fused.token_logprobs(logits, tokens, 5)):
            assert torch.equal(a, b)


def _call(**over):
    a = dict(logits=16, fp32=0, rs=1000, n=4, vocab=1000, tokens=16, top=5, lp=16, h=16, rank=16, tl=16, tt=16, ws=16,
             wsb=1 << 20, stream=None)
    a.update(over)
    return _lib.lib().kvp_token_logprobs(*a.values())


def test_bad_arguments_are_refused_on_the_host():
    E, U = _lib.KVP_EINVAL, _lib.KVP_EUNSUPPORTED
    assert _call(n=0) == _lib.KVP_OK
    for over in (dict(top=65), dict(top=-1), dict(vocab=4, rs=8)):
        assert _call(**over) == U, over
    for over in (dict(n=-1), dict(vocab=0), dict(logits=0), dict(logits=8), dict(rs=1004), dict(rs=992), dict(tokens=0),
                 dict(tokens=4), dict(lp=2), dict(h=0), dict(rank=4), dict(tl=0), dict(tt=4), dict(ws=8),
                 dict(fp32=1, rs=1002)):
        assert _call(**over) == E, over
    assert _call(ws=0) == _lib.KVP_EWORKSPACE and _call(wsb=100) == _lib.KVP_EWORKSPACE
    assert max(_lib.lib().kvp_token_logprobs_workspace_bytes(n) for n in range(2000)) <= 1 << 20


@pytest.mark.gpu
def test_wrapper_checks_types_and_shapes(cuda_device):
    x, t = torch.zeros(4, 64, device=cuda_device), torch.zeros(4, dtype=torch.int64, device=cuda_device)
    assert fused.token_logprobs(x, t)[3].shape == (4, 0)
    assert fused.token_logprobs(x[:0], t[:0], 3)[4].shape == (0, 3)
    for bad in ((x.half(), t), (x[0], t), (x.cpu(), t), (x, t.int()), (x, t[:3]), (x, t.cpu()), (x, t, -1),
                (x.t(), t.repeat(16))):
        with pytest.raises(ValueError):
            fused.token_logprobs(*bad)
    for bad in ((x, t, 65), (torch.zeros(4, 65, device=cuda_device), t)):
        with pytest.raises(_lib.KVPathError):
            fused.token_logprobs(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 5, 5), (2, 63, 63), (255, 70, 64), (256, 70, 64), (16, 40, 33),
                                            (1, 200003, 64)])
def test_small_vocabularies_and_the_bounds_of_the_split(cuda_device, dtype, rows, vocab, top):
    g = gen(7 * rows + vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    check(run(logits, tokens, top), logits, tokens, top)
