"""Verification of drafted tokens against the 64-bit oracle: equal counts, paths and tokens.

Sums that decide about drafts are in 32 bits.  Of 2^t the exponent is rounded to 2^-24 of itself, three times, the
exponential is off by 2^-23, and a thread adds at most vocab / 256 + 16 values one after the other before a tree of twelve
additions: a row's sum is off by at most (vocab / 256 + 32 + 3 |t|) 2^-24 of itself, with |t| <= 40 wherever 2^t
matters, so a decision is the oracle's where its two sides are further apart than twice that.  Next tokens come from 64-bit
sums of weights that are off by 2^-46 of the largest one at most: the oracle's where the number lies more than vocab times
that, and 1e-12 for the sums, from a border.  Inputs nearer to a border would be no test: the oracle says how near
they come, and the seeds are such that none does.
"""

import math
import random

import pytest
import torch

from kavor_amd import _lib
from kavor_amd.layers import fused
from oracle import drafts_oracle as oracle
from tests.helpers import gen

BELOW_ONE = 1 - 2.0 ** -24


def reach(vocab):
    """How far the two sides of a decision have to be apart, and the drawn number from a border."""
    return 2 * (vocab / 256 + 32 + 120) * 2.0 ** -24, vocab * 2.0 ** -46 + 1e-12


def trees(lens, rng):
    """Masks of a random tree for each sequence, and each row's parent."""
    masks, parents = [], []
    for n in lens:
        own = []
        for i in range(n):
            parent = rng.randint(max(0, i - 4), i - 1) if i else -1
            own.append((own[parent] if i else 0) | 1 << i)
            parents.append(parent)
        masks += own
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64), parents


class Batch:
    """Drafts that have a fair chance: sampled from a distribution near the target's, or from its best tokens."""

    def __init__(self, lens, vocab, dtype, form, seed=0, greedy=0.3, width=6.0):
        g, rng = gen(seed), random.Random(seed)
        T = sum(lens)
        self.cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
        self.max_q = max(lens + [1])
        self.logits = (torch.randn(T, vocab, generator=g) * torch.rand(T, 1, generator=g) * width).to(dtype)
        self.temps = torch.rand(len(lens), generator=g) + 0.4
        self.temps[torch.rand(len(lens), generator=g) < greedy] = 0.0
        self.uniforms = torch.rand(T, generator=g)
        self.draft = self.mask = None
        if form == "tree":
            self.mask, parents = trees(lens, rng)
        else:
            parents = [i - 1 for n in lens for i in range(n)]
        near = self.logits.float() + 0.5 * torch.randn(T, vocab, generator=g)
        if form == "sampled":
            self.draft = near.to(dtype)
        first = [q for q, n in zip(self.cu.tolist(), lens) for _ in range(n)]
        above = torch.tensor([f + max(p, 0) for f, p in zip(first, parents)], dtype=torch.int64)
        seq = [b for b, n in enumerate(lens) for _ in range(n)]
        self.tokens = torch.zeros(T, dtype=torch.int64)
        for r in range(T):
            up, temp = int(above[r]), float(self.temps[seq[r]])
            if form == "sampled":
                p = oracle.softmax(self.draft[up], temp) if temp > 0 else None
                self.tokens[r] = int(torch.multinomial(p, 1, generator=g)) if p is not None else oracle.greedy(self.draft[up])
            else:
                best = near[up].topk(min(3, vocab)).indices
                self.tokens[r] = int(best[rng.randrange(len(best))])

    def args(self):
        return dict(logits=self.logits, tokens=self.tokens, uniforms=self.uniforms, temperatures=self.temps,
                    cu_seqlens_q=self.cu, max_seqlen_q=self.max_q, tree_mask=self.mask, draft_logits=self.draft)

    def on_gpu(self):
        """Rows padded to a multiple of 8 whose padding is not to be read."""
        a = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in self.args().items()}
        for name in ("logits", "draft_logits"):
            if a[name] is not None:
                n, vocab = a[name].shape
                room = torch.full((n, -(-vocab // 8) * 8 + 8), math.nan, dtype=a[name].dtype, device="cuda")
                room[:, :vocab] = a[name]
                a[name] = room[:, :vocab]
        return a

    def want(self):
        *want, decided, drawn = oracle.verify_drafts(**self.args())
        apart, off = reach(self.logits.shape[1])
        assert decided > apart and drawn > off, (decided, apart, drawn, off)
        return want


def same(got, want):
    for name, x, y in zip(("accepted", "path", "out_tokens"), got, want):
        x = x.cpu()
        assert x.dtype == y.dtype and torch.equal(x, y), f"{name}:\n{x}\n{y}"


def many(a, want):
    """The batch again and again, in one call of 100 MB of logits and more, which takes another way through the rows."""
    rows, vocab = a["logits"].shape
    times = -(-230_000_000 // (rows * vocab * a["logits"].element_size()))
    seqs = len(a["temperatures"])
    if times * seqs > 20_000:
        return
    wide = {name: t if not isinstance(t, torch.Tensor) else t.repeat(times, *[1] * (t.dim() - 1)) for name, t in a.items()}
    for name in ("logits", "draft_logits"):
        if wide[name] is not None:
            room = torch.full((rows * times, -(-vocab // 8) * 8), math.nan, dtype=a[name].dtype, device="cuda")
            room[:, :vocab] = wide[name]
            wide[name] = room[:, :vocab]
    cu = a["cu_seqlens_q"]
    steps = torch.arange(times, device="cuda", dtype=torch.int32)[:, None] * rows
    wide["cu_seqlens_q"] = torch.cat(((cu[:-1] + steps).view(-1), cu[-1:] + steps[-1]))
    same(fused.verify_drafts(**wide), [w.repeat(times, *[1] * (w.dim() - 1)) for w in want])


def check(batch):
    want = batch.want()
    a = batch.on_gpu()
    same(fused.verify_drafts(**a), want)
    many(a, want)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["sampled", "chosen", "tree"])
@pytest.mark.parametrize("lens,vocab", [
    ([1], 1), ([2], 1), ([3, 1], 2), ([5], 7), ([2, 0, 4], 8), ([8] * 9, 100), ([1, 9, 3, 0, 0], 513), ([16, 5, 7], 1013),
    ([64], 300), ([64, 63, 1, 33], 4099), ([4] * 33, 4096), ([6, 2], 32_003), ([5], 151_936)])
def test_batches_match_the_oracle(cuda_device, dtype, form, lens, vocab):
    check(Batch(lens, vocab, dtype, form, seed=len(lens) + vocab, greedy=0.3 if len(lens) > 1 else 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["sampled", "chosen", "tree"])
@pytest.mark.parametrize("seqs,rows", [(300, 4), (40, 30), (700, 2)])
def test_many_rows_match_the_oracle(cuda_device, form, seqs, rows):
    lens = [random.Random(i).randint(0, rows) for i in range(seqs)]
    want = check(Batch(lens, 700, torch.bfloat16, form, seed=seqs, width=9.0))
    # with 0 to 2 rows a third of the sequences have a draft, and one of the three best tokens, not the best one, passes
    # about one time in four: a twelfth of the sequences keep one
    assert want[0].sum() > seqs / 16


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["sampled", "chosen", "tree"])
def test_the_output_is_distributed_as_the_target(cuda_device, form):
    """50,000 sequences with the same rows and drafts drawn anew: the first token's frequencies against p, by the
    chi-squared statistic over 11 degrees of freedom (48 is passed once in 1e6)."""
    n, vocab, g = 50_000, 12, gen(4)
    z, y = torch.randn(vocab, generator=g) * 1.5, torch.randn(vocab, generator=g) * 1.5
    p, q = torch.softmax(z.bfloat16().double() / 0.8, 0), torch.softmax(y.bfloat16().double() / 0.8, 0)
    rows = {"sampled": 2, "chosen": 2, "tree": 4}[form]
    logits = torch.zeros(n, rows, 16, dtype=torch.bfloat16)
    logits[:, :, :vocab] = z.bfloat16()
    logits = logits.view(-1, 16).cuda()[:, :vocab]
    draft = torch.zeros(n * rows, 16, dtype=torch.bfloat16, device="cuda")
    draft[:, :vocab] = y.bfloat16().cuda()
    tokens = torch.zeros(n, rows, dtype=torch.int64)
    if form == "sampled":
        tokens[:, 1] = torch.multinomial(q, n, replacement=True, generator=g)
    else:
        tokens[:, 1:] = torch.topk(p, 3).indices[torch.randint(0, 3, (n, rows - 1), generator=g)]
    cu = torch.arange(0, n * rows + 1, rows, dtype=torch.int32).cuda()
    mask = torch.tensor([1, 3, 5, 9]).repeat(n).cuda() if form == "tree" else None
    _, _, out = fused.verify_drafts(logits, tokens.view(-1).cuda(), torch.rand(n * rows, generator=g).cuda(),
                                    torch.full((n,), 0.8).cuda(), cu, rows, mask, draft[:, :vocab] if form == "sampled" else None)
    seen = torch.bincount(out[:, 0].cpu(), minlength=vocab).double()
    assert float(((seen - n * p) ** 2 / (n * p)).sum()) < 48


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["sampled", "chosen", "tree"])
def test_rows_without_a_softmax_and_hidden_tokens(cuda_device, dtype, form):
    x = Batch([4] * 12, 3000, dtype, form, seed=2, greedy=0.0)
    low = torch.finfo(dtype).min
    x.logits[0, 77] = math.nan
    x.logits[4] = -math.inf
    x.logits[8, [5, 2000]] = math.inf
    x.logits[12, 10:] = -math.inf
    x.logits[16] = low
    x.logits[20, 1:] = low
    x.logits[24] = math.nan
    x.logits[28, 100] = torch.finfo(dtype).max
    x.temps[7] = 0.0                  # row 28: greedy
    x.logits[32, 2999], x.logits[32, 3] = math.inf, math.nan
    x.tokens[13], x.tokens[33] = 11, 3
    if form == "sampled":
        x.draft[36, 9] = math.nan
        x.draft[40] = -math.inf
        x.draft[44, 20:] = -math.inf
        x.tokens[45] = 30             # q(x) = 0: kept if p(x) > 0
        x.draft[3::4] = math.nan      # no draft behind these
    check(x)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["sampled", "chosen", "tree"])
def test_temperatures_and_numbers_at_their_ends(cuda_device, form):
    x = Batch([3] * 16, 500, torch.float32, form, seed=5, greedy=0.0)
    x.temps[:8] = torch.tensor([0.0, -1.0, math.nan, math.inf, 1e-30, 1e30, 1e-42, 0.02])
    x.logits[18, 40] = x.logits[18].max()  # at a temperature near 0: the first of two equal ones, or both
    x.uniforms[24:36] = 0.0
    x.uniforms[36:48] = BELOW_ONE
    want = oracle.verify_drafts(**x.args())[:3]
    same(fused.verify_drafts(**x.on_gpu()), want)
    many(x.on_gpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_draft_model_that_is_the_target_keeps_everything(cuda_device, dtype):
    x = Batch([8] * 20, 5003, dtype, "sampled", seed=3, greedy=0.0)
    x.draft = x.logits.clone()
    for r in range(len(x.tokens)):
        if r % 8:
            p = oracle.softmax(x.draft[r - 1], float(x.temps[r // 8]))
            x.tokens[r] = int(torch.multinomial(p, 1, generator=gen(r)))
    x.uniforms.view(20, 8)[:, 1:] = BELOW_ONE
    got = fused.verify_drafts(**x.on_gpu())
    assert (got[0] == 7).all()
    want = oracle.verify_drafts(**x.args())[:3]
    same(got, want)
    many(x.on_gpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [37, 4099, 70_001])
def test_what_is_left_between_equal_distributions_is_never_a_hidden_token(cuda_device, dtype, vocab):
    """Drafts that neither model can give, from a draft model that is the target but for a shift, exact or rounded: what is
    left of p - q is nothing, or roundings.  Whatever the number, the next token is one that the target can give."""
    seqs, g = 130, gen(vocab)
    logits = torch.randn(2 * seqs, vocab, generator=g)
    logits[::4] *= 12  # rows with all but a few weights small
    logits[:, ::2] = -math.inf
    logits = logits.to(dtype)
    shift = torch.where(torch.arange(2 * seqs) % 8 < 4, 0.0, 3.7)[:, None]
    a = dict(logits=logits, draft_logits=(logits.float() + shift).to(dtype),
             tokens=2 * torch.randint((vocab + 1) // 2, (2 * seqs,), generator=g),
             uniforms=torch.linspace(0, 1, 2 * seqs).clamp(max=BELOW_ONE), temperatures=torch.ones(seqs),
             cu_seqlens_q=2 * torch.arange(seqs + 1, dtype=torch.int32))
    room = {}
    for name, t in a.items():
        room[name] = t.cuda()
        if t.dim() == 2:
            wide = torch.full((2 * seqs, -(-vocab // 8) * 8), math.nan, dtype=dtype, device="cuda")
            wide[:, :vocab] = room[name]
            room[name] = wide[:, :vocab]
    for few in (seqs, 3):  # both ways to the sums
        n = dict(room, cu_seqlens_q=room["cu_seqlens_q"][:few + 1])
        accepted, path, out = fused.verify_drafts(**n, max_seqlen_q=2)
        assert int(accepted.abs().sum()) == 0 and bool((path == -1).all()) and bool((out[:, 1] == -1).all())
        assert bool((out[:, 0] % 2 == 1).all()), out[:, 0].tolist()


@pytest.mark.gpu
def test_siblings_and_what_is_left_of_them(cuda_device):
    """Siblings with one token, siblings that have nearly all of p, a row that sees no row, masks with bits above."""
    x = Batch([6, 6, 6, 6, 3], 64, torch.float32, "tree", seed=8, greedy=0.0)
    star = torch.tensor([1] + [1 | 1 << i for i in range(1, 6)])
    x.mask[:24] = star.repeat(4)
    x.tokens[:6] = torch.tensor([0, 9, 9, 9, 4, 9])          # twins: the later ones never pass
    x.logits[6] = torch.where(torch.arange(64) < 5, 10.0, -20.0)
    x.tokens[6:12] = torch.tensor([0, 0, 1, 2, 3, 4])
    x.uniforms[6:12] = torch.tensor([0.5] + [BELOW_ONE] * 5)  # 1e-13 of p is left behind them
    x.logits[12] = -math.inf
    x.logits[12, 7] = 1.0                                    # p is one token, refused as none has it
    x.tokens[12:18] = torch.tensor([0, 1, 2, 3, 4, 5])
    x.mask[19] = 0                                           # sees nothing: not kept, nobody's child
    x.mask[20] |= 1 << 40
    x.tokens[20] = x.logits[18].argmax()
    x.uniforms[20] = 0.0
    x.temps[4] = 0.0
    x.mask[24:27] = torch.tensor([1, 3, 7])
    x.tokens[25], x.tokens[26] = x.logits[24].argmax(), x.logits[25].argmax()
    # the decisions with numbers just below 1 are 2^-24 from their borders, and exact: five weights of 1 among others of 1e-13
    want = oracle.verify_drafts(**x.args())[:3]
    same(fused.verify_drafts(**x.on_gpu()), want)
    many(x.on_gpu(), want)
    assert want[1][3, 0] == 2 and want[0][4] == 2


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary_are_refused(cuda_device):
    for form in ("sampled", "chosen", "tree"):
        x = Batch([3] * 6, 1000, torch.bfloat16, form, seed=1)
        x.tokens[1::3] = torch.tensor([-1, 1000, 1 << 40, -(1 << 60), (1 << 32) + 5, 5])
        check(x)


@pytest.mark.gpu
def test_sequences_that_are_no_batch(cuda_device):
    """More rows than announced, rows outside the tensor, falling offsets: nothing kept, no token; the others as ever."""
    x = Batch([3, 5, 2, 4], 200, torch.bfloat16, "chosen", seed=6)
    x.max_q = 4
    want = x.want()
    assert want[0][1] == 0 and (want[2][1] == -1).all()
    same(fused.verify_drafts(**x.on_gpu()), want)
    for ends in ([0, 3, 3, 20, 14], [-2, 3, 8, 10, 14], [0, 8, 3, 10, 14]):
        x.cu = torch.tensor(ends, dtype=torch.int32)
        same(fused.verify_drafts(**x.on_gpu()), oracle.verify_drafts(**x.args())[:3])
    a = x.on_gpu()
    empty = {k: v[:0].contiguous() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    empty["cu_seqlens_q"] = a["cu_seqlens_q"][:1] * 0
    assert [t.shape for t in fused.verify_drafts(**empty)] == [(0,), (0, 4), (0, 4)]
    empty["cu_seqlens_q"], empty["temperatures"] = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda")
    got = fused.verify_drafts(**empty)
    assert (got[0] == 0).all() and (got[1] == -1).all() and (got[2] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["sampled", "tree"])
def test_rows_far_apart(cuda_device, form):
    """Rows more than 2^32 bytes from the first one."""
    x = Batch([3], 400, torch.bfloat16, form, seed=4, greedy=0.0)
    want = x.want()
    a = x.on_gpu()
    stride = (5 << 28) + 64
    for name in ("logits", "draft_logits"):
        if a[name] is not None:
            room = torch.empty(2 * stride + 400, dtype=torch.bfloat16, device="cuda")
            a[name] = room.as_strided((3, 400), (stride, 1)).copy_(a[name])
    same(fused.verify_drafts(**a), want)


@pytest.mark.gpu
def test_other_streams_and_captured_graphs(cuda_device):
    first, second = (Batch([5, 0, 9, 2], 3001, torch.bfloat16, "sampled", seed=s) for s in (1, 2))
    second.cu = first.cu
    wants = [b.want() for b in (first, second)]
    side = torch.cuda.Stream()
    a = first.on_gpu()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = fused.verify_drafts(**a)
    side.synchronize()
    same(got, wants[0])
    fused.reserve_verify_workspace(4, 9, 3001, cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fused.verify_drafts(**a)
    for batch, want in ((second, wants[1]), (first, wants[0]), (second, wants[1])):
        for k, v in batch.on_gpu().items():
            if isinstance(v, torch.Tensor):
                a[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        same(got, want)
        same(fused.verify_drafts(**a), want)  # eager calls in between have a buffer of their own


@pytest.mark.gpu
def test_two_graphs_in_turn(cuda_device):
    """Graphs of different sizes share the captured workspace; replays in turn keep their results."""
    batches = [Batch([4, 2], 2000, torch.float32, "sampled", seed=1), Batch([64, 9, 1], 900, torch.bfloat16, "tree", seed=2)]
    fused.reserve_verify_workspace(4, 64, 2000, cuda_device)
    made = []
    for b in batches:
        a, graph = b.on_gpu(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = fused.verify_drafts(**a)
        made.append((graph, a, got, b.want()))
    for _ in range(3):
        for graph, _, got, want in made:
            for t in got:
                t.fill_(-7)
            graph.replay()
            torch.cuda.synchronize()
            same(got, want)


def test_refusals_on_the_host():
    lib = _lib.lib()
    args = dict(logits=16, fp32=0, rs=1000, total=10, vocab=1000, draft=None, drs=0, tokens=16, uniforms=16, temps=16,
                cu=16, seqs=2, max_q=8, mask=None, accepted=16, path=16, out=16, ws=16, wsb=1 << 30, stream=None)

    def call(**over):
        return lib.kvp_verify_drafts(*dict(args, **over).values())

    assert call(seqs=0) == _lib.KVP_OK
    for bad in (dict(seqs=-1), dict(total=-1), dict(vocab=0), dict(logits=None), dict(tokens=None), dict(uniforms=None),
                dict(temps=None), dict(cu=None), dict(accepted=None), dict(path=None), dict(out=None), dict(logits=24),
                dict(rs=996), dict(rs=1004), dict(fp32=1, rs=1001), dict(draft=16, drs=992), dict(draft=8, drs=1000),
                dict(tokens=12), dict(uniforms=18), dict(cu=18), dict(mask=20), dict(out=20), dict(ws=24)):
        assert call(**bad) == _lib.KVP_EINVAL, bad
    for bad in (dict(max_q=0), dict(max_q=65), dict(seqs=65536), dict(vocab=(1 << 30) + 1, rs=1 << 31),
                dict(draft=16, drs=1000, mask=16)):
        assert call(**bad) == _lib.KVP_EUNSUPPORTED, bad
    assert call(wsb=64) == _lib.KVP_EWORKSPACE and call(ws=None) == _lib.KVP_EWORKSPACE
    assert b"kvp_verify_drafts" in lib.kvp_last_error()


def test_workspace_sizes_grow_with_every_argument():
    size = _lib.lib().kvp_verify_workspace_bytes
    grid = [(b, n, v) for b in (1, 2, 7, 64, 300) for n in (1, 5, 64) for v in (1, 1000, 151_936)]
    for small in grid:
        for large in grid:
            if all(x <= y for x, y in zip(small, large)):
                assert size(*small) <= size(*large)
    assert size(0, 1, 1) == size(1, 65, 1) == size(65536, 1, 1) == size(1, 1, 0) == 0


def test_refusals_of_the_python_layer():
    logits, ids = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        fused.verify_drafts(logits, ids, torch.zeros(3), torch.ones(1), torch.tensor([0, 3], dtype=torch.int32), 3)


@pytest.mark.gpu
def test_refusals_of_wrong_tensors(cuda_device):
    good = Batch([3, 2], 64, torch.bfloat16, "sampled", seed=1).on_gpu()
    for name, value, match in (
            ("logits", good["logits"].half(), "bf16"), ("logits", good["logits"].t(), "contiguous|tokens"),
            ("tokens", good["tokens"].int(), "tokens"), ("tokens", good["tokens"][:4], "tokens"),
            ("tokens", good["tokens"].cpu(), "tokens"), ("uniforms", good["uniforms"].double(), "uniforms"),
            ("uniforms", good["uniforms"][::2], "uniforms"), ("temperatures", good["temperatures"][:1], "temperatures"),
            ("cu_seqlens_q", good["cu_seqlens_q"].long(), "cu_seqlens_q"), ("cu_seqlens_q", good["cu_seqlens_q"][:0], "cu_seqlens_q"),
            ("draft_logits", good["draft_logits"].float(), "draft_logits"), ("draft_logits", good["draft_logits"][:3], "draft_logits"),
            ("tree_mask", torch.ones(5, dtype=torch.int64, device="cuda"), "chain")):
        with pytest.raises(ValueError, match=match):
            fused.verify_drafts(**{**good, name: value})
    for mask in (torch.ones(5, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError, match="tree_mask"):
            fused.verify_drafts(**{**good, "draft_logits": None, "tree_mask": mask})
    for rows in (0, 65, -1):
        with pytest.raises(_lib.KVPathError, match="max_seqlen_q"):
            fused.verify_drafts(**{**good, "max_seqlen_q": rows})


@pytest.mark.gpu
def test_offsets_that_wrap_are_no_rows(cuda_device):
    """Ends past 2^31 that would make a short sequence of two far apart numbers."""
    x = Batch([3, 2, 4], 100, torch.bfloat16, "chosen", seed=2)
    x.cu = torch.tensor([2 ** 31 - 3, -2 ** 31 + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    got = fused.verify_drafts(**x.on_gpu())
    assert (got[0] == 0).all() and (got[1] == -1).all() and (got[2] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 2_500_000), (torch.float32, 1_200_003)])
@pytest.mark.parametrize("form", ["sampled", "chosen"])
def test_vocabularies_of_more_ranges_than_threads(cuda_device, dtype, vocab, form):
    check(Batch([3, 1], vocab, dtype, form, seed=9, greedy=0.0, width=3.0))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["sampled", "chosen", "tree"])
def test_results_do_not_depend_on_another_threads_calls(cuda_device, form):
    """Two threads on one stream, whose calls share the workspace: one reads its rows in one pass, one in several."""
    import threading

    small, large = Batch([5, 9, 2], 4000, torch.bfloat16, form, seed=1), Batch([64] * 24, 1500, torch.float32, form, seed=2)
    calls = [b.on_gpu() for b in (small, large)]
    for k in ("logits", "draft_logits", "tokens", "uniforms", "tree_mask"):
        if calls[1][k] is not None:
            t = calls[1][k].repeat(14, *[1] * (calls[1][k].dim() - 1))
            calls[1][k] = torch.nn.functional.pad(t, (0, 4))[:, :t.shape[1]] if t.dim() == 2 else t
    calls[1]["cu_seqlens_q"] = torch.arange(0, 64 * 24 * 14 + 1, 64, dtype=torch.int32, device="cuda")
    calls[1]["temperatures"] = calls[1]["temperatures"].repeat(14)
    want = [[t.clone() for t in fused.verify_drafts(**a)] for a in calls]
    got, errors, start = [[], []], [], threading.Barrier(2)

    def work(i):
        try:
            start.wait()
            for _ in range(60):
                got[i].append(fused.verify_drafts(**calls[i]))
        except Exception as e:  # reported by the test itself
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(2):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["sampled", "chosen"])
def test_numbers_that_fall_among_small_weights(cuda_device, dtype, form):
    """Rows that are sure of one token, and numbers behind it, among weights of some 2^-28.3 that are taken in 32 bits: they
    are 3e-9 wide, 200 times as much as the sum of 1000 of them may be off."""
    n, vocab, g = 20, 1000, gen(6)
    x = Batch([2] * n, vocab, dtype, "chosen", seed=7, greedy=0.0)
    x.logits[:] = (-19.5 - 0.3 * torch.rand(2 * n, vocab, generator=g)).to(dtype)
    x.logits[:, 123] = 0.0
    x.temps[:] = 1.0
    if form == "sampled":  # what is left of p behind a refused draft lies at the one token and among the others
        x.draft = (-19.5 - 0.3 * torch.rand(2 * n, vocab, generator=g)).to(dtype)
        x.draft[:, 123], x.draft[:, 900] = 0.0, 9.0
        x.tokens[1::2] = 900
    else:
        x.tokens[1::2] = 124
    x.uniforms.view(n, 2)[:, 1] = BELOW_ONE
    x.uniforms.view(n, 2)[:, 0] = 1 - (1 + torch.arange(n)) * 2.0 ** -24
    want = check(x)
    assert (want[0] == 0).all() and len(set(want[2][:, 0].tolist())) > n / 2


def test_results_in_an_inputs_place_are_refused():
    """Some kernels write a sequence's results while others still read these."""
    lib = _lib.lib()
    at = dict(logits=1 << 24, draft=2 << 24, tokens=1 << 12, temps=2 << 12, cu=3 << 12, accepted=4 << 12, path=5 << 12, out=6 << 12)
    sizes = dict(logits=2 * (9 * 1008 + 1000), draft=2 * (9 * 1008 + 1000), tokens=8 * 10, temps=8, cu=12, accepted=8,
                 path=4 * 16, out=8 * 16)

    def call(**over):  # 10 rows of 1000 values at a stride of 1008, two sequences of at most 8 rows
        p = dict(at, **over)
        return lib.kvp_verify_drafts(p["logits"], 0, 1008, 10, 1000, p["draft"], 1008, p["tokens"], 1 << 20, p["temps"], p["cu"],
                                     2, 8, None, p["accepted"], p["path"], p["out"], 1 << 30, 1 << 30, None)

    for result in ("accepted", "path", "out"):
        for other in at:
            if other == result:
                continue
            for place in (at[other], at[other] + (sizes[other] - 1) // 8 * 8, at[other] - sizes[result] + 8):
                assert call(**{result: place}) == _lib.KVP_EINVAL, (result, other, place)
                assert b"share" in lib.kvp_last_error(), (result, other, lib.kvp_last_error())


def test_the_oracle_draws_from_the_target_where_no_draft_was_sampled():
    """p = (.5, .3, .2), q = (.7, .2, .1): behind a row's filler the next token follows p, behind a refused draft
    max(p - q, 0), which has nothing of the first token."""
    p, q = torch.tensor([0.5, 0.3, 0.2]), torch.tensor([0.7, 0.2, 0.1])
    args = dict(logits=p.log().repeat(2, 1), temperatures=torch.ones(1), cu_seqlens_q=torch.tensor([0, 2]), max_seqlen_q=2,
                draft_logits=q.log().repeat(2, 1))
    for u, filler, refused in ((0.0, 0, 1), (0.49, 0, 1), (0.51, 1, 2), (0.79, 1, 2), (0.81, 2, 2)):
        for token, want in ((-1, filler), (3, filler), (1 << 40, filler), (0, refused)):
            got = oracle.verify_drafts(tokens=torch.tensor([0, token]), uniforms=torch.tensor([u, 0.99]), **args)
            assert got[0] == 0 and got[2].tolist() == [[want, -1]], (u, token)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [40_000, 40])
def test_rows_padded_with_tokens_that_are_none_follow_the_target(cuda_device, seqs):
    """A draft model that stopped early: the next token is distributed as the target's, by the chi-squared statistic over 11
    degrees of freedom (48 is passed once in 1e6), or as the oracle has it."""
    n, vocab, g = seqs, 12, gen(11)
    z, y = torch.randn(vocab, generator=g) * 1.5, torch.randn(vocab, generator=g) * 1.5
    x = Batch([3], vocab, torch.bfloat16, "sampled", seed=1)
    x.logits, x.draft = z.bfloat16().repeat(3 * n, 1), y.bfloat16().repeat(3 * n, 1)
    x.temps, x.uniforms = torch.full((n,), 0.8), torch.rand(3 * n, generator=g)
    x.cu, x.max_q = torch.arange(0, 3 * n + 1, 3, dtype=torch.int32), 3
    x.tokens = torch.zeros(n, 3, dtype=torch.int64)
    x.tokens[:, 1] = torch.where(torch.arange(n) % 2 == 0, -1, vocab)
    x.tokens = x.tokens.view(-1)
    got = fused.verify_drafts(**x.on_gpu())
    assert int(got[0].abs().sum()) == 0
    if n < 100:
        same(got, x.want())
        return
    p = torch.softmax(z.bfloat16().double() / 0.8, 0)
    seen = torch.bincount(got[2][:, 0].cpu(), minlength=vocab).double()
    assert float(((seen - n * p) ** 2 / (n * p)).sum()) < 48


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["sampled", "chosen", "tree"])
@pytest.mark.parametrize("rest,cold", [(0.0, 1.0), (2.0 ** -27, 1.0), (0.0, 1e-2), (0.0, 5e-4)])
def test_rows_that_are_sure_of_their_token(cuda_device, dtype, form, rest, cold):
    """p of a token is 1 but for 2^-26, or much less, and its number the last one below 1: it stays.

    Sums of weights relative to the largest: an addition to 1 and more is rounded by no more than what is added, be it
    that it is lost or rounded up, so the sum lies between 1 and 1 + 2^-25, and p of the token above 1 - 2^-24.  At low
    temperatures the largest logit over T is large, and a rounding of it no longer small."""
    n, vocab, g = 48, 20_011, gen(12)
    x = Batch([3] * n, 32, dtype, form, seed=12, greedy=0.0)
    x.temps = (torch.rand(n, generator=g) + 0.4) * cold
    heat = x.temps.repeat_interleave(3)[:, None]
    top = torch.randint(0, vocab, (3 * n,), generator=g)
    at = torch.rand(3 * n, 1, generator=g) * 300 - 100  # where a row's largest value lies
    low = math.log(rest / vocab) if rest else -95.0
    fall = heat / cold * (low - 3 * torch.rand(3 * n, vocab, generator=g))
    x.logits = (at.to(dtype) + fall).to(dtype)
    x.logits.scatter_(1, top[:, None], at.to(dtype))
    weights = ((x.logits.double() - at.to(dtype).double()) / heat).exp().sum(1) - 1
    assert float(weights.max()) < (2.0 ** -26 if rest else 1e-30)
    if form == "sampled":
        x.draft = x.logits.clone()
    row = torch.arange(3 * n).view(n, 3)
    parents = torch.tensor([-1, 0, 1]) if form != "tree" else torch.tensor([-1, 0, 0])
    x.tokens = torch.zeros(n, 3, dtype=torch.int64)
    for i in (1, 2):
        x.tokens[:, i] = top[row[:, int(parents[i])]]
    x.tokens = x.tokens.view(-1)
    x.mask = torch.tensor([1, 3, 5]).repeat(n) if form == "tree" else None
    x.uniforms = torch.full((3 * n,), BELOW_ONE)
    x.uniforms[::3] = torch.rand(n, generator=g)
    want = oracle.verify_drafts(**x.args())[:3]
    assert bool((want[0] == (1 if form == "tree" else 2)).all())
    same(fused.verify_drafts(**x.on_gpu()), want)
    many(x.on_gpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("few", [False, True])
def test_where_siblings_have_all_of_p_nothing_else_is_drawn(cuda_device, dtype, few):
    """Two siblings with all of p but 2^-100: the first is refused, the second has the last number below 1.  Its share of
    what is left is 1, which sums in 32 bits may miss by 2^-24 and more: where it is refused the next token follows p, and
    is one of the two."""
    n, vocab, g = 2000, 1500, gen(13)
    logits = -80.0 - 20.0 * torch.rand(n, vocab, generator=g)
    pair = torch.stack([torch.randperm(vocab, generator=g)[:2] for _ in range(n)])
    logits.scatter_(1, pair, torch.stack([torch.zeros(n), -2.0 * torch.rand(n, generator=g)], 1))
    logits = torch.nn.functional.pad(logits, (0, -vocab % 8), value=math.nan).to(dtype).repeat_interleave(3, 0)
    uniforms = torch.tensor([0.0, 0.95, BELOW_ONE]).repeat(n)
    uniforms[::3] = torch.linspace(0, 1, n).clamp(max=BELOW_ONE)
    tokens = torch.zeros(n, 3, dtype=torch.int64)
    tokens[:, 1:] = pair
    cu = torch.arange(0, 3 * n + 1, 3, dtype=torch.int32)
    mask = torch.tensor([1, 3, 5]).repeat(n)
    step = 20 if few else n  # sequences of a call: both ways to the sums
    for b in range(0, 400 if few else n, step):
        r = slice(3 * b, 3 * (b + step))
        accepted, path, out = (t.cpu() for t in fused.verify_drafts(
            logits[r].cuda()[:, :vocab], tokens.view(-1)[r].cuda(), uniforms[r].cuda(), torch.ones(step, device="cuda"),
            cu[:step + 1].cuda(), 3, mask[r].cuda()))
        first = out[:, :1]
        assert bool((first == pair[b:b + step]).any(1).all()), (b, first[~(first == pair[b:b + step]).any(1)].view(-1).tolist())
        kept = accepted == 1
        assert bool((kept | (accepted == 0)).all()) and bool((path[kept, 0] == 2).all())


@pytest.mark.gpu
def test_sizes_that_pass_32_bits_are_refused(cuda_device):
    """Not taken as what is left of them."""
    good = Batch([3, 2], 64, torch.bfloat16, "chosen", seed=1).on_gpu()
    with pytest.raises(ValueError, match="2\\^31"):
        fused.verify_drafts(**{**good, "max_seqlen_q": (1 << 32) + 8})
    row = torch.empty(1, (1 << 32) + 8, dtype=torch.bfloat16, device="cuda")
    one = dict(logits=row, tokens=good["tokens"][:1], uniforms=good["uniforms"][:1], temperatures=good["temperatures"][:1],
               cu_seqlens_q=torch.tensor([0, 1], dtype=torch.int32, device="cuda"), max_seqlen_q=1)
    with pytest.raises(ValueError, match="2\\^31"):
        fused.verify_drafts(**one)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,form,lens,vocab,times,steps", [
    (torch.bfloat16, "tree", [62] * 20, 4000, 45, 3),       # 446 MB: rows 0, 1 and 2 steps behind, the rest
    (torch.bfloat16, "tree", [62] * 20, 4000, 87, 7),       # 863 MB: 3 to 6 steps behind as well
    (torch.bfloat16, "chosen", [12] * 20, 4000, 450, 7),    # 864 MB
    (torch.bfloat16, "sampled", [12] * 20, 4000, 230, 7),   # 442 MB and as much of the draft model's
    (torch.float32, "sampled", [9] * 20, 4001, 160, 7),     # 461 MB and as much
    (torch.bfloat16, "tree", [62, 61, 64, 60], 151_936, 6, 3),  # 450 MB in 24 sequences, whose ways the sums' kernel finds
    (torch.float32, "tree", [64] * 8, 7, 7400, 1)])         # 106 MB of the shortest rows that get to several passes
def test_batches_that_take_their_rows_in_several_passes(cuda_device, dtype, form, lens, vocab, times, steps):
    """Limits of 200 MB (100 MB without a draft model's logits) for the last pass, each taking half of what was left."""
    x = Batch(lens, vocab, dtype, form, seed=vocab + len(lens), greedy=0.2, width=9.0)
    x.uniforms *= 0.2  # ways of some length
    x.uniforms[x.cu[:-1].long()] *= 5.0
    rng = random.Random(vocab)
    for q0, n in zip(x.cu.tolist(), lens):
        for i in range(1, n):
            up = q0 + (i - 1 if x.mask is None else (int(x.mask[q0 + i]) & (1 << i) - 1).bit_length() - 1)
            if form != "sampled" and rng.random() < 0.85:  # most drafts are the best behind their rows, but for later siblings
                x.logits[up, x.tokens[q0 + i]] = x.logits[up].max() + 4.0
    want = x.want()
    rows, width = len(x.tokens), -(-vocab // 8) * 8
    passes = 1 + sum(rows * times * vocab * x.logits.element_size() * (2 if form == "sampled" else 1) >= at << 20
                     for at in ((200, 400, 800) if form == "sampled" else (100, 400, 800)))
    assert passes >= {1: 2, 3: 3, 7: 4}[steps] and bool((want[0] >= steps).any()), (passes, want[0])
    a = x.on_gpu()
    for name in ("logits", "draft_logits"):
        if a[name] is not None:
            room = torch.full((rows * times, width), math.nan, dtype=dtype, device="cuda")
            room[:, :vocab] = a[name].repeat(times, 1)
            a[name] = room[:, :vocab]
    for name in ("tokens", "uniforms", "temperatures", "tree_mask"):
        a[name] = a[name].repeat(times) if a[name] is not None else None
    cu, steps_of = a["cu_seqlens_q"], torch.arange(times, device="cuda", dtype=torch.int32)[:, None] * rows
    a["cu_seqlens_q"] = torch.cat(((cu[:-1] + steps_of).view(-1), cu[-1:] + steps_of[-1]))
    same(fused.verify_drafts(**a), [w.repeat(times, *[1] * (w.dim() - 1)) for w in want])
