"""Prefill at a softmax scale of zero: the mean of V over the keys that a row sees."""

import numpy as np
import pytest
import torch

from kavor_amd.layers.attention import varlen_prefill
from tests.helpers import TOL, gen, randn_bf16


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1e-60])
@pytest.mark.parametrize("causal", [True, False])
def test_a_scale_of_zero_gives_the_mean(cuda_device, scale, causal):
    g, qlens, klens, hq, hkv = gen(1), [1, 70, 9], [40, 70, 200], 4, 2
    q = randn_bf16((sum(qlens), hq, 128), g)
    k, v = (randn_bf16((sum(klens), hkv, 128), g) for _ in range(2))
    cq, ck = (torch.tensor(np.cumsum([0] + n), dtype=torch.int32) for n in (qlens, klens))
    d = cuda_device
    got = varlen_prefill(q.to(d), k.to(d), v.to(d), max_seqlen_q=70, cu_seqlens_q=cq.to(d), max_seqlen_k=200,
                         cu_seqlens_k=ck.to(d), softmax_scale=scale, causal=causal).cpu()
    for s in range(3):
        mine = v[ck[s]:ck[s + 1]].double().repeat_interleave(hq // hkv, 1)
        for i in range(qlens[s]):
            n = i + 1 + klens[s] - qlens[s] if causal else klens[s]
            torch.testing.assert_close(got[cq[s] + i].double(), mine[:n].mean(0), **TOL)
