"""The weights of a sequence that has no new tokens in a call: none, whatever it holds."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from .test_cache_gpu import _filled, _ints, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D, N, rep", [(128, 1, 4), (128, 3, 5), (128, 8, 4), (128, 20, 4), (256, 1, 4), (256, 3, 5), (256, 20, 4)])
@pytest.mark.parametrize("causal", [True, False])
def test_no_new_tokens_no_weights(causal, D, N, rep):
    lengths, counts = [200, 131, 70], [0, N, 0]
    cache, _, table = _filled(lengths, 32, 2, D, seed=N)
    cache.k8.view(torch.uint8)[int(table[0, 1]), 1, 7] = 0x7F    # a NaN key in a sequence that has nothing to ask
    q = _rand(torch.Generator().manual_seed(N), 3, N, 2 * rep, D).cuda()
    for accumulate in (False, True):
        w = torch.full((3, 2, table.shape[1] * 32), 0.5, device="cuda")
        o, lse = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda(), q_counts=_ints(counts).cuda(), causal=causal, weights=w, accumulate=accumulate, return_lse=True)
        ops.check_status("cuda")
        for b in (0, 2):
            assert torch.equal(w[b], torch.full_like(w[b], 0.5 if accumulate else 0.0))
            assert not bool(o[b].any()) and bool((lse[b] == -torch.inf).all())
        assert bool(w[1].isfinite().all()) and bool(o[1].isfinite().all())
