"""Block tables with far more room than is held, as a loop keeps that captures its step once for the longest length."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from .test_cache_gpu import _filled, _ints, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D, N, rep, T", [(128, 1, 4, 300), (128, 6, 4, 300), (128, 512, 4, 1 << 20), (256, 1, 4, 300), (256, 256, 4, 1 << 20)])
def test_room_to_spare(D, N, rep, T):
    lengths = [700, 64]
    cache, _, table = _filled(lengths, 64, 2, D, seed=N)
    q = _rand(torch.Generator().manual_seed(N), 2, N, 2 * rep, D).cuda()
    wide = torch.full((2, T), -7, dtype=torch.int32, device="cuda")      # what lies beyond the lengths names no page
    wide[:, :table.shape[1]] = table.cuda()
    want = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda(), return_lse=True)
    got = dm.dm_cache_attn(q, cache, wide, _ints(lengths).cuda(), return_lse=True)
    ops.check_status("cuda")
    seen = want[1].isfinite()
    # the same sums in another order, rounded to bf16 once
    assert torch.allclose(got[0].float(), want[0].float(), rtol=2.0 ** -7, atol=2.0 ** -9 * float(want[0].abs().max()))
    assert torch.equal(got[1].isfinite(), seen) and torch.allclose(got[1][seen], want[1][seen], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("D, N, rep", [(128, 1, 4), (128, 4, 4), (128, 7, 4), (128, 12, 4), (256, 1, 4), (256, 12, 4)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weights_with_room_to_spare(accumulate, D, N, rep):
    lengths = [700, 64]
    cache, _, table = _filled(lengths, 64, 2, D, seed=N)
    q = _rand(torch.Generator().manual_seed(N), 2, N, 2 * rep, D).cuda()
    wide = torch.full((2, 200), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table.cuda()
    out = []
    for t in (table.cuda(), wide):
        w = torch.full((2, 2, t.shape[1] * 64 + 33), 0.25, device="cuda")
        dm.dm_cache_attn(q, cache, t, _ints(lengths).cuda(), weights=w, accumulate=accumulate)
        out.append(w)
    ops.check_status("cuda")
    for b, n in enumerate(lengths):
        assert torch.allclose(out[1][b, :, :n], out[0][b, :, :n], rtol=1e-4, atol=1e-6)
        for w in out:
            assert bool((w[b, :, n:] == (0.25 if accumulate else 0.0)).all())
