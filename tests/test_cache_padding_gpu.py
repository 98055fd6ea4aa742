"""Queries behind q_counts are no rows: whatever they hold, outputs and weights have the bits that zeros there give."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from .test_cache_gpu import _filled, _ints, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D, N, rep", [(128, 4, 2), (128, 4, 4), (128, 8, 3), (128, 16, 4), (128, 90, 3), (256, 8, 2), (256, 16, 4), (256, 50, 3)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_what_lies_behind_q_counts_is_not_seen(D, N, rep, accumulate):
    lengths = [300, 700, 129, 64, 40]
    counts = [N // 2 + 1, 1, N - 1, 0, N]
    cache, _, table = _filled(lengths, 64, 2, D, seed=N)
    q = _rand(torch.Generator().manual_seed(N), len(lengths), N, 2 * rep, D).cuda()
    behind = (torch.arange(N)[None] >= _ints(counts)[:, None]).cuda()
    got = []
    for fill in (0.0, float("nan"), float("inf"), float("-inf"), 3e38):
        w = torch.full((len(lengths), 2, table.shape[1] * 64 + 70), 0.5, device="cuda")
        o, lse = dm.dm_cache_attn(torch.where(behind[..., None, None], torch.tensor(fill, dtype=q.dtype, device="cuda"), q), cache, table.cuda(), _ints(lengths).cuda(),
                                  q_counts=_ints(counts).cuda(), weights=w, accumulate=accumulate, return_lse=True)
        got.append((o, lse, w))
    ops.check_status("cuda")
    assert all(bool(t.isfinite().all()) for t in (got[0][0], got[0][2]))
    for i, other in enumerate(got[1:]):
        for name, x, y in zip(("o", "lse", "weights"), got[0], other):
            assert torch.equal(x, y), (i, name)
    # a sequence's weights add up to its rows that see anything, and nothing is added behind what it holds
    rows = torch.minimum(_ints(counts), _ints(lengths)).double()
    sums = got[0][2].double().sum(2).cpu() - (0.5 * got[0][2].shape[2] if accumulate else 0.0)
    assert torch.allclose(sums, rows[:, None].expand(-1, 2) * rep, atol=1e-3)
