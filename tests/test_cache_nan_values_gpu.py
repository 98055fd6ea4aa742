"""A NaN among the held values belongs to its channel of the rows that see its token: a draft's or a prompt's later token must not reach an earlier row through a product
with zero."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from .test_cache_gpu import _filled, _ints, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D, N, rep", [(128, 1, 4), (128, 4, 2), (128, 5, 3), (128, 8, 4), (128, 9, 4), (128, 70, 4), (256, 1, 4), (256, 3, 2), (256, 5, 3), (256, 9, 2), (256, 45, 3)])
@pytest.mark.parametrize("n", [96, 331])
@pytest.mark.parametrize("causal", [True, False])
def test_a_nan_value_reaches_the_rows_that_see_it(causal, n, D, N, rep):
    Hk, lengths = 2, [n, n, n]
    counts = [N, N, max(1, N - 2)]
    cache, _, table = _filled(lengths, 32, Hk, D, seed=N)
    q = _rand(torch.Generator().manual_seed(2), 3, N, rep * Hk, D).cuda()
    args = dict(q_counts=_ints(counts).cuda(), causal=causal)
    clean = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda(), **args)
    assert bool(clean.isfinite().all())
    want = torch.zeros_like(clean, dtype=torch.bool)
    see = lambda b, j: torch.arange(N) + n - counts[b] >= j if causal else torch.ones(N, dtype=torch.bool)
    # (sequence, token, kv head, channel, code): the last token, one in the middle of the new ones, the first, an old one
    for b, j, h, ch, code in ((0, n - 1, 0, 5, 0x7F), (0, n - (counts[0] + 1) // 2, 1, D - 1, 0xFF), (2, n - counts[2], 1, 64, 0x7F), (2, 40, 0, 77, 0xFF), (2, n - 1, 0, 78, 0x7F)):
        cache.v8.view(torch.uint8)[int(table[b, j // 32]), h, j % 32, ch] = code
        rows = see(b, j) & (torch.arange(N) < counts[b])
        want[b, rows.cuda(), h * rep:(h + 1) * rep, ch] = True
    o = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda(), **args)
    ops.check_status("cuda")
    assert torch.equal(o.isnan(), want)
    assert torch.equal(o[1], clean[1])
    # what is not NaN is what it was, but for a code's worth where that token is seen, and the roundings of another order of the sum
    assert torch.allclose(o[~want].float(), clean[~want].float(), rtol=2.0 ** -6, atol=2.0 ** -7 * float(clean.abs().max()))


@pytest.mark.parametrize("D, N, rep", [(128, 5, 3), (128, 40, 2), (256, 5, 3), (256, 40, 2)])
def test_only_nan_tokens_unseen(D, N, rep):
    """Every new token's V is NaN but the first's: the first row sees none of them."""
    n = 200
    cache, _, table = _filled([n], 64, 1, D, seed=1)
    q = _rand(torch.Generator().manual_seed(3), 1, N, rep, D).cuda()
    clean = dm.dm_cache_attn(q, cache, table.cuda(), _ints([n]).cuda())
    for j in range(n - N + 1, n):
        cache.v8.view(torch.uint8)[int(table[0, j // 64]), 0, j % 64] = 0x7F
    o, lse = dm.dm_cache_attn(q, cache, table.cuda(), _ints([n]).cuda(), return_lse=True)
    ops.check_status("cuda")
    assert torch.allclose(o[0, 0].float(), clean[0, 0].float(), rtol=2.0 ** -6, atol=2.0 ** -7 * float(clean.abs().max()))
    assert bool(o[0, 1:].isnan().all()) and bool(lse.isfinite().all())
