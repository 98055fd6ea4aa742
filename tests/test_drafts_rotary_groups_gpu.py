"""dm_cache_append_rotary where a CTA takes more heads than it has warps: calls of many blocks of tokens, in which fewer CTAs share out the heads, down to one for all of them."""
import pytest
import torch

import delta_matching_b200 as dm

from . import cache_ref as ref
from . import drafts_ref as dref
from .test_cache_gpu import _filled, _ints, _rand
from .test_drafts_gpu import _appended, _freqs

pytestmark = pytest.mark.gpu
WARPS = 8                                                        # heads that a CTA takes at a time


def _groups(B, N, H, Hk, sms=148):
    """(heads of a CTA, CTAs that share out the heads) as csrc/dm_cache_rotary.cu lays a call out: 8 CTAs an SM wanted, whole rounds of a head a warp."""
    heads, blocks, want = 2 * Hk + H, (N + 30) // 32 + 1, 8 * sms
    rounds = -(-heads // WARPS)
    parts = min(rounds, max(1, -(-want // (B * blocks))))
    group = -(-rounds // parts) * WARPS
    return group, -(-heads // group)


@pytest.mark.parametrize("B, N, H, Hk, D, F, interleaved, group, groups", [
    (64, 577, 6, 2, 128, 64, False, 16, 1),                      # 1216 blocks: ten heads, all in one CTA, the second round not full
    (64, 609, 12, 3, 128, 24, True, 24, 1),
    (32, 641, 16, 4, 128, 64, True, 16, 2),                      # about 700 blocks: three rounds, in two CTAs
    (40, 500, 14, 2, 256, 128, False, 16, 2),
    (64, 600, 9, 1, 256, 40, True, 16, 1)])
def test_more_heads_than_warps(B, N, H, Hk, D, F, interleaved, group, groups):
    """Ragged, with starts on, before and behind a block's edge, positions by index and by offsets."""
    assert _groups(B, N, H, Hk, torch.cuda.get_device_properties(0).multi_processor_count) == (group, groups)
    start = _ints([(0, 5, 31, 32, 45)[b % 5] for b in range(B)])
    counts = _ints([N - 7 * (b % 4) if b % 9 else b for b in range(B)])
    T = -(-(45 + N) // 64)
    g = torch.Generator().manual_seed(B)
    cache, pools, table = _filled(start.tolist(), 64, Hk, D, seed=N, T=T)
    offsets = (torch.arange(N) // 3 + 40 * torch.arange(B)[:, None]).to(torch.int32) if interleaved else None
    _appended(cache, pools, table, _rand(g, B, N, H, D), _rand(g, B, N, Hk, D, scale=3.0), _rand(g, B, N, Hk, D), start, _freqs(F), offsets, counts, interleaved)
