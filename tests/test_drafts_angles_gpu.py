"""dm_cache_append_rotary: angles at which a channel all but vanishes, where an angle rounded to 32 bits would show in the first digits."""
import math

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("quarter", [False, True])
def test_channels_that_almost_vanish(quarter, interleaved):
    """Positions up to 2^20 at which the angle of some frequency lies 2^-20 ... 2^-17 from an odd multiple of pi / 2 (quarter) or a multiple of pi: the pair (x, 0) becomes
    (x cos, x sin), one of them as small as that.

    The angle is counted in turns in 64 bits: three roundings, 2^-51 of itself.  Cosine and sine are then exact to a few units of their own, 2^-20, and the channel is rounded to bf16, 2^-8."""
    F, D, most = 8, 128, 48
    freqs = torch.tensor([1.0, 0.97, 0.81, 0.77, 0.63, 0.59, 0.43, 0.31])
    t = torch.arange(1, 1 << 20, device="cuda").double()
    pick = []                                                    # (position, pair)
    for j in range(F):
        a = t * freqs[j].double().cuda()
        small = (a.cos() if quarter else a.sin()).abs()
        at = ((small > 2.0 ** -20) & (small < 2.0 ** -17)).nonzero()[:most // F, 0]
        pick += [(int(t[i]), j) for i in at]
    assert len(pick) > 16
    N = len(pick)
    pos = torch.tensor([p for p, _ in pick], dtype=torch.int32)
    q = torch.zeros(1, N, 2, D)
    first = lambda j: 2 * j if interleaved else j
    second = lambda j: 2 * j + 1 if interleaved else j + F
    for i, (_, j) in enumerate(pick):
        q[0, i, 0, first(j)] = 1.0 + (i % 16) / 16
    q = q.to(torch.bfloat16).cuda()
    k = torch.zeros(1, N, 1, D, device="cuda", dtype=torch.bfloat16)
    cache = dm.KVCache8.empty(2, 64, 1, D)
    out, _ = dm.dm_cache_append_rotary(cache, q, k, k, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), freqs.cuda(),
                                       offsets=pos.cuda()[None], interleaved=interleaved)
    ops.check_status("cuda")
    for i, (p, j) in enumerate(pick):
        x, a = float(q[0, i, 0, first(j)]), p * float(freqs[j])
        for at, want in ((first(j), x * math.cos(a)), (second(j), x * math.sin(a))):
            got = float(out[0, i, 0, at])
            assert abs(got - want) <= (2.0 ** -8 + 2.0 ** -20) * abs(want) + x * a * 2.0 ** -51, (p, j, got, want)
