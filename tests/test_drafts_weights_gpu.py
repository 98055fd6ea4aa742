"""How exactly dm_cache_attn_tree holds the weights of its second product: rows whose values cancel, so that the rounding of the output hides nothing."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from . import drafts_ref as dref
from .test_cache_gpu import _ints

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("N, H, Hk, D", [(5, 12, 3, 128), (15, 4, 1, 128), (64, 8, 2, 128), (7, 8, 2, 256), (16, 4, 1, 256), (100, 4, 1, 256)])
def test_weights_of_values_that_cancel(N, H, Hk, D):
    """Each row sees two keys whose logits lie close together anywhere between -8 and 8, and whose values are 1 and -1.

    A weight is held with the largest of its block of 32 keys brought to 2^7 ... 2^8.  Of x in 2^e ... 2^(e + 1) the first code is x rounded to four bits, which leaves 2^(e - 4) at most, and
    the second code of four bits is off by half of its step, 2^(e - 9): 2^-9 of x.  Where the codes are below 2^-6 each is off by 2^-10 at most, 2^-16 of the block's largest together.
    The logits are exact to 2^-19 of their size, exp2 and the sums to 2^-19; o is rounded to bf16, 2^-8 of itself."""
    B = 6
    g = torch.Generator().manual_seed(N)
    q = torch.zeros(B, N, H, D)
    q[..., 0] = torch.rand(B, N, H, generator=g) * 16 - 8
    q[..., 1] = torch.rand(B, N, H, generator=g) * 0.25 - 0.125
    q = q.to(BF)
    k, v = torch.zeros(B, N + 1, Hk, D, dtype=BF), torch.ones(B, N + 1, Hk, D, dtype=BF)
    k[..., 0], k[:, 1:, :, 1], v[:, 1:] = 1.0, 1.0, -1.0
    T = -(-(N + 1) // 64)
    cache, table = dm.KVCache8.empty(B * T, 64, Hk, D), torch.arange(B * T, dtype=torch.int32).view(B, T).cuda()
    n = dm.dm_cache_append(cache, k.cuda(), v.cuda(), table, _ints([0] * B).cuda())
    tree = dm.dm_draft_tree(torch.full((B, N), -1, dtype=torch.int32, device="cuda"))
    o = dm.dm_cache_attn_tree(q.cuda(), cache, table, n, tree, softmax_scale=1.0).cpu().double()
    ops.check_status("cuda")
    s0 = q[..., 0].double()
    s1 = s0 + q[..., 1].double()
    p0, p1 = torch.sigmoid(s0 - s1), torch.sigmoid(s1 - s0)
    want = (p0 - p1)[..., None].expand(o.shape)
    off = 2.0 ** -8 * want.abs() + 2.0 ** -9 + 2.0 ** -16 + 2 * (2.0 ** -19 * s0.abs().amax() + 2.0 ** -19)
    assert bool(((o - want).abs() <= off).all()), float(((o - want).abs() / off).max())
