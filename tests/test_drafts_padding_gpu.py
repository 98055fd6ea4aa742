"""dm_cache_attn_tree over sequences that begin with zeros (padding on the left): the reference that a row's products count in comes from there, and the rest is far above it."""
import ctypes
import math

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import _lib, ops

from . import cache_ref as ref
from . import drafts_ref as dref
from .test_cache_gpu import _ints, _rand
from .test_drafts_divided_gpu import SHAPES, _divided, _plan, _wide
from .test_drafts_gpu import _attended

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _padded(B, n, Hk, D, head, kind, seed, P=64):
    """A cache of n[b] tokens of which the first `head` are zeros in V, and in K too where kind says so; or all V zero, or as small as codes get."""
    g = torch.Generator().manual_seed(seed)
    k, v = _rand(g, B, max(n), Hk, D), _rand(g, B, max(n), Hk, D)
    if kind == "values":
        v[:, :head] = 0
    elif kind == "both":
        k[:, :head], v[:, :head] = 0, 0
    elif kind == "all":
        v[:] = 0
    elif kind == "tiny":                                         # the head's values 2^-120 of the others', which begin inside a block
        v[:, :head] *= 2.0 ** -120
    elif kind == "all tiny":
        v *= 2.0 ** -118
    T = -(-max(n) // P)
    cache, table = ref.make_cache(B * T, P, Hk, D), ref.make_table(B, T, B * T, seed)
    dm.dm_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"), counts=_ints(n).cuda())
    return cache, table


@pytest.mark.parametrize("kind", ["values", "both", "all", "tiny", "all tiny"])
@pytest.mark.parametrize("divided", [False, True])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_zeros_first(N, H, Hk, D, rows, divided, kind):
    """The definition, with logits up to about 25 above those of the padding."""
    n = [N + 20, N + 70, N + 300, N + 900]
    cache, table = _padded(4, n, Hk, D, 70, kind, N)
    if divided:
        table = _wide(table, 64)
        _divided(4, N, H, Hk, D, table, 64, rows)
    else:
        assert _plan(4, N, H, Hk, D, table, 64)[0] > 0
    g = torch.Generator().manual_seed(N)
    _attended(_rand(g, 4, N, H, D, scale=8.0), cache, table, _ints(n), None, dref.make_parents("any", 4, N, seed=1))


@pytest.mark.parametrize("kind", ["values", "both", "all"])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_rows_behind_padding_are_not_made_one_by_one(N, H, Hk, D, rows, kind):
    """Many whole units whose logits rise far above the padding's: rows are marked only where fp32 has no room for their products.

    In powers of two: a padding's logits are 0 or more, its V scale counts as -86, and 40 above its products, at -46 or above, lies the reference u of all products.  A row is marked for products above
    u + 95, 49 at least: its largest logit, rounded up to a whole number, plus the exponent of a block's V scale is above that.  Its LSE is not below its largest logit."""
    B, P, head = 200, 64, 70
    n = [N + 100 + b % 60 for b in range(B)]
    cache, table = _padded(B, n, Hk, D, head, kind, N)
    _divided(B, N, H, Hk, D, table, P, rows)
    g = torch.Generator().manual_seed(N)
    q = _rand(g, B, N, H, D, scale=8.0).cuda()
    table, lengths = table.cuda(), _ints(n).cuda()
    tree = dm.dm_draft_tree(dref.make_parents("any", B, N, seed=1).cuda())
    L = _lib.lib()
    size, at = L.dm_cache_attn_tree_workspace_bytes(B, N, H, Hk, D, table.shape[1], P), L.dm_dbg_cache_tree_plan(B, N, H, Hk, D, table.shape[1], P, 3)
    ws = torch.zeros(size, device="cuda", dtype=torch.uint8)
    o, lse = torch.empty(B, N, H, D, device="cuda", dtype=BF), torch.empty(B, H, N, device="cuda")
    from delta_matching_b200.cache import _c_cache, _check_cache
    _lib.check(L.dm_cache_attn_tree(ctypes.byref(_c_cache(cache, *_check_cache(cache))), q.data_ptr(), *q.stride()[:3], B, N, H, table.data_ptr(), table.stride(0), table.shape[1],
                                    lengths.data_ptr(), None, tree.seen.data_ptr(), *tree.seen.stride()[:2], D ** -0.5, o.data_ptr(), lse.data_ptr(), ws.data_ptr(), size,
                                    ops.status_word(q.device).data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    ops.check_status("cuda")
    assert at + B * H * N <= size
    marked = ws[at:at + B * H * N].view(B, H, N) != 0
    most = float(cache.vs.nan_to_num(0.0).max().log2())
    assert not bool((marked & (lse < (48.0 - most) * math.log(2.0))).any())
    assert kind == "all" or float((lse > 15.0).float().mean()) > 0.5          # (the logits do rise)
    want, lse2 = dm.dm_cache_attn_tree(q, cache, table, lengths, tree, return_lse=True)
    assert torch.equal(o, want) and torch.equal(lse, lse2)
