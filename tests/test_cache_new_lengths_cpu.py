"""The C functions that write new lengths refuse a buffer that shares memory with what their kernels read meanwhile: other heads' CTAs would take the new length for the old one."""
import ctypes

import pytest
import torch

from delta_matching_b200 import _lib

from .test_cache_cpu import FINE, _c

B, N, T, M = 3, 5, 4, 6
AT = dict(lengths=0x20000, before=0x30000, counts=0x40000, offsets=0x50000, path=0x60000, table=0x70000, new_table=0x80000)
ENTRIES = dict(lengths=B, before=B, counts=B, offsets=2 * 7 + N, path=2 * 8 + M, table=2 * 9 + T, new_table=2 * 9 + T)      # from the first row's first to the last row's last


def _append(new):
    return _lib.lib().dm_cache_append(ctypes.byref(_c()), FINE, 768, 256, 128, FINE, 768, 256, 128, B, N, AT["table"], 9, T, AT["lengths"], AT["counts"], new, None, None)


def _append_rotary(new):
    return _lib.lib().dm_cache_append_rotary(ctypes.byref(_c()), *(FINE, 768, 256, 128) * 3, B, N, 4, FINE, 64, 0, AT["table"], 9, T, AT["lengths"], AT["offsets"], 7, AT["counts"], FINE, new,
                                             None, None)


def _evict(new):
    return _lib.lib().dm_cache_evict(ctypes.byref(_c()), B, AT["table"], 9, T, AT["lengths"], FINE, 512, 256, AT["new_table"], 9, T, 100, 10, new, FINE, FINE, None, None)


def _keep(new):
    return _lib.lib().dm_cache_keep(ctypes.byref(_c()), B, AT["table"], 9, T, AT["before"], AT["lengths"], AT["path"], 8, M, AT["counts"], new, None, None)


@pytest.mark.parametrize("call, names", [(_append, ("lengths", "counts", "table")), (_append_rotary, ("lengths", "counts", "offsets", "table")), (_evict, ("lengths", "table", "new_table")),
                                         (_keep, ("before", "lengths", "counts", "path", "table"))])
def test_shared_buffers_are_refused(call, names):
    for name in names:
        first, end = AT[name], AT[name] + 4 * ENTRIES[name]
        for new in (first, first - 4 * (B - 1), end - 4):        # the same; the last entry in it; its last entry
            assert call(new) == -1
            assert "new lengths must not share memory with " + name.replace("table", "block table").replace("_", " ") in _lib.last_error(), (name, hex(new))
        if torch.cuda.is_available():                            # (these are no real addresses)
            continue
        for new in (first - 4 * B, end):                         # beside it: what is refused is the device
            assert call(new) != 0
            assert "share memory" not in _lib.last_error(), (name, hex(new))


@pytest.mark.skipif(torch.cuda.is_available(), reason="these are no real addresses")
@pytest.mark.parametrize("call, name, row, n", [(_append, "table", 9, T), (_append_rotary, "offsets", 7, N), (_keep, "path", 8, M), (_keep, "table", 9, T), (_evict, "new_table", 9, T)])
def test_between_rows_is_a_buffer_of_its_own(call, name, row, n):
    """Where the gap between two rows has room for the new lengths they may lie there; one entry further on they may not."""
    for b in range(B - 1):
        first, last = AT[name] + 4 * (b * row + n), AT[name] + 4 * ((b + 1) * row - B)
        for new in range(first - 4, last + 8, 4):
            assert call(new) != 0
            assert ("share memory" in _lib.last_error()) == (not first <= new <= last), (b, hex(new))
