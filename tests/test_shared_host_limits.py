"""The shared prefixes' calls on the host: refusals and fallbacks at the ends of their ranges."""

from __future__ import annotations

import ctypes

from pagedserve_b200 import _native


def _buffer():
    keep = ctypes.create_string_buffer(4096)
    return keep, ctypes.cast(keep, ctypes.c_void_p).value + 15 & -16


def test_no_groups_need_their_one_bound_all_the_same():
    lib = _native.load()
    keep, p = _buffer()
    call = lambda cu, pre: lib.psb_paged_decode_shared(p, 896, 64, p, 896, 64, p, p, p, 4, p, cu, pre, 2, 0, 14, 0, 1, 9, 2, 16, 64, 2, 64, 0.1, None, 0,
                                                       None, None)
    assert call(None, None) == _native.PSB_ERR_INVALID and call(None, p) == _native.PSB_ERR_INVALID
    assert call(p, None) == _native.PSB_ERR_WORKSPACE  # the lengths of no prefix may be missing
