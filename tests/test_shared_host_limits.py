"""The shared prefixes' calls on the host: refusals and fallbacks at the ends of their ranges."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

from pagedserve_b200 import _native, ops


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


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.fixture
def one_by_one(monkeypatch):
    """paged_decode's arguments where paged_decode_shared leaves a batch to it, on the CPU."""
    calls = []

    def decode(q, k, v, tables, lens, layer, **kw):
        calls.append(dict(kw, q=q, tables=tables, lens=lens, layer=layer))
        kw["out"].zero_()
    monkeypatch.setattr(ops, "_cuda_index", lambda *tensors: 0)
    monkeypatch.setattr(ops, "paged_decode", decode)
    monkeypatch.setattr(torch.cuda, "device", lambda *_: contextlib.nullcontext())
    return calls


def _batch(d=96, batch=3):
    pool = torch.zeros(2, 9, 2, 16, d, dtype=torch.bfloat16)
    return [torch.zeros(batch, 14, d, dtype=torch.bfloat16), pool, pool, torch.zeros(batch, 4, dtype=torch.int32), _i32([5 + i % 7 for i in range(batch)]),
            _i32([0, 2]), _i32([3]), 1]


@pytest.mark.parametrize("args", [_batch(), _batch(64, 2049)], ids=["dims", "sequences"])
def test_what_is_answered_one_by_one_has_work_of_the_stream_in_front(one_by_one, args):
    """paged_decode reads lengths before its predecessor has ended: it gets a copy of them, which is made behind that."""
    out = ops.paged_decode_shared(*args)
    call, = one_by_one
    assert torch.equal(call["lens"], args[4]) and call["lens"].data_ptr() != args[4].data_ptr()
    assert call["layer"] == 1 and call["tables"] is args[3] and call["out"].data_ptr() == out.data_ptr() and call["max_context"] == 64


def test_scratch_of_what_is_answered_one_by_one(one_by_one, monkeypatch):
    """The caller's where it is large enough, else the allocator's: never the buffer that every stream's paged_decode uses."""
    args = _batch()
    need = ops.decode_workspace_bytes(3, 14, 2, 96, 16, 64, torch.bfloat16)
    assert need > 0
    own, small = torch.empty(need, dtype=torch.uint8), torch.empty(16, dtype=torch.uint8)
    for given in (own, small, None):
        ops.paged_decode_shared(*args, workspace=given)
    first, second, third = (c["workspace"] for c in one_by_one)
    assert first is own and second is not small and second.nbytes >= need and third.nbytes >= need
    with pytest.raises(ValueError, match="16 bytes"):
        ops.paged_decode_shared(*args, workspace=torch.empty(need + 8, dtype=torch.uint8)[8:])


def test_groups_are_checked_where_each_sequence_is_answered_by_itself(one_by_one, monkeypatch):
    args, seen = _batch(), []
    monkeypatch.setattr(ops, "_call", lambda dev, fn, what, *a: seen.append(a))
    err = torch.zeros(1, dtype=torch.int32)
    ops.paged_decode_shared(*args, error_flag=err)
    assert seen == [(args[5].data_ptr(), args[6].data_ptr(), 3, 1, err.data_ptr())]
    ops.paged_decode_shared(*args)  # nobody to tell
    assert len(seen) == 1 and len(one_by_one) == 2


def test_check_groups_refuses():
    lib = _native.load()
    keep, p = _buffer()
    inv = _native.PSB_ERR_INVALID
    assert lib.psb_check_groups(None, p, 1, 1, p, None) == inv and lib.psb_check_groups(p, None, 1, 1, p, None) == inv
    assert lib.psb_check_groups(p, p, -1, 1, p, None) == inv and lib.psb_check_groups(p, p, 1, -1, p, None) == inv
    assert lib.psb_check_groups(p, None, 1, 0, None, None) == 0


def test_verify_tokens_writes_over_none_of_its_inputs():
    logits, u, heat = torch.zeros(5, 30), torch.zeros(5, 2), torch.ones(2)
    ids, bounds = torch.zeros(16, dtype=torch.int64), torch.zeros(16, dtype=torch.int32)
    bounds[:3] = _i32([0, 2, 5])
    new, counts = torch.zeros(5, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    for out in ((ids[1:6], counts), (ids[4:9], counts), (new, bounds[1:3]), (new, bounds[2:4]), (u.view(torch.int64).view(-1), counts),
                (new, heat.view(torch.int32)), (new, new.view(torch.int32)[4:6])):
        with pytest.raises(ValueError, match="overlap"):
            ops.verify_tokens(logits, ids[:5], bounds[:3], u, heat, out=out)
    for out in ((ids[5:10], counts), (new, bounds[3:5])):  # side by side is apart
        with pytest.raises(ValueError, match="CUDA"):
            ops.verify_tokens(logits, ids[:5], bounds[:3], u, heat, out=out)
    with pytest.raises(ValueError, match="CUDA"):  # nothing shares nothing
        ops.verify_tokens(logits[:0], ids[4:4], torch.zeros(3, dtype=torch.int32), u[:0], heat, out=(ids[6:6], counts))
    assert not ops._overlap(ids[6:6], ids) and ops._overlap(ids[6:7], ids)
