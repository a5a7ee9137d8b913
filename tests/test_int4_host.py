"""Refusals of the 4-bit pool's and the block tables' entry points, without a GPU."""

from __future__ import annotations

import pytest
import torch

from pagedserve_b200 import _native, ops


def _pools(dtype=torch.bfloat16, layers=1, blocks=4, hkv=2, bs=16, d=64):
    return (torch.zeros(layers, blocks, hkv, 2, bs, d // 2, dtype=torch.uint8),
            torch.zeros(layers, blocks, hkv, 2, bs, 2, dtype=dtype))


def _rows(t=3, h=2, d=64, dtype=torch.bfloat16):
    return torch.zeros(t, h, d, dtype=dtype)


SLOTS = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("change,message", [
    (dict(codes=torch.zeros(1, 4, 2, 2, 16, 32)), "kv_codes must be uint8"),
    (dict(codes=torch.zeros(1, 4, 2, 3, 16, 32, dtype=torch.uint8)), "kv_codes must be uint8"),
    (dict(params=torch.zeros(1, 4, 2, 2, 16, 3)), "kv_params must be"),
    (dict(params=torch.zeros(1, 4, 2, 2, 16, 2, dtype=torch.float64)), "Unsupported dtype"),
    (dict(codes=torch.zeros(1, 4, 2, 2, 16, 64, dtype=torch.uint8)[..., ::2]), "contiguous"),
    (dict(codes=torch.zeros(1, 4, 2, 2, 16, 129, dtype=torch.uint8)), "head_dim up to"),
    (dict(key=_rows(h=3)), r"key/value must be \[T, 2, 64\]"),
    (dict(value=_rows(t=4)), "key/value must be"),
    (dict(key=_rows(dtype=torch.float16)), "dtype must match"),
    (dict(key=torch.zeros(3, 2, 128, dtype=torch.bfloat16)[..., ::2]), "unit stride"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "slot_mapping must be int64"),
    (dict(slots=torch.zeros(4, dtype=torch.int64)), "slot_mapping must be int64"),
    (dict(layer=1), "Invalid layer"), (dict(layer=-1), "Invalid layer"),
    (dict(flag=torch.zeros(1)), "error_flag"),
    (dict(), "requires CUDA"),
])
def test_write_refusals(change, message):
    codes, params = _pools()
    a = dict(codes=codes, params=params, key=_rows(), value=_rows(), slots=SLOTS, layer=0, flag=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        ops.reshape_and_cache_int4(a["key"], a["value"], a["codes"], a["params"], a["slots"], a["layer"],
                                   error_flag=a["flag"])
    q = _rows(h=4)
    cs = torch.zeros(3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=message):
        ops.rope_reshape_and_cache_int4(q, a["key"], a["value"], cs, cs, a["codes"], a["params"], a["slots"],
                                        a["layer"], error_flag=a["flag"])


@pytest.mark.parametrize("change,message", [
    (dict(q=_rows(h=4, d=32)), "query must be"), (dict(q=_rows(t=2, h=4)), "key/value must be"),
    (dict(q=_rows(h=4, dtype=torch.float32)), "dtype must match"),
    (dict(cos=torch.zeros(2, 64, dtype=torch.bfloat16)), "one .* row per token"),
    (dict(cos=torch.zeros(3, 64)), "dtype must match"),
])
def test_rope_refusals(change, message):
    codes, params = _pools()
    cs = torch.zeros(3, 64, dtype=torch.bfloat16)
    a = dict(q=_rows(h=4), cos=cs)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        ops.rope_reshape_and_cache_int4(a["q"], _rows(), _rows(), a["cos"], cs, codes, params, SLOTS, 0)


def test_gather_refusals():
    codes, params = _pools()
    with pytest.raises(ValueError, match="slot_mapping"):
        ops.gather_cache_int4(codes, params, torch.zeros(2, 2, dtype=torch.int64), 0)
    with pytest.raises(ValueError, match="Invalid layer"):
        ops.gather_cache_int4(codes, params, SLOTS, 5)
    with pytest.raises(ValueError, match="requires CUDA"):
        ops.gather_cache_int4(codes, params, SLOTS, 0)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(2, 4, 32, dtype=torch.bfloat16)), "query must be"),
    (dict(q=torch.zeros(0, 4, 64, dtype=torch.bfloat16)), "Batch must not be empty"),
    (dict(q=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), "divisible"),
    (dict(q=torch.zeros(2, 0, 64, dtype=torch.bfloat16)), "divisible"),
    (dict(q=torch.zeros(2, 4, 64)), "dtype"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "block_tables"),
    (dict(table=torch.zeros(3, 3, dtype=torch.int32)), "block_tables"),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), "context_lens"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "context_lens"),
    (dict(layer=7), "Invalid layer"), (dict(max_context=49), "max_context"), (dict(max_context=-1), "max_context"),
    (dict(error_flag=torch.zeros(1, dtype=torch.int64)), "error_flag"),
    (dict(), "requires CUDA"),
])
def test_decode_refusals(change, message):
    codes, params = _pools()
    a = dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16), table=torch.zeros(2, 3, dtype=torch.int32),
             lens=torch.zeros(2, dtype=torch.int32), layer=0)
    a.update(change)
    rest = {k: v for k, v in a.items() if k in ("max_context", "error_flag")}
    with pytest.raises(ValueError, match=message):
        ops.paged_decode_int4(a["q"], codes, params, a["table"], a["lens"], a["layer"], **rest)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(5, 4, 32, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(5, 3, 64, dtype=torch.bfloat16)), "divisible"),
    (dict(q=torch.zeros(5, 4, 64, dtype=torch.float16)), "dtype"),
    (dict(cu=torch.zeros(3, dtype=torch.int64)), "cu_seqlens"),
    (dict(table=torch.zeros(3, 3, dtype=torch.int32)), "block_tables"),
    (dict(lens=torch.zeros(1, dtype=torch.int32)), "context_lens"),
    (dict(layer=-1), "Invalid layer"), (dict(max_context=100), "max_context"), (dict(most=60), "max_seqlen"),
    (dict(), "requires CUDA"),
])
def test_prefill_refusals(change, message):
    codes, params = _pools()
    a = dict(q=torch.zeros(5, 4, 64, dtype=torch.bfloat16), table=torch.zeros(2, 3, dtype=torch.int32),
             lens=torch.zeros(2, dtype=torch.int32), cu=torch.zeros(3, dtype=torch.int32), layer=0, most=5)
    a.update(change)
    rest = {k: v for k, v in a.items() if k == "max_context"}
    with pytest.raises(ValueError, match=message):
        ops.paged_prefill_int4(a["q"], codes, params, a["table"], a["lens"], a["cu"], a["most"], a["layer"], **rest)


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("change,message", [
    (dict(store=torch.zeros(4, 8)), "table_store"), (dict(store=_i32(4, 8).t()), "table_store"),
    (dict(store=_i32(1, 8).expand(4, 8)), "table_store"),
    (dict(rows=_i32(3)), "must be int32"), (dict(rows=torch.zeros(2, dtype=torch.int64)), "req_rows"),
    (dict(first=_i32(2, 1)), "must be int32"), (dict(second=_i32(1)), "must be int32"),
    (dict(free=torch.zeros(9)), "free_blocks"), (dict(free=_i32(0)), "free_blocks"),
    (dict(state=_i32(2)), "free_state"), (dict(block=0), "block_size"), (dict(), "requires CUDA"),
])
def test_tables_refusals(change, message):
    a = dict(store=_i32(4, 8), rows=_i32(2), first=_i32(2), second=_i32(2), free=_i32(9), state=_i32(4), block=16)
    a.update(change)
    args = (a["store"], a["rows"], a["first"], a["second"], a["free"], a["state"])
    with pytest.raises(ValueError, match=message):
        ops.extend_step(*args, 0, a["block"])
    with pytest.raises(ValueError, match=message):
        ops.trim_tables(*args, a["block"])


def test_free_list():
    ids, state = ops.free_list(5, "cpu", [3, 1, 0, 2, 4])
    assert ids.tolist() == [3, 1, 0, 2, 4] and state.tolist() == [0, 5, 0, 0]
    assert ids.dtype == state.dtype == torch.int32
    for bad in ([0, 1], [0, 1, 2, 3, 3]):
        with pytest.raises(ValueError, match="permutation"):
            ops.free_list(5, "cpu", bad)
    with pytest.raises(ValueError, match="positive"):
        ops.free_list(0, "cpu")


def test_c_entries_check_their_arguments():
    """Null pointers and impossible geometries are answered before any CUDA call; nothing to do is PSB_OK."""
    lib = _native.load()
    inv, ok, bf = _native.PSB_ERR_INVALID, _native.PSB_OK, _native.PSB_BF16

    def write(tokens=1, d=64, hkv=2, bs=16, dtype=bf, layer=0):
        return lib.psb_reshape_and_cache_int4(None, 0, 0, None, 0, 0, None, None, None, tokens, layer, 1, 8, hkv, bs,
                                              d, dtype, None, None)

    assert write() == inv and write(tokens=0) == ok and write(tokens=-1) == inv
    for bad in (dict(d=63), dict(d=258), dict(d=0), dict(hkv=0), dict(bs=0), dict(dtype=7), dict(layer=1)):
        assert write(tokens=0, **bad) == inv
    assert lib.psb_rope_reshape_and_cache_int4(None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, None,
                                               0, None, None, None, 1, 2, 0, 1, 8, 2, 16, 64, bf, None, None) == inv
    assert lib.psb_gather_cache_int4(None, None, None, None, 0, 0, None, 0, 0, 3, 0, 1, 8, 2, 16, 64, bf, None,
                                     None) == inv
    assert lib.psb_gather_cache_int4(None, None, None, None, 0, 0, None, 0, 0, 0, 0, 1, 8, 2, 16, 64, bf, None,
                                     None) == ok
    size = lib.psb_paged_decode_int4_workspace_size
    assert size(4, 14, 2, 64, 16, 4096, bf) > 0
    for bad in ((0, 14, 2, 64, 16, 64, bf), (4, 14, 3, 64, 16, 64, bf), (4, 14, 2, 65, 16, 64, bf),
                (4, 14, 2, 64, 0, 64, bf), (4, 14, 2, 64, 16, -1, bf), (4, 14, 2, 64, 16, 64, 9),
                (4, 14, 2, 512, 16, 64, bf)):
        assert size(*bad) == 0
    assert lib.psb_paged_decode_int4(None, 0, 0, None, 0, 0, None, None, None, 4, None, 1, 14, 0, 1, 8, 2, 16, 64, bf,
                                     64, 0.125, None, 0, None, None) == inv
    assert lib.psb_paged_prefill_int4(None, 0, 0, None, None, None, 4, None, None, 0, 0, None, 1, 5, 5, 64, 14, 0, 1,
                                      8, 2, 16, 64, bf, 0.125, None, 0, None, None) == inv
    assert lib.psb_paged_prefill_int4(None, 0, 0, None, None, None, 4, None, None, 0, 0, None, 0, 0, 0, 64, 14, 0, 1,
                                      8, 2, 16, 64, bf, 0.125, None, 0, None, None) == ok
    assert lib.psb_paged_prefill_int4(None, 0, 0, None, None, None, 3, None, None, 0, 0, None, 0, 0, 0, 64, 14, 0, 1,
                                      8, 2, 16, 64, bf, 0.125, None, 0, None, None) == inv  # tables narrower than max_context
    psize = lib.psb_paged_prefill_int4_workspace_size
    assert psize(100, 2, 14, 2, 64, 16, 4096, bf) > 0 and psize(100, 2, 14, 3, 64, 16, 4096, bf) == 0
    assert psize(100, 2, 14, 2, 63, 16, 4096, bf) == 0 and psize(-1, 2, 14, 2, 64, 16, 4096, bf) == 0
    assert lib.psb_extend_step(None, 4, 1, 4, None, None, None, 0, None, 5, None, 0, 16, None, None, None, None, None,
                               4, None, None) == ok
    assert lib.psb_extend_step(None, 4, 1, 4, None, None, None, 2, None, 5, None, 0, 16, None, None, None, None, None,
                               4, None, None) == inv
    assert lib.psb_extend_step(None, 3, 1, 4, None, None, None, 0, None, 5, None, 0, 16, None, None, None, None, None,
                               4, None, None) == inv
    assert lib.psb_trim_tables(None, 4, 1, 4, None, None, None, 0, None, 5, None, 16, None, None) == ok
    assert lib.psb_trim_tables(None, 4, 1, 4, None, None, None, 1, None, 5, None, 16, None, None) == inv
