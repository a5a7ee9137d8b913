"""The 4-bit cache's bookkeeping and refusals, without a GPU."""

from __future__ import annotations

import pytest
import torch

from pagedserve_b200 import KVCache, PagedKVCache, paged_decode_attention
from pagedserve_b200.model_runner import PagedModelRunner, QwenConfig


def _cache(**kw):
    args = dict(num_blocks=4, num_layers=2, num_kv_heads=2, head_dim=64, block_size=16, dtype=torch.bfloat16,
                device="cpu", kv_bits=4)
    args.update(kw)
    return PagedKVCache(**args)


def test_int4_pools_and_bytes():
    kv = _cache().kv_cache
    assert kv.k_cache is None and kv.v_cache is None and kv.kv_bits == 4
    assert kv.kv_codes.shape == (2, 4, 2, 2, 16, 32) and kv.kv_codes.dtype == torch.uint8
    assert kv.kv_params.shape == (2, 4, 2, 2, 16, 2) and kv.kv_params.dtype == torch.bfloat16
    assert kv.block_bytes == 2 * 2 * 2 * 16 * (32 + 4) and kv.total_bytes == 4 * kv.block_bytes
    assert kv.total_bytes == kv.kv_codes.nbytes + kv.kv_params.nbytes
    plain = KVCache(num_blocks=4, num_layers=2, num_kv_heads=2, head_dim=64, dtype=torch.bfloat16, device="cpu")
    assert plain.kv_bits == 16 and plain.kv_codes is None and plain.kv_params is None


@pytest.mark.parametrize("change,message", [
    (dict(kv_bits=8), "kv_bits must be 4 or 16"), (dict(head_dim=63), "even head_dim"),
    (dict(head_dim=258), "even head_dim"), (dict(dtype=torch.float64), "Unsupported dtype"),
])
def test_int4_pool_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        _cache(**change)


def test_int4_rows_need_a_cuda_device():
    cache = _cache()
    cache.allocate("A", 17)
    row = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA device"):
        cache.write_token("A", 0, 16, row, row)
    with pytest.raises(ValueError, match="CUDA device"):
        cache.read_token("A", 0, 16)
    with pytest.raises(ValueError, match="Expected K/V shape"):
        cache.write_token("A", 0, 16, row[:1], row)
    with pytest.raises(ValueError, match="dtype"):
        cache.write_token("A", 0, 16, row.float(), row)
    with pytest.raises(IndexError):
        cache.write_token("A", 0, 17, row, row)
    block = torch.zeros(2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA device"):
        cache.kv_cache.write_block(0, 0, block, block)
    with pytest.raises(ValueError, match="CUDA device"):
        cache.kv_cache.read_block(0, 0)
    with pytest.raises(IndexError):
        cache.kv_cache.read_block(0, 4)
    with pytest.raises(ValueError, match="requires CUDA"):
        paged_decode_attention(torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16), cache, ["A"], [16], 0)


class _Weights:
    cfg = QwenConfig(layers=2)
    dtype = torch.bfloat16
    device = torch.device("cpu")


@pytest.mark.parametrize("change,message", [
    (dict(kv_bits=8), "kv_bits must be 4 or 16"), (dict(kv_bits=16), "pools do not match"),
    (dict(codes=torch.zeros(2, 4, 2, 2, 16, 64, dtype=torch.uint8)), "pools do not match"),
    (dict(codes=torch.zeros(3, 4, 2, 2, 16, 32, dtype=torch.uint8)), "pools do not match"),
    (dict(codes=torch.zeros(2, 4, 2, 2, 16, 32)), "pools do not match"),
    (dict(params=torch.zeros(2, 5, 2, 2, 16, 2, dtype=torch.bfloat16)), "pools do not match"),
    (dict(params=torch.zeros(2, 4, 2, 2, 16, 2)), "dtypes differ"), (dict(block_size=32), "pools do not match"),
])
def test_runner_refuses_other_pools(change, message):
    kv = _cache().kv_cache
    a = dict(codes=kv.kv_codes, params=kv.kv_params, block_size=16, kv_bits=4)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        PagedModelRunner(_Weights, a["codes"], a["params"], a["block_size"], kv_bits=a["kv_bits"])
