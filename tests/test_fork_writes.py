"""Writes through requests that share blocks: what others hold too is not changed."""

from __future__ import annotations

import pytest
import torch

from pagedserve_b200 import PagedKVCache, paged_decode_attention_with_write, rope_and_write_tokens, write_tokens


def _forked(device="cpu", bits=16):
    cache = PagedKVCache(12, 2, 1, 8 if device == "cpu" else 64, block_size=4 if device == "cpu" else 16,
                         dtype=torch.float32 if device == "cpu" else torch.bfloat16, device=device, kv_bits=bits)
    bs = cache.block_size
    cache.allocate("p", 2 * bs + 1)
    cache.fork("p", ["a", "b"])
    return cache, bs


def test_write_token_refuses_a_shared_block():
    cache, bs = _forked()
    row = torch.ones(1, 8)
    cache.kv_cache.k_cache.zero_()
    for name in ("p", "a", "b"):
        for pos in (0, bs - 1, 2 * bs - 1):
            with pytest.raises(ValueError, match="held by other requests"):
                cache.write_token(name, 0, pos, row, row)
        cache.write_token(name, 1, 2 * bs, row, row)  # its own
    assert not cache.kv_cache.k_cache[0].any()
    cache.free("p")
    with pytest.raises(ValueError, match="held by other requests"):
        cache.write_token("a", 0, 0, row, row)
    cache.free("b")
    cache.write_token("a", 0, 0, row, row)  # alone again
    assert cache.read_token("a", 0, 0)[0].eq(1).all()


def test_batched_writes_refuse_a_shared_block():
    cache, bs = _forked()
    key = torch.ones(2, 1, 8)
    with pytest.raises(ValueError, match="of request 'b' is held by other requests"):
        write_tokens(cache, ["a", "b"], [2 * bs, 1], 0, key, key)
    with pytest.raises(ValueError, match="of request 'a' is held by other requests"):
        rope_and_write_tokens(torch.ones(2, 2, 1, 8), key, key, torch.ones(2, 8), torch.ones(2, 8), cache, ["a", "b"], [0, 2 * bs], 0)
    cache.check_writable(["a", "b"], [2 * bs, 2 * bs])
    cache.check_writable([], [])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_writes_on_the_device(bits):
    cache, bs = _forked("cuda", bits)
    kv = cache.kv_cache
    pools = (kv.kv_codes, kv.kv_params) if bits == 4 else (kv.k_cache, kv.v_cache)
    for pool in pools:
        pool.zero_()
    q, key = torch.ones(2, 2, 1, 64, device="cuda").bfloat16(), torch.ones(2, 1, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="of request 'b' is held by other requests"):
        paged_decode_attention_with_write(q, key, key, cache, ["a", "b"], [2 * bs, 3], 0)
    with pytest.raises(ValueError, match="held by other requests"):
        write_tokens(cache, ["b", "a"], [3, 2 * bs], 0, key, key)
    assert not any(pool.any() for pool in pools)
    for _ in range(2):
        out = paged_decode_attention_with_write(q, key, key, cache, ["a", "b"], [2 * bs, 2 * bs], 0)
    write_tokens(cache, ["p", "a"], [2 * bs, 2 * bs], 1, key, key)
    assert torch.isfinite(out).all() and all(pool.any() for pool in pools)
