"""Requests that share the blocks of one prompt: the host's bookkeeping, on a CPU pool."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from pagedserve_b200 import BlockManager, PagedKVCache


def _cache(blocks=12, bs=4):
    return PagedKVCache(blocks, 2, 1, 8, block_size=bs, dtype=torch.float32, device="cpu")


def _fill(cache, request_id, first, last, seed):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(2, last, 2, 1, 8, generator=g)  # [layer, token, k or v, head, dim]
    for layer in range(2):
        for i in range(first, last):
            cache.write_token(request_id, layer, i, rows[layer, i, 0], rows[layer, i, 1])
    return rows


def _read(cache, request_id, layer, n):
    return torch.stack([torch.stack(cache.read_token(request_id, layer, i)) for i in range(n)]) if n else torch.empty(0, 2, 1, 8)


def test_manager_shares_whole_blocks():
    m = BlockManager(6, 4)
    assert m.allocate("a", 10) == [0, 1, 2]
    assert m.fork("a", "b", 10) == ([0, 1, 3], (2, 3))
    assert m.fork("a", "c", 8) == ([0, 1], None)
    assert m.fork("b", "d", 3) == ([4], (0, 4))
    assert m.fork("a", "e", 0) == ([], None)
    assert [m.holders(x) for x in (0, 1, 2, 3, 4)] == [3, 3, 1, 1, 1] and m.free_blocks == 1
    m.free("a")
    assert [m.holders(x) for x in (0, 1)] == [2, 2] and m.free_blocks == 2
    m.free("c")
    m.free("b")
    m.free("e")
    assert list(m._free) == [5, 2, 0, 1, 3] and not m._shares
    m.free("d")
    assert m.free_blocks == 6


def test_manager_refuses_a_fork():
    m = BlockManager(3, 4)
    m.allocate("a", 9)
    with pytest.raises(KeyError):
        m.fork("x", "b", 4)
    with pytest.raises(ValueError, match="already has blocks"):
        m.fork("a", "a", 4)
    with pytest.raises(ValueError, match="fewer than"):
        m.fork("a", "b", 13)
    with pytest.raises(ValueError, match="negative"):
        m.fork("a", "b", -1)
    with pytest.raises(RuntimeError, match="Not enough KV blocks"):
        m.fork("a", "b", 9)
    assert m.holders(0) == 1 and not m.has_request("b")  # nothing was shared by the fork that failed
    m.free("a")
    assert m.free_blocks == 3


@pytest.mark.parametrize("n", [0, 1, 3, 4, 5, 8, 9])
def test_children_go_their_own_way(n):
    cache = _cache()
    cache.allocate("p", 9)
    rows = _fill(cache, "p", 0, 9, 0)
    cache.fork("p", ["a", "b"], n)
    for name, seed in (("a", 1), ("b", 2), ("p", 3)):
        held = cache.token_count(name)
        cache.append_tokens(name, 3)
        own = _fill(cache, name, held, held + 3, seed)
        for layer in range(2):
            got = _read(cache, name, layer, held + 3)
            torch.testing.assert_close(got[:held], rows[layer, :held], rtol=0, atol=0)
            torch.testing.assert_close(got[held:], own[layer, held:], rtol=0, atol=0)
    for layer in range(2):  # and nobody's tokens were written over
        for name, held in (("a", n), ("b", n), ("p", 9)):
            torch.testing.assert_close(_read(cache, name, layer, held), rows[layer, :held], rtol=0, atol=0)
    for name in ("p", "b", "a"):
        cache.free(name)
    assert cache.free_blocks == 12


def test_fork_refuses_whole():
    cache = _cache(blocks=4)
    cache.allocate("p", 9)
    for ids, n, err in ((["p"], 4, ValueError), (["a", "a"], 4, ValueError), (["a"], 10, ValueError), (["a"], -1, ValueError),
                        (["a", "b"], 9, RuntimeError)):
        with pytest.raises(err):
            cache.fork("p", ids, n)
    with pytest.raises(KeyError):
        cache.fork("x", ["a"])
    with pytest.raises(KeyError):
        cache.token_count("a")
    cache.fork("p", [])
    cache.fork("p", ["a", "b"], 8)
    assert cache.free_blocks == 1 and cache.token_count("a") == 8


def test_shared_prefixes():
    cache = _cache(blocks=64)
    cache.allocate("p", 18)
    cache.fork("p", ["a", "b"])          # 4 whole blocks shared
    cache.fork("p", ["c"], 8)            # 2 of them
    cache.allocate("x", 9)
    cache.allocate("y", 0)
    cache.fork("x", ["z"], 7)
    for ids, cu, prefix in (([], [0], []), (["x"], [0, 1], [0]), (["y", "y"], [0, 1, 2], [0, 0]),
                            (["a", "b"], [0, 2], [16]), (["a", "b", "p", "c"], [0, 4], [8]),
                            (["a", "x", "b"], [0, 1, 2, 3], [0, 0, 0]),
                            (["c", "a", "y", "x", "z"], [0, 2, 3, 5], [8, 0, 4])):
        got = cache.shared_prefixes(ids)
        assert [g.dtype for g in got] == [np.int32, np.int32]
        assert got[0].tolist() == cu and got[1].tolist() == prefix, ids
    with pytest.raises(KeyError):
        cache.shared_prefixes(["nobody"])


def test_random_forks_and_frees_keep_the_books():
    rng = random.Random(0)
    cache, live = _cache(blocks=200), []
    for step in range(400):
        if live and rng.random() < 0.45:
            cache.free(live.pop(rng.randrange(len(live))))
        elif live and rng.random() < 0.6:
            parent = rng.choice(live)
            n = rng.randint(0, cache.token_count(parent))
            if cache.free_blocks:
                cache.fork(parent, [f"r{step}"], n)
                live.append(f"r{step}")
        elif cache.free_blocks >= 10:
            cache.allocate(f"r{step}", rng.randint(0, 40))
            live.append(f"r{step}")
        held = {}
        for name in live:
            for blk in cache.get_block_table(name).get_blocks():
                held[blk] = held.get(blk, 0) + 1
        assert cache.used_blocks == len(held)
        assert all(cache.block_manager.holders(blk) == n for blk, n in held.items())
        assert not set(held) & set(cache.block_manager._free)
    for name in live:
        cache.free(name)
    assert cache.free_blocks == 200 and not cache.block_manager._shares
