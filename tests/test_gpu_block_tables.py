"""extend_step / trim_tables against the host-side BlockManager and pack_step."""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


def _dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bs,blocks,rows,width", [(16, 400, 40, 32), (1, 300, 9, 64), (32, 64, 300, 8)])
def test_follows_the_block_manager(bs, blocks, rows, width):
    """Random admissions, growth, partial and full releases over a shuffled
    pool: the same ids as BlockManager, the same free list, pack_step's outputs."""
    from pagedserve_b200 import ops
    from pagedserve_b200.paged_kv import BlockManager
    rng = random.Random(bs + blocks)
    order = list(range(blocks))
    rng.shuffle(order)
    bm = BlockManager(blocks, bs, free_order=order)
    free, state = ops.free_list(blocks, "cuda", order)
    store = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
    held = {}
    err = _flag()
    for step in range(25):
        batch = rng.sample(range(rows), rng.randint(1, min(rows, 24)))
        plan = []
        room = bm.free_blocks
        for r in batch:
            n = rng.randint(0, 3 * bs)
            n = min(n, width * bs - held.get(r, 0))
            need = bm.blocks_needed(held.get(r, 0) + n) - bm.blocks_needed(held.get(r, 0))
            if need > room:
                n = 0
            else:
                room -= need
            plan.append(n)
        starts = [held.get(r, 0) for r in batch]
        cu, ctx, slots, pos, tables = ops.extend_step(store, _dev(batch), _dev(starts), _dev(plan), free, state,
                                                      sum(plan), bs, error_flag=err)
        for r, s, n in zip(batch, starts, plan):
            name = f"r{r}"
            extra = bm.blocks_needed(s + n) - bm.blocks_needed(s)
            if not bm.has_request(name):
                bm.allocate(name, s + n)
            elif extra:
                bm.allocate_blocks(name, extra)
            held[r] = s + n
        for r in range(rows):
            ids = bm.get_blocks(f"r{r}") if bm.has_request(f"r{r}") else []
            assert store[r].tolist() == ids + [0] * (width - len(ids))
        pcu, pctx, pslots, ppos, ptab = ops.pack_step(store, _dev(batch), _dev(starts), _dev(plan), sum(plan), bs)
        for a, b in ((cu, pcu), (ctx, pctx), (slots, pslots), (pos, ppos), (tables, ptab)):
            assert a.dtype == b.dtype and torch.equal(a, b)
        # release some requests, whole
        gone = [r for r in held if rng.random() < 0.3]
        if gone:
            ops.trim_tables(store, _dev(gone), _dev([held[r] for r in gone]), _dev([0] * len(gone)), free, state, bs,
                            error_flag=err)
            for r in gone:
                bm.free(f"r{r}")
                del held[r]
        head, count, ticket, _ = state.tolist()
        assert ticket == 0 and count == bm.free_blocks
        ring = free.tolist()
        assert [ring[(head + i) % blocks] for i in range(count)] == list(bm._free)
    assert int(err.item()) == 0


def test_trim_to_a_shorter_length():
    """A rejected draft: blocks past the kept length come back, the rest stays."""
    from pagedserve_b200 import ops
    bs, blocks = 16, 20
    free, state = ops.free_list(blocks, "cuda")
    store = torch.zeros(4, 8, dtype=torch.int32, device="cuda")
    rows = _dev([2, 0])
    ops.extend_step(store, rows, _dev([0, 0]), _dev([50, 40]), free, state, 90, bs)
    assert store[2, :5].tolist() == [0, 1, 2, 3, 0] and store[0, :4].tolist() == [4, 5, 6, 0]
    ops.trim_tables(store, rows, _dev([50, 40]), _dev([17, 33]), free, state, bs)
    assert store[2, :5].tolist() == [0, 1, 0, 0, 0] and store[0, :4].tolist() == [4, 5, 6, 0]
    assert state.tolist() == [7, 15, 0, 0]
    assert [free.tolist()[(7 + i) % blocks] for i in range(15)] == list(range(7, 20)) + [2, 3]


def test_padding_entries_and_out_buffers():
    from pagedserve_b200 import ops
    bs = 4
    free, state = ops.free_list(10, "cuda")
    store = torch.zeros(3, 6, dtype=torch.int32, device="cuda")
    rows, starts, new = _dev([1, -1, 0, -1]), _dev([0, 0, 0, 7]), _dev([5, 3, 1, 2])
    out = (torch.full((5,), 9, dtype=torch.int32, device="cuda"), torch.full((4,), 9, dtype=torch.int32, device="cuda"),
           torch.full((11,), 9, dtype=torch.int64, device="cuda"), torch.full((11,), 9, dtype=torch.int64, device="cuda"),
           torch.full((4, 3), 9, dtype=torch.int32, device="cuda"))
    err = _flag()
    got = ops.extend_step(store, rows, starts, new, free, state, 11, bs, out_width=3, error_flag=err, out=out)
    assert all(a is b for a, b in zip(got, out))
    assert out[0].tolist() == [0, 5, 8, 9, 11] and out[1].tolist() == [5, 0, 1, 0]
    assert out[2].tolist() == [0, 1, 2, 3, 4, -1, -1, -1, 8, -1, -1]
    assert out[3].tolist() == [0, 1, 2, 3, 4, 0, 0, 0, 0, 0, 0]
    assert out[4].tolist() == [[0, 1, 0], [0, 0, 0], [2, 0, 0], [0, 0, 0]]
    assert int(err.item()) == 0 and state.tolist() == [3, 7, 0, 0]


REFUSED = [
    (dict(new=[40, 45]), 128),                         # 6 blocks of 16 wanted, 5 free
    (dict(rows=[1, 1]), 256),                          # a row twice
    (dict(rows=[1, 4]), 4), (dict(starts=[0, -1]), 4), (dict(new=[5, -1]), 4),
    (dict(new=[5, 16 * 6 + 1]), 4),                    # more than the row holds
    (dict(total=7), 32),
    (dict(starts=[0, 2 ** 31 - 1]), 4),
]


@pytest.mark.parametrize("change,bit", REFUSED)
def test_a_refused_step_changes_nothing(change, bit):
    from pagedserve_b200 import ops
    plan = dict(rows=[1, 2], starts=[0, 0], new=[5, 7])
    plan.update({k: v for k, v in change.items() if k != "total"})
    total = change.get("total", sum(plan["new"]))
    free, state = ops.free_list(5, "cuda", [4, 2, 0, 1, 3])
    store = torch.full((4, 6), -3, dtype=torch.int32, device="cuda")
    err = _flag()
    cu, ctx, slots, pos, tables = ops.extend_step(store, _dev(plan["rows"]), _dev(plan["starts"]), _dev(plan["new"]),
                                                  free, state, total, 16, error_flag=err)
    assert int(err.item()) & bit
    assert bool((store == -3).all()) and state.tolist() == [0, 5, 0, 0] and free.tolist() == [4, 2, 0, 1, 3]
    assert bool((slots == -1).all()) and bool((ctx == 0).all()) and bool((tables == 0).all())
    # the next step is carried out
    err.zero_()
    ops.extend_step(store, _dev([0]), _dev([0]), _dev([17]), free, state, 17, 16, error_flag=err)
    assert int(err.item()) == 0 and store[0, :2].tolist() == [4, 2] and state.tolist() == [2, 3, 0, 0]


@pytest.mark.parametrize("rows,held,keep,bit", [([1, 1], [16, 16], [0, 0], 256), ([0, 5], [16, 16], [0, 0], 4),
                                                ([0, 1], [16, 16], [0, 17], 4), ([0, 1], [16, 16], [0, -1], 4),
                                                ([0, 1], [16, 200], [0, 0], 4), ([0, 1], [64, 64], [0, 0], 128)])
def test_a_refused_trim_changes_nothing(rows, held, keep, bit):
    from pagedserve_b200 import ops
    free, state = ops.free_list(5, "cuda")
    store = torch.zeros(3, 6, dtype=torch.int32, device="cuda")
    ops.extend_step(store, _dev([0, 1]), _dev([0, 0]), _dev([16, 16]), free, state, 32, 16)
    before = store.clone(), free.clone(), state.clone()
    err = _flag()
    ops.trim_tables(store, _dev(rows), _dev(held), _dev(keep), free, state, 16, error_flag=err)
    assert int(err.item()) == bit
    assert torch.equal(store, before[0]) and torch.equal(free, before[1]) and torch.equal(state, before[2])


def test_large_step_in_a_graph():
    """A captured extend + trim replayed: the ring turns, the ids stay a
    permutation, several CTAs see the same ring."""
    from pagedserve_b200 import ops
    bs, batch, blocks = 16, 256, 9000
    free, state = ops.free_list(blocks, "cuda")
    store = torch.zeros(300, 600, dtype=torch.int32, device="cuda")
    rng = random.Random(2)
    rows = _dev(rng.sample(range(300), batch))
    new = [rng.randint(1, 500) for _ in range(batch)]
    zero, add = _dev([0] * batch), _dev(new)
    err = _flag()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cu, ctx, slots, pos, tables = ops.extend_step(store, rows, zero, add, free, state, sum(new), bs, error_flag=err)
        ops.trim_tables(store, rows, add, zero, free, state, bs, error_flag=err)
    taken = sum(-(-n // bs) for n in new)
    for step in range(5):
        g.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0 and state.tolist() == [(step + 1) * taken % blocks, blocks, 0, 0]
        assert bool((store == 0).all())
        assert sorted(free.tolist()) == list(range(blocks))
        live = slots.cpu()
        assert bool((live >= 0).all()) and len(set(live.tolist())) == sum(new)


def test_empty_batch():
    from pagedserve_b200 import ops
    free, state = ops.free_list(5, "cuda")
    store = torch.zeros(3, 6, dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    cu, ctx, slots, pos, tables = ops.extend_step(store, none, none, none, free, state, 0, 16)
    assert cu.tolist() == [0] and ctx.numel() == slots.numel() == tables.numel() == 0
    ops.trim_tables(store, none, none, none, free, state, 16)
    assert state.tolist() == [0, 5, 0, 0]
