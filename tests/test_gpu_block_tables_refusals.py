"""Refused table calls as a whole: ids outside the pool, a refused extend_step
followed by the calls that were planned behind it, and lengths past 2^31."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK_RANGE, CONTEXT, POOL, REFUSED = 1, 4, 128, 512


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


def _dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


class _Tables:
    def __init__(self, blocks, rows, width, bs=16, order=None):
        from pagedserve_b200 import ops
        self.ops, self.bs = ops, bs
        self.free, self.state = ops.free_list(blocks, "cuda", order)
        self.store = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
        self.err = _flag()

    def extend(self, rows, starts, new, flag=True):
        return self.ops.extend_step(self.store, _dev(rows), _dev(starts), _dev(new), self.free, self.state, sum(new),
                                    self.bs, error_flag=self.err if flag else None)

    def trim(self, rows, held, keep):
        self.ops.trim_tables(self.store, _dev(rows), _dev(held), _dev(keep), self.free, self.state, self.bs,
                             error_flag=self.err)

    def copy(self):
        return self.store.tolist(), self.ring(), self.state.tolist()

    def same(self, before):
        return self.copy() == before

    def ring(self):
        head, count = self.state.tolist()[:2]
        ids = self.free.tolist()
        return [ids[(head + i) % len(ids)] for i in range(count)]


@pytest.mark.parametrize("bad", [-1, 400, 1 << 30])
@pytest.mark.parametrize("batch,width,new", [(2, 6, 40), (40, 300, 150)])
def test_trim_of_an_id_outside_the_pool_changes_nothing(bad, batch, width, new):
    """Whichever entry it is found in, and however many CTAs the call has."""
    t = _Tables(400, batch, width)
    rows = list(range(batch))
    t.extend(rows, [0] * batch, [new] * batch)
    last = -(-new // 16) - 1
    for row, col in ((0, 0), (batch - 1, last)):
        good = t.store[row, col].item()
        t.store[row, col] = bad
        before = t.copy()
        t.trim(rows, [new] * batch, [0] * batch)
        assert int(t.err.item()) == BLOCK_RANGE and t.same(before)
        t.err.zero_()
        t.store[row, col] = good
    # an id that is kept is not looked at
    t.store[0, 0] = bad
    t.trim(rows, [new] * batch, [16] * batch)
    assert int(t.err.item()) == 0 and t.store[0, 0].item() == bad
    assert len(t.ring()) == 400 - batch and all(0 <= i < 400 for i in t.ring())


@pytest.mark.parametrize("bad", [-1, 9, 1 << 30])
def test_extend_over_an_id_outside_the_pool_changes_nothing(bad):
    t = _Tables(9, 3, 6, order=[4, 2, 0, 1, 3, 5, 6, 7, 8])
    t.free[2] = bad
    t.state.copy_(_dev([7, 9, 0, 0]))  # 7, 8, 4, 2, bad, ...
    before = t.copy()
    cu, ctx, slots, pos, tables = t.extend([0, 2], [0, 0], [33, 20])  # 3 + 2 blocks
    assert int(t.err.item()) & BLOCK_RANGE and t.same(before)
    assert bool((slots == -1).all()) and bool((ctx == 0).all()) and bool((tables == 0).all())
    t.err.zero_()
    t.extend([0, 2], [0, 0], [33, 16])  # the four before it
    assert int(t.err.item()) == 0 and t.store[0, :4].tolist() == [7, 8, 4, 0] and t.store[2, 0].item() == 2


@pytest.mark.parametrize("captured", [False, True])
def test_what_follows_a_refused_step_changes_nothing(captured):
    """extend_step, then the planned trim_tables: when the step was refused for
    lack of blocks, the trim does not hand out blocks the request never got
    (block 0 belongs to another request), nor does a next step whose starts
    have moved on use them; once the flag is cleared all goes on."""
    t = _Tables(6, 4, 8)
    t.extend([3], [0], [16 * 4])                  # request 3: blocks 0 .. 3
    t.extend([1], [0], [10])                      # request 1: block 4
    assert int(t.err.item()) == 0 and t.ring() == [5]
    rows, starts, new, zero = _dev([1]), _dev([10]), _dev([30]), _dev([0])  # two blocks more: one is there
    before = t.copy()

    def step():
        out = t.ops.extend_step(t.store, rows, starts, new, t.free, t.state, 30, 16, error_flag=t.err)
        t.ops.trim_tables(t.store, rows, starts + new, zero, t.free, t.state, 16, error_flag=t.err)
        return out

    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
            new.fill_(1)  # (the next replay's plan: 30 tokens are not its total)
        new.fill_(30)
        torch.cuda.synchronize()
        g.replay()
    else:
        out = step()
    assert int(t.err.item()) == POOL | REFUSED and t.same(before)
    # the step behind it, planned as if the first had been carried out
    cu, ctx, slots, pos, tables = t.extend([1], [40], [1])
    assert bool((slots == -1).all()) and bool((ctx == 0).all()) and bool((tables == 0).all())
    assert int(t.err.item()) == POOL | REFUSED and t.same(before)
    # the host has seen it: request 3 makes room, request 1 goes on where it was
    t.err.zero_()
    t.trim([3], [64], [0])
    t.extend([1], [10], [30])
    assert int(t.err.item()) == 0
    assert t.store[1, :4].tolist() == [4, 5, 0, 0] and t.ring() == [1, 2, 3]


def test_held_lengths_from_the_step_itself():
    """Without a flag: a trim whose held lengths are the step's context_lens
    gives nothing back when the step was refused."""
    t = _Tables(6, 4, 8)
    t.extend([3, 1], [0, 0], [64, 10])
    before = t.copy()
    _, lens, _, _, _ = t.extend([1], [10], [30], flag=False)
    t.ops.trim_tables(t.store, _dev([1]), lens, _dev([0]), t.free, t.state, 16)
    assert t.same(before)
    _, lens, _, _, _ = t.extend([1], [10], [20], flag=False)
    t.ops.trim_tables(t.store, _dev([1]), lens, _dev([0]), t.free, t.state, 16)
    assert t.ring() == [4, 5]


def test_a_length_past_31_bits_is_refused():
    bs = 1 << 20
    t = _Tables(4, 2, 4096, bs=bs)
    before = t.copy()
    _, ctx, slots, _, _ = t.extend([0, 1], [0, 2 ** 31 - 16], [5, 16])
    assert int(t.err.item()) & CONTEXT and t.same(before)
    assert bool((ctx == 0).all()) and bool((slots == -1).all())
    t.err.zero_()
    _, ctx, _, pos, _ = t.extend([0, 1], [0, 2 ** 31 - 16], [5, 15])
    assert int(t.err.item()) == 0 and ctx.tolist() == [5, 2 ** 31 - 1] and pos[-1].item() == 2 ** 31 - 2
