"""Forked pages and decode over shared prefixes at their limits: tables and plans
larger than shared memory, many sequences and groups, several streams, repeated rows."""

from __future__ import annotations

import random

import pytest
import torch

from tests.test_gpu_shared_decode import Batch, _i32, _same
from tests.test_gpu_shared_pages import Device, Host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


# ---------------------------------------------------------------- pages
@pytest.mark.parametrize("kids,tokens", [(3, 300), (130, 4000 * 16 + 5), (64, 9000)])
def test_tables_that_do_and_do_not_fit_shared_memory(kids, tokens):
    """Up to 520000 entries: one cluster keeps some 400000 blocks between its phases, and reads more again."""
    own = -(-tokens // 16)
    blocks = own + kids + 2
    order = list(range(blocks))
    random.Random(kids).shuffle(order)
    host, dev = Host(order, 16), Device(blocks, order, kids + 3, own + 5, 16)
    host.grow(0, tokens)
    dev.grow([0], [0], [tokens])
    rows = list(range(1, kids + 1))
    lens = [tokens - (i % 3) * 7 for i in range(kids)]
    assert dev.fork([0] * kids, rows, lens) == host.fork([0] * kids, rows, lens)
    dev.same_as(host)
    # a count that says less than the tables do: refused, and nothing has changed
    blk = host.rows[0][0][0]
    dev.shares[0, blk] -= 1
    before = [x.clone() for x in (dev.store, dev.shares, dev.free, dev.state)]
    dev.release(rows + [0], lens + [tokens], [0] * (kids + 1))
    assert int(dev.err) == 128
    assert all(torch.equal(a, b) for a, b in zip(before, (dev.store, dev.shares, dev.free, dev.state)))
    dev.shares[0, blk] += 1
    dev.err.zero_()
    # an id outside the pool: the same
    dev.store[kids, 3] = blocks
    before = [x.clone() for x in (dev.store, dev.shares, dev.free, dev.state)]
    dev.release(rows + [0], lens + [tokens], [0] * (kids + 1))
    assert int(dev.err) == 1
    assert all(torch.equal(a, b) for a, b in zip(before, (dev.store, dev.shares, dev.free, dev.state)))
    dev.store[kids, 3] = host.rows[kids][0][3]
    dev.err.zero_()
    random.Random(1).shuffle(rows)
    part = rows[: kids // 2]
    keeps = [16 * (r % 5) for r in part]
    host.release(part, keeps)
    dev.release(part, [lens[r - 1] for r in part], keeps)
    dev.same_as(host)
    rest = [r for r in rows if r not in part] + [0] + part
    held = [lens[r - 1] if r and r not in part else tokens if r == 0 else 16 * (r % 5) for r in rest]
    host.release(rest, [0] * len(rest))
    dev.release(rest, held, [0] * len(rest))
    dev.same_as(host)
    assert len(host.free) == blocks


def test_many_entries_and_a_batch_beyond_the_plan():
    host, dev = Host(range(9000), 16), Device(9000, range(9000), 5000, 5, 16)
    parents = list(range(50))
    for r in parents:
        host.grow(r, 1 + r % 70)
    dev.grow(parents, [0] * 50, [1 + r % 70 for r in parents])
    kids = list(range(50, 5000))
    of = [k % 50 for k in kids]
    lens = [(k * 7) % (2 + p % 70) for k, p in zip(kids, of)]
    assert dev.fork(of, kids, lens) == host.fork(of, kids, lens)
    dev.same_as(host)
    rows = parents + kids
    random.Random(0).shuffle(rows)
    host_held = [host.rows[r][1] for r in rows]
    host.release(rows, [0] * 5000)
    dev.release(rows, host_held, [0] * 5000)
    dev.same_as(host)
    before = [x.clone() for x in (dev.store, dev.shares, dev.free, dev.state)]
    with pytest.raises((RuntimeError, ValueError)):
        dev.fork([0] * 30000, [-1] * 30000, [0] * 30000)
    assert all(torch.equal(a, b) for a, b in zip(before, (dev.store, dev.shares, dev.free, dev.state)))


# ---------------------------------------------------------------- decode
def test_many_sequences_in_one_group():
    Batch([_same(75, [i % 19 for i in range(1500)])], hq=4, hkv=2, seed=1).check()


def test_many_groups():
    Batch([_same(17 + g % 60, [g % 5, 3]) for g in range(400)], alone=(5, 0, 33), hq=4, hkv=2, seed=2).check()


def test_a_plan_beyond_shared_memory_is_answered_one_by_one():
    from pagedserve_b200 import ops
    assert ops.decode_shared_workspace_bytes(2000, 1000, 4, 2, 64, 16, 256, torch.bfloat16) == 0
    Batch([_same(17 + g % 60, [g % 5, 3]) for g in range(1000)], hq=4, hkv=2, seed=2).check()


@pytest.mark.parametrize("d,hq,hkv,bs", [(64, 14, 2, 16), (128, 8, 2, 32), (128, 32, 8, 64), (64, 16, 1, 16)])
@pytest.mark.parametrize("seed", range(6))
def test_pairs_and_single_tiles_in_any_order(d, hq, hkv, bs, seed):
    """Steps of single tiles and of pairs, in odd and even numbers, follow one another in a CTA's list:
    a stage of keys and values then goes from one stream of products to the other."""
    rng = random.Random(100 * d + seed)
    tile = 128 // (hq // hkv)
    groups = []
    for _ in range(rng.randint(2, 5)):
        n = rng.choice([2, tile - 1, tile, tile + 1, 2 * tile, 2 * tile + 1, 3 * tile])
        prefix = rng.choice([1, 63, 64, 65, 64 * 3, 64 * 5 + 7, 64 * 9])
        groups.append(_same(prefix, [rng.choice([0, 1, 20]) for _ in range(n)]))
    if seed == 0:  # short ones of a step each between long ones
        groups = [g for p in (64 * 3, 64, 1) for g in (_same(p, [1] * tile), _same(64, [0] * (tile + 1)), _same(64 * 2 + 1, [2, 0]))]
    Batch(groups, hq=hq, hkv=hkv, d=d, bs=bs, seed=seed).check()


def test_many_long_runs_of_single_tiles():
    """As the above, with prefixes from beyond the cache, over and over: every result is the first one's, bit by bit."""
    from pagedserve_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    batch, blocks = 96, 1100
    k, v = (torch.randn(1, blocks, 8, 32, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    table = torch.arange(938, dtype=torch.int32, device="cuda").repeat(batch, 1)
    table[:, 937] = torch.arange(938, 938 + batch, device="cuda")
    q = torch.randn(batch, 32, 128, generator=g, device="cuda").to(torch.bfloat16)
    ctx = torch.full((batch,), 30000, dtype=torch.int32, device="cuda")
    first = ops.paged_decode_shared(q, k, v, table, ctx, _i32([0, batch]), _i32([937 * 32]), 0)
    big = torch.empty(200 << 20, dtype=torch.uint8, device="cuda")
    for i in range(60):
        if i % 2:
            big.zero_()
        got = ops.paged_decode_shared(q, k, v, table, ctx, _i32([0, batch]), _i32([937 * 32]), 0)
        assert torch.equal(got, first)


def test_repeated_tables_and_an_output_over_the_query():
    from pagedserve_b200 import ops
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(1, 40, 2, 16, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    row = torch.randperm(40, generator=g)[:12].int().cuda()
    q = torch.randn(1, 14, 64, generator=g).to(torch.bfloat16).cuda()
    one = ops.paged_decode(q, k, v, row[None], _i32([180]), 0)
    many = q.repeat(30, 1, 1)
    got = ops.paged_decode_shared(many, k, v, row[None].expand(30, 12), _i32([180] * 30), _i32([0, 30]), _i32([180]), 0)
    assert (got == got[:1]).all()
    # two roundings to bf16 of the probabilities and of the result each
    assert ((got[0].double() - one[0].double()).abs() <= 4 * 2.0 ** -8 * v.double().abs().max()).all()
    again = ops.paged_decode_shared(many, k, v, row[None].expand(30, 12), _i32([180] * 30), _i32([0, 30]), _i32([180]), 0, out=many)
    assert again is many and torch.equal(many, got)


def test_two_streams_at_once_and_graphs_that_share_a_workspace():
    from pagedserve_b200 import ops
    cases = [Batch([_same(700, [5, 90, 33, 0, 1])], alone=(50,), seed=4), Batch([_same(64 * 9, [1] * 40), _same(100, [3, 3])], seed=5)]
    args = [(b.q.cuda(), b.k.cuda(), b.v.cuda(), b.table.cuda(), _i32(b.lens), _i32(b.cu), _i32(b.prefix), b.layer) for b in cases]
    want = [ops.paged_decode_shared(*a) for a in args]
    for b, w in zip(cases, want):
        exact, tol = b.expected()
        assert ((w.cpu().double() - exact).abs() <= tol).all()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(20):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(ops.paged_decode_shared(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    need = max(ops.decode_shared_workspace_bytes(len(b.lens), len(b.prefix), b.hq, b.hkv, b.d, b.bs, b.table.shape[1] * b.bs, b.dtype)
               for b in cases)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    graphs, outs = [], []
    for a in args:
        out = torch.empty_like(a[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_decode_shared(*a, out=out, workspace=ws)
        graphs.append(g), outs.append(out)
    for i in (0, 1, 0, 0, 1, 1, 0):
        outs[i].zero_()
        ws.fill_(255)
        graphs[i].replay()
        assert torch.equal(outs[i], want[i])
    with pytest.raises((RuntimeError, ValueError)):
        ops.paged_decode_shared(*args[0], workspace=ws[:64])
    with pytest.raises(ValueError, match="16 bytes"):
        ops.paged_decode_shared(*args[0], workspace=ws[8:])
