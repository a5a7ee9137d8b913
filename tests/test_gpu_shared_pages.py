"""fork_tables / copy_blocks / release_tables against bookkeeping on the host."""

from __future__ import annotations

import collections
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


class Host:
    """The same bookkeeping with a counter per block."""

    def __init__(self, order, bs):
        self.free, self.bs, self.rows = collections.deque(order), bs, {}
        self.holders = collections.Counter()

    def grow(self, row, n):
        t, held = self.rows.setdefault(row, ([], 0))
        new = [self.free.popleft() for _ in range(-(-(held + n) // self.bs) - len(t))]
        for x in new:
            self.holders[x] = 1
        self.rows[row] = (t + new, held + n)

    def fork(self, parents, children, lens):
        src, dst = [], []
        for p, c, n in zip(parents, children, lens):
            if c < 0:
                src.append(-1), dst.append(-1)
                continue
            whole = self.rows[p][0][:n // self.bs]
            for x in whole:
                self.holders[x] += 1
            t = list(whole)
            if n % self.bs:
                src.append(self.rows[p][0][n // self.bs])
                dst.append(self.free.popleft())
                self.holders[dst[-1]] = 1
                t.append(dst[-1])
            else:
                src.append(-1), dst.append(-1)
            self.rows[c] = (t, n)
        return src, dst

    def release(self, rows, keeps):
        for r, keep in zip(rows, keeps):
            if r < 0:
                continue
            t, _ = self.rows[r]
            k = -(-keep // self.bs)
            for x in t[k:]:
                self.holders[x] -= 1
                if self.holders[x] == 0:
                    self.free.append(x)
            self.rows[r] = (t[:k], keep)


class Device:
    def __init__(self, blocks, order, rows, width, bs):
        from pagedserve_b200 import ops
        self.ops, self.bs, self.blocks = ops, bs, blocks
        self.free, self.state = ops.free_list(blocks, "cuda", order)
        self.store = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
        self.shares = ops.share_counts(blocks, "cuda")
        self.err = _flag()

    def same_as(self, host):
        head, count, ticket, _ = self.state.tolist()
        ring = self.free.tolist()
        assert ticket == 0 and [ring[(head + i) % self.blocks] for i in range(count)] == list(host.free)
        table = self.store.cpu()
        want = torch.zeros_like(table)
        for r, (t, _) in host.rows.items():
            want[r, :len(t)] = torch.tensor(t, dtype=torch.int32)
        assert torch.equal(table, want)
        shares = self.shares.cpu()
        assert not shares[1].any()
        assert shares[0].tolist() == [max(0, host.holders[x] - 1) for x in range(self.blocks)]
        assert int(self.err) == 0

    def grow(self, rows, starts, ns):
        self.ops.extend_step(self.store, _dev(rows), _dev(starts), _dev(ns), self.free, self.state, sum(ns), self.bs, error_flag=self.err)

    def fork(self, parents, children, lens):
        src, dst = self.ops.fork_tables(self.store, _dev(parents), _dev(children), _dev(lens), self.shares, self.free, self.state, self.bs,
                                        error_flag=self.err)
        return src.tolist(), dst.tolist()

    def release(self, rows, helds, keeps):
        self.ops.release_tables(self.store, _dev(rows), _dev(helds), _dev(keeps), self.shares, self.free, self.state, self.bs, error_flag=self.err)


@pytest.mark.parametrize("bs,blocks,rows,width", [(16, 600, 60, 40), (1, 500, 30, 64), (12, 900, 200, 33)])
def test_follows_a_counter_per_block(bs, blocks, rows, width):
    """Random growth, forks (children of children among them) and whole and partial releases: the same ids, counts and free list."""
    rng = random.Random(bs + blocks)
    order = list(range(blocks))
    rng.shuffle(order)
    host, dev = Host(order, bs), Device(blocks, order, rows, width, bs)
    for step in range(40):
        live = [r for r in host.rows if host.rows[r][0]]
        idle = [r for r in range(rows) if r not in live]
        room = len(host.free)
        if step % 3 == 0 and idle:
            grow = rng.sample(idle, min(len(idle), rng.randint(1, 4))) + rng.sample(live, min(len(live), 3))
            starts, ns = [], []
            for r in grow:
                held = host.rows.get(r, ([], 0))[1] if r in live else 0
                n = rng.randint(1, 5 * bs)
                n = min(n, width * bs - held, max(0, room - 8) * bs - bs)
                n = max(n, 0)
                room -= -(-(held + n) // bs) - -(-held // bs)
                starts.append(held), ns.append(n)
                if r in idle:
                    host.rows.pop(r, None)
            for r, n in zip(grow, ns):
                host.grow(r, n)
            dev.grow(grow, starts, ns)
        elif step % 3 == 1 and live and idle:
            children = rng.sample(idle, min(len(idle), rng.randint(1, 20), room))
            parents = [rng.choice(live) for _ in children]
            lens = [rng.randint(0, host.rows[p][1]) for p in parents]
            at = rng.randrange(len(children) + 1)
            children.insert(at, -1), parents.insert(at, 0), lens.insert(at, 5)
            for c in children:
                host.rows.pop(c, None)
            assert dev.fork(parents, children, lens) == host.fork(parents, children, lens)
        elif live:
            out = rng.sample(live, rng.randint(1, len(live)))
            helds = [host.rows[r][1] for r in out]
            keeps = [rng.choice([0, 0, h, h // bs * bs]) for h in helds]
            host.release(out, keeps)
            dev.release(out, helds, keeps)
        dev.same_as(host)


def test_a_block_released_by_all_its_holders_at_once():
    """The last of them in entry order returns it, in one CTA or over many."""
    for n, tokens in ((2, 20), (40, 1000), (300, 700)):
        blocks = -(-tokens // 16) + n + 3
        host, dev = Host(range(blocks), 16), Device(blocks, range(blocks), n + 4, 70, 16)
        host.grow(0, tokens)
        dev.grow([0], [0], [tokens])
        kids = list(range(1, n))
        random.Random(n).shuffle(kids)
        assert dev.fork([0] * (n - 1), kids, [tokens] * (n - 1)) == host.fork([0] * (n - 1), kids, [tokens] * (n - 1))
        dev.same_as(host)
        rows = kids[: n // 2] + [0] + kids[n // 2:]
        host.release(rows, [0] * n)
        dev.release(rows, [tokens] * n, [0] * n)
        dev.same_as(host)
        assert len(host.free) == blocks


def test_rolling_back_own_blocks_and_refusing_shared_ones():
    host, dev = Host(range(40), 16), Device(40, range(40), 6, 8, 16)
    host.grow(0, 50)
    dev.grow([0], [0], [50])
    host.fork([0, 0], [1, 2], [50, 33])
    dev.fork([0, 0], [1, 2], [50, 33])
    # inside the block of its own: kept in part
    host.release([1], [49])
    dev.release([1], [50], [49])
    dev.same_as(host)
    before = [x.clone() for x in (dev.store, dev.shares, dev.free, dev.state)]
    dev.release([1], [49], [40])  # inside a block that rows 0 and 2 hold
    assert int(dev.err) == 1024
    assert all(torch.equal(a, b) for a, b in zip(before, (dev.store, dev.shares, dev.free, dev.state)))
    dev.err.zero_()
    dev.release([1, 2, 0], [49, 33, 50], [40, 0, 0])  # the others let go in the same call
    host.release([1, 2, 0], [40, 0, 0])
    dev.same_as(host)


REFUSED = [
    ("child out of range", lambda d: ([0], [99], [5]), 4),
    ("parent out of range", lambda d: ([-1], [2], [5]), 4),
    ("length", lambda d: ([0], [2], [-1]), 4),
    ("width", lambda d: ([0], [2], [8 * 16 + 1]), 4),
    ("child twice", lambda d: ([0, 0], [2, 2], [5, 5]), 256),
    ("child is a parent", lambda d: ([0, 2], [2, 3], [5, 5]), 256),
    ("too few blocks", lambda d: ([0] * 4, [2, 3, 4, 5], [5] * 4), 128),
    ("id outside", lambda d: (d.store[0, 1].fill_(77), ([0], [2], [40]))[1], 1),
    ("copied id outside", lambda d: (d.store[0, 2].fill_(-7), ([0], [2], [40]))[1], 1),
    ("id on the ring outside", lambda d: (d.free[3].fill_(1000), ([0], [2], [40]))[1], 1),
]


@pytest.mark.parametrize("name,plan,bit", REFUSED, ids=[r[0] for r in REFUSED])
def test_fork_is_refused_as_a_whole(name, plan, bit):
    d = Device(6, range(6), 6, 8, 16)
    d.grow([0], [0], [40])  # three of six blocks
    args = plan(d)
    before = [x.clone() for x in (d.store, d.shares, d.free, d.state)]
    src, dst = d.fork(*args)
    assert int(d.err) == bit | 512
    assert src == dst == [-1] * len(src)
    assert all(torch.equal(a, b) for a, b in zip(before, (d.store, d.shares, d.free, d.state)))
    # and what is planned behind it, until the flag is cleared
    assert d.fork([0], [2], [5]) == ([-1], [-1])
    d.release([0], [40], [0])
    d.grow([0], [40], [1])
    assert all(torch.equal(a, b) for a, b in zip(before, (d.store, d.shares, d.free, d.state)))


@pytest.mark.parametrize("rows,helds,keeps,bit", [
    ([9], [40], [0], 4), ([0], [40], [41], 4), ([0], [40], [-1], 4), ([0], [8 * 16 + 1], [0], 4), ([0, 0], [40, 40], [0, 0], 256),
    ([0, 1], [40, 40], [0, 0], 128)])
def test_release_is_refused_as_a_whole(rows, helds, keeps, bit):
    d = Device(6, range(6), 6, 8, 16)
    d.grow([0], [0], [40])
    d.store[1] = d.store[0]  # a row that was never forked: its blocks have one holder
    before = [x.clone() for x in (d.store, d.shares, d.free, d.state)]
    d.release(rows, helds, keeps)
    assert int(d.err) == bit
    assert all(torch.equal(a, b) for a, b in zip(before, (d.store, d.shares, d.free, d.state)))
    d.err.zero_()
    d.store[0, 1] = 55
    before = [x.clone() for x in (d.store, d.shares, d.free, d.state)]
    d.release([0], [40], [0])
    assert int(d.err) == 1
    assert all(torch.equal(a, b) for a, b in zip(before, (d.store, d.shares, d.free, d.state)))


def test_empty_batches():
    d = Device(6, range(6), 6, 8, 16)
    assert d.fork([], [], []) == ([], [])
    d.release([], [], [])
    assert d.fork([0, 3], [-1, -1], [5, 5]) == ([-1, -1], [-1, -1])
    d.grow([0], [0], [40])
    assert d.fork([0], [1], [0]) == ([-1], [-1])  # nothing is shared
    assert int(d.err) == 0 and not d.shares.any()


@pytest.mark.parametrize("shapes,dtypes", [
    ([(3, 50, 2, 16, 64)] * 2, [torch.bfloat16] * 2),
    ([(2, 40, 2, 2, 16, 32), (2, 40, 2, 2, 16, 2)], [torch.uint8, torch.float16]),
    ([(1, 9, 1, 3, 5)], [torch.float16]),       # 30 bytes a block
    ([(2, 9, 1, 3, 5), (2, 9, 7)], [torch.float32, torch.uint8]),
    ([(24, 300, 2, 16, 64)] * 2, [torch.bfloat16] * 2),
])
def test_copy_blocks(shapes, dtypes):
    from pagedserve_b200 import ops
    g = torch.Generator().manual_seed(1)
    pools = [(torch.randint(0, 255, s, generator=g)).to(t).cuda() for s, t in zip(shapes, dtypes)]
    n = shapes[0][1]
    perm = torch.randperm(n, generator=g).tolist()
    m = n // 3
    dst = perm[:m] + [-1, 3]
    src = [perm[m + i % (n - m)] for i in range(m)] + [2, -5]  # sources may repeat
    if m > 1:
        src[1] = src[0]
    want = [x.clone() for x in pools]
    for x in want:
        for a, b in zip(src[:m], dst[:m]):
            x[:, b] = x[:, a]
    err = _flag()
    ops.copy_blocks(pools, _dev(src), _dev(dst), error_flag=err)
    assert int(err) == 0 and all(torch.equal(a, b) for a, b in zip(pools, want))
    ops.copy_blocks(pools, _dev([0, n, 1]), _dev([n + 5, 0, -1]), error_flag=err)
    assert int(err) == 1 and all(torch.equal(a, b) for a, b in zip(pools, want))
    ops.copy_blocks(pools, _dev([]), _dev([]))


def test_captured_cycle():
    """Fork, copy and release in one graph, replayed: every replay takes the blocks the one before gave back."""
    d = Device(30, range(30), 8, 8, 16)
    ops = d.ops
    d.grow([0], [0], [40])
    pool = torch.randn(2, 30, 2, 16, 64, device="cuda")
    kids, zero, held = _dev([3, 1, 2]), _dev([0, 0, 0]), _dev([40, 33, 32])

    def cycle():
        src, dst = ops.fork_tables(d.store, zero, kids, held, d.shares, d.free, d.state, 16, error_flag=d.err)
        ops.copy_blocks((pool,), src, dst, error_flag=d.err)
        table = d.store.clone()
        ops.release_tables(d.store, kids, held, zero, d.shares, d.free, d.state, 16, error_flag=d.err)
        return src, dst, table
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cycle()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        src, dst, table = cycle()
    host = Host(range(30), 16)
    host.grow(0, 40)
    host.fork([0] * 3, [3, 1, 2], [40, 33, 32])
    host.release([3, 1, 2], [0, 0, 0])
    for _ in range(25):
        want = host.fork([0] * 3, [3, 1, 2], [40, 33, 32])
        tables = {r: list(t) for r, (t, _) in host.rows.items()}
        host.release([3, 1, 2], [0, 0, 0])
        graph.replay()
        assert (src.tolist(), dst.tolist()) == want
        for r, t in tables.items():
            assert table[r, :len(t)].tolist() == t
        for a, b in zip(*want):
            if a >= 0:
                assert torch.equal(pool[:, a], pool[:, b])
        d.same_as(host)
