"""paged_decode_shared against attention in 64 bits, over batches whose sequences share prefixes."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Batch:
    """Groups ``[(prefix, [context lengths])]``, then ``alone`` context lengths of no group.

    Whole blocks of a prefix are shared; where it ends inside a block every
    sequence holds a copy of its rows.  Whatever no sequence reaches is NaN."""

    def __init__(self, groups, alone=(), hq=14, hkv=2, d=64, bs=16, dtype=torch.bfloat16, layers=2, layer=1, seed=0, extra_blocks=3):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.bs, self.dtype, self.layer = hq, hkv, d, bs, dtype, layer
        self.lens = [n for _, ns in groups for n in ns] + list(alone)
        self.prefix = [p for p, _ in groups]
        cu = [0]
        for _, ns in groups:
            cu.append(cu[-1] + len(ns))
        self.cu = cu
        tables, at, copies = [], 0, []  # copies: (from block, to block, rows)
        total = sum(-(-n // bs) for n in self.lens) + sum(p // bs + 1 for p in self.prefix) + extra_blocks
        perm = torch.randperm(total, generator=g).tolist()
        for p, ns in groups:
            whole = min(p, max(ns, default=0)) // bs
            shared = perm[at:at + whole]
            at += whole
            begun = []  # (block the prefix ends in, its prefix rows)
            for n in ns:
                own = max(0, -(-n // bs) - whole)
                tables.append(shared[:-(-n // bs)] + perm[at:at + own])
                at += own
                if own:
                    begun.append((tables[-1][whole], min(p, n) - whole * bs))
            full = max(begun, key=lambda c: c[1], default=None)
            copies += [(full[0], blk, rows) for blk, rows in begun if blk != full[0]]
        for n in alone:
            need = -(-n // bs)
            tables.append(perm[at:at + need])
            at += need
        width = max(1, max((len(t) for t in tables), default=1)) + 1
        self.table = torch.full((len(self.lens), width), total + 7, dtype=torch.int32)  # never to be read
        for i, t in enumerate(tables):
            self.table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        shape = (layers, total, hkv, bs, d)
        k = torch.randn(shape, generator=g).to(dtype)
        v = torch.randn(shape, generator=g).to(dtype)
        for a, b, rows in copies:
            k[:, b, :, :rows] = k[:, a, :, :rows]
            v[:, b, :, :rows] = v[:, a, :, :rows]
        used = torch.zeros(total, bs, dtype=torch.bool)
        for t, n in zip(tables, self.lens):
            for j, blk in enumerate(t):
                used[blk, :max(0, min(bs, n - j * bs))] = True
        for pool in (k, v):
            pool.masked_fill_(~used[None, :, None, :, None], math.nan)
            for other in range(layers):
                if other != layer:
                    pool[other] = math.nan
        self.tables = tables
        self.k, self.v = k, v
        self.q = torch.randn(len(self.lens), hq, d, generator=g).to(dtype)

    def expected(self, scale=None, q=None):
        """(output, tolerance) in float64, sequence by sequence through its own table."""
        q = self.q if q is None else q
        scale = self.d ** -0.5 if scale is None else scale
        group = self.hq // self.hkv
        out = torch.zeros(q.shape, dtype=torch.float64)
        tol = torch.zeros_like(out)
        u = HALF_STEP[self.dtype]
        for i, n in enumerate(self.lens):
            if n == 0:
                continue
            t = torch.tensor(self.tables[i])
            k, v = (x[self.layer, t].transpose(0, 1).reshape(self.hkv, -1, self.d)[:, :n].double() for x in (self.k, self.v))
            for h in range(self.hkv):
                qq = q[i, h * group:(h + 1) * group].double()
                s = qq @ k[h].T * scale
                p = torch.softmax(s, -1)
                o = p @ v[h]
                out[i, h * group:(h + 1) * group] = o
                # each score: d products and sums in fp32; each probability then off by twice that, by the
                # exponential (2^-22) and sums and joins (below 2^-20 together), and by its rounding to the type;
                # the result by its rounding; f16 probabilities are at least 1 at the maximum, and below 2^-14 off by
                # 2^-25 each
                ds = (self.d + 4) * 2.0 ** -24 * (qq.abs() @ k[h].abs().T * scale).amax(-1, keepdim=True)
                room = (u * 1.01 if self.dtype != torch.float32 else 0) + 2 * ds + 2.0 ** -19
                tiny = n * 2.0 ** -25 * v[h].abs().amax() if self.dtype == torch.float16 else 0.0
                tol[i, h * group:(h + 1) * group] = room * (p @ v[h].abs()) + u * o.abs() + tiny + 1e-9
        return out, tol

    def run(self, **kw):
        from pagedserve_b200 import ops
        return ops.paged_decode_shared(self.q.cuda(), self.k.cuda(), self.v.cuda(), self.table.cuda(), _i32(self.lens), _i32(self.cu),
                                       _i32(self.prefix), self.layer, **kw)

    def check(self, **kw):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = self.run(error_flag=err, **kw).cpu().double()
        want, tol = self.expected()
        assert int(err) == 0
        assert torch.isfinite(got).all()
        worst = ((got - want).abs() / tol.clamp(min=1e-300)).max() if got.numel() else torch.zeros(())
        assert ((got - want).abs() <= tol).all(), float(worst)
        return got


def _same(prefix, owns):
    return (prefix, [prefix + o for o in owns])


SHAPES = [
    # the smallest prefixes, and own parts of none to a few tokens
    dict(groups=[_same(1, [0, 1])]),
    dict(groups=[_same(5, [1, 2, 30])]),
    dict(groups=[_same(16, [0, 0, 1, 16, 17])]),
    # prefixes at the edges of blocks and of the 64-key steps
    dict(groups=[_same(63, [1, 5])]),
    dict(groups=[_same(64, [1, 5])]),
    dict(groups=[_same(65, [1, 5])]),
    dict(groups=[_same(128, [0, 3])]),
    dict(groups=[_same(200, [7] * 18)]),   # a whole tile of sequences
    dict(groups=[_same(200, [7] * 19)]),   # one more
    dict(groups=[_same(333, list(range(37)))]),
    # idle rows, the first of the group among them; rows that end inside the prefix; a prefix longer than every row
    dict(groups=[(100, [0, 110, 0, 130]), (64, [0, 0]), (70, [71, 0])]),
    dict(groups=[(100, [3, 50, 99, 100, 101, 64, 120])]),
    dict(groups=[(1000, [30, 77, 77, 16])]),
    # groups of one, of none, without a prefix; sequences of no group
    dict(groups=[(50, [60]), (40, []), (0, [33, 34]), _same(48, [1, 2])], alone=[5, 0, 300]),
    # many groups of ragged prefixes
    dict(groups=[_same(17 + 29 * i, [3 + i, 1, 40]) for i in range(23)]),
    # long, with more steps than CTAs
    dict(groups=[_same(5000, [3 * i for i in range(40)])]),
    dict(groups=[_same(3001, [1] * 130), _same(700, [400, 900])]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
def test_bf16_against_64_bits(shape):
    Batch(**shape).check()


@pytest.mark.parametrize("hq,hkv,d,bs,dtype", [
    (14, 2, 64, 16, torch.float16), (32, 8, 128, 32, torch.bfloat16), (32, 8, 128, 16, torch.float16), (8, 8, 64, 64, torch.bfloat16),
    (16, 1, 64, 16, torch.bfloat16), (10, 5, 64, 32, torch.float16), (28, 4, 128, 128, torch.bfloat16), (3, 1, 128, 64, torch.bfloat16),
    (24, 2, 64, 16, torch.bfloat16), (9, 3, 64, 192, torch.bfloat16), (1, 1, 64, 16, torch.bfloat16)])
def test_geometries(hq, hkv, d, bs, dtype):
    Batch([_same(530, [0, 1, 90, 33, 700]), (70, [0, 71, 20, 90])], alone=[45], hq=hq, hkv=hkv, d=d, bs=bs, dtype=dtype).check()
    Batch([_same(129, [5] * 70)], hq=hq, hkv=hkv, d=d, bs=bs, dtype=dtype, seed=1).check()


@pytest.mark.parametrize("hq,hkv,d,bs,dtype", [
    (14, 2, 64, 16, torch.float32), (14, 2, 64, 8, torch.bfloat16), (6, 2, 96, 16, torch.bfloat16), (40, 2, 64, 16, torch.float16)])
def test_geometries_that_are_answered_one_by_one(hq, hkv, d, bs, dtype):
    Batch([_same(130, [0, 1, 90, 33]), (70, [0, 71, 20, 90])], alone=[45], hq=hq, hkv=hkv, d=d, bs=bs, dtype=dtype).check()


def test_strides_outputs_and_scale():
    from pagedserve_b200 import ops
    b = Batch([_same(150, [3, 60, 0, 9]), _same(64, [1, 1])])
    k, v, lens, cu, pre = b.k.cuda(), b.v.cuda(), _i32(b.lens), _i32(b.cu), _i32(b.prefix)
    n = len(b.lens)
    wide = torch.randn(n, 18 * 64 + 8, device="cuda").to(b.dtype)
    q = wide[:, 8:8 + 14 * 64].unflatten(1, (14, 64))  # rows of a fused projection
    table = torch.full((n, b.table.shape[1] + 5), 9999, dtype=torch.int32, device="cuda")[:, 2:2 + b.table.shape[1]]
    table.copy_(b.table)
    out = torch.full((n, 14, 1, 70), 7.0, device="cuda", dtype=b.dtype)
    got = ops.paged_decode_shared(q[:, :, None], k, v, table, lens, cu, pre, b.layer, scale=0.3, out=out[..., :64])
    assert got.data_ptr() == out.data_ptr() and bool((out[..., 64:] == 7).all())
    want, tol = b.expected(scale=0.3, q=q.cpu())
    assert ((got[:, :, 0].cpu().double() - want).abs() <= tol).all()
    # a base or a stride off 16 bytes, heads far apart, a given workspace, a bound on the context
    odd = torch.randn(n, 14 * 65 + 1, device="cuda").to(b.dtype)[:, 1:].unflatten(1, (14, 65))[..., :64]
    ws = torch.empty(ops.decode_shared_workspace_bytes(n, 2, 14, 2, 64, 16, 400, b.dtype), dtype=torch.uint8, device="cuda")
    got = ops.paged_decode_shared(odd, k, v, torch.nn.functional.pad(b.table, (0, 20)).cuda(), lens, cu, pre, b.layer, max_context=400, workspace=ws)
    want, tol = b.expected(q=odd.cpu())
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_large_scores():
    b = Batch([_same(200, [30, 0, 5])], seed=3)
    b.q *= 40  # scores of several hundred: exponents' references move, most probabilities vanish
    b.check()
    b = Batch([_same(200, [30, 0, 5])], seed=4)
    b.k[..., 5] += 300.0
    b.q[..., 5] = -1.0
    b.check()


def test_what_is_not_a_number_reaches_the_rows_that_see_it():
    b = Batch([_same(100, [20, 40, 3]), _same(80, [2, 2])])
    blk, row = b.tables[1][6], 10  # position 106: the second sequence's own
    b.v[b.layer, blk, 0, row, 3] = math.inf
    got = b.run().cpu()
    assert bool(torch.isinf(got[1, :7, 3]).all())
    got[1, :7, 3] = 0
    assert bool(torch.isfinite(got).all())
    b.k[b.layer, b.tables[0][2], 1, 4] = math.nan  # position 36: the first group's prefix
    got = b.run().cpu()
    assert bool(got[:3, 7:].isnan().all()) and bool(torch.isfinite(got[3:]).all())


def test_pool_past_4_gb():
    from pagedserve_b200 import ops
    b = Batch([_same(100, [20, 40, 3])], layers=1, layer=0)
    blocks = (1 << 32) // (2 * 16 * 64 * 2) + 100
    pools = []
    for x in (b.k, b.v):
        big = torch.empty(1, blocks, 2, 16, 64, dtype=b.dtype, device="cuda")
        big[0, blocks - x.shape[1]:] = x[0].cuda()
        pools.append(big)
    table = b.table.cuda() + (blocks - b.k.shape[1])
    got = ops.paged_decode_shared(b.q.cuda(), *pools, table, _i32(b.lens), _i32(b.cu), _i32(b.prefix), 0).cpu().double()
    want, tol = b.expected()
    assert ((got - want).abs() <= tol).all()


def test_what_is_wrong_is_flagged_and_never_read():
    from pagedserve_b200 import ops
    b = Batch([_same(100, [20, 40, 3]), _same(80, [2, 2])], alone=[33])
    want, tol = b.expected()
    args = lambda **kw: [b.q.cuda(), b.k.cuda(), b.v.cuda(), kw.get("table", b.table).cuda(), _i32(kw.get("lens", b.lens)), _i32(kw.get("cu", b.cu)),
                         _i32(kw.get("prefix", b.prefix)), b.layer]
    ok = lambda got, rows: ((got.cpu().double() - want).abs() <= tol)[rows].all()

    def flagged(**kw):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = ops.paged_decode_shared(*args(**kw), error_flag=err)
        return got, int(err)
    # groups that are not in order: flagged, and every sequence is read on its own
    for cu in ([0, 5, 3], [-1, 3, 5], [0, 3, 99]):
        got, bits = flagged(cu=cu)
        assert bits == 32 and ok(got, slice(None))
    got, bits = flagged(prefix=[-5, 80])
    assert bits == 4 and ok(got, slice(None))
    lens = list(b.lens)
    lens[4], lens[5] = -3, 10 ** 6
    got, bits = flagged(lens=lens, table=b.table.clamp(max=b.k.shape[1] - 1))
    assert bits == 4 and ok(got, slice(0, 4)) and bool((got[4] == 0).all())
    for where, hit in (((1, 7), [1]), ((4, 5), [4])):  # a block of a sequence's own
        table = b.table.clone()
        table[where] = b.k.shape[1] + 3
        got, bits = flagged(table=table)
        assert bits == 1 and ok(got, [i for i in range(6) if i not in hit])
    table = b.table.clone()
    table[1, 2] = -4  # in the longest sequence's table: the first group's prefix
    got, bits = flagged(table=table)
    assert bits == 1 and ok(got, slice(3, 6))


def test_captured_and_replayed_with_other_lengths_and_groups():
    from pagedserve_b200 import ops
    a = Batch([_same(100, [20, 40, 3]), _same(80, [2, 2])], alone=[33], seed=5)
    q, k, v, table = a.q.cuda(), a.k.cuda(), a.v.cuda(), a.table.cuda()
    lens, cu, pre = _i32(a.lens), _i32(a.cu), _i32(a.prefix)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_decode_shared(q, k, v, table, lens, cu, pre, a.layer, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_decode_shared(q, k, v, table, lens, cu, pre, a.layer, out=out)
    want, tol = a.expected()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert ((out.cpu().double() - want).abs() <= tol).all()
    # idle rows, another division of the same batch
    a.lens[1] = a.lens[5] = 0
    lens.copy_(_i32(a.lens))
    cu.copy_(_i32([0, 2, 6]))
    pre.copy_(_i32([64, 0]))
    graph.replay()
    want, tol = a.expected()
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_behind_writes_and_a_chain_of_calls():
    """Each call's query is the call before's output, and the new token's rows are written right in front of it."""
    from pagedserve_b200 import ops
    b = Batch([_same(96, [20] * 9), _same(333, [5] * 4)], seed=6, layers=1, layer=0)
    k, v, table, lens, cu, pre = b.k.cuda(), b.v.cuda(), b.table.cuda(), _i32(b.lens), _i32(b.cu), _i32(b.prefix)
    k.nan_to_num_()
    v.nan_to_num_()
    n = len(b.lens)
    slots = torch.tensor([b.tables[i][(m - 1) // 16] * 16 + (m - 1) % 16 for i, m in enumerate(b.lens)], device="cuda")
    rows = [torch.randn(n, 2, 64, device="cuda").to(b.dtype) for _ in range(6)]
    q = b.q.cuda()
    outs = []
    for r in rows:
        ops.reshape_and_cache(r, r, k, v, slots, 0)
        q = ops.paged_decode_shared(q, k, v, table, lens, cu, pre, 0)
        outs.append(q)
    q = b.q
    for r, got in zip(rows, outs):
        kk, vv = b.k.clone(), b.v.clone()
        for pool in (kk, vv):
            pool.view(1, -1, 2, 16, 64)[0, slots.cpu() // 16, :, slots.cpu() % 16] = r.cpu()
        b.k, b.v = kk, vv
        want, tol = b.expected(q=q)
        assert ((got.cpu().double() - want).abs() <= tol).all()
        q = got.cpu()
