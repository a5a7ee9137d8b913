"""Attention over the 4-bit pool against the plain 64-bit form, with the
tolerance int4_reference.attend derives; every row outside the sequences
holds NaN parameters and random codes, and unused table entries point past
the pool."""

from __future__ import annotations

import math

import pytest
import torch

from tests import int4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


def _decode_case(seed, lens, hq, hkv, d, bs, dtype, layers=2, layer=1, spread=None, qscale=1.0):
    gen = torch.Generator().manual_seed(seed)
    table, blocks = ref.shuffled_tables(gen, lens, bs)
    codes, params = ref.make_pool(gen, layers, blocks, hkv, bs, d, dtype, spread)
    pc, pp = ref.poison(codes, params, layer, table, lens, bs)
    q = (torch.randn(len(lens), hq, d, generator=gen) * qscale).to(dtype)
    return dict(q=q, codes=codes, params=params, pc=pc, pp=pp, table=table, lens=lens, layer=layer, bs=bs, d=d)


def _decode(c, **kw):
    from pagedserve_b200 import ops
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.paged_decode_int4(c["q"].cuda(), c["pc"].cuda(), c["pp"].cuda(), c["table"].cuda(),
                                torch.tensor(c["lens"], dtype=torch.int32, device="cuda"), c["layer"], error_flag=err,
                                **kw)
    torch.cuda.synchronize()
    return out.cpu(), int(err.item())


def _want_decode(c, scale=None, lens=None, rows=None):
    scale = c["d"] ** -0.5 if scale is None else scale
    outs, tols = [], []
    for b in range(len(c["lens"])) if rows is None else rows:
        n = (lens or c["lens"])[b]
        o, t = ref.attend(c["q"][b:b + 1], c["codes"], c["params"], c["layer"], c["table"][b], n, c["bs"], n - 1, scale)
        outs.append(o)
        tols.append(t)
    return torch.cat(outs), torch.cat(tols)


def _close(got, want, tol):
    worst = ((got.double() - want).abs() / tol.clamp(min=1e-300)).max()
    assert bool(((got.double() - want).abs() <= tol).all()), f"{float(worst):.2f} times the tolerance"


RAGGED = [1, 0, 15, 16, 17, 33, 64, 100, 257, 1000, 0, 31]
#         hq, hkv, d, bs
SHAPES = [(14, 2, 64, 16), (7, 1, 64, 16), (8, 8, 64, 16), (32, 8, 128, 32), (28, 4, 128, 16), (16, 1, 64, 64),
          (24, 2, 64, 16), (40, 1, 128, 16), (9, 3, 64, 48), (6, 2, 80, 16), (4, 2, 64, 8), (3, 3, 32, 16),
          (2, 1, 256, 16), (5, 5, 2, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_decode_ragged(dtype, hq, hkv, d, bs):
    c = _decode_case(hq * 100 + d + bs, RAGGED, hq, hkv, d, bs, dtype)
    got, err = _decode(c)
    want, tol = _want_decode(c)
    assert err == 0
    _close(got, want, tol)
    assert bool((got[1] == 0).all())  # a sequence of no tokens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (32, 8, 128, 32)])
def test_decode_rows_of_very_different_size(dtype, hq, hkv, d, bs):
    """Steps and offsets over many powers of two: the scores' terms cancel and
    the largest rows dominate."""
    c = _decode_case(77, [40, 300, 1, 129], hq, hkv, d, bs, dtype, spread=3, qscale=0.5)
    got, err = _decode(c)
    want, tol = _want_decode(c)
    assert err == 0
    _close(got, want, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_many_sequences(dtype):
    """A served batch: lengths that put sequence ends everywhere in the split."""
    gen = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 700, (257,), generator=gen).tolist()
    lens[3] = 5000
    c = _decode_case(6, lens, 14, 2, 64, 16, dtype, layers=1, layer=0)
    got, err = _decode(c)
    rows = [0, 1, 2, 3, 4, 100, 101, 200, 255, 256]
    want, tol = _want_decode(c, rows=rows)
    assert err == 0
    _close(got[rows], want, tol)
    # two independent roundings, each uniform within half a step: the norm stays inside one half step
    assert float((got[rows].double() - want).norm() / want.norm()) <= ref.HALF_STEP[dtype]
    assert not bool(torch.isnan(got).any())


@pytest.mark.parametrize("dtype,d,bs", [(torch.bfloat16, 64, 16), (torch.float16, 128, 16)])
def test_decode_long_context(dtype, d, bs):
    c = _decode_case(8, [40001, 3], 14, 2, d, bs, dtype, layers=1, layer=0)
    got, err = _decode(c)
    want, tol = _want_decode(c)
    assert err == 0
    _close(got, want, tol)


def test_decode_peaked_and_flat_scores():
    """Queries large enough that one token takes all, and zero queries (a plain mean)."""
    c = _decode_case(9, [500, 500, 33], 14, 2, 64, 16, torch.bfloat16, qscale=30.0)
    c["q"][1] = 0
    got, err = _decode(c)
    want, tol = _want_decode(c)
    assert err == 0
    _close(got, want, tol)


@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (4, 2, 64, 8)])
def test_decode_scale_strides_and_4d(hq, hkv, d, bs):
    """Query and output as strided slices, a wider table's slice, a given scale, [B, Hq, 1, D]."""
    from pagedserve_b200 import ops
    c = _decode_case(10, [70, 5, 200], hq, hkv, d, bs, torch.bfloat16)
    wide = torch.zeros(3, (hq + 3) * d, dtype=torch.bfloat16)
    wide[:, d:d + hq * d] = c["q"].reshape(3, -1)
    dw = wide.cuda()
    q = dw[:, d:d + hq * d].view(3, hq, d)
    store = torch.full((3, 3, d + 8, hq), 7.0, dtype=torch.bfloat16, device="cuda")
    buf = torch.full((3, hq, 2 * d), 7.0, dtype=torch.bfloat16, device="cuda")
    tab = torch.cat([c["table"], c["table"]], 1).cuda()[:, :c["table"].shape[1]]
    lens = torch.tensor(c["lens"], dtype=torch.int32, device="cuda")
    pc, pp = c["pc"].cuda(), c["pp"].cuda()
    ops.paged_decode_int4(q, pc, pp, tab, lens, c["layer"], scale=0.3, out=buf[:, :, :d])
    want, tol = _want_decode(c, scale=0.3)
    _close(buf[:, :, :d].cpu(), want, tol)
    assert bool((buf[:, :, d:] == 7).all()) and bool((store == 7).all())
    out4 = ops.paged_decode_int4(q.unsqueeze(2), pc, pp, tab, lens, c["layer"], scale=0.3)
    assert out4.shape == (3, hq, 1, d)
    assert torch.equal(out4.squeeze(2), buf[:, :, :d])


def test_decode_unaligned_query():
    """Rows that start on an odd element."""
    from pagedserve_b200 import ops
    c = _decode_case(11, [70, 5, 200], 14, 2, 64, 16, torch.bfloat16)
    flat = torch.zeros(3 * 14 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    q = flat[1:].view(3, 14, 64)
    q.copy_(c["q"])
    out = torch.zeros(3 * 14 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 14, 64)
    ops.paged_decode_int4(q, c["pc"].cuda(), c["pp"].cuda(), c["table"].cuda(),
                          torch.tensor(c["lens"], dtype=torch.int32, device="cuda"), c["layer"], out=out)
    want, tol = _want_decode(c)
    _close(out.cpu(), want, tol)


@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (4, 2, 64, 8)])
def test_decode_bad_blocks_and_lengths(hq, hkv, d, bs):
    """A block id outside the pool is skipped and flagged; a length past
    max_context is cut there and flagged, a negative one is empty."""
    lens = [70, 50, 90]
    c = _decode_case(12, lens, hq, hkv, d, bs, torch.bfloat16)
    good = c["table"].clone()
    c["table"][0, 1] = 1 << 20
    c["table"][2, 0] = -1
    got, err = _decode(c)
    assert err == 1
    c["table"] = good
    for b, col in ((0, 1), (2, 0)):
        keep = torch.ones(lens[b], dtype=torch.bool)
        keep[col * bs:(col + 1) * bs] = False
        want, tol = ref.attend(c["q"][b:b + 1], c["codes"], c["params"], c["layer"], c["table"][b], lens[b], bs,
                               lens[b] - 1, d ** -0.5, keep)
        _close(got[b:b + 1], want, tol)
    c["lens"] = [70, -5, 90]
    got, err = _decode(c, max_context=80)
    assert err == 4
    want, tol = _want_decode(c, lens=[70, 0, 80])
    _close(got, want, tol)


def test_decode_non_finite_rows():
    """A row stored as NaN makes its sequence's outputs NaN, and no other's."""
    c = _decode_case(13, [40, 40, 40], 14, 2, 64, 16, torch.bfloat16)
    c["pp"][c["layer"], c["table"][1, 1], 0, 1, 3, 1] = math.nan  # a V row of kv head 0
    got, _ = _decode(c)
    assert bool(torch.isnan(got[1, :7]).all()) and not bool(torch.isnan(got[[0, 2]]).any())
    assert not bool(torch.isnan(got[1, 7:]).any())


def test_decode_repeats_bit_for_bit():
    c = _decode_case(14, [3000, 17, 900, 0, 64], 14, 2, 64, 16, torch.bfloat16)
    first, _ = _decode(c)
    for _ in range(3):
        again, _ = _decode(c)
        assert torch.equal(first, again)


def test_decode_two_streams_and_graphs():
    """Two captured calls replayed at once on two streams, and an eager call
    beside them: none shares scratch with another."""
    from pagedserve_b200 import ops
    cases = [_decode_case(20 + i, [2000, 33, 700], 14, 2, 64, 16, torch.bfloat16) for i in range(2)]
    args = [(c["q"].cuda(), c["pc"].cuda(), c["pp"].cuda(), c["table"].cuda(),
             torch.tensor(c["lens"], dtype=torch.int32, device="cuda"), c["layer"]) for c in cases]
    eager = [ops.paged_decode_int4(*a) for a in args]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_decode_int4(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        side = ops.paged_decode_int4(*args[0])
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        assert torch.equal(o, e)
    assert torch.equal(side, eager[0])


# -- prefill -----------------------------------------------------------------------------------------------------


def _prefill_case(seed, qlens, ctxs, hq, hkv, d, bs, dtype, layers=2, layer=1, spread=None):
    c = _decode_case(seed, ctxs, hq, hkv, d, bs, dtype, layers, layer, spread)
    gen = torch.Generator().manual_seed(seed + 1)
    c["q"] = torch.randn(sum(qlens), hq, d, generator=gen).to(dtype)
    c["qlens"] = qlens
    c["cu"] = torch.tensor([0] + qlens).cumsum(0).to(torch.int32)
    return c


def _prefill(c, **kw):
    from pagedserve_b200 import ops
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.paged_prefill_int4(c["q"].cuda(), c["pc"].cuda(), c["pp"].cuda(), c["table"].cuda(),
                                 torch.tensor(c["lens"], dtype=torch.int32, device="cuda"), c["cu"].cuda(),
                                 max(c["qlens"]), c["layer"], error_flag=err, **kw)
    torch.cuda.synchronize()
    return (out if kw.get("out") is not None else out).cpu(), int(err.item())


def _want_prefill(c, scale=None):
    scale = c["d"] ** -0.5 if scale is None else scale
    outs, tols = [], []
    cu = c["cu"].tolist()
    for b, (n, ctx) in enumerate(zip(c["qlens"], c["lens"])):
        o, t = ref.attend(c["q"][cu[b]:cu[b + 1]], c["codes"], c["params"], c["layer"], c["table"][b], ctx, c["bs"],
                          ctx - n, scale)
        outs.append(o)
        tols.append(t)
    return torch.cat(outs), torch.cat(tols)


CHUNKS = [([1], [1]), ([8], [28]), ([1, 17, 0, 130, 64], [1, 40, 9, 130, 1000]), ([37, 129, 5], [700, 300, 5]),
          ([4] * 9, [16, 17, 63, 64, 65, 127, 128, 129, 500])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (8, 8, 64, 16), (16, 1, 64, 16), (10, 5, 64, 16),
                                         (8, 2, 128, 16), (4, 2, 64, 32), (2, 1, 80, 8), (48, 1, 64, 16)])
@pytest.mark.parametrize("qlens,ctxs", CHUNKS)
def test_prefill_chunks(dtype, hq, hkv, d, bs, qlens, ctxs):
    c = _prefill_case(sum(qlens) * 7 + d, qlens, ctxs, hq, hkv, d, bs, dtype)
    got, err = _prefill(c)
    want, tol = _want_prefill(c)
    assert err == 0
    _close(got, want, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill_long_and_mixed(dtype):
    c = _prefill_case(31, [300, 2, 513], [6000, 3000, 513], 14, 2, 64, 16, dtype, layers=1, layer=0, spread=2)
    got, err = _prefill(c)
    want, tol = _want_prefill(c)
    assert err == 0
    _close(got, want, tol)
    assert float((got.double() - want).norm() / want.norm()) <= ref.HALF_STEP[dtype]


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (4, 2, 80)])
def test_prefill_rows_behind_the_last_sequence_keep_their_values(hq, hkv, d):
    c = _prefill_case(32, [5, 20], [30, 20], hq, hkv, d, 16, torch.bfloat16)
    c["q"] = torch.cat([c["q"], torch.randn(40, hq, d).bfloat16()])
    out = torch.full((65, hq, 2 * d), 3.0, dtype=torch.bfloat16, device="cuda")
    got, err = _prefill(c, out=out[:, :, :d], scale=0.2)
    want, tol = _want_prefill(c, scale=0.2)
    assert err == 0
    _close(got[:25], want, tol)
    assert bool((out[25:] == 3).all()) and bool((out[:, :, d:] == 3).all())


def test_prefill_equals_decode_for_single_rows():
    """One new token per sequence: the same attention as decode, within both tolerances."""
    ctxs = [1, 16, 100, 333]
    c = _prefill_case(33, [1] * 4, ctxs, 14, 2, 64, 16, torch.bfloat16)
    got, _ = _prefill(c)
    dec, _ = _decode(c)
    want, tol = _want_prefill(c)
    _close(got, want, tol)
    _close(dec, want, tol)


def test_prefill_bad_blocks_lengths_and_seqlens():
    c = _prefill_case(34, [20, 30], [100, 90], 14, 2, 64, 16, torch.bfloat16)
    good = c["table"].clone()
    c["table"][0, 2] = 1 << 28
    got, err = _prefill(c)
    assert err == 1
    c["table"] = good
    keep = torch.ones(100, dtype=torch.bool)
    keep[32:48] = False
    want, tol = ref.attend(c["q"][:20], c["codes"], c["params"], c["layer"], c["table"][0], 100, 16, 80, 0.125, keep)
    _close(got[:20], want, tol)
    c["lens"] = [10, 90]  # fewer tokens than query rows: flagged
    _, err = _prefill(c)
    assert err == 4
    c["lens"] = [100, 90]
    c["cu"] = torch.tensor([0, 60, 50], dtype=torch.int32)
    _, err = _prefill(c)
    assert err & 32


def test_prefill_graph_and_second_stream():
    from pagedserve_b200 import ops
    c = _prefill_case(35, [40, 7], [200, 300], 14, 2, 64, 16, torch.bfloat16)
    a = (c["q"].cuda(), c["pc"].cuda(), c["pp"].cuda(), c["table"].cuda(),
         torch.tensor(c["lens"], dtype=torch.int32, device="cuda"), c["cu"].cuda(), 40, c["layer"])
    eager = ops.paged_prefill_int4(*a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.paged_prefill_int4(*a)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        g.replay()
        other = ops.paged_prefill_int4(*a)
    torch.cuda.synchronize()
    assert torch.equal(out, eager) and torch.equal(other, eager)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("which", [0, 1])
def test_prefill_non_finite_rows_stay_behind_the_mask(which, dtype):
    """A key or value stored as NaN reaches the rows that see its position and
    no others, in its kv head alone."""
    c = _prefill_case(35, [130, 70], [200, 70], 14, 2, 64, 16, dtype)
    at = 150  # row 80 of the first sequence is the first that sees it
    want, tol = _want_prefill(c)
    c["pp"][c["layer"], c["table"][0, at // 16], 1, which, at % 16, 0] = 0.0
    c["pp"][c["layer"], c["table"][0, at // 16], 1, which, at % 16, 1] = math.nan
    got, err = _prefill(c)
    assert err == 0
    hit = torch.zeros(200, 14, dtype=torch.bool)
    hit[80:130, 7:] = True
    assert bool(torch.isnan(got[hit]).all())
    _close(got[~hit], want[~hit], tol[~hit])


@pytest.mark.parametrize("power", [118, -100])
@pytest.mark.parametrize("qlens,ctxs", [([70], [300]), ([1, 1], [77, 2000])])
def test_values_at_the_ends_of_bf16(power, qlens, ctxs):
    """V rows scaled by a power of two up to 2^118 (values to 1e36) or down to
    2^-100 give results scaled by it: no sum inside over- or underflows."""
    c = _prefill_case(36, qlens, ctxs, 14, 2, 64, 16, torch.bfloat16)
    want, tol = _want_prefill(c)
    c["pp"][:, :, :, 1] = (c["pp"][:, :, :, 1].double() * 2.0 ** power).bfloat16()
    got, err = _prefill(c)
    assert err == 0
    _close(got.double() * 2.0 ** -power, want, tol)
    if max(qlens) == 1:
        got, err = _decode(c)
        assert err == 0
        _close(got.double() * 2.0 ** -power, want, tol)


def test_offsets_past_32_bits():
    """A pool whose codes are past 4 GB: rows written to its last blocks are
    read back and attended to as from a small pool, bit for bit."""
    from pagedserve_b200 import ops
    gen = torch.Generator().manual_seed(37)
    hq, hkv, d, bs, n, blocks = 14, 2, 64, 16, 100, 2_200_000
    k, v = (torch.randn(n, hkv, d, generator=gen).bfloat16().cuda() for _ in range(2))
    q = torch.randn(40, hq, d, generator=gen).bfloat16().cuda()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    outs = []
    for num, ids in ((blocks, [blocks - 1 - 3 * i for i in range(7)]), (9, [8, 2, 3, 7, 0, 1, 5])):
        codes = torch.empty(1, num, hkv, 2, bs, d // 2, dtype=torch.uint8, device="cuda")
        params = torch.empty(1, num, hkv, 2, bs, 2, dtype=torch.bfloat16, device="cuda")
        blk = torch.tensor(ids, device="cuda")
        pos = torch.arange(n, device="cuda")
        slots = blk[pos // bs] * bs + pos % bs
        ops.reshape_and_cache_int4(k, v, codes, params, slots, 0)
        table = blk.to(torch.int32)[None]
        outs.append([*ops.gather_cache_int4(codes, params, slots, 0),
                     ops.paged_decode_int4(q[:1], codes, params, table, lens, 0),
                     ops.paged_prefill_int4(q, codes, params, table, lens, cu, 40, 0)])
        del codes, params
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,qlens", [(14, 2, [18, 19, 36, 37, 72, 73]), (8, 1, [16, 17, 32, 33, 48]),
                                          (128, 1, [1, 2, 3, 5]), (3, 3, [128, 129, 256, 257])])
def test_prefill_tile_boundaries(dtype, hq, hkv, qlens):
    """Chunks that end at, just behind and between the ends of the tiles of
    128 rows (128 / group tokens) and of their pairs, alone and together."""
    ctxs = [n + 61 * i for i, n in enumerate(qlens)]
    c = _prefill_case(38, qlens, ctxs, hq, hkv, 64, 16, dtype)
    got, err = _prefill(c)
    want, tol = _want_prefill(c)
    assert err == 0
    _close(got, want, tol)
    for i in (1, len(qlens) - 1):
        one = _prefill_case(39 + i, [qlens[i]], [ctxs[i] + 700], hq, hkv, 64, 16, dtype)
        got, err = _prefill(one)
        want, tol = _want_prefill(one)
        assert err == 0
        _close(got, want, tol)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-3])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 80)])
def test_scales_of_either_sign(scale, dtype, d):
    c = _prefill_case(50, [70, 1, 40], [300, 77, 40], 14, 2, d, 16, dtype)
    got, err = _prefill(c, scale=scale)
    want, tol = _want_prefill(c, scale=scale)
    assert err == 0
    _close(got, want, tol)
    c["q"] = c["q"][:3]
    got, err = _decode(c, scale=scale)
    want, tol = _want_decode(c, scale=scale)
    assert err == 0
    _close(got, want, tol)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128), (24, 2, 64)])
@pytest.mark.parametrize("power", [-110, 90, 105, 120])
def test_decode_queries_at_the_ends_of_bf16(power, hq, hkv, d):
    """Queries scaled by a power of two up to 2^120 (values to 2^122) and keys
    by its inverse: the same scores, so the same outputs."""
    c = _decode_case(40, [77, 2000, 16], hq, hkv, d, 16, torch.bfloat16)
    want, tol = _want_decode(c)
    c["q"] = (c["q"].double() * 2.0 ** power).bfloat16()
    c["pp"][:, :, :, 0] = (c["pp"][:, :, :, 0].double() * 2.0 ** -power).bfloat16()
    got, err = _decode(c)
    assert err == 0
    _close(got, want, tol)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("power", [60, 114])
def test_decode_scores_as_large_as_they_may_be(power, hq, hkv, d):
    """Keys to 2^116, so scores to 2^117: where one score is ahead of the
    others by more than their roundings, its value row is the result."""
    c = _decode_case(41, [77, 2000, 5], hq, hkv, d, 16, torch.bfloat16)
    for name in ("params", "pp"):
        c[name][:, :, :, 0] = (c[name][:, :, :, 0].double() * 2.0 ** power).bfloat16()
    got, err = _decode(c)
    assert err == 0 and bool(torch.isfinite(got).all())
    h, seen = ref.HALF_STEP[torch.bfloat16], 0
    for b, n in enumerate(c["lens"]):
        (k, _, _, _), (v, dev, _, _) = ref.sequence_rows(c["codes"], c["params"], c["layer"], c["table"][b], n, 16)
        for a in range(hq):
            kh = a // (hq // hkv)
            s = (c["q"][b, a].double() @ k[kh].T) * d ** -0.5
            best = s.topk(2)
            # sums of D + 8 fp32 products of codes up to 15 and offsets: 2^-10 of the largest is far above their roundings
            if best.values[0] - best.values[1] < 2.0 ** -10 * s.abs().max():
                continue
            seen += 1
            at = int(best.indices[0])
            tol = h * v[kh, at].abs() + h * dev[kh, at].abs() + 2.0 ** -20 * v[kh, at].abs() + 1e-12
            assert bool(((got[b, a].double() - v[kh, at]).abs() <= tol).all())
    assert seen > hq
