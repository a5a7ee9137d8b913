"""Writes into the 4-bit pool and its read-back: codes and parameters equal
the plain form's, rows no slot names stay as they were, and the values read
back are within half a quantisation step of what was written."""

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


GEOMETRIES = [(14, 2, 64, 16), (32, 8, 128, 32), (4, 4, 80, 8), (3, 1, 2, 1), (2, 1, 256, 16), (6, 3, 96, 64)]


def _pool(gen, layers, blocks, hkv, bs, d, dtype):
    codes = torch.randint(0, 256, (layers, blocks, hkv, 2, bs, d // 2), generator=gen, dtype=torch.uint8)
    params = torch.randn(layers, blocks, hkv, 2, bs, 2, generator=gen).to(dtype)
    return codes, params


def _expect(codes, params, layer, slots, k, v, bs):
    codes, params = codes.clone(), params.clone()
    for i, x in enumerate((k, v)):
        c, step, mid = ref.quantize(x)
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                codes[layer, s // bs, :, i, s % bs] = ref.pack(c[t])
                params[layer, s // bs, :, i, s % bs, 0:1] = step[t]
                params[layer, s // bs, :, i, s % bs, 1:2] = mid[t]
    return codes, params


def _same(a, b):
    """Equal bit for bit, any NaN equal to any NaN."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, 0.0), torch.nan_to_num(b, 0.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d,bs", GEOMETRIES)
@pytest.mark.parametrize("tokens", [1, 37])
def test_write_and_gather(dtype, hq, hkv, d, bs, tokens):
    from pagedserve_b200 import ops
    gen = torch.Generator().manual_seed(d * 1000 + bs * 10 + tokens)
    blocks, layers, layer = -(-tokens // bs) + 3, 2, 1
    codes, params = _pool(gen, layers, blocks, hkv, bs, d, dtype)
    qkv = (torch.randn(tokens, (hq + 2 * hkv) * d + 8, generator=gen) * 3 + 1).to(dtype)
    k = qkv[:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
    v = qkv[:, (hq + hkv) * d:(hq + 2 * hkv) * d].view(tokens, hkv, d)
    v[0, 0] = 0.75  # a constant row is kept exactly
    slots = torch.randperm(blocks * bs, generator=gen)[:tokens]
    if tokens > 3:
        slots[2] = -1
    want_c, want_p = _expect(codes, params, layer, slots, k, v, bs)
    dc, dp, ds, dq = codes.cuda(), params.cuda(), slots.cuda(), qkv.cuda()
    dk = dq[:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
    dv = dq[:, (hq + hkv) * d:(hq + 2 * hkv) * d].view(tokens, hkv, d)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.reshape_and_cache_int4(dk, dv, dc, dp, ds, layer, error_flag=err)
    gk, gv = ops.gather_cache_int4(dc, dp, ds, layer, error_flag=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert torch.equal(dc.cpu(), want_c)
    assert torch.equal(dp.cpu(), want_p)
    live = slots >= 0
    for got, x, i in ((gk, k, 0), (gv, v, 1)):
        s = slots[live]
        val = ref.values(want_c[layer, s // bs, :, i, s % bs], want_p[layer, s // bs, :, i, s % bs])
        # one fp32 rounding and one of the type
        tol = val.abs() * (ref.HALF_STEP[dtype] + 2.0 ** -23) + 2.0 ** -25
        assert bool(((got.cpu()[live].double() - val).abs() <= tol).all())
        assert bool((got.cpu()[~live] == 0).all())
        step = want_p[layer, s // bs, :, i, s % bs, 0:1].double()
        mid = want_p[layer, s // bs, :, i, s % bs, 1:2].double()
        # half a step, the clipped end (7.5 steps off by a rounding of step) and the rounding of x^
        limit = step * (0.5 + 7.5 * 2 * ref.HALF_STEP[dtype]) + tol + step.abs() * 2.0 ** -20 + mid.abs() * 2.0 ** -23
        assert bool(((got.cpu()[live].double() - x[live].double()).abs() <= limit).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d,bs", [(14, 2, 64, 16), (32, 8, 128, 32), (3, 1, 80, 8), (1, 1, 2, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_write(dtype, hq, hkv, d, bs, in_place):
    """Rotated query and key bit-identical to the full-precision pool's
    operator, the pool to the plain form on that key."""
    from pagedserve_b200 import ops
    gen = torch.Generator().manual_seed(d + bs)
    tokens, layers, layer = 29, 2, 0
    blocks = -(-tokens // bs) + 2
    codes, params = _pool(gen, layers, blocks, hkv, bs, d, dtype)
    q = torch.randn(tokens, hq, d, generator=gen).to(dtype)
    k = torch.randn(tokens, hkv, d, generator=gen).to(dtype)
    v = torch.randn(tokens, hkv, d, generator=gen).to(dtype)
    ang = torch.rand(tokens, d, generator=gen, dtype=torch.float64) * 6.3
    cos, sin = ang.cos().to(dtype), ang.sin().to(dtype)
    slots = torch.randperm(blocks * bs, generator=gen)[:tokens]
    slots[5] = -1
    qr, kr = ref.rotate(q, cos[:, None], sin[:, None]), ref.rotate(k, cos[:, None], sin[:, None])
    want_c, want_p = _expect(codes, params, layer, slots, kr, v, bs)
    dq, dk, dc, dp = q.cuda(), k.cuda(), codes.cuda(), params.cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    oq, ok = ops.rope_reshape_and_cache_int4(dq, dk, v.cuda(), cos.cuda(), sin.cuda(), dc, dp, slots.cuda(), layer,
                                             query_out=dq if in_place else None, key_out=dk if in_place else None,
                                             error_flag=err)
    kc = torch.zeros(1, blocks, hkv, bs, d, dtype=dtype, device="cuda")
    fq, fk = ops.rope_reshape_and_cache(q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), kc, kc.clone(),
                                        slots.cuda(), 0)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert torch.equal(oq, fq) and torch.equal(ok, fk)
    assert torch.equal(oq.cpu(), qr) and torch.equal(ok.cpu(), kr)
    assert torch.equal(dc.cpu(), want_c) and torch.equal(dp.cpu(), want_p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_extreme_rows(dtype):
    """Infinities and NaN make their row NaN and no other; zeros, the largest
    values, subnormals and one-sided rows are quantised as the format says."""
    from pagedserve_b200 import ops
    hkv, d, bs = 2, 64, 16
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    gen = torch.Generator().manual_seed(3)
    rows = [torch.zeros(d), torch.full((d,), -big), torch.linspace(-big, big, d), torch.linspace(0, tiny, d),
            torch.randn(d, generator=gen).abs() + 100, torch.randn(d, generator=gen) * 1e-3,
            torch.linspace(-1, 1, d) * big]
    bad = [torch.randn(d, generator=gen) for _ in range(4)]
    bad[0][3], bad[1][63], bad[2][0], bad[3][17] = math.inf, -math.inf, math.nan, math.nan
    bad[3][18] = math.inf
    x = torch.stack([torch.stack([r, r.flip(0)]) for r in rows + bad]).to(dtype)
    t = x.shape[0]
    codes, params = _pool(gen, 1, 2, hkv, bs, d, dtype)
    slots = torch.randperm(2 * bs, generator=gen)[:t]
    want_c, want_p = _expect(codes, params, 0, slots, x, x.flip(0), bs)
    dc, dp = codes.cuda(), params.cuda()
    ops.reshape_and_cache_int4(x.cuda(), x.flip(0).cuda(), dc, dp, slots.cuda(), 0)
    k, _ = ops.gather_cache_int4(dc, dp, slots.cuda(), 0)
    torch.cuda.synchronize()
    assert torch.equal(dc.cpu(), want_c) and _same(dp.cpu(), want_p)
    # (a linspace over the whole range of an 8-bit exponent overflows to non-finite inputs itself: 2 max > the fp32 maximum)
    broken = ~torch.isfinite(x.float()).all(-1, keepdim=True)
    assert torch.equal(torch.isnan(k.cpu()), broken.expand(x.shape))
    assert bool(broken[len(rows):].any(1).all()) and not bool(broken[[0, 1, 3, 4, 5, 6]].any())


def test_slots_past_the_pool_are_flagged_and_skipped():
    from pagedserve_b200 import ops
    gen = torch.Generator().manual_seed(9)
    codes, params = _pool(gen, 1, 4, 2, 16, 64, torch.bfloat16)
    k = torch.randn(3, 2, 64, generator=gen).bfloat16()
    slots = torch.tensor([5, 64, 1 << 40])
    want_c, want_p = _expect(codes, params, 0, torch.tensor([5, -1, -1]), k, k, 16)
    dc, dp = codes.cuda(), params.cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.reshape_and_cache_int4(k.cuda(), k.cuda(), dc, dp, slots.cuda(), 0, error_flag=err)
    assert int(err.item()) == 2
    assert torch.equal(dc.cpu(), want_c) and torch.equal(dp.cpu(), want_p)
    err.zero_()
    gk, _ = ops.gather_cache_int4(dc, dp, slots.cuda(), 0, error_flag=err)
    assert int(err.item()) == 2 and bool((gk[1:] == 0).all()) and bool((gk[0] != 0).any())


def test_no_tokens():
    from pagedserve_b200 import ops
    codes, params = _pool(torch.Generator().manual_seed(1), 1, 2, 2, 16, 64, torch.bfloat16)
    dc, dp = codes.cuda(), params.cuda()
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.empty(0, dtype=torch.int64, device="cuda")
    ops.reshape_and_cache_int4(none, none, dc, dp, slots, 0)
    k, v = ops.gather_cache_int4(dc, dp, slots, 0)
    assert k.shape == (0, 2, 64) and v.shape == (0, 2, 64)
    assert torch.equal(dc.cpu(), codes)


def test_side_stream_and_graph():
    """The same bytes on another stream and from a replayed capture with new inputs in the same buffers."""
    from pagedserve_b200 import ops
    gen = torch.Generator().manual_seed(4)
    codes, params = _pool(gen, 1, 8, 2, 16, 64, torch.bfloat16)
    slots = torch.randperm(128, generator=gen)[:50]
    a, b = (torch.randn(50, 2, 64, generator=gen).bfloat16() for _ in range(2))
    want_c, want_p = _expect(codes, params, 0, slots, b, a, 16)
    dc, dp, dk, dv, ds = codes.cuda(), params.cuda(), a.cuda(), a.cuda(), slots.cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.reshape_and_cache_int4(dk, dv, dc, dp, ds, 0)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ops.reshape_and_cache_int4(dk, dv, dc, dp, ds, 0)
        gk, gv = ops.gather_cache_int4(dc, dp, ds, 0)
    dk.copy_(b)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(dc.cpu(), want_c) and torch.equal(dp.cpu(), want_p)
    k2, v2 = ops.gather_cache_int4(dc, dp, ds, 0)
    assert torch.equal(gk, k2) and torch.equal(gv, v2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("hq,hkv,d,tokens", [(14, 2, 64, 1), (14, 2, 64, 3), (14, 2, 64, 7), (3, 1, 128, 1),
                                             (5, 3, 32, 5), (1, 1, 256, 1)])
def test_last_row_of_a_partly_filled_warp(dtype, rope, hq, hkv, d, tokens):
    """A token count whose pieces do not fill the last warp, the last slot live
    and the last V row's extremes outside its last piece: the row's codes are
    the whole row's, whichever lanes hold copies of that piece."""
    from pagedserve_b200 import ops
    gen = torch.Generator().manual_seed(d + tokens)
    bs, layers, layer = 16, 2, 1
    codes, params = _pool(gen, layers, 3, hkv, bs, d, dtype)
    q = torch.randn(tokens, hq, d, generator=gen).to(dtype)
    k = torch.randn(tokens, hkv, d, generator=gen).to(dtype)
    v = torch.randn(tokens, hkv, d, generator=gen).to(dtype)
    v[-1, -1, 0], v[-1, -1, d // 2] = 9.0, -7.0
    ang = torch.rand(tokens, d, generator=gen, dtype=torch.float64) * 6.3
    cos, sin = ang.cos().to(dtype), ang.sin().to(dtype)
    slots = torch.randperm(3 * bs, generator=gen)[:tokens]
    kw = ref.rotate(k, cos[:, None], sin[:, None]) if rope else k
    want_c, want_p = _expect(codes, params, layer, slots, kw, v, bs)
    for _ in range(3):
        dc, dp = codes.cuda(), params.cuda()
        if rope:
            oq, ok = ops.rope_reshape_and_cache_int4(q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), dc, dp,
                                                     slots.cuda(), layer)
            assert torch.equal(oq.cpu(), ref.rotate(q, cos[:, None], sin[:, None])) and torch.equal(ok.cpu(), kw)
        else:
            ops.reshape_and_cache_int4(k.cuda(), v.cuda(), dc, dp, slots.cuda(), layer)
        assert torch.equal(dc.cpu(), want_c) and torch.equal(dp.cpu(), want_p)
