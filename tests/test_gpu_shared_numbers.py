"""paged_decode_shared where scores are infinite or no numbers: it gives what its definition does."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_shared_decode import Batch, _same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


GEOMETRIES = [dict(), dict(dtype=torch.float16), dict(hq=16, hkv=1), dict(hq=32, hkv=8, d=128, bs=32), dict(hq=12, hkv=1, d=128, bs=64)]


@pytest.mark.parametrize("kw", GEOMETRIES, ids=range(len(GEOMETRIES)))
@pytest.mark.parametrize("where", ["own", "prefix", "whole own part"])
def test_scores_of_minus_infinity_have_no_weight(kw, where):
    """Keys whose scores leave fp32's range below (or are -infinity as f16 holds them), among others and by themselves."""
    b = Batch([_same(200, [1, 40, 300, 17]), _same(90, [2, 65])], alone=[70], **kw)
    dtype, channel, group = b.dtype, 5, b.hq // b.hkv
    b.q[..., channel] = 8.0
    # scores of the finite keys: d products and sums in fp32; probabilities, sums and the result as in Batch.expected,
    # each at most its bound times the largest value
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    pools = b.k[b.layer].nan_to_num(0).abs().max().item() * b.q.abs().sum(-1).max().item() * b.d ** -0.5
    room = u * 1.01 + 2 * (b.d + 4) * 2.0 ** -24 * pools + 2.0 ** -19
    low = -3e38 if dtype == torch.bfloat16 else -math.inf
    hit = {"own": [(0, 200), (1, 203), (1, 239), (2, 200), (2, 216), (2, 217), (3, 204), (4, 91), (6, 0), (6, 16), (6, 63)] + [(2, 400 + i) for i in range(40)],
           "prefix": [(0, 0), (0, 64), (0, 65), (4, 3), (4, 89)] + [(0, 100 + i) for i in range(64)],
           "whole own part": [(1, 200 + i) for i in range(40)] + [(4, 90 + i) for i in range(2)]}[where]
    for i, pos in hit:
        for j in ([i] if pos >= 200 or i == 6 or (i >= 4 and pos >= 90) else range(4) if i < 4 else (4, 5)):
            b.k[b.layer, b.tables[j][pos // b.bs], :, pos % b.bs, channel] = low
    got = b.run().cpu().double()
    v_max = 0.0
    want = torch.zeros_like(got)
    for i, n in enumerate(b.lens):
        t = torch.tensor(b.tables[i])
        k, v = (x[b.layer, t].transpose(0, 1).reshape(b.hkv, -1, b.d)[:, :n].double() for x in (b.k, b.v))
        v_max = max(v_max, v.abs().max().item())
        for h in range(b.hkv):
            want[i, h * group:(h + 1) * group] = torch.softmax(b.q[i, h * group:(h + 1) * group].double() @ k[h].T * b.d ** -0.5, -1) @ v[h]
    assert bool(torch.isfinite(want).all())
    tiny = max(b.lens) * 2.0 ** -25 * v_max if dtype == torch.float16 else 0.0
    assert bool(((got - want).abs() <= room * v_max + u * want.abs() + tiny).all())


@pytest.mark.parametrize("kw", GEOMETRIES, ids=range(len(GEOMETRIES)))
def test_nothing_but_scores_of_minus_infinity(kw):
    b = Batch([_same(80, [3, 20])], alone=[5, 40], **kw)
    b.q[..., 5] = 8.0
    want = b.run().cpu()
    for i in (1, 2):
        for pos in range(b.lens[i]):
            b.k[b.layer, b.tables[i][pos // b.bs], :, pos % b.bs, 5] = -math.inf
    got = b.run().cpu()
    # the second sequence's prefix is the first one's too, whose last three tokens alone are left to it
    assert bool((got[1:3] == 0).all()) and torch.equal(got[3], want[3]) and bool(torch.isfinite(got[0]).all())


def _same_but(b, got, want, rows):
    """The other rows are what they were."""
    keep = torch.ones(want.shape[:2], dtype=torch.bool)
    for where in rows:
        keep[where] = False
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("kw", GEOMETRIES, ids=range(len(GEOMETRIES)))
def test_an_own_part_of_one_token_that_is_no_number(kw):
    """The first token behind a fork: its key is NaN, so is the row, however finite the prefix's part is."""
    b = Batch([_same(160, [1, 1, 30, 0])], alone=[1, 40], **kw)
    group = b.hq // b.hkv
    want = b.run().cpu()
    assert bool(torch.isfinite(want).all())
    h = b.hkv - 1
    heads = slice(h * group, (h + 1) * group)
    for i, pos in ((1, 160), (4, 0)):
        blk = b.tables[i][pos // b.bs]
        b.k[b.layer, blk, h, pos % b.bs] = math.nan
    got = b.run().cpu()
    assert bool(got[1, heads].isnan().all()) and bool(got[4, heads].isnan().all())
    _same_but(b, got, want, [(1, heads), (4, heads)])


@pytest.mark.parametrize("kw", GEOMETRIES, ids=range(len(GEOMETRIES)))
def test_a_prefix_of_one_token_that_is_no_number(kw):
    b = Batch([_same(1, [0, 5, 40]), _same(64, [3, 3])], **kw)
    group = b.hq // b.hkv
    want = b.run().cpu()
    for t in b.tables[:3]:  # every sequence holds a copy of the block the prefix ends in
        b.k[b.layer, t[0], 0, 0] = math.nan
    got = b.run().cpu()
    assert bool(got[:3, :group].isnan().all())
    _same_but(b, got, want, [(slice(0, 3), slice(0, group))])


@pytest.mark.parametrize("kw", GEOMETRIES, ids=range(len(GEOMETRIES)))
@pytest.mark.parametrize("shape", [dict(groups=[_same(300, [0, 20, 33]), _same(70, [1] * 20)], alone=[50]), dict(groups=[_same(4000, [5, 600])])], ids=["short", "long"])
def test_queries_that_are_no_numbers(kw, shape):
    b = Batch(**shape, **kw)
    want = b.run().cpu()
    b.q[1, 0, 7] = math.nan
    b.q[0, b.hq - 1] = math.nan
    b.q[-1] = math.nan
    got = b.run().cpu()
    assert bool(got[1, 0].isnan().all()) and bool(got[0, -1].isnan().all()) and bool(got[-1].isnan().all())
    _same_but(b, got, want, [(1, 0), (0, b.hq - 1), (-1,)])


@pytest.mark.parametrize("kw", GEOMETRIES, ids=range(len(GEOMETRIES)))
def test_idle_rows_whose_queries_are_no_numbers(kw):
    b = Batch([(200, [0, 230, 0, 201, 199]), (64, [0, 0])], alone=[0, 40], **kw)
    want = b.run().cpu()
    idle = [i for i, n in enumerate(b.lens) if n == 0]
    b.q[idle] = math.nan
    got = b.run().cpu()
    assert bool((got[idle] == 0).all()) and torch.equal(got, want)
