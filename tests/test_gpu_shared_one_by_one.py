"""paged_decode_shared where it leaves a batch to paged_decode: what it promises holds there too."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_shared_decode import Batch, _i32, _same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


def test_no_groups():
    Batch([], alone=[5, 0, 300, 64, 17]).check()
    Batch([], alone=[5, 0, 300], hq=32, hkv=8, d=128, bs=32).check()


@pytest.mark.parametrize("d,batch", [(64, 2100), (96, 300)])
def test_directly_behind_a_step_that_writes_tables(d, batch):
    """extend_step's lengths and tables are read as it left them, with no other launch in between."""
    from pagedserve_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(d)
    hq, hkv, bs, steps = 4, 2, 16, 12
    blocks = batch * 3
    assert ops.decode_shared_workspace_bytes(batch, 1, hq, hkv, d, bs, 3 * bs, torch.bfloat16) == 0
    k, v = (torch.randn(1, blocks, hkv, bs, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    store = torch.zeros(batch, 3, dtype=torch.int32, device="cuda")
    free, state = ops.free_list(blocks, "cuda", order=torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).tolist())
    rows = torch.arange(batch, dtype=torch.int32, device="cuda")
    held = torch.zeros(batch, dtype=torch.int32, device="cuda")
    groups = _i32([0, batch]), _i32([0])
    q = torch.randn(steps, batch, hq, d, generator=g, device="cuda").to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got, seen = [], []
    for i in range(steps):
        new = torch.full((batch,), 3 if i % 2 else 4, dtype=torch.int32, device="cuda")
        total = batch * (3 if i % 2 else 4)
        torch.cuda.synchronize()
        _, ctx, _, _, tables = ops.extend_step(store, rows, held, new, free, state, total, bs, error_flag=err)
        got.append(ops.paged_decode_shared(q[i], k, v, tables, ctx, *groups, 0, error_flag=err))
        seen.append((tables, ctx))
        held = ctx
    torch.cuda.synchronize()
    assert int(err) == 0
    for i, (tables, ctx) in enumerate(seen):
        want = ops.paged_decode(q[i], k, v, tables, ctx, 0)
        assert torch.equal(got[i], want) and int(ctx[0]) == 7 * (i // 2) + 4 + 3 * (i % 2)


@pytest.mark.parametrize("batch", [dict(hq=4, hkv=2, d=96), dict(hq=14, hkv=2, dtype=torch.float32), dict(hq=4, hkv=2)], ids=["dims", "f32", "plan"])
def test_two_streams_at_once(batch):
    """Calls on two streams, and one with a workspace of the caller's: each has its own scratch."""
    from pagedserve_b200 import ops
    pairs = batch == dict(hq=4, hkv=2)
    cases = [Batch([_same(17, [1500 + g % 60, 3]) for g in range(1100 if pairs else 20)], seed=s, **batch) for s in (1, 2)]
    args = [(b.q.cuda(), b.k.cuda(), b.v.cuda(), b.table.cuda(), _i32(b.lens), _i32(b.cu), _i32(b.prefix), b.layer) for b in cases]
    for b in cases:
        assert ops.decode_shared_workspace_bytes(len(b.lens), len(b.prefix), b.hq, b.hkv, b.d, b.bs, b.table.shape[1] * b.bs, b.dtype) == 0
    b = cases[0]
    need = ops.decode_workspace_bytes(len(b.lens), b.hq, b.hkv, b.d, b.bs, b.table.shape[1] * b.bs, b.dtype)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    want = [ops.paged_decode(*a[:5], a[7]) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(10):
        got = []
        for s, a, w in zip(streams, args, (ws, None)):
            with torch.cuda.stream(s):
                got.append(ops.paged_decode_shared(*a, workspace=w))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("d", [64, 96])
@pytest.mark.parametrize("cu,prefix,bits", [([0, 3, 5], [100, 80], 0), ([0, 5, 3], [100, 80], 32), ([-1, 3, 5], [100, 80], 32), ([0, 3, 99], [100, 80], 32),
                                            ([0, 3, 5], [-5, 80], 4), ([0, 7, 5], [4, -1], 36), ([0], [], 0), ([7], [], 32), ([-1], [], 32)])
def test_malformed_groups_are_flagged(d, cu, prefix, bits):
    """Whichever kernel answers: the flag is the same, and every sequence is read on its own."""
    from pagedserve_b200 import ops
    b = Batch([_same(100, [20, 40, 3]), _same(80, [2, 2])], alone=[33], d=d, hq=4)
    want, tol = b.expected()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_decode_shared(b.q.cuda(), b.k.cuda(), b.v.cuda(), b.table.cuda(), _i32(b.lens), _i32(cu), _i32(prefix), b.layer, error_flag=err)
    assert int(err) == bits and ((got.cpu().double() - want).abs() <= tol).all()
    many = torch.arange(1000, dtype=torch.int32, device="cuda")  # more groups than threads
    err.zero_()
    many[701] = 5
    ops.paged_decode_shared(b.q.cuda(), b.k.cuda(), b.v.cuda(), b.table.cuda(), _i32(b.lens), many.clamp(max=6), torch.zeros(999, dtype=torch.int32, device="cuda"),
                            b.layer, error_flag=err)
    assert int(err) == 32
