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
