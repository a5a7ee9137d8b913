"""The shared prefixes' calls through csrc/calls.cpp and through the checks in ops.py:
the same results, and what the first does not take goes on to the second."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


class _Declines:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    import pagedserve_b200._native as native
    native.calls()
    if request.param == "python":
        monkeypatch.setattr(native, "_calls", _Declines())
    return request.param


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _spread(x):
    """The same values, every other element of a wider tensor."""
    y = torch.stack([x, torch.zeros_like(x)], -1).flatten(-2)[..., ::2]
    assert not y.is_contiguous() or y.numel() < 2
    return y


@pytest.mark.parametrize("spread", [False, True])
def test_pages(path, spread):
    from pagedserve_b200 import ops
    look = _spread if spread else (lambda x: x)
    free, state = ops.free_list(20, "cuda")
    store, shares = torch.zeros(4, 6, dtype=torch.int32, device="cuda"), ops.share_counts(20, "cuda")
    ops.extend_step(store, _i32([0]), _i32([0]), _i32([40]), free, state, 40, 16)
    pool = torch.randn(2, 20, 1, 16, 8, device="cuda")
    before = pool.clone()
    src, dst = ops.fork_tables(store, look(_i32([0, 0])), look(_i32([1, 2])), look(_i32([40, 32])), shares, free, state, 16)
    assert (src.tolist(), dst.tolist()) == ([2, -1], [3, -1]) and shares[0, :4].tolist() == [2, 2, 0, 0]
    ops.copy_blocks([pool], look(src), look(dst))
    before[:, 3] = before[:, 2]
    assert torch.equal(pool, before)
    ops.release_tables(store, look(_i32([1, 0])), look(_i32([40, 40])), look(_i32([0, 32])), shares, free, state, 16)
    assert store.tolist() == [[0, 1, 0, 0, 0, 0], [0] * 6, [0, 1, 0, 0, 0, 0], [0] * 6]
    assert shares[0, :4].tolist() == [1, 1, 0, 0] and int(state[1]) == 18


@pytest.mark.parametrize("spread", [False, True])
@pytest.mark.parametrize("unit", [False, True])
def test_decode(path, spread, unit):
    from pagedserve_b200 import ops
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 12, 2, 16, 64, generator=g).to(torch.float16).cuda() for _ in range(2))
    q = torch.randn(5, 14, 64, generator=g).to(torch.float16).cuda()
    table = _i32([[0, 1, 2, 3 + i] for i in range(5)])
    lens, cu, pre = _i32([50, 60, 48, 64, 7]), _i32([0, 4]), _i32([48])
    want = ops.paged_decode(q, k, v, table, lens, 1, scale=0.25)
    if spread:
        lens, cu, pre, table = _spread(lens), _spread(cu), _spread(pre), _spread(table)
    if unit:
        q = q[:, :, None]
    out = torch.empty(5, 14, 128, dtype=torch.float16, device="cuda")[..., :64]
    for kw in ({}, {"out": out[:, :, None] if unit else out}, {"max_context": 64}, {"workspace": torch.empty(1 << 25, dtype=torch.uint8, device="cuda")}):
        got = ops.paged_decode_shared(q, k, v, table, lens, cu, pre, 1, scale=0.25, **kw)
        assert got.shape == q.shape
        # each of the two rounds its probabilities and its result to f16: four half steps of the largest value, and the
        # fp32 scores' 2^-20 or so
        assert ((got.reshape(want.shape).double() - want.double()).abs() <= 4.1 * 2.0 ** -11 * v.abs().max().double()).all()


@pytest.mark.parametrize("spread", [False, True])
def test_verify(path, spread):
    from pagedserve_b200 import ops
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(7, 300, generator=g).cuda()
    tokens = torch.randint(0, 300, (7,), generator=g).cuda()
    cu, u = _i32([0, 3, 7]), torch.rand(7, 2, generator=g).cuda()
    heat = torch.tensor([0.0, 0.8], device="cuda")
    probs = torch.softmax(logits * 0.5, -1)
    tokens[1] = logits[0].argmax()
    import pagedserve_b200._native as native
    from tests.test_gpu_verify_tokens import _rule
    want, counts = _rule(logits.cpu(), tokens.cpu(), cu.tolist(), u.cpu(), heat.cpu(), probs.cpu())
    args = [logits, tokens, cu, u, heat]
    if spread:
        args = [_spread(x) for x in args]
        probs = _spread(probs)
    new, n = ops.verify_tokens(*args, draft_probs=probs)
    assert torch.equal(new.cpu(), want) and torch.equal(n.cpu(), counts)
    new, n = ops.verify_tokens(*args, draft_probs=probs, out=(torch.empty_like(new), torch.empty_like(n)))
    assert torch.equal(new.cpu(), want) and torch.equal(n.cpu(), counts)
    assert native.load() is not None


def test_what_is_wrong_is_refused_by_either(path):
    from pagedserve_b200 import ops
    free, state = ops.free_list(20, "cuda")
    store, shares = torch.zeros(4, 6, dtype=torch.int32, device="cuda"), ops.share_counts(20, "cuda")
    one = _i32([0])
    with pytest.raises(ValueError, match="shares"):
        ops.fork_tables(store, one, one, one, shares[:, :5], free, state, 16)
    with pytest.raises(ValueError, match="block_size"):
        ops.release_tables(store, one, one, one, shares, free, state, 0)
    with pytest.raises(ValueError):
        ops.fork_tables(store, one.long(), one, one, shares, free, state, 16)
    pool = torch.zeros(1, 20, 8, device="cuda")
    with pytest.raises(ValueError, match="int32"):
        ops.copy_blocks((pool,), one.long(), one)
    with pytest.raises(ValueError, match="one to four"):
        ops.copy_blocks((pool,) * 5, one, one)
    with pytest.raises(ValueError):
        ops.copy_blocks((pool.cpu(),), one, one)
    k = torch.zeros(1, 4, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    for kw, text in (({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"max_context": 99}, "max_context"), ({"layer": 1}, "layer")):
        with pytest.raises(ValueError, match=text):
            ops.paged_decode_shared(q, k, k, _i32([[0]]), one, _i32([0, 1]), one, **{"layer": 0, **kw})
    with pytest.raises(ValueError, match="uniforms"):
        ops.verify_tokens(torch.zeros(1, 5, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), _i32([0, 1]),
                          torch.zeros(1, 3, device="cuda"), torch.zeros(1, device="cuda"))
