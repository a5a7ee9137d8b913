"""verify_tokens against its rule in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


def _rule(logits, tokens, cu, u, heat, probs):
    """(new tokens, counts) as the rule says, row by row in float64."""
    out, counts = torch.full((tokens.shape[0],), -1, dtype=torch.int64), []
    v = logits.shape[1]
    u = u.double()
    for b in range(len(cu) - 1):
        counts.append(0)
        for r in range(cu[b], cu[b + 1]):
            x = logits[r].double()
            if heat[b] > 0:
                e = torch.exp((x - x.max()) / float(heat[b]))
                p = e / e.sum()
            else:
                p = torch.zeros(v, dtype=torch.float64)
                p[int((x == x.max()).nonzero()[0])] = 1
            d = int(tokens[r + 1]) if r + 1 < cu[b + 1] else -1
            counts[-1] += 1
            w = p
            if 0 <= d < v:
                q = torch.zeros(v, dtype=torch.float64)
                if probs is None:
                    q[d] = 1
                else:
                    q = probs[r].double().nan_to_num(0, posinf=math.inf).clamp(min=0)
                if float(u[r, 0] * q[d]) < float(p[d]):
                    out[r] = d
                    continue
                w = (p - q).clamp(min=0)
                if float(w.sum()) == 0:
                    w = p
            c = w.cumsum(0)
            out[r] = int(torch.searchsorted(c, (u[r, 1] * c[-1])[None], right=True).clamp(max=int(w.nonzero()[-1])))
            break
    return out, torch.tensor(counts, dtype=torch.int32)


def _inputs(ns, vocab, dtype, probs_dtype, seed, heat=None, spread=2.0):
    """Rows of spread-out logits with one token that stands out; drafts from another draw of the same rows."""
    g = torch.Generator().manual_seed(seed)
    cu = [0]
    for n in ns:
        cu.append(cu[-1] + n)
    t = cu[-1]
    logits = (torch.randn(t, vocab, generator=g) * spread).to(dtype)
    if vocab > 2 and t:
        peak = torch.randint(0, vocab, (t, 1), generator=g)
        logits.scatter_(1, peak, torch.full((t, 1), math.log(vocab) + spread ** 2 / 2).to(dtype))
    u = torch.rand(t, 2, generator=g)
    if heat is None:
        heat = torch.rand(len(ns), generator=g) + 0.5
        heat[torch.rand(len(ns), generator=g) < 0.2] = 0
    heat = torch.as_tensor(heat, dtype=torch.float32)
    probs = None
    tokens = torch.randint(0, vocab, (t,), generator=g)
    if t:
        z = logits.double() + 0.7 * torch.randn(t, vocab, generator=g)
        q = torch.softmax(z, -1)
        if probs_dtype is not None:
            probs = q.to(probs_dtype)
            tokens[1:] = torch.multinomial(probs.double(), 1, generator=g)[:-1, 0]
        else:
            guess = torch.where(torch.rand(t, generator=g) < 0.8, logits.double().argmax(-1), tokens)
            tokens[1:] = guess[:-1]
    return logits, tokens, cu, u, heat, probs


def _run(logits, tokens, cu, u, heat, probs, **kw):
    from pagedserve_b200 import ops
    c = lambda x: None if x is None else x.cuda()
    new, counts = ops.verify_tokens(c(logits), c(tokens), torch.tensor(cu, dtype=torch.int32, device="cuda"), c(u), c(heat), draft_probs=c(probs), **kw)
    return new.cpu(), counts.cpu()


def _check(*args):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    new, counts = _run(*args, error_flag=err)
    want, want_counts = _rule(*args)
    assert int(err) == 0
    assert torch.equal(counts, want_counts)
    assert torch.equal(new, want)
    return new, counts


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("probs", [None, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ns,vocab", [([1], 1), ([3], 2), ([2, 1, 5], 7), ([1, 0, 6, 0, 0, 2], 33), ([4] * 30, 1000), ([9, 8, 17, 1], 4099), ([6, 3], 32003)])
def test_types_and_sizes(ns, vocab, dtype, probs):
    for seed in range(3):
        _check(*_inputs(ns, vocab, dtype, probs, seed))


@pytest.mark.parametrize("ns,probs", [([1] * 3, None), ([6], torch.float32), ([1] * 80, None), ([5] * 20, torch.bfloat16), ([21], None)])
def test_a_large_vocabulary(ns, probs):
    _check(*_inputs(ns, 151936, torch.bfloat16, probs, len(ns)))


@pytest.mark.parametrize("batch", [1, 9, 10, 18, 19, 37, 74, 75, 150, 300, 1000])
def test_every_size_of_cluster(batch):
    """Batches at which the number of CTAs a sequence has changes."""
    _check(*_inputs([2] * batch, 517, torch.bfloat16, torch.float32, batch))


def test_many_samples_of_one_row():
    """Rows that differ in their random numbers alone: uniforms spread over the whole range fall on the tokens they belong to."""
    n, vocab = 4096, 5000
    logits = (torch.randn(1, vocab, generator=torch.Generator().manual_seed(1)) * 2).to(torch.float16).expand(n, vocab).contiguous()
    u = torch.zeros(n, 2)
    u[:, 1] = torch.arange(n) / n
    u[-1, 1] = 1 - 2.0 ** -24
    new, _ = _check(logits, torch.zeros(n, dtype=torch.int64), list(range(n + 1)), u, torch.full((n,), 0.9), None)
    assert bool((new[1:] >= new[:-1]).all()) and int(new[0]) == 0


@pytest.mark.parametrize("probs", [False, True])
def test_tokens_are_distributed_as_the_target(probs):
    """First tokens of many sequences: accepted drafts and replacements together follow p.  The counts' distance from
    their expectation, sum (n - E)^2 / E, has mean 7 and variance 14 for 8 tokens: below 35 but for 1 in 10^5."""
    n, v = 40000, 8
    g = torch.Generator().manual_seed(3)
    row = torch.randn(1, v, generator=g)
    p = torch.softmax(row.double() / 0.8, -1)[0]
    q = torch.softmax(torch.randn(1, v, generator=g), -1)
    drafts = torch.multinomial(q.double(), n, replacement=True, generator=g)[0] if probs else torch.randint(0, v, (n,), generator=g)
    logits = row.expand(2 * n, v).contiguous()
    tokens = torch.stack([torch.zeros(n, dtype=torch.int64), drafts], 1).reshape(-1)
    u = torch.rand(2 * n, 2, generator=g)
    new, counts = _run(logits, tokens, list(range(0, 2 * n + 1, 2)), u, torch.full((n,), 0.8), q.expand(2 * n, v).contiguous() if probs else None)
    seen = torch.bincount(new[::2], minlength=v).double()
    assert float(((seen - n * p) ** 2 / (n * p)).sum()) < 35
    assert 0 < int((counts == 2).sum()) < n


def test_temperature_zero_takes_the_first_maximum():
    logits = torch.tensor([[1.0, 5, 5, 2], [7, 7, 7, 7], [-math.inf, -1, -math.inf, -1], [0, 1, 2, 3]]).to(torch.bfloat16)
    tokens, u = torch.tensor([9, 1, 0, 3]), torch.tensor([[0.99, 0.99]] * 4)
    args = (logits, tokens, [0, 4], u, torch.zeros(1), None)
    new, counts = _check(*args)
    assert new.tolist() == [1, 0, 1, -1] and counts.tolist() == [3]  # the third draft (3) is the second of two maxima


def test_masked_tokens_are_never_drawn():
    args = list(_inputs([4] * 50, 300, torch.float32, None, 5, heat=torch.full((50,), 1.0)))
    args[0][:, ::3] = -math.inf
    args[3][:, 1] = torch.where(torch.rand(200, generator=torch.Generator().manual_seed(2)) < 0.5, 0.0, 1 - 2.0 ** -24)
    new, _ = _check(*args)
    assert not bool((new[new >= 0] % 3 == 0).any())
    args[0][:] = -math.inf
    args[0][:, 77] = -5.0  # all of p on one token
    new, _ = _check(*args)


def test_drafts_that_are_none():
    args = list(_inputs([5, 4, 3], 100, torch.bfloat16, torch.float32, 8, heat=torch.ones(3)))
    args[1][2] = -1      # behind row 1
    args[1][7] = 100     # past the vocabulary
    _check(*args)


def test_equal_distributions_are_always_taken():
    args = list(_inputs([6] * 20, 700, torch.float32, torch.float32, 9, heat=torch.ones(20)))
    args[5] = torch.softmax(args[0], -1)
    args[1][1:] = torch.multinomial(args[5], 1, generator=torch.Generator().manual_seed(0))[:-1, 0]
    args[3][:, 0] = args[3][:, 0].clamp(max=0.999)
    _, counts = _check(*args)
    assert counts.tolist() == [6] * 20


def test_nothing_left_of_the_target():
    """p below q everywhere: drawn from p itself."""
    args = list(_inputs([2] * 8, 50, torch.float32, torch.float32, 10, heat=torch.ones(8)))
    args[5].fill_(1.0)
    args[3][:, 0] = 0.9999
    _check(*args)


def test_rows_without_probabilities_are_flagged():
    for value, heat, first in ((math.nan, 1.0, 7), (math.inf, 0.7, 7), (-math.inf, 1.0, 0)):
        args = list(_inputs([1, 1, 1], 40, torch.float32, None, 11, heat=torch.tensor([1.0, heat, 0.0])))
        if value == -math.inf:
            args[0][1] = value
        else:
            args[0][1, [7, 9]] = value
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        new, counts = _run(*args, error_flag=err)
        assert int(err) == 2048 and int(new[1]) == first and counts.tolist() == [1, 1, 1]
        args[0][1] = 0
        want, _ = _rule(*args)
        assert new[0] == want[0] and new[2] == want[2]
    for heat in (-1.0, math.nan, math.inf):
        args = list(_inputs([2, 1], 40, torch.float32, None, 12, heat=torch.tensor([heat, 1.0])))
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = _run(*args, error_flag=err)
        args[4] = torch.tensor([0.0, 1.0])
        want = _rule(*args)
        assert int(err) == 2048 and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_probabilities_that_are_none_count_as_nothing():
    args = list(_inputs([3] * 10, 60, torch.bfloat16, torch.float32, 13, heat=torch.ones(10)))
    args[5][:, ::7] = -0.5
    args[5][:, 3::7] = math.nan
    _check(*args)


def test_strides_padding_and_given_outputs():
    from pagedserve_b200 import ops
    logits, tokens, cu, u, heat, probs = _inputs([3, 2, 4], 1001, torch.float16, torch.bfloat16, 14)
    wide = torch.full((9 + 5, 1100), 9.0, dtype=torch.float16, device="cuda")
    wide[:9, 3:1004] = logits.cuda()
    wide_q = torch.zeros(14, 1003, dtype=torch.bfloat16, device="cuda")
    wide_q[:9, 1:1002] = probs.cuda()
    pad = lambda x: torch.cat([x, torch.zeros((5,) + x.shape[1:], dtype=x.dtype)]).cuda()
    out = (torch.full((14,), 55, dtype=torch.int64, device="cuda"), torch.full((4,), 55, dtype=torch.int32, device="cuda"))
    # rows behind the last sequence hold no token; a sequence of no rows has none
    new, counts = ops.verify_tokens(wide[:, 3:1004], pad(tokens), torch.tensor(cu + [9], dtype=torch.int32, device="cuda"), pad(u), pad(heat)[:4],
                                    draft_probs=wide_q[:, 1:1002], out=out)
    assert new is out[0] and counts is out[1]
    want, want_counts = _rule(logits, tokens, cu, u, heat, probs)
    assert torch.equal(new[:9].cpu(), want) and bool((new[9:] == -1).all()) and counts.tolist() == want_counts.tolist() + [0]
    column = torch.empty(1001, 14, dtype=torch.float16, device="cuda").t()
    column[:9] = logits.cuda()
    new, _ = ops.verify_tokens(column, pad(tokens), torch.tensor(cu, dtype=torch.int32, device="cuda"), pad(u), pad(heat)[:3], draft_probs=wide_q[:, 1:1002])
    assert torch.equal(new[:9].cpu(), want)


def test_malformed_sequences_are_flagged():
    logits, tokens, _, u, heat, _ = _inputs([3, 3, 3], 100, torch.bfloat16, None, 15)
    for cu, bad in (([0, 5, 3, 9], 1), ([-2, 3, 6, 9], 0), ([0, 3, 6, 99], 2)):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        new, counts = _run(logits, tokens, cu, u, heat, None, error_flag=err)
        assert int(err) == 32 and int(counts[bad]) == 0
    new, counts = _run(logits[:0], tokens[:0], [0, 0, 0], u[:0], heat[:2], None)
    assert new.shape == (0,) and counts.tolist() == [0, 0]


def test_captured_and_replayed():
    from pagedserve_b200 import ops
    a = _inputs([4] * 12, 2000, torch.bfloat16, torch.float32, 16)
    dev = [x.cuda() if torch.is_tensor(x) else x for x in a]
    cu = torch.tensor(a[2], dtype=torch.int32, device="cuda")
    call = lambda: ops.verify_tokens(dev[0], dev[1], cu, dev[3], dev[4], draft_probs=dev[5])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, counts = call()
    for seed in range(3):
        b = _inputs([4] * 12, 2000, torch.bfloat16, torch.float32, 17 + seed)
        for i in (0, 1, 3, 4, 5):
            dev[i].copy_(b[i])
        graph.replay()
        want, want_counts = _rule(*b)
        assert torch.equal(new.cpu(), want) and torch.equal(counts.cpu(), want_counts)
