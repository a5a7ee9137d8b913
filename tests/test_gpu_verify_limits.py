"""verify_tokens at the ends of its range: temperatures, random numbers and drafts that its fp32 weights do not decide."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_verify_tokens import _check, _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


LOW = [0.5, 0.3, 0.1, 1e-2, 1e-3, 1e-5, 1e-7, 1e-8, 1e-9, 1e-10, 1e-20, 1e-30, 1e-37]


@pytest.mark.parametrize("heat", LOW)
@pytest.mark.parametrize("probs", [None, torch.float32])
@pytest.mark.parametrize("dtype,shift", [(torch.float32, 20.0), (torch.float32, -20.0), (torch.float32, 0.0), (torch.bfloat16, 0.0), (torch.float16, 5.0)])
def test_low_temperatures(heat, probs, dtype, shift):
    """The maximum always has weight, however steep the weights beside it are; equal maxima have it alike."""
    args = list(_inputs([3, 1, 6, 2, 1, 4], 777, dtype, probs, 21, heat=torch.full((6,), heat)))
    args[0] = (args[0].float() + shift).to(dtype)
    args[0][5, [9, 70, 500]] = args[0][5].max()
    top = args[0].float().argmax(-1)
    args[1][1:13] = top[:12]  # drafts that are taken, and some that are not
    args[1][8] = (top[7] + 1) % 777
    _check(*args)


@pytest.mark.parametrize("heat", [0.2, 1e-8, 1e-9, 1e-10, 1e-37])
@pytest.mark.parametrize("probs", [None, torch.float32])
def test_low_temperatures_of_many_sequences(heat, probs):
    """Draws that are left for a second launch."""
    ns = [2] * 80 if probs else [1] * 160
    args = list(_inputs(ns, 50000, torch.float32, probs, 22, heat=torch.full((len(ns),), heat)))
    args[0] -= 7.0
    _check(*args)


def test_neighbours_of_the_maximum_at_low_temperatures():
    """Logits one and two units in the last place below the maximum, at temperatures of that size: with a random number
    of 0 the first token of any weight is drawn, down to weights of 2^-793 of the largest."""
    top = torch.tensor(20.5)
    down = [top]
    for _ in range(3):
        down.append(torch.nextafter(down[-1], torch.tensor(-1e9)))
    step = float(top - down[1])
    rows = torch.full((8, 40), -3.0)
    for r in range(8):
        rows[r, 30] = top
        rows[r, 20] = down[1]
        rows[r, 10] = down[2]
        rows[r, 5] = down[3]
    # octaves a step: 1.44 step / t
    heat = torch.tensor([step, step / 10, step / 100, step / 400, step / 550, step / 760, step / 1e4, step * 3])
    for u1 in (0.0, 0.5, 0.99):
        u = torch.full((8, 2), u1)
        _check(rows, torch.zeros(8, dtype=torch.int64), list(range(9)), u, heat, None)


def _borders():
    """Rows whose fp32 weights are off by nearly all that they can be, with random numbers next to a border.

    A logit of 0 at the end, equal ones some 60 octaves below it in front: the k-th of them ends at k w of the sum.  Their
    fp32 weight is off by the rounding of c = log2(e) / t, times 60, and by that of their exponent: temperatures and logits
    are looked for where both are large and of one sign.  The random number is a hair beside the border."""
    import numpy as np
    rng = np.random.default_rng(0)
    found = []
    heats = np.float32(1.4426950408889634 / (1.0 + rng.random(4000) / 64))
    c = 1.4426950408889634 / heats.astype(np.float64)
    of_c = c.astype(np.float32).astype(np.float64) / c - 1
    for sign in (1, -1):  # weights too large, too small
        for i in np.argsort(sign * of_c)[:12]:  # c32 below c: weights above theirs
            x = -(np.float32(62.0) + rng.random(4000).astype(np.float32) * 2)
            y = x.astype(np.float64) * c[i].astype(np.float32).astype(np.float64)
            up = y.astype(np.float32).astype(np.float64) - y
            x = x[np.argmax(sign * up)]
            w = np.exp(np.float64(x) / np.float64(heats[i]))
            total = 1 + 12800 * w
            for k in range(24, 48):  # the random number that is closest to the border on the wrong side
                u = np.float32(k * w / total)
                while sign * (np.float64(u) * total - k * w) <= 2e-8 * k * w:
                    u = np.nextafter(u, np.float32(sign))
                if sign * (np.float64(u) * total / (k * w) - 1) < 7e-8:
                    found.append((float(heats[i]), float(x), float(u)))
                    break
    return found


def test_next_to_borders_where_fp32_is_worst():
    cases = _borders()
    assert len(cases) > 16
    cases = (cases * 10)[:150]  # so many that one CTA has a row: its first warp's first tokens are cut no further
    logits = torch.full((len(cases), 12801), 0.0)
    u = torch.zeros(len(cases), 2)
    for r, (_, x, u1) in enumerate(cases):
        logits[r, :12800] = x
        u[r, 1] = u1
    new, _ = _check(logits, torch.zeros(len(cases), dtype=torch.int64), list(range(len(cases) + 1)), u, torch.tensor([h for h, _, _ in cases]), None)
    assert bool((new >= 23).all()) and bool((new <= 48).all())


@pytest.mark.parametrize("probs", [None, torch.float32])
@pytest.mark.parametrize("u1", [0.0, 1e-30, 1e-18, 2.0 ** -40, 1e-9, 1e-6, 1e-4, 2e-3, 1 - 2.0 ** -24])
def test_small_random_numbers(u1, probs):
    """They fall on the first tokens, however little weight those have."""
    for heat, vocab, ns in ((0.25, 3001, [1, 3, 2, 5] * 4), (1.0, 60000, [1, 2] * 3), (0.7, 777, [2] * 40)):
        args = list(_inputs(ns, vocab, torch.float32, probs, 23, heat=torch.full((len(ns),), heat), spread=4.0))
        args[3][:, 1] = u1
        _check(*args)


@pytest.mark.parametrize("near", [1e-7, 1e-6, 1e-5, 1e-4, 1e-2])
@pytest.mark.parametrize("batch,vocab", [(60, 400), (5, 9001), (80, 50000)])
def test_drafts_from_nearly_the_target(near, batch, vocab):
    """Probabilities within ``near`` of the target's, drafts refused all the same: the token is drawn from the little that is left.

    The target and its weights' sum are good to 3e-12 each, against what is left in all, about near / 4; next to a border
    of the 64-bit rule by no more than that a token's neighbour may be drawn."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(2 * batch, vocab, generator=g) * 1.5
    p = torch.softmax(logits.double() / 0.9, -1)
    probs = (p * (1 + near * (2 * torch.rand(p.shape, generator=g, dtype=torch.float64) - 1))).float()
    over = (probs.double() / p - 1)[::2]
    tokens = torch.zeros(2 * batch, dtype=torch.int64)
    tokens[1::2] = over.argmax(-1)
    u = torch.rand(2 * batch, 2, generator=g)
    u[:, 0] = 1 - 2.0 ** -24
    assert bool((over.amax(-1) > 1.2e-7).all())  # u0 q is above p, by 2^-24 of it at least
    heat = torch.full((batch,), 0.9)
    p = torch.softmax(logits.double() / heat[0].double(), -1)
    new, counts = _run(logits, tokens, list(range(0, 2 * batch + 1, 2)), u, heat, probs)
    assert counts.tolist() == [1] * batch
    w = (p - probs.double()).clamp(min=0)[::2]
    c = w.cumsum(-1)
    all_, at = c[:, -1], new[::2, None]
    assert bool((w.gather(1, at)[:, 0] > 0).all())
    target, room = u[::2, 1].double() * all_, 2 * 6e-12 + 1e-9 * all_
    assert bool((c.gather(1, at)[:, 0] + room > target).all()) and bool(((c - w).gather(1, at)[:, 0] - room <= target).all())


@pytest.mark.parametrize("heat", [1e-37, 1.1e-38, 1e-39, 1e-42, 2.0 ** -149])
@pytest.mark.parametrize("batch", [3, 200])
def test_the_least_temperatures(heat, batch):
    """Any temperature above 0 is one: equal maxima share p, and logits that differ by the least fp32 values by e or so."""
    vocab = 70000 if batch == 200 else 50
    logits = torch.full((batch, vocab), -2.0)
    logits[:, [7, 20, 33]] = 3.0
    # all tokens about 0, the first ones a few temperatures below
    logits[1::2] = -1e30
    logits[1::2, 5:15] = -float(torch.tensor(heat)) * torch.arange(9, -1, -1, dtype=torch.float64).float()
    u = torch.rand(batch, 2, generator=torch.Generator().manual_seed(4))
    args = (logits, torch.zeros(batch, dtype=torch.int64), list(range(batch + 1)), u, torch.full((batch,), heat), None)
    new, _ = _check(*args)
    assert batch == 3 or len(set(new[::2].tolist())) == 3 and len(set(new[1::2].tolist())) > 2


@pytest.mark.parametrize("probs", [None, torch.float16])
def test_a_vocabulary_beyond_the_fp32_weights(probs):
    """More tokens than fp32's sums are asked about: all of it in 64 bits."""
    vocab = (1 << 25) + 3
    g = torch.Generator().manual_seed(6)
    logits = (torch.rand(2, vocab, generator=g) * 3).half()
    tokens = torch.tensor([0, 12345678])
    q = None
    if probs is not None:
        q = torch.zeros(2, vocab, dtype=probs)
        q[0, 100:2100] = 5e-4
    for u in ([[0.5, 0.3], [0.1, 0.99999]], [[0.0, 0.7], [0.9, 1e-7]]):
        _check(logits, tokens, [0, 2], torch.tensor(u), torch.tensor([0.8]), q)
