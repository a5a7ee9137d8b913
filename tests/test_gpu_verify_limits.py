"""verify_tokens at the ends of its range: temperatures, random numbers and drafts that its fp32 weights do not decide."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_verify_tokens import _check, _inputs

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
