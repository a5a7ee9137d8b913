"""paged_decode_shared with 9 to 16 q heads per kv head, at both head sizes."""

from __future__ import annotations

import random

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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,bs", [(16, 1, 16), (9, 1, 32), (32, 2, 64), (24, 2, 128), (30, 3, 16), (88, 8, 32)])
@pytest.mark.parametrize("d", [64, 128])
def test_geometries(hq, hkv, bs, d, dtype):
    Batch([_same(530, [0, 1, 90, 33, 700]), (70, [0, 71, 20, 90])], alone=[45], hq=hq, hkv=hkv, d=d, bs=bs, dtype=dtype).check()
    Batch([_same(129, [5] * 33)], hq=hq, hkv=hkv, d=d, bs=bs, dtype=dtype, seed=1).check()


@pytest.mark.parametrize("hq,hkv", [(16, 1), (24, 2), (11, 1)])
@pytest.mark.parametrize("seed", range(4))
def test_pairs_and_single_tiles_in_any_order(hq, hkv, seed):
    rng = random.Random(hq + seed)
    tile = 128 // (hq // hkv)
    groups = [_same(rng.choice([1, 63, 64, 65, 64 * 3, 64 * 5 + 7, 64 * 9]),
                    [rng.choice([0, 1, 20]) for _ in range(rng.choice([2, tile - 1, tile, tile + 1, 2 * tile, 2 * tile + 1, 3 * tile]))])
              for _ in range(rng.randint(2, 5))]
    Batch(groups, hq=hq, hkv=hkv, d=128, bs=16, seed=seed).check()


def test_long_prefixes_and_own_parts():
    Batch([_same(5000, [37 * i for i in range(20)])], alone=[3000], hq=32, hkv=2, d=128, bs=32, seed=2).check()
