"""PagedModelRunner's refusals of grouped decode steps, on the CPU."""

from __future__ import annotations

import pytest
import torch

from pagedserve_b200.model_runner import PagedModelRunner


def test_a_four_bit_step_with_groups_is_refused_before_it_writes(monkeypatch):
    runner = object.__new__(PagedModelRunner)
    runner.kv_bits, runner.block_size = 4, 16
    monkeypatch.setattr(PagedModelRunner, "_layers", lambda *a, **kw: pytest.fail("the step has begun"))
    z, i = torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="16-bit pool"):
        runner.decode(z, z, i[None], i + 1, z, groups=(i, i[:0]))
