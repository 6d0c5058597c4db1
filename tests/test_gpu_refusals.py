"""Refusals that come before anything is allocated for the result."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("experts", [0, -1, 1025, 1 << 40, (1 << 63) - 1, -(1 << 63)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_numbers_of_experts(experts, dtype):
    with pytest.raises(ValueError):
        mb.expert_sort(torch.zeros(4, 2, dtype=dtype, device=DEV), experts)
