"""CPU: the router's refusal of a tangent names the router's operators, the sort's names its own."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

import metalblas_b200 as mb

IDS = torch.zeros(4, 2, dtype=torch.int32)


@pytest.mark.parametrize("call,name", [
    (lambda t: mb.expert_route(t, 2), "expert_route"), (lambda t: mb.expert_balance(t, IDS), "expert_balance"),
    (lambda t: mb.expert_gather(t, mb.ExpertOrder(IDS, IDS, IDS[:, 0])), "expert_gather"),
    (lambda t: mb.expert_combine(t, None, mb.ExpertOrder(IDS, IDS, IDS[:, 0])), "expert_combine")])
def test_the_operator_is_named(call, name):
    with fwd.dual_level(), pytest.raises(NotImplementedError, match=f"{name}.*forward-mode"):
        call(fwd.make_dual(torch.zeros(4, 8), torch.ones(4, 8)))
