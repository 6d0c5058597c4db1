"""CPU: arguments that are no tensors are refused by the framework's own assertions, with or
without the host fast path in front of them."""
from __future__ import annotations

import pytest
import torch

import metalblas_b200 as mb
from metalblas_b200 import experts, quantized

I8, F32 = torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
IDS = torch.zeros(4, 2, dtype=torch.int64)
ORDER = mb.ExpertOrder(torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32),
                       torch.zeros(3, dtype=torch.int32))
ROWS = torch.zeros(8, 8)


@pytest.mark.parametrize("call", [
    lambda x: mb.quantize(x), lambda x: mb.scaled_mm(x, I8.t(), F32, F32), lambda x: mb.scaled_mm(I8, x, F32, F32),
    lambda x: mb.scaled_mm(I8, I8.t(), x, F32), lambda x: mb.scaled_mm(I8, I8.t(), F32, x),
    lambda x: mb.scaled_mm(I8, I8.t(), F32, F32, bias=x), lambda x: mb.scaled_mm(I8, I8.t(), F32, F32, out=x),
    lambda x: mb.grouped_scaled_mm(I8, I8.t()[None], F32, F32[None], x),
    lambda x: mb.expert_sort(x, 4), lambda x: mb.expert_gather(x, ORDER), lambda x: mb.expert_gather_quantize(x, ORDER),
    lambda x: mb.expert_combine(x, None, ORDER), lambda x: mb.expert_combine(ROWS, x, ORDER),
    lambda x: mb.expert_gather_backward(x, ORDER), lambda x: mb.expert_combine_backward(x, ROWS, IDS, ORDER),
    lambda x: mb.expert_combine_backward(ROWS[:4], x, IDS.float(), ORDER)])
@pytest.mark.parametrize("x", [0.5, [1.0, 2.0], "x"])
def test_no_tensor(call, x):
    with pytest.raises(AssertionError):
        call(x)


@pytest.mark.parametrize("kw,name", [(dict(scale_a=0.5), "scale_a"), (dict(scale_b=[1.0]), "scale_b"),
                                     (dict(bias=1.0), "bias"), (dict(out=3), "out")])
def test_the_argument_is_named(kw, name):
    """Past the device check, which needs no device here: the function behind it."""
    args = dict(a=I8, b=torch.zeros(16, 4, dtype=torch.int8), scale_a=F32, scale_b=F32, bias=None, out_dtype=None,
                out=None, _plan=None)
    with pytest.raises(AssertionError, match=name):
        quantized._scaled_mm.__wrapped__(**{**args, **kw})


def test_the_argument_is_named_by_group():
    args = dict(a=I8, b=torch.zeros(1, 16, 4, dtype=torch.int8), scale_a=F32, scale_b=F32[None], offsets=[0, 4],
                out_dtype=None, out=None, _plan=None)
    with pytest.raises(AssertionError, match="offsets"):
        quantized._grouped_scaled_mm.__wrapped__(**args)
    with pytest.raises(AssertionError, match="weights"):
        experts._combine.__wrapped__(ROWS, [1.0], ORDER)
    with pytest.raises(AssertionError, match="rows"):
        experts._combine_backward.__wrapped__(ROWS[:4], [1.0], IDS.float(), ORDER)


@pytest.mark.parametrize("out", [torch.zeros(3, 2, 4).transpose(0, 1), torch.zeros(2, 5, 4)[:, :3]])
def test_an_output_that_is_no_matrix_of_rows(out):
    """Leading dimensions of out that do not fold into one stride."""
    a, b = torch.zeros(2, 3, 16, dtype=torch.int8), torch.zeros(16, 4, dtype=torch.int8)
    with pytest.raises(AssertionError, match="out"):
        quantized._scaled_mm.__wrapped__(a, b, torch.ones(2, 3), torch.ones(4), None, torch.float32, out, None)
