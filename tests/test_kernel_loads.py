"""CPU: kernels that may start beside their predecessor read memory by coherent loads.

A kernel launched with programmatic serialization can be resident while the kernel before it
still writes what it is about to read; ``griddepcontrol.wait`` makes those writes visible to
ordinary loads.  The non-coherent form (``ld.global.nc``, ``__ldg``) is defined only for memory
that nobody writes during the kernel's life, so it is left to kernels launched in plain order.
"""
from __future__ import annotations

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "metalblas_b200", "csrc")
OPERATORS = ("quantize.cuh", "experts.cuh", "scaled_tc.cuh", "scaled_gemv.cuh")


PRODUCTS = ("gemv.cuh", "tc_gemm.cuh")


def code_of(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", OPERATORS)
def test_operators_load_coherently(name):
    code = code_of(name)
    assert "ld.global.nc" not in code and "__ldg" not in code


@pytest.mark.parametrize("name", PRODUCTS)
def test_products_load_coherently(name):
    code = code_of(name)
    assert "ld.global.nc" not in code and "__ldg" not in code
