"""metalblas_b200 — B200 (sm_100a) matmul / addmm / bmm with the metalBLAS API.

Drop-in for the reference's public names (metalblas/__init__.py:1-19):

    import metalblas_b200 as metalblas
    c = metalblas.matmul(a, b)          # a, b are CUDA tensors

The compute runs in ``libmetalblas_b200.so`` through the C ABI declared in
``include/metalblas_b200.h``; there is no CPU fallback.
"""
from . import kernels
from .dispatch import (
    addbmm,
    addmm,
    baddbmm,
    bmm,
    dot,
    gemm,
    ger,
    matmul,
    mv,
    outer,
    vdot,
)
# This package's own operators, which the reference does not have (``__all__`` is the
# reference's list of names).
from .experts import (  # noqa: F401
    ExpertOrder,
    expert_combine,
    expert_combine_backward,
    expert_gather,
    expert_gather_backward,
    expert_gather_quantize,
    expert_sort,
)
from .int4 import dequantize_int4, grouped_int4_mm, int4_mm, quantize_int4  # noqa: F401
from .quantized import grouped_scaled_mm, quantize, scaled_mm  # noqa: F401
from .router import (  # noqa: F401
    ExpertBalance,
    expert_balance,
    expert_balance_backward,
    expert_route,
    expert_route_backward,
)

__all__ = [
    "matmul", "gemm", "addmm", "bmm", "baddbmm", "addbmm",
    "dot", "vdot", "outer", "ger", "mv", "kernels",
]
