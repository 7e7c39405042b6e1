"""MI355X-native fused MoE (FP8 block-scaled, DeepSeek routing) for gfx950.

``flashinfer_amd.kernel.run`` is the drop-in for the reference's
``kernel.py::run``; the compute lives in ``libmi_moe.so`` (HIP, gfx950).
``flashinfer_amd.experts`` and ``flashinfer_amd.int8`` are operators for
experts of a caller's own (``libmi_experts.so``), ``flashinfer_amd.layer`` and
``flashinfer_amd.int4`` what stands inside a layer of them (``libmi_layer.so``).
"""
from .kernel import run, route  # noqa: F401
from .experts import ExpertPlan, permute, sort_experts, unpermute  # noqa: F401
from .int8 import (int8_grouped_matmul, int8_matmul, quantize_int8,  # noqa: F401
                   swiglu_quantize_int8)
from .layer import balance_loss, swiglu  # noqa: F401
from .int4 import (Int4Weights, int4_grouped_matmul, int4_matmul, pack_int4,  # noqa: F401
                   quantize_int4)

__all__ = ["run", "route", "ExpertPlan", "sort_experts", "permute", "unpermute", "quantize_int8",
           "swiglu_quantize_int8", "int8_matmul", "int8_grouped_matmul", "balance_loss", "swiglu",
           "Int4Weights", "pack_int4", "quantize_int4", "int4_matmul", "int4_grouped_matmul"]
