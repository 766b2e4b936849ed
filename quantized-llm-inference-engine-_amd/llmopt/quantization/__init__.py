"""Weight quantization: RTN, GPTQ, packed storage and ``QuantLinear``.

Exports the same names as the reference's ``src/llmopt/quantization/__init__.py:30-49``, plus
the fused projections of :mod:`llmopt.quantization.fused`, the packed checkpoint of
:mod:`llmopt.quantization.checkpoint` and 8-bit floating point (:mod:`llmopt.quantization.float8`) (which have no counterpart there).
"""

from __future__ import annotations

from llmopt.quantization.calibration import (
    CalibrationHarness,
    CalibrationResult,
    HessianCollector,
    apply_quantization,
)
from llmopt.quantization.checkpoint import is_quantized_checkpoint, load_quantized_, save_quantized
from llmopt.quantization.float8 import (
    Float8Linear,
    Float8SwiGLU,
    Float8Tensor,
    FusedFloat8Linear,
    float8_linear,
    float8_swiglu,
    quantize_float8,
    quantize_model_float8_,
    rmsnorm_float8,
)
from llmopt.quantization.fused import FusedQuantLinear, QuantSwiGLU, concat_rows, interleave_gate_up
from llmopt.quantization.quant_linear import (
    QuantLinear,
    QuantLinearConfig,
    quantize_model_,
    replace_linear_modules,
)
from llmopt.quantization.quantizers import (
    GPTQQuantizer,
    QuantizedTensor,
    Quantizer,
    RoundToNearestQuantizer,
    build_quantizer,
    choose_qparams,
    dequantize,
    pack_int4,
    quantize_to_codes,
    unpack_int4,
)

__all__ = [
    "CalibrationHarness",
    "CalibrationResult",
    "Float8Linear",
    "Float8SwiGLU",
    "Float8Tensor",
    "FusedFloat8Linear",
    "FusedQuantLinear",
    "GPTQQuantizer",
    "HessianCollector",
    "QuantLinear",
    "QuantLinearConfig",
    "QuantSwiGLU",
    "QuantizedTensor",
    "Quantizer",
    "RoundToNearestQuantizer",
    "apply_quantization",
    "build_quantizer",
    "choose_qparams",
    "concat_rows",
    "dequantize",
    "float8_linear",
    "float8_swiglu",
    "interleave_gate_up",
    "is_quantized_checkpoint",
    "load_quantized_",
    "pack_int4",
    "quantize_float8",
    "quantize_model_",
    "quantize_model_float8_",
    "quantize_to_codes",
    "replace_linear_modules",
    "rmsnorm_float8",
    "save_quantized",
    "unpack_int4",
]
