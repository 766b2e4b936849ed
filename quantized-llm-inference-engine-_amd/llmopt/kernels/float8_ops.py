"""Torch-facing wrappers over the entry points of ``include/llmopt_float8.h``: quantizing, RMSNorm with a quantized output,
the projection and the gated MLP product in 8-bit floating point. The checks, errors and streams are those of
:mod:`llmopt.kernels.ops`; :mod:`llmopt.quantization.float8` is what a user calls. The plain form of a call has its checks,
allocations and launch in native code (:func:`native`)."""

from __future__ import annotations

import math

import torch

from llmopt.kernels._lib import DTYPE_CODES, call, load_binding, load_library
from llmopt.kernels.ops import _launching_on, _same_device, _stream_handle

__all__ = ["as_rows", "linear", "native", "quantize", "rmsnorm", "rmsnorm_supported", "swiglu"]

GROUP = 128


def _groups(n: int) -> int:
    return -(-n // GROUP)


def as_rows(x: torch.Tensor) -> torch.Tensor:
    """``[..., K]`` as a matrix, also where ``K`` is 0 (the number of rows is not left to be found)."""
    return x.reshape(math.prod(x.shape[:-1]), x.shape[-1]) if x.dim() != 2 else x


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``[..., K]`` as a matrix with a unit inner stride and rows that do not overlap; a view where that is possible."""
    x = as_rows(x)
    rows, cols = x.shape
    if (cols > 1 and x.stride(1) != 1) or (rows > 1 and x.stride(0) < cols):
        x = x.contiguous()
    return x


def _ld(x: torch.Tensor) -> int:
    return max(x.stride(0), x.shape[1]) if x.shape[0] > 1 else x.shape[1]


class _NoBinding:
    """Where the native path is not built: every call takes the general one."""

    @staticmethod
    def _none(*_args: object) -> None:
        return None

    f8_check = f8_quantize = f8_rmsnorm = f8_linear = f8_swiglu = _none


_NO_BINDING = _NoBinding()


def native():  # noqa: ANN201 - the extension module
    """The native path: ``f8_check(codes, scales, block_rows)``, ``f8_quantize(x, block_rows)``, ``f8_rmsnorm(x, weight, eps,
    residual)``, ``f8_linear(codes, scales, codes, scales, bias, dtype)`` and ``f8_swiglu``, of which each gives what the function
    of its name here does for the plain form of a call -- contiguous or row-strided tensors that belong together, on the current
    device, without derivatives -- and None for any other form, which those functions take."""
    return load_binding() or _NO_BINDING


def quantize(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes of ``x [..., cols]`` and their scales (``llmopt_f8_quantize``)."""
    lead = x.shape[:-1]
    if x.dtype not in DTYPE_CODES:
        x = x.to(torch.float32)
    x = _rows(x)
    rows, cols = (int(d) for d in x.shape)
    codes = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(rows if block_rows == 1 else _groups(rows), _groups(cols), dtype=torch.float8_e8m0fnu, device=x.device)
    if codes.numel():
        with _launching_on(x.device):
            call(
                load_library().llmopt_f8_quantize(
                    x.data_ptr(), _ld(x), DTYPE_CODES[x.dtype], rows, cols, block_rows, codes.data_ptr(), cols,
                    scales.data_ptr(), int(scales.shape[1]), _stream_handle(x.device),
                ),
                "llmopt_f8_quantize",
            )
    return (codes.view(*lead, cols), scales.view(*lead, _groups(cols))) if block_rows == 1 else (codes, scales)


def rmsnorm_supported(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None) -> bool:
    """Whether :func:`rmsnorm` takes these tensors (fp16 or bf16 of one type on one HIP device)."""
    return (x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and weight.dtype == x.dtype
            and weight.device == x.device and x.dim() > 0 and weight.dim() == 1 and weight.shape[0] == x.shape[-1]
            and (residual is None or (residual.dtype == x.dtype and residual.shape == x.shape
                                      and residual.device == x.device)))


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None
            ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Codes of ``x``'s shape, their scales, and ``residual + x`` (``llmopt_f8_rmsnorm``)."""
    shape = x.shape
    x = _rows(x)
    rows, hidden = (int(d) for d in x.shape)
    codes = torch.empty(rows, hidden, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(rows, _groups(hidden), dtype=torch.float8_e8m0fnu, device=x.device)
    h = res = None
    if residual is not None:
        res = _rows(residual)
        h = torch.empty(rows, hidden, dtype=x.dtype, device=x.device)
    if codes.numel():
        weight = weight.contiguous()
        with _launching_on(x.device):
            call(
                load_library().llmopt_f8_rmsnorm(
                    x.data_ptr(), _ld(x), None if res is None else res.data_ptr(), 0 if res is None else _ld(res),
                    None if h is None else h.data_ptr(), hidden, weight.data_ptr(), codes.data_ptr(), hidden,
                    scales.data_ptr(), int(scales.shape[1]), rows, hidden, float(eps), DTYPE_CODES[x.dtype],
                    _stream_handle(x.device),
                ),
                "llmopt_f8_rmsnorm",
            )
    return codes.view(shape), scales.view(*shape[:-1], _groups(hidden)), None if h is None else h.view(shape)


def linear(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
           bias: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    """``[..., N]`` of ``dtype``: codes ``x [..., K]`` with scales ``[..., ceil(K / 128)]`` times codes ``w [N, K]`` with scales
    ``[ceil(N / 128), ceil(K / 128)]``, plus ``bias [N]`` of ``dtype`` (``llmopt_f8_linear``)."""
    _same_device(x, x_scales, w, w_scales, bias)
    lead = x.shape[:-1]
    x, w, x_scales, w_scales = _rows(x), _rows(w), _rows(x_scales), _rows(w_scales)
    (m, k), n = x.shape, int(w.shape[0])
    y = torch.empty(m, n, dtype=dtype, device=x.device)
    if y.numel():
        bias = None if bias is None else bias.contiguous()
        lib = load_library()
        with _launching_on(x.device):
            ws_bytes = lib.llmopt_f8_linear_workspace(m, n, k)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
            call(
                lib.llmopt_f8_linear(
                    x.data_ptr(), _ld(x), x_scales.data_ptr(), _ld(x_scales), m, k, w.data_ptr(), _ld(w),
                    w_scales.data_ptr(), _ld(w_scales), None if bias is None else bias.data_ptr(), y.data_ptr(), n, n,
                    DTYPE_CODES[dtype], None if ws is None else ws.data_ptr(), ws_bytes, _stream_handle(x.device),
                ),
                "llmopt_f8_linear",
            )
    return y.view(*lead, n)


def swiglu(x: torch.Tensor, x_scales: torch.Tensor, gate: torch.Tensor, gate_scales: torch.Tensor, up: torch.Tensor,
           up_scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes ``[..., N]`` and scales of ``silu(x gate^T) * (x up^T)`` (``llmopt_f8_swiglu``)."""
    lead = x.shape[:-1]
    _same_device(x, x_scales, gate, gate_scales, up, up_scales)
    x, gate, up = _rows(x), _rows(gate), _rows(up)
    x_scales, gate_scales, up_scales = _rows(x_scales), _rows(gate_scales), _rows(up_scales)
    (m, k), n = x.shape, int(gate.shape[0])
    codes = torch.empty(m, n, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(m, _groups(n), dtype=torch.float8_e8m0fnu, device=x.device)
    if codes.numel():
        lib = load_library()
        with _launching_on(x.device):
            ws_bytes = lib.llmopt_f8_swiglu_workspace(m, n, k)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
            call(
                lib.llmopt_f8_swiglu(
                    x.data_ptr(), _ld(x), x_scales.data_ptr(), _ld(x_scales), m, k, gate.data_ptr(), _ld(gate),
                    gate_scales.data_ptr(), _ld(gate_scales), up.data_ptr(), _ld(up), up_scales.data_ptr(),
                    _ld(up_scales), n, codes.data_ptr(), n, scales.data_ptr(), int(scales.shape[1]),
                    None if ws is None else ws.data_ptr(), ws_bytes, _stream_handle(x.device),
                ),
                "llmopt_f8_swiglu",
            )
    return codes.view(*lead, n), scales.view(*lead, _groups(n))
