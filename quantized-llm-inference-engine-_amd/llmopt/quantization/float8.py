"""Weights and activations in 8-bit floating point: half the bytes of a 16-bit layer, and products at twice its rate.

A number is held as a ``float8_e4m3fn`` code times a ``float8_e8m0fnu`` scale, a power of two. Activations ``[..., K]`` have
one scale for each row and 128 columns, ``[..., ceil(K / 128)]``; weights ``[N, K]`` one for each block of 128 x 128. A group
whose largest magnitude is ``amax`` takes ``2^e`` for the smallest ``e >= -127`` with ``amax <= 448 2^e``, and a number ``x``
the code ``x / 2^e`` rounded to the nearest, ties to even; a group that holds an infinity or NaN gets the scale NaN and reads
as NaN. So a code times its scale is exact in bf16 and fp32, and the matrix cores take codes and scales as they are. A
checkpoint with other scales is quantized anew from its numbers.

* :func:`quantize_float8`: activations, or with ``block_rows=128`` a weight;
* :func:`rmsnorm_float8`: RMSNorm, with the residual's addition in front of it, its output quantized;
* :func:`float8_linear`: a projection of quantized activations by a quantized weight;
* :func:`float8_swiglu`: ``silu(x gate^T) * (x up^T)``, quantized for the projection behind it;
* :class:`Float8Linear`, :class:`FusedFloat8Linear`, :class:`Float8SwiGLU` and :func:`quantize_model_float8_`: the layers made
  of them.

On HIP devices each is hand-written kernels (``include/llmopt_float8.h``); on the host the same definitions run in torch.
Products of the matrix cores are sums in fp32 but for what lies below 2^-13 of the largest of eight neighbouring products: 1.5e-5
to 2.7e-5 of a typical sum, and up to 1e-4, half of what rounding to fp16 brings, where a few channels are 100 times as strong as the
rest and more. Results are 16-bit numbers, rounded once. Codes carry no derivative; a :class:`Float8Linear` passes a gradient straight through the rounding of its input. The reference's linears hold integer
codes only (``src/llmopt/quantization/quant_linear.py``), so none of this has a counterpart there.
"""

from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch
from torch import nn

from llmopt.kernels import float8_ops
from llmopt.quantization.quant_linear import replace_linear_modules
from llmopt.utils.autograd import is_differentiated

__all__ = [
    "Float8Linear",
    "Float8SwiGLU",
    "Float8Tensor",
    "FusedFloat8Linear",
    "float8_linear",
    "float8_swiglu",
    "quantize_float8",
    "quantize_model_float8_",
    "rmsnorm_float8",
]

GROUP = 128
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
OUT_DTYPES = (torch.float16, torch.bfloat16)
_DTYPE_CODES = {torch.float16: 1, torch.bfloat16: 2}


def _groups(n: int) -> int:
    return -(-n // GROUP)


@dataclass
class Float8Tensor:
    """Codes with their scales.

    Attributes:
        codes: ``float8_e4m3fn [..., K]``.
        scales: ``float8_e8m0fnu``; with ``block_rows`` 1 ``[..., ceil(K / 128)]``, with 128 (``codes [N, K]``) ``[ceil(N / 128), ceil(K /
            128)]``.
        block_rows: rows that share a scale, 1 (activations) or 128 (weights).
    """

    codes: torch.Tensor
    scales: torch.Tensor
    block_rows: int = 1

    def __post_init__(self) -> None:
        codes, scales = self.codes, self.scales
        if codes.is_cuda and float8_ops.native().f8_check(codes, scales, self.block_rows):
            return  # what is checked here, in native code
        if codes.dtype != F8 or scales.dtype != E8:
            raise TypeError(f"expected float8_e4m3fn codes and float8_e8m0fnu scales, got {codes.dtype} and {scales.dtype}")
        if self.block_rows == 1 and codes.dim() > 0:
            want = (*codes.shape[:-1], _groups(codes.shape[-1]))
        elif self.block_rows == GROUP and codes.dim() == 2:
            want = (_groups(codes.shape[0]), _groups(codes.shape[1]))
        else:
            raise ValueError(f"a scale covers 1 row of codes [..., K] or 128 of codes [N, K], not block_rows="
                             f"{self.block_rows} of {tuple(codes.shape)}")
        if tuple(scales.shape) != want:
            raise ValueError(f"codes {tuple(codes.shape)} with block_rows={self.block_rows} have scales {want}, not "
                             f"{tuple(scales.shape)}")
        if codes.device != scales.device:
            raise RuntimeError(f"Expected all tensors to be on the same device, but found at least two devices, "
                               f"{codes.device} and {scales.device}!")

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    def dim(self) -> int:
        return self.codes.dim()

    def to(self, device: torch.device | str) -> Float8Tensor:
        return Float8Tensor(self.codes.to(device), self.scales.to(device), self.block_rows)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The numbers, code times scale, rounded to ``dtype``."""
        k = self.codes.shape[-1]
        scales = self.scales.float().repeat_interleave(GROUP, dim=-1)[..., :k]
        if self.block_rows != 1:
            scales = scales.repeat_interleave(GROUP, dim=0)[: self.codes.shape[0]]
        return (self.codes.float() * scales).to(dtype)


def _float(x: torch.Tensor, what: str) -> None:
    if not x.is_floating_point() or x.element_size() < 2:
        raise TypeError(f"{what} must be a 16- or 32-bit floating-point tensor, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError(f"{what} must have at least one dimension")


def _quantize_torch(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The definition, on fp32 numbers ``[rows, K]``."""
    x = x.detach().float()
    rows, k = x.shape
    groups = nn.functional.pad(x, (0, -k % GROUP, 0, -rows % block_rows))
    groups = groups.view(groups.shape[0] // block_rows, block_rows, _groups(k), GROUP)
    finite = groups.isfinite().all(3).all(1)
    amax = groups.abs().amax((1, 3)) if groups.numel() else groups.new_zeros(groups.shape[0], groups.shape[2])
    m, p = torch.frexp(torch.where(finite, amax, 0.0))  # amax = m 2^p with m in [0.5, 1), and 448 = 0.875 2^9
    e = torch.where(m > 0, p - 9 + (m > 0.875).to(p.dtype), -127).clamp(min=-127)
    codes = torch.where(finite[:, None, :, None], torch.ldexp(groups, -e[:, None, :, None]), 0.0)
    codes = codes.reshape(groups.shape[0] * block_rows, _groups(k) * GROUP)[:rows, :k].to(F8)
    return codes.contiguous(), torch.where(finite, e + 127, 255).to(torch.uint8).view(E8)


def _made(codes: torch.Tensor, scales: torch.Tensor, block_rows: int = 1) -> Float8Tensor:
    """Codes and scales that a kernel made: nothing to check."""
    out = Float8Tensor.__new__(Float8Tensor)
    out.codes, out.scales, out.block_rows = codes, scales, block_rows
    return out


def quantize_float8(x: torch.Tensor, block_rows: int = 1) -> Float8Tensor:
    """Quantize activations ``x [..., K]``, or with ``block_rows=128`` a weight ``[N, K]`` (see the module)."""
    made = float8_ops.native().f8_quantize(x, block_rows) if x.is_cuda else None
    if made is not None:
        return _made(*made, block_rows)
    _float(x, "x")
    if block_rows not in (1, GROUP):
        raise ValueError(f"a scale covers 1 or {GROUP} rows, not {block_rows}")
    if block_rows == GROUP and x.dim() != 2:
        raise ValueError(f"expected a 2D weight, got shape {tuple(x.shape)}")
    if x.is_cuda:
        return _made(*float8_ops.quantize(x, block_rows), block_rows)
    codes, scales = _quantize_torch(float8_ops.as_rows(x), block_rows)
    if block_rows == 1:
        codes, scales = codes.view(x.shape), scales.view(*x.shape[:-1], scales.shape[1])
    return _made(codes, scales, block_rows)


def rmsnorm_float8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None
                   ) -> tuple[Float8Tensor, torch.Tensor]:
    """``(norm(h), h)`` with ``h = residual + x`` rounded to their type (``x`` without a residual): ``norm(h) = h /
    sqrt(mean(h^2) + eps) * weight`` in fp32, quantized by rows without another rounding."""
    made = float8_ops.native().f8_rmsnorm(x, weight, eps, residual) if x.is_cuda else None
    if made is not None:
        return _made(made[0], made[1]), x if residual is None else made[2]
    _float(x, "x")
    if weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"a norm of {tuple(x.shape)} needs a weight of [{x.shape[-1]}], got {tuple(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"the residual must be {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")
    if not is_differentiated(x, *(() if residual is None else (residual,))) and float8_ops.rmsnorm_supported(x, weight, residual):
        codes, scales, h = float8_ops.rmsnorm(x, weight, eps, residual)
        return _made(codes, scales), x if h is None else h
    h = x if residual is None else residual + x
    h32 = h.detach().float()
    y = h32 * torch.rsqrt(h32.pow(2).mean(-1, keepdim=True) + eps) * weight.detach().float()
    return quantize_float8(y), h


def _check_product(x: Float8Tensor, w: Float8Tensor, what: str = "the weight") -> None:
    if x.block_rows != 1 or w.block_rows != GROUP:
        raise ValueError(f"expected activations with a scale per row and {what} with a scale per {GROUP} x {GROUP}, got "
                         f"block_rows {x.block_rows} and {w.block_rows}")
    if x.shape[-1] != w.shape[1]:
        raise RuntimeError(f"mat1 and mat2 shapes cannot be multiplied ({x.codes.numel() // max(1, x.shape[-1])}x"
                           f"{x.shape[-1]} and {w.shape[1]}x{w.shape[0]})")


def _product_torch(x: Float8Tensor, w: Float8Tensor) -> torch.Tensor:
    if x.device != w.device:
        raise RuntimeError("Expected all tensors to be on the same device, but found at least two devices, "
                           f"{x.device} and {w.device}!")
    return torch.matmul(float8_ops.as_rows(x.dequantize()), w.dequantize().t())


def float8_linear(x: Float8Tensor, w: Float8Tensor, bias: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x w^T + bias`` of activations ``[..., K]`` and a weight ``[N, K]``: ``[..., N]`` of ``dtype`` (fp16 or bf16, also the
    bias's). With a bias that has to carry a derivative the product runs in torch."""
    if x.codes.is_cuda and x.block_rows == 1 and w.block_rows == GROUP:
        y = float8_ops.native().f8_linear(x.codes, x.scales, w.codes, w.scales, bias, _DTYPE_CODES.get(dtype, 0))
        if y is not None:
            return y
    _check_product(x, w)
    n = int(w.shape[0])
    if dtype not in OUT_DTYPES:
        raise TypeError(f"float8_linear gives float16 or bfloat16, not {dtype}")
    if bias is not None:
        if bias.dtype != dtype:
            raise RuntimeError(f"self and mat2 must have the same dtype, but got {bias.dtype} and {dtype}")
        if tuple(bias.shape) != (n,):
            raise ValueError(f"a bias of [{n}] expected, got {tuple(bias.shape)}")
    if x.is_cuda and (bias is None or not is_differentiated(bias)):
        return float8_ops.linear(x.codes, x.scales, w.codes, w.scales, bias, dtype)
    y = _product_torch(x, w)
    return (y if bias is None else y + bias.float()).to(dtype).view(*x.shape[:-1], n)


def float8_swiglu(x: Float8Tensor, gate: Float8Tensor, up: Float8Tensor) -> Float8Tensor:
    """``silu(x gate^T) * (x up^T)`` of activations ``[..., K]`` and two weights ``[N, K]``, in fp32 up to its quantizing by
    rows: ``[..., N]``."""
    if x.codes.is_cuda and x.block_rows == 1 and gate.block_rows == up.block_rows == GROUP:
        made = float8_ops.native().f8_swiglu(x.codes, x.scales, gate.codes, gate.scales, up.codes, up.scales)
        if made is not None:
            return _made(*made)
    _check_product(x, gate, "gate")
    _check_product(x, up, "up")
    if gate.shape != up.shape:
        raise ValueError(f"gate and up have different shapes: {tuple(gate.shape)}, {tuple(up.shape)}")
    if x.is_cuda:
        return _made(*float8_ops.swiglu(x.codes, x.scales, gate.codes, gate.scales, up.codes, up.scales))
    g = _product_torch(x, gate)
    y = g / (1.0 + torch.exp(-g)) * _product_torch(x, up)
    return quantize_float8(y.view(*x.shape[:-1], gate.shape[0]))


# ---- layers -----------------------------------------------------------------------------------------


class Float8Linear(nn.Module):
    """A linear layer whose weight is held in 8-bit floating point, and whose input is quantized on its way in.

    ``forward(x)`` takes ``x [..., in_features]`` in ``compute_dtype``, or activations that are quantized already
    (:class:`Float8Tensor`, from :func:`rmsnorm_float8` or :func:`float8_swiglu`), and returns ``compute_dtype``. Where ``x``
    has to carry a derivative, the product runs in torch on the same numbers, and the derivative passes straight through
    the rounding of ``x``.

    Attributes:
        weight_codes: ``float8_e4m3fn [out_features, in_features]``.
        weight_scales: ``float8_e8m0fnu [ceil(out_features / 128), ceil(in_features / 128)]``.
        bias: of ``compute_dtype``, or None.
    """

    def __init__(self, weight: Float8Tensor, bias: torch.Tensor | None = None,
                 compute_dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        if weight.block_rows != GROUP:
            raise ValueError("a Float8Linear needs a weight with a scale per 128 x 128 (quantize_float8(..., block_rows=128))")
        if compute_dtype not in OUT_DTYPES:
            raise TypeError(f"Float8Linear computes float16 or bfloat16, not {compute_dtype}")
        self.out_features, self.in_features = (int(d) for d in weight.shape)
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError(f"a bias of [{self.out_features}] expected, got {tuple(bias.shape)}")
        self.compute_dtype = compute_dtype
        self.register_buffer("weight_codes", weight.codes)
        self.register_buffer("weight_scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().to(compute_dtype))

    @classmethod
    def from_float(cls, linear: nn.Linear, compute_dtype: torch.dtype | None = None) -> Float8Linear:
        """The quantized form of ``linear``, computing in its weight's type."""
        return cls(quantize_float8(linear.weight.detach(), block_rows=GROUP), linear.bias,
                   compute_dtype or linear.weight.dtype)

    def _apply(self, fn, recurse: bool = True):  # noqa: ANN001, ANN202 - nn.Module signature
        # module.to(dtype) converts floating-point buffers: the codes and their scales keep their types.
        kept = {name: self._buffers[name] for name in ("weight_codes", "weight_scales")}
        super()._apply(fn, recurse)
        for name, old in kept.items():
            if self._buffers[name].dtype != old.dtype:
                self._buffers[name] = old.to(self._buffers[name].device)
        if self.bias is not None and self.bias.dtype != self.compute_dtype:
            self.bias = self.bias.to(self.compute_dtype)
        return self

    def weight_tensor(self) -> Float8Tensor:
        return Float8Tensor(self.weight_codes, self.weight_scales, GROUP)

    def forward(self, x: torch.Tensor | Float8Tensor) -> torch.Tensor:
        if isinstance(x, torch.Tensor):
            if x.dtype != self.compute_dtype:
                raise RuntimeError(f"expected m1 and m2 to have the same dtype, but got: {x.dtype} != {self.compute_dtype}")
            if is_differentiated(x):
                y = nn.functional.linear(_straight_through(x), self.weight_tensor().dequantize())
                return (y if self.bias is None else y + self.bias.float()).to(self.compute_dtype)
            x = quantize_float8(x)
        return float8_linear(x, self.weight_tensor(), self.bias, self.compute_dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class FusedFloat8Linear(nn.Module):
    """Several :class:`Float8Linear` over one input as one weight (q, k and v): ``forward(x)`` returns ``tuple(part(x) for part
    in parts)``, column slices of one tensor, from one product. All but the last part need a multiple of 128 rows, so that no
    scale covers two of them."""

    def __init__(self, parts: Sequence[Float8Linear]) -> None:
        super().__init__()
        reason = self.refusal(parts)
        if reason is not None:
            raise ValueError(reason)
        first = parts[0]
        bias = None
        if any(p.bias is not None for p in parts):
            bias = torch.cat([torch.zeros(p.out_features, dtype=p.compute_dtype, device=p.weight_codes.device)
                              if p.bias is None else p.bias for p in parts])
        codes = torch.cat([p.weight_codes.view(torch.uint8) for p in parts]).view(F8)
        scales = torch.cat([p.weight_scales.view(torch.uint8) for p in parts]).view(E8)
        self.linear = Float8Linear(Float8Tensor(codes, scales, GROUP), bias, first.compute_dtype)
        self.out_features = [p.out_features for p in parts]

    @staticmethod
    def refusal(parts: Sequence[Float8Linear]) -> str | None:
        """Why ``parts`` cannot be fused; None where they can."""
        if not parts:
            return "nothing to fuse"
        if any(p.in_features != parts[0].in_features or p.compute_dtype != parts[0].compute_dtype for p in parts):
            return "fused layers need the same in_features and compute dtype"
        if any(p.out_features % GROUP for p in parts[:-1]):
            return f"all but the last of the fused layers need a multiple of {GROUP} rows"
        return None

    def forward(self, x: torch.Tensor | Float8Tensor) -> tuple[torch.Tensor, ...]:
        return tuple(torch.split(self.linear(x), self.out_features, dim=-1))

    def extra_repr(self) -> str:
        return f"out_features={self.out_features}"


def _straight_through(x: torch.Tensor) -> torch.Tensor:
    """``x`` as its quantized numbers (fp32), with ``x``'s derivative."""
    x32 = x.float()
    return x32 + (quantize_float8(x).dequantize() - x32).detach()


class Float8SwiGLU(nn.Module):
    """``silu(gate(x)) * up(x)`` of two :class:`Float8Linear` without biases, quantized for the layer behind it
    (:class:`Float8Tensor`). Where ``x`` has to carry a derivative, an unquantized tensor comes back, from the two layers."""

    def __init__(self, gate: Float8Linear, up: Float8Linear) -> None:
        super().__init__()
        reason = self.refusal(gate, up)
        if reason is not None:
            raise ValueError(reason)
        self.gate_proj, self.up_proj = gate, up

    @staticmethod
    def refusal(gate: Float8Linear, up: Float8Linear) -> str | None:
        """Why ``gate`` and ``up`` cannot be one product; None where they can."""
        if gate.weight_codes.shape != up.weight_codes.shape or gate.compute_dtype != up.compute_dtype:
            return "gate and up need the same shape and compute dtype"
        if gate.bias is not None or up.bias is not None:
            return "gate and up must have no bias"
        return None

    def forward(self, x: torch.Tensor | Float8Tensor) -> torch.Tensor | Float8Tensor:
        if isinstance(x, torch.Tensor):
            if is_differentiated(x):
                return nn.functional.silu(self.gate_proj(x)) * self.up_proj(x)
            if x.dtype != self.gate_proj.compute_dtype:
                raise RuntimeError(f"expected m1 and m2 to have the same dtype, but got: {x.dtype} != "
                                   f"{self.gate_proj.compute_dtype}")
            x = quantize_float8(x)
        return float8_swiglu(x, self.gate_proj.weight_tensor(), self.up_proj.weight_tensor())


def quantize_model_float8_(model: nn.Module, *, ignore_layers: tuple[str, ...] = ("lm_head", "embed_tokens")) -> nn.Module:
    """Swap every ``nn.Linear`` of ``model`` whose qualified name contains none of ``ignore_layers`` for a
    :class:`Float8Linear`, in place, and return the model (as :func:`quantize_model_` does with integer codes). The layers
    must be fp16 or bf16."""
    swaps = {module: Float8Linear.from_float(module) for name, module in model.named_modules()
             if isinstance(module, nn.Linear) and not any(tok in name for tok in ignore_layers)}
    return replace_linear_modules(model, swaps)
