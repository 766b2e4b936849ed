"""The operators of 8-bit floating point in 64 bits, from their definitions and without the package: what tests compare with,
and how far a result may be off."""

from __future__ import annotations

import torch

GROUP = 128


def spread(groups: torch.Tensor, rows: int, shape) -> torch.Tensor:  # noqa: ANN001
    """A group's value for each number of a matrix."""
    return groups.repeat_interleave(rows, 0)[: shape[0]].repeat_interleave(GROUP, 1)[:, : shape[1]]


def numbers(codes: torch.Tensor, scales: torch.Tensor, rows: int) -> torch.Tensor:
    return codes.double() * spread(scales.double(), rows, codes.shape)


def scales_of(x: torch.Tensor, rows: int) -> torch.Tensor:
    """The scales of a matrix ``x`` (float64, finite): the smallest powers of two from 2^-127 on with amax <= 448 scale."""
    x = torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % GROUP, 0, -x.shape[0] % rows))
    amax = x.view(x.shape[0] // rows, rows, -1, GROUP).amax((1, 3))
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448.0).clamp(min=-127.0)))
    scale = torch.where(amax > 448.0 * scale, 2 * scale, scale)
    return torch.where((scale > 2.0**-127) & (amax <= 224.0 * scale), scale / 2, scale)


def check_quantized(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, off, rows: int = 1) -> None:  # noqa: ANN001
    """``codes`` and ``scales`` are those of numbers that are at most ``off`` from ``x`` (float64; ``off`` a number or of x's
    shape): a scale is that of a group whose numbers are off by as much, and a number is off by half a step of its code
    and by ``off``."""
    off = torch.as_tensor(off, dtype=torch.float64, device=x.device).expand(x.shape)
    # the largest magnitude of a group lies between those of the numbers at their least and at their most
    least, most = scales_of((x.abs() - off).clamp(min=0), rows), scales_of(x.abs() + off, rows)
    got = scales.double()
    assert scales.shape == least.shape and bool(((got >= least) & (got <= most)).all())
    numbers_ = numbers(codes, scales, rows)
    step = torch.maximum((x.abs() + off) * 2.0**-4, spread(got, rows, x.shape) * 2.0**-10)
    assert bool(((numbers_ - x).abs() <= step + off).all())


def product(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x w^T`` in 64 bits, and how far the matrix cores' sums may be off: of eight neighbouring products what is below
    2^-13 of the largest is dropped, from seven of them at most, so each term may bring 7 * 2^-13 of its magnitude with it;
    and the sums of eight are added in fp32, each addition off by a step of 2^-23 of the terms' sum at most."""
    terms = x.abs() @ w.abs().t().contiguous()
    return x @ w.t().contiguous(), terms * (7 * 2.0**-13 + (-(-x.shape[1] // 8) + 8) * 2.0**-23)


def swiglu(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``silu(x gate^T) * (x up^T)`` in 64 bits, and how far fp32 may be off: |silu'| < 1.1, and a few steps of the
    exponential (8, and 2^-22 |g| of its argument), the sum, the division and the product."""
    g, dg = product(x, gate)
    u, du = product(x, up)
    s = g * torch.sigmoid(g)
    return s * u, 1.1 * dg * u.abs() + s.abs() * du + (s * u).abs() * (16 + 4 * g.abs()) * 2.0**-24 + 1.1 * dg * du
