"""A linear layer on a weight of 8 bits in 64 bits, on the CPU or where its operands lie: the checker of linear_fp8.  The numbers of e4m3 are
written down from the format (sign, 4 bits of exponent with bias 7, 3 of mantissa, subnormals, no infinities, 0x7f NaN).  No counterpart in the
reference, whose weights have 16 bits."""
from __future__ import annotations

import torch

E4M3 = [(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127]


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """The nearest numbers of e4m3 to v (|v| <= 448), the even one of two that are as near."""
    table = torch.tensor(E4M3, dtype=torch.float64, device=v.device)
    middle = (table[1:] + table[:-1]) / 2
    low, high = torch.bucketize(v.abs(), middle), torch.bucketize(v.abs(), middle, right=True)
    return torch.sign(v) * table[torch.where(low % 2 == 0, low, high)]


def quantize_rows(x: torch.Tensor) -> torch.Tensor:
    """x with every block of 128 columns of a row rounded to e4m3 numbers times the least power of two (at least 2^-126) that holds it."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for k in range(0, x.size(1), 128):
        part = x[:, k:k + 128].double()
        most = part.abs().amax(1)
        unit = torch.tensor([_unit(float(v)) for v in most], dtype=torch.float64, device=x.device)[:, None]
        rounded = round_e4m3(torch.nan_to_num(part / unit, 0.0, 0.0, 0.0)) * unit
        out[:, k:k + 128] = torch.where(torch.isfinite(most)[:, None], rounded, torch.full_like(rounded, float("nan")))
    return out


def _unit(most: float) -> float:
    unit = 2.0 ** -126
    if most != most or most == float("inf"):
        return 1.0
    while most > 448.0 * unit:
        unit *= 2.0
    return unit


def dequantize(weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    n, k = weight.shape
    return weight.double() * scale.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def linear(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, bias=None):
    """(x . (weight times its scales)^T + bias, the sums of the products' magnitudes), without a rounding behind the rows'."""
    rows, w = quantize_rows(x), dequantize(weight, scale)
    y = rows @ w.t().contiguous()
    size = torch.nan_to_num(rows.abs()) @ w.abs().t().contiguous()
    return (y if bias is None else y + bias.double()), size
