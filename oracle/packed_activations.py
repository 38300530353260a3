"""CPU checker of the packed activations: E4M3 with a power-of-two scale per 128 features, the
root-mean-square norm, its gradients and a linear layer's weight gradient, from their definitions
in 64 bits.  Test infrastructure only; written for plainness, not speed."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

BLOCK = 128


def e4m3_values() -> torch.Tensor:
    """The 256 numbers of OCP E4M3 by their definition: sign, 4 exponent bits biased by 7, 3
    significand bits; subnormals in steps of 2^-9, 0x7f and 0xff are NaN, no infinities."""
    out = torch.empty(256, dtype=torch.float64)
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        v = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        if code & 0x7F == 0x7F:
            v = math.nan
        out[code] = -v if code & 0x80 else v
    return out


_MAGNITUDES = e4m3_values()[:127]  # 0 .. 448, ascending


def to_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Codes of the nearest numbers; halfway goes to the even code.  |v| <= 448 or NaN."""
    mag = torch.nan_to_num(v.abs(), nan=0.0)
    hi = torch.searchsorted(_MAGNITUDES, mag).clamp(max=126)  # first that is >= mag
    lo = (hi - 1).clamp(min=0)
    below, above = mag - _MAGNITUDES[lo], _MAGNITUDES[hi] - mag
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    code = torch.where(torch.isnan(v), torch.tensor(127), code)
    return torch.where(torch.signbit(v), code | 128, code).to(torch.uint8)


def pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes [rows, features], biased exponents [rows, blocks]) of a matrix."""
    x = x.double()
    rows, features = x.shape
    codes = torch.zeros(rows, features, dtype=torch.uint8)
    exponents = torch.zeros(rows, -(-features // BLOCK), dtype=torch.uint8)
    for r in range(rows):
        for j in range(exponents.shape[1]):
            b = x[r, j * BLOCK:(j + 1) * BLOCK]
            finite = b[torch.isfinite(b)]
            top = float(finite.abs().max()) if finite.numel() else 0.0
            k = -117
            while k < 119 and top > math.ldexp(448.0, k):
                k += 1
            v = torch.where(torch.isfinite(b), b, torch.full_like(b, math.nan)) * 2.0 ** -k
            codes[r, j * BLOCK:(j + 1) * BLOCK] = to_e4m3(v.clamp(-448.0, 448.0))
            exponents[r, j] = k + 127
    return codes, exponents


def unpack(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    scale = torch.exp2(exponents.double() - 127).repeat_interleave(BLOCK, dim=1)
    return e4m3_values()[codes.long()] * scale[:, : codes.shape[1]]


def rms_norm(x, weight, eps, residual=None):
    """(y, h, n, rstd) in 64 bits; h is the sum rounded to x's type, as the norm's input is."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    wide = h.double()
    rstd = 1.0 / (wide.pow(2).mean(dim=1) + eps).sqrt()
    n = wide * rstd[:, None]
    return n if weight is None else n * weight.double(), h, n, rstd


def rms_norm_backward(grad_y, n, rstd, weight, grad_h=None):
    gy, n, rstd = grad_y.double(), n.double(), rstd.double()
    g = gy if weight is None else gy * weight.double()
    grad_x = rstd[:, None] * (g - n * (g * n).mean(dim=1, keepdim=True))
    if grad_h is not None:
        grad_x = grad_x + grad_h.double()
    return grad_x, (gy * n).sum(dim=0)


def linear_weight_grad(grad_out, x, column_scale: Optional[torch.Tensor] = None):
    out = grad_out.double().t() @ x.double()
    return out if column_scale is None else out * column_scale.double()


def bf16_parts(v: torch.Tensor, parts: int) -> torch.Tensor:
    """What ``parts`` bf16 numbers, each cut off from what the ones before leave, add up to."""
    left, total = v.float(), torch.zeros(v.shape, dtype=torch.float64)
    for _ in range(parts):
        cut = (left.view(torch.int32) & -65536).view(torch.float32)
        total += cut.double()
        left = left - cut
    return total


def weight_grad_bound(grad_out, x, parts: int):
    """How far sums in fp32 may be off, products being exact.  Matrix instructions of 16 tokens align
    what they add to the largest of it: every product and the sum so far may lose a step of 2^-23.
    Tokens of zeros add nothing; pieces of the sum are joined by at most a rounding each."""
    groups = -(-grad_out.shape[0] // 16)
    steps = parts * (grad_out.shape[0] + groups) + groups
    return linear_weight_grad(grad_out.abs(), x.abs()) * steps * 2.0 ** -23
