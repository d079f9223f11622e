"""CPU oracle: the store of embeddings held in 4 or 8 bits, in 64 bits (no counterpart in the reference).

TEST INFRASTRUCTURE ONLY -- see oracle/__init__.py.
"""
from __future__ import annotations

import torch

__all__ = ["store_values", "store_pack"]


def _padded(x: torch.Tensor) -> torch.Tensor:
    n, d = x.shape
    out = torch.zeros(n, -(-d // 128) * 128, dtype=torch.float64)
    out[:, :d] = x.double()
    return out


def _fp4(x: torch.Tensor, group: int):
    """(levels [n, width] signed fp64, scales [n, width / group] fp64); a group that is not finite: levels 0, scale NaN."""
    full = _padded(x)
    g = full.view(full.shape[0], -1, group)
    top = g.abs().amax(2)
    bad = ~torch.isfinite(g).all(2)
    scale = (torch.where(bad, 0.0, top).float() / 6).bfloat16().double()                  # fp32 division is correctly rounded on the CPU
    scale = scale.clamp(min=2.0 ** -120)
    y = torch.where(bad[:, :, None], 0.0, g.abs()) / scale[:, :, None]
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    level = ((y / step).round() * step).clamp(max=6.0) * torch.where(g < 0, -1.0, 1.0)
    level = torch.where(bad[:, :, None], 0.0, level)
    return level.reshape(full.shape), torch.where(bad, float("nan"), scale)


def _i8(x: torch.Tensor):
    x = x.float()
    top = x.abs().amax(1)
    bad = ~torch.isfinite(x).all(1)
    scale = torch.where(top / 127 > 0, top / 127, 1.0)
    scale[bad] = 1.0
    code = torch.where(bad[:, None], 0.0, x)
    code = (code / scale[:, None]).round().clamp(-127, 127)
    scale[bad] = float("nan")
    return code, scale


def store_values(x: torch.Tensor, group: int) -> torch.Tensor:
    """The values (fp64 [n, d]) that a store holds for the rows of x; group 0 = the 8-bit form."""
    if group == 0:
        code, scale = _i8(x)
        return code.double() * scale.double()[:, None]
    level, scale = _fp4(x, group)
    n = level.shape[0]
    return (level.view(n, -1, group) * scale[:, :, None]).view(n, -1)[:, : x.shape[1]]


def store_pack(x: torch.Tensor, group: int):
    """(data, scale) as the store lays them out."""
    if group == 0:
        code, scale = _i8(x)
        out = torch.zeros(x.shape[0], -(-x.shape[1] // 128) * 128, dtype=torch.int8)
        out[:, : x.shape[1]] = code.to(torch.int8)
        return out, scale
    level, scale = _fp4(x, group)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    code = (level.abs()[:, :, None] == table).int().argmax(2) + 8 * (torch.signbit(level) & (_padded(x) < 0)).int()
    n, w = code.shape
    out = torch.zeros(n, w // 2, dtype=torch.int32)
    k = torch.arange(w)
    piece, r = k // 128, k % 128
    nibble = 32 * ((r % 32) // 8) + 8 * (r // 32) + r % 8                                  # m = r / 32, c = (r % 32) / 8, j = r % 8
    for half in (0, 1):
        pick = nibble % 2 == half
        out[:, (64 * piece + nibble // 2)[pick]] += code[:, pick].int() << (4 * half)
    return out.to(torch.uint8), scale.to(torch.bfloat16)
