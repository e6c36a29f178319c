"""The microscaled formats in 64 bits, by search instead of by exponent arithmetic, for the tests."""

from __future__ import annotations

import torch

LARGEST = {"mxfp8": 448.0, "mxfp4": 6.0}


def grid(fmt: str) -> torch.Tensor:
    """Magnitudes by code: subnormals, then (1 + m / 2^bits) * 2^e; the e4m3 code 127 is a NaN."""

    bits, bias, codes = (3, 7, 127) if fmt == "mxfp8" else (1, 1, 8)
    values = []
    for c in range(codes):
        e, m = c >> bits, c & ((1 << bits) - 1)
        values.append(m / (1 << bits) * 2.0 ** (1 - bias) if e == 0 else (1 + m / (1 << bits)) * 2.0 ** (e - bias))
    return torch.tensor(values, dtype=torch.float64)


def blocks_of(x: torch.Tensor) -> torch.Tensor:
    """[rows, cols] -> [rows, steps * 4, 32] float64, zeros past the last column."""

    rows, cols = x.shape
    out = torch.zeros(rows, -(-cols // 128) * 128, dtype=torch.float64)
    out[:, :cols] = x.double().cpu()
    return out.view(rows, -1, 32)


def quantize(x: torch.Tensor, fmt: str):
    """float [rows, cols] -> (values [rows, padded] with the scale applied, scale bytes [rows, blocks]); a
    block that is not finite gives byte 255 and NaN."""

    blocks = blocks_of(x)
    amax = blocks.abs().amax(-1)
    table = 2.0 ** torch.arange(-127, 128, dtype=torch.float64)
    byte = torch.searchsorted(table * LARGEST[fmt], torch.nan_to_num(amax, 0.0, 0.0))  # first that is >= amax
    scale = table[byte][..., None]
    g = grid(fmt)
    unit = torch.nan_to_num(blocks / scale, 0.0, 0.0, 0.0)
    upper = torch.searchsorted(g, unit.abs()).clamp(max=len(g) - 1)
    lower = (upper - 1).clamp(min=0)
    up, down = g[upper] - unit.abs(), unit.abs() - g[lower]
    code = torch.where(up < down, upper, torch.where(down < up, lower, torch.where(upper % 2 == 0, upper, lower)))
    values = torch.copysign(g[code], unit) * scale
    bad = ~torch.isfinite(blocks).all(-1)
    values[bad] = float("nan")
    return values.view(x.shape[0], -1), torch.where(bad, 255, byte).to(torch.uint8)


def scale_bytes(scales: torch.Tensor, rows: int) -> torch.Tensor:
    """Scale tiles -> [rows of all tiles, blocks], first checking nothing; index arithmetic of the layout."""

    scales = scales.cpu()
    total, blocks = scales.shape[0] * 128, scales.shape[1] * 4
    r, b = torch.arange(total)[:, None], torch.arange(blocks)[None, :]
    return scales[r // 128, b // 4, r % 32, r // 32 % 4, b % 4]


def decode(codes: torch.Tensor, scales: torch.Tensor, fmt: str, rows: int, cols: int) -> torch.Tensor:
    """float64 [rows, cols]."""

    codes = codes.cpu().long()
    if fmt == "mxfp4":
        codes = torch.stack((codes & 15, codes >> 4), -1).view(rows, -1)
    half = 128 if fmt == "mxfp8" else 8
    g = torch.cat((grid(fmt), torch.tensor([float("nan")] if fmt == "mxfp8" else [], dtype=torch.float64)))
    values = torch.where(codes >= half, -1.0, 1.0) * g[codes % half]
    byte = scale_bytes(scales, rows)[:rows].double()
    scale = torch.where(byte == 255, float("nan"), 2.0 ** (byte - 127))
    return (values * scale.repeat_interleave(32, 1))[:, :cols]
