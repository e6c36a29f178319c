"""The definition of tests/mx_reference.py on the device of its inputs, for sizes that a host takes long over."""

from __future__ import annotations

import torch

from tests import mx_reference as ref


def powers(device) -> torch.Tensor:
    """2^(byte - 127) in float64 (by the host: a power worked out by the device may be off by a last place)."""

    return torch.tensor([2.0 ** (b - 127) for b in range(255)], dtype=torch.float64).to(device)


def scale_byte(amax: torch.Tensor, fmt: str) -> torch.Tensor:
    """Byte of the smallest power of two that keeps finite magnitudes (float64) in range."""

    return torch.searchsorted(powers(amax.device) * ref.LARGEST[fmt], amax)


def blocks_of(x: torch.Tensor) -> torch.Tensor:
    rows, cols = x.shape
    return torch.nn.functional.pad(x.double(), (0, -cols % 128)).view(rows, -1, 32)


def tiles_to_rows(scales: torch.Tensor) -> torch.Tensor:
    """Scale tiles -> [rows of all tiles, blocks], int64."""

    r = torch.arange(scales.shape[0] * 128, device=scales.device)[:, None]
    b = torch.arange(scales.shape[1] * 4, device=scales.device)[None, :]
    return scales[r // 128, b // 4, r % 32, r // 32 % 4, b % 4].long()


def elements(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    """float64 [rows, padded], without scales."""

    rows, codes = codes.shape[0], codes.long()
    if fmt == "mxfp4":
        codes = torch.stack((codes & 15, codes >> 4), -1).view(rows, -1)
    half = 128 if fmt == "mxfp8" else 8
    g = torch.cat((ref.grid(fmt), torch.full((1,), float("nan"), dtype=torch.float64))).to(codes.device)
    return torch.where(codes >= half, -1.0, 1.0) * g[codes % half]


def check_container(q):
    """Scale rows past the last are zero; returns the bytes [rows, blocks] and the elements [rows, padded]."""

    byte = tiles_to_rows(q.scales)
    assert not byte[q.rows:].any()
    return byte[:q.rows], elements(q.codes, q.format)


def check_quantized(q, x: torch.Tensor) -> None:
    """Scales and element values of finite ``x`` [rows, cols], bit for bit, and zeros past the last column."""

    byte, got = check_container(q)
    blocks = blocks_of(x)
    want = scale_byte(blocks.abs().amax(-1), q.format)
    assert torch.equal(byte, want)
    unit = (blocks / powers(x.device)[want][..., None]).view(q.rows, -1)
    g = ref.grid(q.format).to(x.device)
    code = torch.searchsorted((g[1:] + g[:-1]) / 2, unit.abs())  # ties to the lower one
    tie = (code < len(g) - 1) & (unit.abs() == ((g[1:] + g[:-1]) / 2)[code.clamp(max=len(g) - 2)])
    code += (tie & (code % 2 == 1)).long()  # unless the upper one is even
    want = torch.copysign(g[code], unit)
    assert torch.equal(got, want)
