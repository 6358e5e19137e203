"""The block-scaled formats in 64 bits, written from their definition (no code shared
with the package): decoding stored codes and scales, and the nearest value a format has."""
from __future__ import annotations

import torch

BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}
TOP = {"mxfp8": 448.0, "mxfp4": 6.0, "nvfp4": 6.0}


def e4m3(byte: torch.Tensor) -> torch.Tensor:
    """Value of an e4m3 byte: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f is NaN."""
    byte = byte.long()
    e, f, sign = (byte >> 3) & 15, byte & 7, byte >> 7
    v = torch.where(e > 0, (8 + f).double() * torch.pow(2.0, (e - 10).double()), f.double() * 2.0 ** -9)
    v = torch.where((byte & 127) == 127, float("nan"), v)
    return torch.where(sign == 1, -v, v)


def e2m1(code: torch.Tensor) -> torch.Tensor:
    """Value of an e2m1 code: sign, 2 exponent bits (bias 1), 1 fraction bit."""
    code = code.long()
    e, f, sign = (code >> 1) & 3, code & 1, code >> 3
    v = torch.where(e > 0, (2 + f).double() * torch.pow(2.0, (e - 2).double()), f.double() * 0.5)
    return torch.where(sign == 1, -v, v)


def scale_bytes(t) -> torch.Tensor:  # noqa: ANN001
    """``[rows, blocks]`` scale bytes picked one by one out of the tiled layout."""
    rows, blocks = t.rows, -(-t.cols // BLOCK[t.fmt])
    tiles = -(-blocks // 4)
    r, c = torch.meshgrid(torch.arange(rows), torch.arange(blocks), indexing="ij")
    at = (r // 128 * tiles + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4
    return t.scales.cpu()[at]


def elements(t) -> torch.Tensor:  # noqa: ANN001
    """``[rows, cols]`` element values without their scales."""
    codes = t.codes.cpu()
    if t.fmt == "mxfp8":
        return e4m3(codes)[:, :t.cols]
    return e2m1(torch.stack((codes & 15, codes >> 4), -1).flatten(1))[:, :t.cols]


def scales(t) -> torch.Tensor:  # noqa: ANN001
    """``[rows, cols]`` full scale (block times tensor scale) of every element."""
    raw = scale_bytes(t)
    s = e4m3(raw) if t.fmt == "nvfp4" else torch.where(raw == 255, float("nan"),
                                                       torch.pow(2.0, raw.double() - 127))
    if t.global_scale is not None:
        s = s * t.global_scale.cpu().double()
    return s.repeat_interleave(BLOCK[t.fmt], 1)[:, :t.cols]


def decode(t) -> torch.Tensor:  # noqa: ANN001
    return elements(t) * scales(t)


def spacing(ratio: torch.Tensor, fmt: str) -> torch.Tensor:
    """Distance between neighbouring elements around ``|ratio|``."""
    least, bits = (-6, 3) if fmt == "mxfp8" else (0, 1)
    e = torch.frexp(ratio.abs().clamp(max=TOP[fmt])).exponent - 1
    return torch.pow(2.0, (e.clamp(min=least) - bits).double())


def round_to(v: torch.Tensor, fmt: str) -> torch.Tensor:
    """Nearest element (ties to even), saturating."""
    unit = spacing(v, fmt)
    return torch.sign(v) * (torch.round(v.abs() / unit) * unit).clamp(max=TOP[fmt])


def power_scale(amax: torch.Tensor, fmt: str) -> torch.Tensor:
    """Exponent of the smallest power of two that keeps ``amax`` within the format's top."""
    s = torch.full(amax.shape, -126, dtype=torch.int64)
    for e in range(-126, 127):
        s = torch.where(amax > TOP[fmt] * 2.0 ** e, e + 1, s)
    return s.clamp(max=126)
