"""Block-scaled ("microscaled") 8- and 4-bit operands: the formats, and the operators on them.

======  ==================  ==========================  =====================
format  element             block scale                 tensor scale
======  ==================  ==========================  =====================
mxfp8   e4m3 (8 bits)       2^s per 32 (e8m0)           -
mxfp4   e2m1 (4 bits)       2^s per 32 (e8m0)           -
nvfp4   e2m1 (4 bits)       e4m3 per 16                 fp32 ``g``
======  ==================  ==========================  =====================

A value is ``code * block scale (* g)``; blocks run along a row, which is the axis a
linear layer reduces over. :func:`quantize` and :func:`dequantize` move between plain
and packed tensors, :func:`add_rmsnorm_mod` adds a residual update, normalises and
writes the packed rows the next linear layer reads, :func:`matmul` multiplies two
packed operands on the tensor cores without unpacking them.

On a CUDA device these launch the sm_100a kernels (``csrc/microscale.cu``,
``csrc/mx_gemm.cu``) on the current stream and never wait for the device; on the CPU
they are the PyTorch restatement below. They have no gradient (sampling and
evaluation run them): an input that requires one is refused while gradients are being
recorded. The reference framework has no counterpart; its low-precision option is a
third-party package's fp8 training (avgen/parallel/precision.py:212-284).

Rounding is to nearest, ties to even, saturating at the format's largest number.

* mxfp8 / mxfp4: a block's ``s`` is the smallest with ``amax <= top * 2^s`` (top = 448
  or 6), so no value saturates, kept within [-126, 126].
* nvfp4: block scale ``amax / (6 g)`` rounded to e4m3. :func:`quantize` makes
  ``g = amax(tensor) / (6 * 448)`` from the tensor's finite values (at least
  ``2^-100``) unless it is given one; :func:`add_rmsnorm_mod` takes ``g = 1`` unless it
  is given one. With ``g = 1`` a block whose largest value is under 0.09 gets a subnormal
  scale (fewer bits), under 0.006 a zero one: rows that a small gain or ``1 + scale``
  takes there want their own ``g``. No row of ``W`` columns needs a larger one than
  ``(sqrt(W) * max|weight * (1 + scale)| + max|shift|) / 2688``, with which nothing
  saturates and blocks keep normal scales down to 1 / 28000 of that bound.
* A block that holds an infinity or a NaN gets a NaN scale. It reads back as NaN and
  every product row it enters is NaN; other blocks are not touched.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from avgen_b200.ops._ext import load
from avgen_b200.ops.kernels import _count

__all__ = ["FORMATS", "MXTensor", "add_rmsnorm_mod", "block_size", "dequantize", "matmul", "quantize"]

_IDS = {"mxfp8": 0, "mxfp4": 1, "nvfp4": 2}
FORMATS = tuple(_IDS)
_F32 = torch.float32
_SCALE_FLOOR = 2.0 ** -100


def _format_id(fmt: str) -> int:
    try:
        return _IDS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"format must be one of {', '.join(FORMATS)}; got {fmt!r}") from None


def block_size(fmt: str) -> int:
    """Columns that share one scale."""
    return 16 if _format_id(fmt) == 2 else 32


def _row_bytes(fmt: str, cols: int) -> int:
    padded = -(-cols // 32) * 32
    return padded if fmt == "mxfp8" else padded // 2


def _scale_bytes(fmt: str, rows: int, cols: int) -> int:
    return -(-rows // 128) * -(-cols // (4 * block_size(fmt))) * 512


@dataclass(slots=True, eq=False)
class MXTensor:
    """A packed matrix ``[rows, cols]``. Its fields are set once, here or by the operators.

    ``codes`` is uint8 ``[rows, bytes]``: one row's codes, columns padded with zero
    codes to a multiple of 32; 4-bit codes two to a byte, the even column in the low
    half. ``scales`` is one flat uint8 array of tiles of 128 rows x 4 blocks: the scale
    of row ``r``, block ``c`` is byte ``r % 32 * 16 + r % 128 // 32 * 4 + c % 4`` of the
    512-byte tile ``(r // 128, c // 4)``, tiles of a row group side by side; bytes past
    the matrix are zero. ``global_scale`` (nvfp4 only) is fp32 ``[1]`` on the same
    device; None stands for 1.
    """

    codes: torch.Tensor
    scales: torch.Tensor
    fmt: str
    cols: int
    global_scale: torch.Tensor | None = None

    def __post_init__(self) -> None:
        _format_id(self.fmt)
        if self.global_scale is not None and self.fmt != "nvfp4":
            raise ValueError(f"{self.fmt} has no tensor scale")
        codes = self.codes
        if (codes.dtype is not torch.uint8 or codes.dim() != 2 or self.cols < 1
                or codes.shape[1] != _row_bytes(self.fmt, self.cols)):
            raise ValueError(f"{self.fmt} codes of {self.cols} columns must be uint8 [rows, "
                             f"{_row_bytes(self.fmt, max(1, self.cols))}]; got {codes.dtype} {tuple(codes.shape)}")
        if self.scales.dtype is not torch.uint8 or self.scales.numel() != _scale_bytes(self.fmt, len(codes), self.cols):
            raise ValueError(f"{self.fmt} scales of a {len(codes)} x {self.cols} matrix must be "
                             f"{_scale_bytes(self.fmt, len(codes), self.cols)} uint8 bytes; got "
                             f"{self.scales.dtype} {tuple(self.scales.shape)}")

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def shape(self) -> tuple[int, int]:
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + (0 if self.global_scale is None else 4)

    def to(self, device: torch.device | str) -> MXTensor:
        g = self.global_scale
        return MXTensor(self.codes.to(device), self.scales.to(device), self.fmt, self.cols,
                        None if g is None else g.to(device))

    def block_scales(self) -> torch.Tensor:
        """fp32 ``[rows, blocks]`` block scales (without the tensor scale)."""
        blocks = -(-self.cols // block_size(self.fmt))
        tiles = -(-blocks // 4)
        raw = self.scales.view(-1, tiles, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, 4 * tiles)
        raw = raw[:self.rows, :blocks].contiguous()
        if self.fmt == "nvfp4":
            return raw.view(torch.float8_e4m3fn).float()
        value = torch.exp2(raw.float() - 127.0)
        return torch.where(raw == 255, torch.full_like(value, float("nan")), value)


def _made(codes: torch.Tensor, scales: torch.Tensor, fmt: str, cols: int, g: torch.Tensor | None) -> MXTensor:
    """An :class:`MXTensor` of what a kernel returned, without checking it again."""
    t = MXTensor.__new__(MXTensor)
    t.codes, t.scales, t.fmt, t.cols, t.global_scale = codes, scales, fmt, cols, g
    return t


def _no_grad_input(what: str, *tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad() or with detached inputs")


def quantize(x: torch.Tensor, fmt: str, *, global_scale: torch.Tensor | None = None) -> MXTensor:
    """Pack ``x[..., cols]`` (bf16, fp16 or fp32; leading dimensions become rows).

    ``global_scale`` (nvfp4): a positive fp32 ``[1]`` tensor scale to use, e.g. a
    calibrated one; without it one pass over ``x`` measures it first."""
    fid = _format_id(fmt)
    if x.requires_grad:
        _no_grad_input("quantize", x)
    if global_scale is not None and fid != 2:
        raise ValueError(f"{fmt} has no tensor scale")
    if not x.is_cuda:
        return _quantize_reference(x, fmt, global_scale)
    codes, scales, g, launches = load().mx_quantize(x, fid, global_scale, fid == 2 and global_scale is None)
    _count(launches)
    return _made(codes, scales, fmt, x.shape[-1], g)


def dequantize(t: MXTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values ``[rows, cols]`` that ``t`` stands for, in bf16, fp16 or fp32."""
    if not t.codes.is_cuda:
        return _dequantize_reference(t).to(dtype)
    out = load().mx_dequantize(t.codes, t.scales, _IDS[t.fmt], t.cols, t.global_scale, dtype)
    _count()
    return out


def add_rmsnorm_mod(
    x: torch.Tensor,
    update: torch.Tensor | None,
    weight: torch.Tensor | None,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    *,
    gate: torch.Tensor | None = None,
    rows_per_batch: int = 1,
    groups: torch.Tensor | None = None,
    eps: float = 1e-6,
    fmt: str = "mxfp8",
    global_scale: torch.Tensor | None = None,
) -> tuple[torch.Tensor, MXTensor]:
    """``x' = x + gate[b] * update`` and ``rmsnorm(x') * weight * (1 + scale[b]) + shift[b]`` packed.

    ``x`` and ``update`` are ``[..., W]`` of one type (bf16, fp16 or fp32); ``weight``
    fp32 ``[W]``; ``scale``, ``shift`` and ``gate`` fp32 ``[B, W]`` rows picked as in
    :func:`avgen_b200.ops.kernels.rmsnorm_mod` (``b = groups[row]``, else ``row //
    rows_per_batch``). Without ``update``, ``x'`` is ``x`` itself. The norm takes the fp32
    sum, so ``x'``'s rounding to its type does not enter it."""
    fid = _format_id(fmt)
    _no_grad_input("add_rmsnorm_mod", x, update, weight, scale, shift, gate)
    if global_scale is not None and fid != 2:
        raise ValueError(f"{fmt} has no tensor scale")
    if not x.is_cuda:
        return _add_rmsnorm_reference(x, update, weight, scale, shift, gate, rows_per_batch, groups, eps, fmt,
                                      global_scale)
    out, codes, scales = load().mx_add_rmsnorm(x, update, weight, scale, shift, gate, groups, rows_per_batch, eps, fid,
                                               global_scale)
    _count()
    return out, _made(codes, scales, fmt, x.shape[-1], global_scale)


def matmul(a: MXTensor, b: MXTensor, *, bias: torch.Tensor | None = None,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a[M, K] @ b[N, K]^T (+ bias[N])`` of two packed operands of one format, accumulated
    in fp32 and rounded once to ``out_dtype`` (bf16, fp16 or fp32)."""
    if a.fmt != b.fmt or a.cols != b.cols:
        raise ValueError(f"operands differ: {a.fmt} {a.shape} and {b.fmt} {b.shape}")
    if bias is not None:
        _no_grad_input("matmul", bias)
    if not a.codes.is_cuda:
        out = _dequantize_reference(a) @ _dequantize_reference(b).t()
        return (out if bias is None else out + bias).to(out_dtype)
    out = load().mx_gemm(a.codes, a.scales, a.global_scale, b.codes, b.scales, b.global_scale, _IDS[a.fmt], a.cols,
                         bias, out_dtype)
    _count()
    return out


# ----------------------------------------------------------------------------- CPU restatement
def _round_e2m1(v: torch.Tensor) -> torch.Tensor:
    """Indices 0..7 of the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, bit 3 the sign."""
    a = v.abs()
    index = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, 2 + torch.round(a), 4 + torch.round(a / 2)))
    return index.clamp(max=7).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)


def _tile_scales(raw: torch.Tensor) -> torch.Tensor:
    rows, blocks = raw.shape
    full = torch.zeros(-(-rows // 128) * 128, -(-blocks // 4) * 4, dtype=torch.uint8)
    full[:rows, :blocks] = raw
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _quantize_reference(x: torch.Tensor, fmt: str, global_scale: torch.Tensor | None) -> MXTensor:
    if x.dtype not in (torch.bfloat16, torch.float16, _F32):
        raise ValueError(f"quantize: x must be bf16, fp16 or fp32; got {x.dtype}")
    cols, block = x.shape[-1], block_size(fmt)
    v = x.reshape(-1, cols).float()
    rows = v.shape[0]
    v = torch.nn.functional.pad(v, (0, -cols % 32)).view(rows, -1, block)
    bad = ~torch.isfinite(v).all(-1)
    amax = torch.where(bad, 0.0, v.abs().amax(-1))
    if fmt == "nvfp4":
        if global_scale is None:
            finite = torch.where(torch.isfinite(v), v.abs(), 0.0)
            g = (finite.amax() * (1.0 / 2688.0) if rows else torch.ones(())).clamp(min=_SCALE_FLOOR).reshape(1)
        else:
            g = global_scale.float()
        scale = (amax / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
        inv = torch.where(scale.float() > 0, 1.0 / (scale.float() * g), 0.0)
        raw = torch.where(bad, torch.tensor(0x7F, dtype=torch.uint8), scale.view(torch.uint8))
    else:
        g = None
        mantissa, exponent = torch.frexp(amax)
        top, bits = (0.875, 9) if fmt == "mxfp8" else (0.75, 3)
        s = torch.where(mantissa <= top, exponent - bits, exponent - bits + 1)
        s = torch.where(amax > 0, s, -126).clamp(-126, 126)
        inv = torch.exp2(-s.float())
        raw = torch.where(bad, 255, s + 127).to(torch.uint8)
    q = torch.where(bad[..., None], torch.zeros(()), v * inv[..., None]).flatten(1)
    if fmt == "mxfp8":
        codes = q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        index = _round_e2m1(q)
        codes = index[:, 0::2] | (index[:, 1::2] << 4)
    return MXTensor(codes.contiguous(), _tile_scales(raw[:, :-(-cols // block)]), fmt, cols, g)


def _dequantize_reference(t: MXTensor) -> torch.Tensor:
    if t.fmt == "mxfp8":
        q = t.codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
        table = torch.cat((table, -table))
        q = torch.stack((table[(t.codes & 15).long()], table[(t.codes >> 4).long()]), -1).flatten(1)
    s = t.block_scales().repeat_interleave(block_size(t.fmt), 1)[:, :t.cols]
    v = q[:, :t.cols] * s
    return v if t.global_scale is None else v * t.global_scale


def _add_rmsnorm_reference(x, update, weight, scale, shift, gate, rows_per_batch, groups, eps,  # noqa: ANN001, ANN202
                           fmt, global_scale):
    cols = x.shape[-1]
    v = x.reshape(-1, cols).float()
    rows = torch.arange(v.shape[0]) // max(1, rows_per_batch) if groups is None else groups.long()
    out = x
    if update is not None:
        u = update.reshape(-1, cols).float()
        v = v + (u if gate is None else gate[rows] * u)
        out = v.to(x.dtype).view(x.shape)
    elif gate is not None:
        raise ValueError("add_rmsnorm_mod: gate needs an update")
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight
    if scale is not None:
        y = y * (1.0 + scale[rows])
    if shift is not None:
        y = y + shift[rows]
    g = torch.ones(1) if fmt == "nvfp4" and global_scale is None else global_scale
    q = _quantize_reference(y, fmt, g)
    return out, MXTensor(q.codes, q.scales, fmt, cols, global_scale)
