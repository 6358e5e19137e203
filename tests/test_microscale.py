"""Block-scaled formats on the CPU: the layout, the rounding and the scale rules against a
64-bit oracle, and what the entry points refuse."""
from __future__ import annotations

import subprocess
import sys

import pytest
import torch

import microscale_oracle as oracle
from avgen_b200.ops import microscale as mx

SHAPES = [(1, 1), (1, 16), (3, 31), (2, 33), (130, 257), (5, 640)]


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_rounds_to_the_nearest_value_of_its_scale(fmt: str, shape: tuple[int, int]) -> None:
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)) * torch.logspace(-3, 3, shape[1])
    t = mx.quantize(x, fmt)
    scale = oracle.scales(t)
    ratio = torch.where(scale > 0, x.double() / scale, torch.zeros(()).double())
    # fp32 scaling moves a ratio by at most three roundings, so the element is within half a
    # spacing of it (plus that much); saturation only where nvfp4 rounded its scale down
    slack = 3 * 2.0 ** -24 * ratio.abs()
    off = (oracle.elements(t) - ratio.clamp(-oracle.TOP[fmt], oracle.TOP[fmt])).abs()
    assert (off <= 0.5 * oracle.spacing(ratio, fmt) + slack).all()
    if fmt != "nvfp4":
        assert (ratio.abs() <= oracle.TOP[fmt]).all()
    assert torch.equal(mx.dequantize(t, torch.float32).double(), oracle.decode(t).float().double())
    codes = t.codes[:, -(-shape[1] * (8 if fmt == "mxfp8" else 4) // 8):]
    assert not codes.any()  # columns past the matrix


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_power_scales_are_the_smallest_that_saturate_nothing(fmt: str) -> None:
    top = oracle.TOP[fmt]
    amax = torch.tensor([0.0, 1e-45, 2.0 ** -130, 2.0 ** -126, 1.0, top, top * 1.0001, top / 2, 3.3e38, 7.0, 6.0,
                         449.0])
    x = torch.zeros(len(amax), 32)
    x[:, 5] = -amax
    t = mx.quantize(x, fmt)
    assert torch.equal(oracle.scale_bytes(t)[:, 0].long() - 127, oracle.power_scale(amax.double(), fmt))


def test_nvfp4_scales() -> None:
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(2))
    x[1] *= 1e-6  # these blocks' scales round to zero against the tensor's largest value
    t = mx.quantize(x, "nvfp4")
    g = x.abs().max().double() / 2688
    assert torch.allclose(t.global_scale.double(), g.reshape(1), rtol=2.0 ** -23)
    assert torch.equal(oracle.scale_bytes(t)[1], torch.zeros(4, dtype=torch.uint8))
    assert not mx.dequantize(t)[1].any()
    fixed = mx.quantize(x, "nvfp4", global_scale=torch.tensor([0.25]))
    assert float(fixed.global_scale) == 0.25
    zero = mx.quantize(torch.zeros(3, 16), "nvfp4")
    assert not mx.dequantize(zero).any()
    assert not mx.dequantize(mx.quantize(torch.zeros(2, 20), "mxfp8")).any()


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_non_finite_blocks_read_back_as_nan_and_spare_the_others(fmt: str) -> None:
    x = torch.randn(3, 96, generator=torch.Generator().manual_seed(3))
    clean = mx.dequantize(mx.quantize(x.clone(), fmt, **_fixed(fmt)))
    x[0, 1], x[1, 40], x[2, 95] = float("inf"), float("nan"), float("-inf")
    back = mx.dequantize(mx.quantize(x, fmt, **_fixed(fmt)))
    block = oracle.BLOCK[fmt]
    bad = (~torch.isfinite(x)).view(3, -1, block).any(-1).repeat_interleave(block, 1)
    assert torch.equal(torch.isnan(back), bad)
    assert torch.equal(back[~bad], clean[~bad])


def _fixed(fmt: str) -> dict:
    return {"global_scale": torch.tensor([0.002])} if fmt == "nvfp4" else {}


def test_measured_tensor_scale_ignores_non_finite_values() -> None:
    x = torch.ones(2, 32)
    x[0, 0], x[1, 31] = float("inf"), float("nan")
    assert torch.allclose(mx.quantize(x, "nvfp4").global_scale, torch.tensor([1 / 2688]))


def test_add_rmsnorm_reference_matches_its_formula() -> None:
    gen = torch.Generator().manual_seed(4)
    x, u = torch.randn(6, 40, generator=gen).bfloat16(), torch.randn(6, 40, generator=gen).bfloat16()
    w, scale, shift, gate = (torch.randn(s, generator=gen) for s in ((40,), (2, 40), (2, 40), (2, 40)))
    groups = torch.tensor([0, 1, 1, 0, 1, 0], dtype=torch.int32)
    out, t = mx.add_rmsnorm_mod(x, u, w, scale, shift, gate=gate, groups=groups, eps=1e-5)
    rows = groups.long()
    s = x.double() + gate[rows].double() * u.double()
    y = s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-5) * w.double() * (1 + scale[rows].double()) + shift[rows]
    assert (out.double() - s).abs().max() <= 2.0 ** -8 * s.abs().max()
    unit = oracle.spacing(y / oracle.scales(t), "mxfp8") * oracle.scales(t)
    assert ((oracle.decode(t) - y).abs() <= 0.5 * unit + 1e-5 * (1 + y.abs())).all()
    same, _ = mx.add_rmsnorm_mod(x, None, w)
    assert same is x


def test_matmul_reference() -> None:
    gen = torch.Generator().manual_seed(5)
    a = mx.quantize(torch.randn(3, 50, generator=gen), "mxfp4")
    b = mx.quantize(torch.randn(7, 50, generator=gen), "mxfp4")
    out = mx.matmul(a, b, bias=torch.arange(7.0), out_dtype=torch.float32)
    want = oracle.decode(a) @ oracle.decode(b).t() + torch.arange(7.0)
    assert (out.double() - want).abs().max() < 1e-5 * (1 + want.abs().max())


def test_refusals() -> None:
    x = torch.randn(4, 64)
    with pytest.raises(ValueError, match="format must be"):
        mx.quantize(x, "fp8")
    with pytest.raises(ValueError, match="no tensor scale"):
        mx.quantize(x, "mxfp4", global_scale=torch.ones(1))
    with pytest.raises(ValueError, match="no tensor scale"):
        mx.add_rmsnorm_mod(x, None, None, fmt="mxfp8", global_scale=torch.ones(1))
    with pytest.raises(RuntimeError, match="no gradient"):
        mx.quantize(x.clone().requires_grad_(), "mxfp8")
    with torch.no_grad():
        mx.quantize(x.clone().requires_grad_(), "mxfp8")
    with pytest.raises(ValueError, match="gate needs an update"):
        mx.add_rmsnorm_mod(x, None, None, gate=torch.ones(1, 64))
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        mx.quantize(x.double(), "mxfp8")
    a, b = mx.quantize(x, "mxfp8"), mx.quantize(x, "mxfp4")
    with pytest.raises(ValueError, match="operands differ"):
        mx.matmul(a, b)
    with pytest.raises(ValueError, match="operands differ"):
        mx.matmul(a, mx.quantize(x[:, :32], "mxfp8"))
    with pytest.raises(ValueError, match="codes of"):
        mx.MXTensor(a.codes, a.scales, "mxfp8", 65)
    with pytest.raises(ValueError, match="scales of"):
        mx.MXTensor(a.codes, a.scales[:-1], "mxfp8", 64)
    with pytest.raises(ValueError, match="no tensor scale"):
        mx.MXTensor(a.codes, a.scales, "mxfp8", 64, torch.ones(1))


def test_extension_error_messages_format_numbers() -> None:
    """A refusal that prints a number is an exception, not a crash of the process (run in a child)."""
    from avgen_b200.ops import _ext

    if not _ext.available():
        pytest.skip("extension not built")
    code = ("import torch; from avgen_b200.ops._ext import load\n"
            "c = torch.zeros(4, 64, dtype=torch.uint8)\n"
            "try: load().mx_dequantize(c, c, 77, 64, None, torch.float32)\n"
            "except RuntimeError as e: print('refused:', e)\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "unknown format 77" in done.stdout


def test_packed_rows_past_32_bits_are_refused() -> None:
    """A row's scales are found by its number in 32 bits: past them it would get another row's."""
    from avgen_b200.ops import _ext

    if not _ext.available():
        pytest.skip("extension not built")
    rows = 2 ** 32 + 1
    codes = torch.zeros(1, 16, dtype=torch.uint8).expand(rows, 16)
    scales = torch.zeros(1, dtype=torch.uint8).expand(-(-rows // 128) * 512)
    with pytest.raises(RuntimeError, match=f"at most {2 ** 32} rows, got {rows}"):
        _ext.load().mx_dequantize(codes, scales, 1, 1, None, torch.float32)


def test_packed_size() -> None:
    t = mx.quantize(torch.zeros(256, 512), "nvfp4")
    assert t.nbytes == 256 * 512 // 2 + 256 * 512 // 16 + 4
    assert t.shape == (256, 512) and t.rows == 256
    assert t.to("cpu").fmt == "nvfp4"
