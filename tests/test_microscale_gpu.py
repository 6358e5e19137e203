"""The block-scaled kernels on a B200 against 64-bit oracles and the CPU restatement."""
from __future__ import annotations

import pytest
import torch

import microscale_oracle as oracle
from avgen_b200.ops import microscale as mx

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _clean() -> None:
    from avgen_b200.ops._ext import check_errors

    assert check_errors() == 0


def _rows(rows: int, cols: int, seed: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(cols, generator=gen))
    return x.to(dtype)


def _same(got: mx.MXTensor, want: mx.MXTensor) -> None:
    assert got.shape == want.shape and got.fmt == want.fmt
    assert torch.equal(got.scales.cpu(), want.scales)
    assert torch.equal(got.codes.cpu(), want.codes)
    if want.global_scale is not None:
        assert torch.equal(got.global_scale.cpu(), want.global_scale)


# ----------------------------------------------------------------------------- quantise
@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 2560), (3, 31), (2, 33), (129, 257), (127, 512), (300, 1000), (5, 8200)])
def test_quantize_equals_the_restatement(fmt: str, dtype: torch.dtype, shape: tuple[int, int]) -> None:
    x = _rows(*shape, seed=shape[1], dtype=dtype)
    got = mx.quantize(x.to(DEV), fmt)
    _same(got, mx.quantize(x, fmt))
    for out in DTYPES:
        assert torch.equal(mx.dequantize(got, out).cpu(), mx.dequantize(mx.quantize(x, fmt), out))


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_quantize_takes_any_layout(fmt: str) -> None:
    base = _rows(96, 200, 7, torch.bfloat16)
    dev = base.to(DEV)
    for view in (lambda t: t[:, 3:131], lambda t: t[::2, :64], lambda t: t.t(), lambda t: t[5:6].expand(40, 200),
                 lambda t: t.view(4, 24, 200), lambda t: t[:, ::2], lambda t: t[0], lambda t: t[:, 8:136]):
        _same(mx.quantize(view(dev), fmt), mx.quantize(view(base), fmt))


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_quantize_edges(fmt: str) -> None:
    x = torch.zeros(8, 160)
    x[1] = 1e-45
    x[2] = torch.linspace(-3.3e38, 3.3e38, 160)
    x[3] = torch.linspace(-6, 6, 160)
    x[4, 3], x[4, 50], x[4, 159] = float("inf"), float("nan"), float("-inf")
    x[5] = torch.arange(160) % 13 * 0.25  # ties
    x[6] = 2.0 ** -126
    x[7] = -0.0
    for g in ([None] if fmt != "nvfp4" else [None, torch.tensor([1e-4]), torch.tensor([2.0])]):
        got = mx.quantize(x.to(DEV), fmt, global_scale=None if g is None else g.to(DEV))
        want = mx.quantize(x, fmt, global_scale=g)
        assert torch.equal(got.scales.cpu(), want.scales)
        a, b = mx.dequantize(got, torch.float32).cpu(), mx.dequantize(want, torch.float32)
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def test_quantize_empty_rows() -> None:
    for fmt in mx.FORMATS:
        t = mx.quantize(torch.empty(0, 64, device=DEV), fmt)
        assert t.shape == (0, 64) and mx.dequantize(t).shape == (0, 64)
        w = mx.quantize(torch.ones(8, 64, device=DEV), fmt)
        assert mx.matmul(t, w).shape == (0, 8) and mx.matmul(w, t).shape == (8, 0)
        out, n = mx.add_rmsnorm_mod(torch.empty(0, 64, device=DEV), None, None, fmt=fmt)
        assert out.shape == (0, 64) and n.shape == (0, 64)


# ----------------------------------------------------------------------------- residual norm
def _norm_case(rows: int, cols: int, dtype: torch.dtype, levels: int, seed: int) -> dict:
    gen = torch.Generator().manual_seed(seed)
    case = {"x": _rows(rows, cols, seed, dtype), "update": _rows(rows, cols, seed + 1, dtype),
            "weight": 1 + 0.1 * torch.randn(cols, generator=gen)}
    for name in ("scale", "shift", "gate"):
        case[name] = 0.3 * torch.randn(levels, cols, generator=gen) if levels else None
    case["groups"] = torch.randint(0, levels, (rows,), generator=gen, dtype=torch.int32) if levels else None
    return case


def _norm_oracle(case: dict, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    rows = case["groups"].long() if case["groups"] is not None else None
    pick = lambda name: case[name].double()[rows] if case[name] is not None else None  # noqa: E731
    s = case["x"].double()
    if case["update"] is not None:
        gate = pick("gate")
        s = s + case["update"].double() * (1.0 if gate is None else gate)
    y = s / torch.sqrt(s.square().mean(1, keepdim=True) + eps)
    if case["weight"] is not None:
        y = y * case["weight"].double()
    if case["scale"] is not None:
        y = y * (1 + pick("scale"))
    if case["shift"] is not None:
        y = y + pick("shift")
    return s, y


def _check_norm(case: dict, fmt: str, eps: float = 1e-6, **more: object) -> None:
    dev = {k: None if v is None else v.to(DEV) for k, v in case.items()}
    out, t = mx.add_rmsnorm_mod(dev["x"], dev["update"], dev["weight"], dev["scale"], dev["shift"], gate=dev["gate"],
                                groups=dev["groups"], eps=eps, fmt=fmt, **more)
    s, y = _norm_oracle(case, eps)
    half_ulp = torch.finfo(out.dtype).eps / 2
    mass = case["x"].double().abs() + (s - case["x"].double()).abs()
    assert ((out.cpu().double() - s).abs() <= half_ulp * s.abs() + 2.0 ** -23 * mass + 2.0 ** -25).all()
    # fp32 arithmetic: a row sum of W squares and four products are off by far less than 1e-5
    # relative; an element is then within half a spacing, at its own block's scale
    cols = y.shape[1]
    block = oracle.BLOCK[fmt]
    amax = torch.nn.functional.pad(y.abs(), (0, -cols % block)).view(len(y), -1, block).amax(-1)
    if fmt == "nvfp4":
        off = (oracle.e4m3(oracle.scale_bytes(t)) - amax / 6).abs()
        assert off.le(amax / 6 * (2.0 ** -4 + 1e-5) + 2.0 ** -10).all()
    else:
        low, high = (oracle.power_scale(amax * f, fmt) for f in (1 - 1e-5, 1 + 1e-5))
        got = oracle.scale_bytes(t).long() - 127
        assert ((got >= low) & (got <= high)).all()
    scale = oracle.scales(t)
    ratio = torch.where(scale > 0, y / scale, torch.zeros(()).double()).clamp(-oracle.TOP[fmt], oracle.TOP[fmt])
    slack = 1e-5 * (1 + y.abs().amax(1, keepdim=True))
    assert ((oracle.elements(t) - ratio).abs() * scale <= 0.5 * oracle.spacing(ratio, fmt) * scale + slack).all()
    rows = torch.arange(t.rows)
    used = torch.zeros_like(t.scales.cpu())
    tiles = -(-t.cols // (4 * block))
    blocks = torch.arange(-(-t.cols // block))
    r, c = torch.meshgrid(rows, blocks, indexing="ij")
    used[(r // 128 * tiles + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4] = 1
    assert not t.scales.cpu()[used == 0].any()
    _clean()


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 2560), (3, 33), (130, 768), (129, 1000), (16, 2560), (5, 5120), (40, 40),
                                   (3, 8192), (2, 13824), (2, 40000), (257, 1537)])
def test_add_rmsnorm_against_64_bits(fmt: str, shape: tuple[int, int]) -> None:
    _check_norm(_norm_case(*shape, torch.bfloat16, 3, seed=sum(shape)), fmt)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [256, 259, 4096])
def test_add_rmsnorm_types_and_missing_parts(dtype: torch.dtype, cols: int) -> None:
    case = _norm_case(70, cols, dtype, 2, seed=cols)
    _check_norm(case, "mxfp8")
    for missing in (("gate",), ("gate", "update"), ("scale",), ("shift",), ("weight",),
                    ("scale", "shift", "gate", "groups"), ("scale", "shift", "gate", "groups", "weight", "update")):
        _check_norm({k: None if k in missing else v for k, v in case.items()}, "mxfp8", eps=1e-5)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [250, 256, 500, 700, 1000, 4096, 9000, 20000])
def test_add_rmsnorm_other_types_to_four_bits(fmt: str, dtype: torch.dtype, cols: int) -> None:
    case = _norm_case(130 if cols < 5000 else 5, cols, dtype, 2, seed=cols)
    _check_norm(case, fmt)
    _check_norm({k: None if k in ("scale", "shift", "gate", "groups") else v for k, v in case.items()}, fmt)


@pytest.mark.parametrize("cols", [640, 1001])
@pytest.mark.parametrize("gain", [1.0, 1e-2, 1e-3])
def test_add_rmsnorm_nvfp4_tensor_scale_of_the_norms_range(cols: int, gain: float) -> None:
    """With the tensor scale that the largest possible value of a row asks for, block scales keep e4m3's
    precision (normal ones 2^-4 of theirs), and values an element's, at gains that differ by 1000."""
    case = _norm_case(70, cols, torch.bfloat16, 3, seed=cols)
    case["shift"] = None
    case["weight"][:cols // 2] *= gain
    reach = cols ** 0.5 * float((case["weight"].abs() * (1 + case["scale"]).abs()).max())
    g = torch.tensor([reach / 2688])
    dev = {k: None if v is None else v.to(DEV) for k, v in case.items()}
    _, t = mx.add_rmsnorm_mod(dev["x"], dev["update"], dev["weight"], dev["scale"], gate=dev["gate"],
                              groups=dev["groups"], fmt="nvfp4", global_scale=g.to(DEV))
    assert torch.equal(t.global_scale.cpu(), g)
    y = _norm_oracle(case, 1e-6)[1]
    amax = torch.nn.functional.pad(y.abs(), (0, -cols % 16)).view(len(y), -1, 16).amax(-1) / (6 * g.double())
    assert ((oracle.e4m3(oracle.scale_bytes(t)) - amax).abs() <= amax * (2.0 ** -4 + 1e-5) + 2.0 ** -10).all()
    scale = oracle.scales(t)
    ratio = torch.where(scale > 0, y / scale, torch.zeros(()).double())
    slack = 1e-5 * amax.repeat_interleave(16, 1)[:, :cols] * 6 * g.double()
    assert ((oracle.elements(t) - ratio.clamp(-6, 6)).abs() * scale
            <= 0.5 * oracle.spacing(ratio, "nvfp4") * scale + slack).all()


def test_add_rmsnorm_rows_per_batch_and_strides() -> None:
    case = _norm_case(64, 640, torch.bfloat16, 4, seed=3)
    case["groups"] = None
    dev = {k: None if v is None else v.to(DEV) for k, v in case.items()}
    wide = torch.randn(4, 6, 640, device=DEV)  # modulation rows as the model keeps them: chunks of one tensor
    wide[:, 0], wide[:, 1], wide[:, 2] = dev["shift"], dev["scale"], dev["gate"]
    xs, us = torch.zeros(64, 700, device=DEV).bfloat16(), torch.zeros(64, 643, device=DEV).bfloat16()
    xs[:, 8:648], us[:, 3:] = dev["x"], dev["update"]
    a, ta = mx.add_rmsnorm_mod(xs[:, 8:648], us[:, 3:], dev["weight"], wide[:, 1], wide[:, 0], gate=wide[:, 2],
                               rows_per_batch=16)
    groups = torch.arange(64, device=DEV, dtype=torch.int32) // 16
    b, tb = mx.add_rmsnorm_mod(dev["x"].view(4, 16, 640), dev["update"].view(4, 16, 640), dev["weight"], dev["scale"],
                               dev["shift"], gate=dev["gate"], groups=groups)
    assert torch.equal(a, b.view(64, 640)) and torch.equal(ta.codes, tb.codes) and torch.equal(ta.scales, tb.scales)


@pytest.mark.parametrize("rows", [1, 4])
def test_add_rmsnorm_scale_and_shift_of_different_strides(rows: int) -> None:
    wide, x = torch.randn(rows, 6, 640, device=DEV), torch.randn(16 * rows, 640, device=DEV).bfloat16()
    plain = wide[:, 0].clone()
    once = torch.randn(640, device=DEV).expand(rows, 640)
    for scale, shift in ((wide[:, 1], plain), (plain, wide[:, 1]), (once, plain), (wide[:, 1], once)):
        _, got = mx.add_rmsnorm_mod(x, None, None, scale, shift, rows_per_batch=16)
        _, want = mx.add_rmsnorm_mod(x, None, None, scale.clone(memory_format=torch.contiguous_format),
                                     shift.clone(memory_format=torch.contiguous_format), rows_per_batch=16)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


def test_add_rmsnorm_edges() -> None:
    x = torch.zeros(5, 96, device=DEV)
    x[1], x[2, 4], x[3, 90] = 1e30, float("nan"), float("inf")
    x[4] = torch.linspace(-1, 1, 96, device=DEV)
    out, t = mx.add_rmsnorm_mod(x, None, None)
    back = mx.dequantize(t, torch.float32)
    assert out is x and not back[0].any()
    assert torch.isnan(back[2]).all() and torch.isnan(back[3, 64:]).all()  # a NaN reaches its row, inf its block
    assert torch.isfinite(back[4]).all()
    _, t4 = mx.add_rmsnorm_mod(x[4:], None, None, fmt="nvfp4", global_scale=torch.tensor([0.01], device=DEV))
    assert (mx.dequantize(t4, torch.float32) - back[4]).abs().max() < 0.5


@pytest.mark.parametrize("rows", [2 ** 31 - 257, 2 ** 31 - 9000])
def test_add_rmsnorm_refuses_rows_past_its_row_numbers(rows: int) -> None:
    """Rows are counted in 32 signed bits: the last row plus one step of the loop (up to 64
    rows an SM) has to fit. One column, repeated without memory of its own."""
    most = 2 ** 31 - 128 - 64 * torch.cuda.get_device_properties(0).multi_processor_count
    x = torch.ones(1, 1, device=DEV).expand(rows, 1)
    with pytest.raises(RuntimeError, match=f"at most {most} rows, got {rows}"):
        mx.add_rmsnorm_mod(x, None, None, fmt="mxfp4")


def test_add_rmsnorm_picks_from_a_modulation_table_of_2_to_the_31_rows() -> None:
    shift = torch.zeros(2 ** 31, 1, device=DEV)
    shift[2 ** 31 - 1], shift[5] = 2.0, 4.0
    groups = torch.tensor([5, 2 ** 31 - 1, 6], dtype=torch.int32, device=DEV)
    _, t = mx.add_rmsnorm_mod(torch.zeros(3, 1, device=DEV), None, None, None, shift, groups=groups)
    assert mx.dequantize(t, torch.float32).flatten().tolist() == [4.0, 2.0, 0.0]
    _, t = mx.add_rmsnorm_mod(torch.zeros(3, 1, device=DEV), None, None, None, shift[:8], rows_per_batch=2 ** 62)
    assert not mx.dequantize(t).any()


# ----------------------------------------------------------------------------- product
PRODUCTS = [(1, 1, 1), (1, 8, 32), (2, 130, 65), (128, 128, 256), (129, 127, 96), (200, 300, 1000), (257, 513, 2570),
            (1, 2560, 2560), (16, 640, 4096), (33, 1024, 160), (64, 200, 13824), (640, 384, 129), (1000, 2568, 512),
            (130, 24, 10240), (3, 7, 30000), (2400, 2100, 160), (4000, 1304, 1100), (300, 20000, 520)]


def _check_product(a: mx.MXTensor, b: mx.MXTensor, bias: torch.Tensor | None, dtype: torch.dtype) -> None:
    got = mx.matmul(a, b, bias=bias, out_dtype=dtype)
    assert got.dtype is dtype and got.is_contiguous()
    va, vb = oracle.decode(a), oracle.decode(b)
    want, mass = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias is not None:
        want, mass = want + bias.cpu().double(), mass + bias.cpu().double().abs()
    # one truncation to 24 bits per accumulated product slice of at least 32 columns, and the tree inside a slice
    fp32 = (a.cols / 32 + 32) * 2.0 ** -23 * mass
    half_ulp = torch.finfo(dtype).eps / 2
    least = {torch.bfloat16: 2.0 ** -130, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}[dtype]
    assert ((got.cpu().double() - want).abs() <= fp32 + half_ulp * (want.abs() + fp32) + least).all()
    _clean()


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("shape", PRODUCTS)
def test_matmul_against_64_bits(fmt: str, shape: tuple[int, int, int]) -> None:
    m, n, k = shape
    a, b = mx.quantize(_rows(m, k, m + k).to(DEV), fmt), mx.quantize(_rows(n, k, n).to(DEV) / k ** 0.5, fmt)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(DEV)
    _check_product(a, b, bias if (m + n) % 2 else None, DTYPES[(m + k) % 3])


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_output_types(fmt: str, dtype: torch.dtype) -> None:
    for n in (264, 261):
        a, b = mx.quantize(_rows(150, 320, 1).to(DEV), fmt), mx.quantize(_rows(n, 320, 2).to(DEV), fmt)
        _check_product(a, b, torch.ones(n, device=DEV), dtype)
        _check_product(a, b, None, dtype)


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_matmul_every_scale_reaches_its_block(fmt: str) -> None:
    """Ones with one block's scale doubled per row: the row's sum says which scale was applied where."""
    block, cols, rows = oracle.BLOCK[fmt], 1024, 272
    x = torch.ones(rows, cols)
    which = torch.arange(rows) % (cols // block)
    for r in range(rows):
        x[r, which[r] * block:(which[r] + 1) * block] = 4.0
    g = {"global_scale": torch.ones(1)} if fmt == "nvfp4" else {}
    packed = mx.quantize(x, fmt, **g)
    probe = torch.zeros(cols // block, cols)
    for c in range(cols // block):
        probe[c, c * block:(c + 1) * block] = 1.0
    probe = mx.quantize(probe, fmt, **g)
    per_block = oracle.decode(packed) @ oracle.decode(probe).t()
    for a, b, ref in ((packed, probe, per_block), (probe, packed, per_block.t())):
        got = mx.matmul(a.to(DEV), b.to(DEV), out_dtype=torch.float32).cpu().double()
        assert (got - ref).abs().max() <= 1e-4 * ref.abs().max()
    _clean()


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_matmul_non_finite_rows_stay_in_their_rows(fmt: str) -> None:
    x, w = _rows(140, 300, 1), _rows(150, 300, 2)
    x[5, 7], w[131, 299] = float("nan"), float("inf")
    g = {"global_scale": torch.tensor([0.01])} if fmt == "nvfp4" else {}
    got = mx.matmul(mx.quantize(x, fmt, **g).to(DEV), mx.quantize(w, fmt, **g).to(DEV), out_dtype=torch.float32).cpu()
    bad = torch.zeros(140, 150, dtype=torch.bool)
    bad[5], bad[:, 131] = True, True
    assert torch.equal(torch.isnan(got), bad)


# one row, few rows, one tile a CTA and one tile a CTA pair
SCALED = [(1, 64, 13824), (3, 130, 64), (100, 200, 1024), (300, 20000, 520), (2400, 2100, 160)]


@pytest.mark.parametrize("shape", SCALED)
@pytest.mark.parametrize("sizes", [(1e-18, 1e-18), (3e-19, 1e-20), (1e-28, 1e-9), (1e15, 1e17), (1e-30, 1e30)])
def test_matmul_of_operands_of_any_size(shape: tuple[int, int, int], sizes: tuple[float, float]) -> None:
    """The tensor scales' product leaves fp32's range, or nearly, where the results do not."""
    m, n, k = shape
    a = mx.quantize((_rows(m, k, m + k) * sizes[0]).to(DEV), "nvfp4")
    b = mx.quantize((_rows(n, k, n) * sizes[1]).to(DEV), "nvfp4")
    _check_product(a, b, None, torch.float32)


@pytest.mark.parametrize("shape", SCALED)
def test_matmul_of_tensor_scales_whose_product_overflows(shape: tuple[int, int, int]) -> None:
    m, n, k = shape
    g, size = torch.tensor([2.0 ** 66], device=DEV), 6 * 2.0 ** -9 * 2.0 ** 66  # code 6, the smallest block scale
    x, w = torch.zeros(m, k, device=DEV), torch.full((n, k), size, device=DEV)
    x[::2, :16] = size
    got = mx.matmul(mx.quantize(x, "nvfp4", global_scale=g), mx.quantize(w, "nvfp4", global_scale=g),
                    out_dtype=torch.float32)
    assert (got[::2] == 16 * size ** 2).all() and not got[1::2].any()


@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("m", [1, 40, 300])
def test_matmul_repeats_bitwise(fmt: str, m: int) -> None:
    a, b = mx.quantize(_rows(m, 5120, 1).to(DEV), fmt), mx.quantize(_rows(640, 5120, 2).to(DEV), fmt)
    first = mx.matmul(a, b)
    for _ in range(3):
        assert torch.equal(mx.matmul(a, b), first)


def test_operators_run_on_the_current_stream_and_in_graphs() -> None:
    x, w = _rows(300, 640, 1, torch.bfloat16).to(DEV), _rows(512, 640, 2).to(DEV)
    packed = mx.quantize(w, "nvfp4")

    def step(t: torch.Tensor) -> torch.Tensor:
        _, n = mx.add_rmsnorm_mod(t, t, None, fmt="nvfp4")
        return mx.matmul(n, packed) + mx.matmul(mx.quantize(t, "nvfp4"), packed)

    want = step(x)
    side = torch.cuda.Stream()
    late = torch.zeros_like(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        got = step(late)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(late)
    late.copy_(2 * x)
    graph.replay()
    assert torch.equal(out, step(2 * x))
    _clean()


def test_device_refusals() -> None:
    x = torch.randn(4, 64, device=DEV)
    a = mx.quantize(x, "nvfp4")
    cases = [
        (lambda: mx.quantize(x.double(), "mxfp8"), "bf16, fp16 or fp32"),
        (lambda: mx.quantize(x[:, :0], "mxfp8"), "at least one column"),
        (lambda: mx.quantize(x, "nvfp4", global_scale=torch.ones(1)), "CUDA|device"),
        (lambda: mx.quantize(x, "nvfp4", global_scale=torch.ones(2, device=DEV)), "one fp32 value"),
        (lambda: mx.dequantize(a, torch.float64), "bf16, fp16 or fp32"),
        (lambda: mx.add_rmsnorm_mod(torch.ones(2, 65537, device=DEV), None, None), "at most 65536 columns"),
        (lambda: mx.dequantize(mx.MXTensor(a.codes.t().contiguous().t(), a.scales, "nvfp4", 64)), "contiguous"),
        (lambda: mx.matmul(a, a, bias=torch.ones(3, device=DEV)), "bias must be"),
        (lambda: mx.matmul(a, a, bias=torch.ones(4, device=DEV).half()), "fp32"),
        (lambda: mx.matmul(a, a, out_dtype=torch.int32), "bf16, fp16 or fp32"),
        (lambda: mx.matmul(a, a.to("cpu")), "CUDA|device"),
        (lambda: mx.add_rmsnorm_mod(x, x.half(), None), "x's shape, type and device"),
        (lambda: mx.add_rmsnorm_mod(x, x[:2], None), "x's shape, type and device"),
        (lambda: mx.add_rmsnorm_mod(x, None, torch.ones(63, device=DEV)), "weight must be"),
        (lambda: mx.add_rmsnorm_mod(x, None, None, torch.ones(1, 64, device=DEV), rows_per_batch=2), "do not cover"),
        (lambda: mx.add_rmsnorm_mod(x, None, None, torch.ones(1, 63, device=DEV)), "scale must be"),
        (lambda: mx.add_rmsnorm_mod(x, None, None, gate=torch.ones(1, 64, device=DEV)), "gate needs an update"),
        (lambda: mx.add_rmsnorm_mod(x, x, None, torch.ones(2, 64, device=DEV), gate=torch.ones(1, 64, device=DEV),
                                    rows_per_batch=4), "differ in their rows"),
        (lambda: mx.add_rmsnorm_mod(x, None, None, torch.ones(1, 64, device=DEV),
                                    groups=torch.zeros(4, device=DEV)), "int32"),
    ]
    for call, message in cases:
        with pytest.raises((RuntimeError, ValueError), match=message):
            call()
    _clean()
