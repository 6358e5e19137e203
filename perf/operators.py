"""Cases of the block-scaled ("microscaled") low-precision operators.

Three operators, each in the formats

    ======  ==================  ==========================  =====================
    name    element             block scale                 tensor scale
    ======  ==================  ==========================  =====================
    mxfp8   e4m3 (8 bits)       2^s per 32 (e8m0)           -
    mxfp4   e2m1 (4 bits)       2^s per 32 (e8m0)           -
    nvfp4   e2m1 (4 bits)       e4m3 per 16                 fp32 ``g``
    ======  ==================  ==========================  =====================

* quantise: rows of bf16 / fp16 / fp32 to codes and scales, and back to the
  values they stand for. The power-of-two scale is the smallest that saturates
  no value of its block; for nvfp4 ``g = amax(tensor) / (6 * 448)`` and a block's
  scale is ``amax(block) / (6 g)`` rounded to e4m3.
* norm: ``x' = x + gate * update`` and ``rmsnorm(x') * w * (1 + scale) + shift``
  in 8 bits (mxfp8): the residual addition and adaLN norm in front of a
  quantised linear layer.
* product: ``A[M, K] . B[N, K]^T (+ bias)`` of two quantised operands.

Quantised operands are kept as codes ``[rows, bytes]`` (columns padded to a
multiple of 32 with zero codes, two 4-bit codes to a byte, the even column in
the low half) and one flat array of scale bytes in 128 x 4 tiles: the scale of
row ``r``, block ``c`` lies in tile ``(r // 128, c // 4)`` (512 bytes, tiles of a
row group side by side) at ``(r % 32) * 16 + (r % 128) // 32 * 4 + c % 4``.

Widths are this repository's video models' (2560 with 10240 hidden units, 5120
with 13824, 768), row counts its clips' token counts.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
G_FLOOR = 2.0 ** -100  # the tensor scale of an all-zero tensor


def listed() -> list[dict]:
    return [
        # one sample's conditioning row on its way into the modulation layer: latency only
        {"name": "quantise row nvfp4", "op": "quantise", "fmt": "nvfp4", "rows": 1, "cols": 2560, "dtype": "bf16"},
        # a 64k-token clip's activations in front of an attention or MLP projection
        {"name": "quantise clip nvfp4", "op": "quantise", "fmt": "nvfp4", "rows": 65536, "cols": 2560, "dtype": "bf16"},
        # fp32 master weights of the wide model's MLP, quantised when a model is loaded
        {"name": "quantise weight mxfp4", "op": "quantise", "fmt": "mxfp4", "rows": 13824, "cols": 5120,
         "dtype": "fp32"},
        # rows and columns of no particular alignment
        {"name": "quantise odd mxfp8", "op": "quantise", "fmt": "mxfp8", "rows": 4099, "cols": 1537, "dtype": "fp16"},
        # a few tokens: a short audio stream or the last sampling step's preview
        {"name": "norm few mxfp8", "op": "norm", "fmt": "mxfp8", "rows": 16, "cols": 2560, "levels": 1, "gated": True},
        # a 64k-token clip with two noise levels (conditioned frames beside noisy ones)
        {"name": "norm clip mxfp8", "op": "norm", "fmt": "mxfp8", "rows": 65536, "cols": 2560, "levels": 2,
         "gated": True},
        # the wide model's un-modulated norm in front of cross-attention, ragged row count
        {"name": "norm wide mxfp8", "op": "norm", "fmt": "mxfp8", "rows": 16387, "cols": 5120, "levels": 0,
         "gated": False},
        # the modulation layer: one conditioning row against 6 x 2560 outputs
        {"name": "product row nvfp4", "op": "product", "fmt": "nvfp4", "m": 1, "n": 15360, "k": 2560, "bias": True,
         "dtype": "bf16"},
        # the MLP's gate and up projections over a 64k-token clip
        {"name": "product gate-up nvfp4", "op": "product", "fmt": "nvfp4", "m": 65536, "n": 20480, "k": 2560,
         "bias": False, "dtype": "bf16"},
        # the MLP's down projection over a 16k-token clip
        {"name": "product down mxfp4", "op": "product", "fmt": "mxfp4", "m": 16384, "n": 2560, "k": 10240,
         "bias": False, "dtype": "bf16"},
        # the wide model's attention output projection
        {"name": "product out mxfp8", "op": "product", "fmt": "mxfp8", "m": 32768, "n": 5120, "k": 5120,
         "bias": False, "dtype": "bf16"},
        # text tokens of two prompts into the model's width, sizes of no alignment, half-precision out
        {"name": "product odd mxfp8", "op": "product", "fmt": "mxfp8", "m": 925, "n": 2567, "k": 4090, "bias": True,
         "dtype": "fp16"},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    if rng.random() < 0.5 and v >= 64:  # half of the sizes are aligned as a model's are
        v -= v % 64
    return v if v != 3072 else 2880


def draw(rng: random.Random) -> dict:
    op = rng.choice(["quantise", "norm", "product"])
    if op == "quantise":
        fmt = rng.choice(["mxfp8", "mxfp4", "nvfp4"])
        cols = _log_int(rng, 64, 13824)
        return {"op": op, "fmt": fmt, "rows": _log_int(rng, 1, min(65536, 100_000_000 // cols)), "cols": cols,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "norm":
        cols = _log_int(rng, 256, 8192)
        rows = _log_int(rng, 1, min(65536, 100_000_000 // cols))
        levels = rng.choice([0, 1, 2, 5])
        return {"op": op, "fmt": "mxfp8", "rows": rows, "cols": cols, "levels": levels,
                "gated": levels > 0 and rng.random() < 0.7}
    fmt = rng.choice(["mxfp8", "mxfp4", "nvfp4"])
    n, k = _log_int(rng, 256, 20480), _log_int(rng, 256, 13824)
    m = _log_int(rng, 1, max(1, min(65536, int(2.5e12 / n / k))))
    return {"op": op, "fmt": fmt, "m": m, "n": n, "k": k, "bias": rng.random() < 0.3,
            "dtype": rng.choice(["bf16", "bf16", "fp16"])}


def _packed_bytes(fmt: str, rows: int, cols: int) -> float:
    bits = 8 if fmt == "mxfp8" else 4
    return rows * cols * bits / 8 + rows * math.ceil(cols / BLOCK[fmt])


def work(case: dict) -> dict:
    if case["op"] == "quantise":
        # the input once, the packed tensor written and read back, the values once
        n, size = case["rows"] * case["cols"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * size + 2 * _packed_bytes(case["fmt"], case["rows"], case["cols"]) + 2 * n, "flops": 4 * n}
    if case["op"] == "norm":
        # x and the update once, x' once, the packed rows written and read back, the values once
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * 3 * n + 2 * _packed_bytes(case["fmt"], case["rows"], case["cols"]) + 2 * n,
                "flops": 12 * n}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": _packed_bytes(case["fmt"], m, k) + _packed_bytes(case["fmt"], n, k) + 2 * m * n,
            "flops": 2 * m * n * k}


# ----------------------------------------------------------------------------- plain forms
def _pow2(s: torch.Tensor) -> torch.Tensor:
    """``2^s`` in fp32 for whole ``s`` in [-126, 127], from its bits."""
    return ((s + 127) << 23).to(torch.int32).view(torch.float32)


def _e2m1(v: torch.Tensor) -> torch.Tensor:
    """Nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), saturating."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.where(v < 0, -1.0, 1.0) * (torch.round(a / step) * step).clamp(max=6.0)


def _e4m3(v: torch.Tensor) -> torch.Tensor:
    return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()


def _blocks(x: torch.Tensor, block: int) -> torch.Tensor:
    """fp32 ``[rows, blocks, block]`` with the columns padded with zeros to a multiple of 32."""
    rows, cols = x.shape
    pad = -(-cols // 32) * 32
    if pad == cols:
        return x.float().view(rows, pad // block, block)
    v = torch.zeros(rows, pad, device=x.device)
    v[:, :cols] = x
    return v.view(rows, pad // block, block)


def _quantise(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Element values ``[rows, blocks, block]``, block scales ``[rows, blocks]`` and the tensor scale."""
    v = _blocks(x, BLOCK[fmt])
    amax = v.abs().amax(-1)
    if fmt == "nvfp4":
        g = (amax.amax() / 2688.0).clamp(min=G_FLOOR)
        s = _e4m3(amax / (6.0 * g))
        inv = torch.where(s > 0, 1.0 / (s * g), 0.0)
        return _e2m1(v * inv[..., None]), s, g
    m, e = torch.frexp(amax)
    top, bits = (0.875, 9) if fmt == "mxfp8" else (0.75, 3)
    s = torch.where(m <= top, e - bits, e - bits + 1)
    s = torch.where(amax > 0, s, -126).clamp(-126, 127)
    q = v * _pow2(-s)[..., None]
    return (_e4m3(q) if fmt == "mxfp8" else _e2m1(q)), _pow2(s), None


def _values(q: torch.Tensor, s: torch.Tensor, g: torch.Tensor | None, cols: int, dtype: torch.dtype) -> torch.Tensor:
    out = q * s[..., None]
    if g is not None:
        out = out * g
    return out.flatten(1)[:, :cols].to(dtype).contiguous()


def _decode(state: dict, which: str) -> torch.Tensor:
    """fp32 values of a stored operand."""
    fmt, codes, rows, cols = state["fmt"], state[which + "_codes"], state[which + "_rows"], state["cols"]
    if fmt == "mxfp8":
        q = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        table = torch.cat((table, -table))
        q = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(1)
    blocks = q.shape[1] // BLOCK[fmt]
    tiles = -(-blocks // 4)
    raw = state[which + "_scales"].view(-1, tiles, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, 4 * tiles)
    raw = raw[:rows, :blocks]
    s = raw.contiguous().view(torch.float8_e4m3fn).float() if fmt == "nvfp4" else _pow2(raw.int() - 127)
    v = (q.view(rows, blocks, BLOCK[fmt]) * s[..., None]).flatten(1)[:, :cols]
    return v if state[which + "_g"] is None else v * state[which + "_g"]


# ----------------------------------------------------------------------------- inputs
def _store(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Codes, scale bytes and tensor scale of ``x`` as a program keeps them."""
    q, s, g = _quantise(x, fmt)
    rows, blocks = s.shape
    if fmt == "mxfp8":
        codes = q.flatten(1).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = q.abs().flatten(1)
        c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
        c = c | ((q.flatten(1) < 0).to(torch.uint8) << 3)
        codes = c[:, 0::2] | (c[:, 1::2] << 4)
    if fmt == "nvfp4":
        raw = s.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        raw = ((s.view(torch.int32) >> 23) & 255).to(torch.uint8)
    full = torch.zeros(-(-rows // 128) * 128, -(-blocks // 4) * 4, dtype=torch.uint8, device=x.device)
    full[:rows, :blocks] = raw
    tiled = full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    return codes.contiguous(), tiled.contiguous(), None if g is None else g.reshape(1)


def _activations(gen: torch.Generator, rows: int, cols: int) -> torch.Tensor:
    """Activations of a transformer: normal, channels of unequal size, a few large ones."""
    size = torch.exp(0.5 * torch.randn(cols, generator=gen, device=DEV))
    size[torch.randint(0, cols, (max(1, cols // 256),), generator=gen, device=DEV)] *= 8.0
    return torch.randn(rows, cols, generator=gen, device=DEV) * size


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case)
    if case["op"] == "quantise":
        state["x"] = _activations(gen, case["rows"], case["cols"]).to(DTYPES[case["dtype"]])
    elif case["op"] == "norm":
        rows, cols, levels = case["rows"], case["cols"], case["levels"]
        state["x"] = _activations(gen, rows, cols).bfloat16()
        state["update"] = (0.5 * _activations(gen, rows, cols)).bfloat16()
        state["weight"] = 1.0 + 0.1 * torch.randn(cols, generator=gen, device=DEV)
        state["scale"] = state["shift"] = state["gate"] = state["groups"] = None
        if levels:
            state["scale"] = 0.3 * torch.randn(levels, cols, generator=gen, device=DEV)
            state["shift"] = 0.3 * torch.randn(levels, cols, generator=gen, device=DEV)
            state["groups"] = torch.randint(0, levels, (rows,), generator=gen, device=DEV, dtype=torch.int32)
            if case["gated"]:
                state["gate"] = 0.5 * torch.randn(levels, cols, generator=gen, device=DEV)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        state.update(cols=k, a_rows=m, b_rows=n)
        state["a_codes"], state["a_scales"], state["a_g"] = _store(_activations(gen, m, k).bfloat16(), case["fmt"])
        weight = torch.randn(n, k, generator=gen, device=DEV) / math.sqrt(k)
        state["b_codes"], state["b_scales"], state["b_g"] = _store(weight, case["fmt"])
        state["bias_row"] = torch.randn(n, generator=gen, device=DEV) if case["bias"] else None
    return state


# ----------------------------------------------------------------------------- one pass
def run(state: dict) -> dict:
    return _run_own(state) if own else _run_plain(state)


def _run_plain(state: dict) -> dict:
    if state["op"] == "quantise":
        return {"values": _values(*_quantise(state["x"], state["fmt"]), state["cols"], torch.bfloat16)}
    if state["op"] == "norm":
        rows = state["groups"].long() if state["groups"] is not None else None
        update = state["update"].float()
        if state["gate"] is not None:
            update = update * state["gate"][rows]
        x = state["x"].float() + update
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * state["weight"]
        if rows is not None:
            y = y * (1.0 + state["scale"][rows]) + state["shift"][rows]
        return {"x": x.bfloat16(),
                "values": _values(*_quantise(y, state["fmt"]), state["cols"], torch.bfloat16)}
    out = _decode(state, "a") @ _decode(state, "b").t()
    if state["bias_row"] is not None:
        out = out + state["bias_row"]
    return {"out": out.to(DTYPES[state["dtype"]])}


def _run_own(state: dict) -> dict:
    from avgen_b200.ops import microscale as mx

    if state["op"] == "quantise":
        return {"values": mx.dequantize(mx.quantize(state["x"], state["fmt"]))}
    if state["op"] == "norm":
        x, y = mx.add_rmsnorm_mod(state["x"], state["update"], state["weight"], state["scale"], state["shift"],
                                  gate=state["gate"], groups=state["groups"], eps=1e-6, fmt=state["fmt"])
        return {"x": x, "values": mx.dequantize(y)}
    a = mx.MXTensor(state["a_codes"], state["a_scales"], state["fmt"], state["cols"], state["a_g"])
    b = mx.MXTensor(state["b_codes"], state["b_scales"], state["fmt"], state["cols"], state["b_g"])
    return {"out": mx.matmul(a, b, bias=state["bias_row"], out_dtype=DTYPES[state["dtype"]])}


# ----------------------------------------------------------------------------- in 64 bits
def _round64(v: torch.Tensor, mantissa: int, least: int, top: float) -> torch.Tensor:
    """Nearest number with ``mantissa`` fraction bits and exponents from ``least`` up, at most ``top``."""
    a = v.abs()
    exponent = torch.frexp(a).exponent - 1
    unit = torch.pow(2.0, (exponent.clamp(min=least) - mantissa).double())
    return torch.sign(v) * (torch.round(a / unit) * unit).clamp(max=top)


def _quantised64(v: torch.Tensor, fmt: str, limit: torch.Tensor | None) -> torch.Tensor:
    """What ``[rows, cols]`` in 64 bits stands for after quantising; ``limit``: the whole tensor's largest value."""
    rows, cols = v.shape
    block = BLOCK[fmt]
    padded = torch.nn.functional.pad(v, (0, -cols % block)).view(rows, -1, block)
    largest = padded.abs().amax(-1, keepdim=True)
    if fmt == "nvfp4":
        g = torch.clamp(limit / (6 * 448), min=G_FLOOR)
        scale = _round64(largest / 6 / g, 3, -6, 448.0) * g
    else:
        top = 448.0 if fmt == "mxfp8" else 6.0
        s = torch.ceil(torch.log2(largest / top)).clamp(min=-126)
        s = torch.where(largest > top * torch.pow(2.0, s), s + 1, s)  # log2 may be off by a rounding
        s = torch.where((largest <= top * torch.pow(2.0, s - 1)) & (s > -126), s - 1, s)
        scale = torch.pow(2.0, s)
    ratio = torch.where(scale > 0, padded / scale, torch.zeros_like(padded))
    q = _round64(ratio, 3, -6, 448.0) if fmt == "mxfp8" else _round64(ratio, 1, 0, 6.0)
    return (q * scale).view(rows, -1)[:, :cols]


def _operand64(state: dict, which: str) -> torch.Tensor:
    fmt, rows = state["fmt"], state[which + "_rows"]
    byte = state[which + "_codes"].long()
    if fmt == "mxfp8":
        e, f, sign = (byte >> 3) & 15, byte & 7, byte >> 7
        q = torch.where(e > 0, (8 + f) * torch.pow(2.0, (e - 10).double()), f * 2.0 ** -9)
    else:
        c = torch.stack((byte % 16, byte // 16), 2).view(rows, -1)
        e, f, sign = (c >> 1) & 3, c & 1, c >> 3
        q = torch.where(e > 0, (2 + f) * torch.pow(2.0, (e - 2).double()), f * 0.5)
    q = q * (1 - 2 * sign)
    count = q.shape[1] // BLOCK[fmt]
    tiles = -(-count // 4)
    r = torch.arange(rows, device=q.device)[:, None]
    c = torch.arange(count, device=q.device)[None, :]
    at = (r // 128 * tiles + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4
    s = state[which + "_scales"][at].long()
    if fmt == "nvfp4":
        e, f = s >> 3, s & 7
        scale = torch.where(e > 0, (8 + f) * torch.pow(2.0, (e - 10).double()), f * 2.0 ** -9)
        scale = scale * state[which + "_g"].double()
    else:
        scale = torch.pow(2.0, (s - 127).double())
    return (q.view(rows, count, -1) * scale[..., None]).view(rows, -1)[:, :state["cols"]]


def exact(case: dict, seed: int) -> dict:
    state = prepare(case, seed)
    if case["op"] == "product":
        a, b = _operand64(state, "a"), _operand64(state, "b")
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device=DEV)
        for i in range(0, case["m"], 8192):
            torch.mm(a[i:i + 8192], b.t(), out=out[i:i + 8192])
        if case["bias"]:
            out += state["bias_row"].double()
        return {"out": out}
    rows = case["rows"]
    values = torch.empty(rows, case["cols"], dtype=torch.float64, device=DEV)
    if case["op"] == "quantise":
        limit = state["x"].double().abs().max()
        for i in range(0, rows, 8192):
            values[i:i + 8192] = _quantised64(state["x"][i:i + 8192].double(), case["fmt"], limit)
        return {"values": values}
    x = torch.empty_like(values)
    for i in range(0, rows, 8192):
        at = slice(i, i + 8192)
        part = state["update"][at].double()
        level = None if state["groups"] is None else state["groups"][at].long()
        if state["gate"] is not None:
            part = part * state["gate"].double()[level]
        x[at] = state["x"][at].double() + part
        y = x[at] / torch.sqrt(x[at].square().mean(1, keepdim=True) + 1e-6) * state["weight"].double()
        if level is not None:
            y = y * (1 + state["scale"].double()[level]) + state["shift"].double()[level]
        values[at] = _quantised64(y, case["fmt"], None)
    return {"x": x, "values": values}
