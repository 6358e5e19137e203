"""DiT blocks with block-scaled 8- or 4-bit linears, for sampling and evaluation.

:func:`quantize_model` packs the weights of every DiT block once; from then on a block
runs

    n1  = rmsnorm(x) * w_a * (1 + scale_a) + shift_a, packed         add_rmsnorm_mod
    qkv = n1 @ Wqkv^T                                                block-scaled product
    O   = attention(rope(qknorm(qkv)))                               the fused block's kernels
    x1  = x + gate_a * (pack(O) @ Wo^T);  n2 = rmsnorm(x1), packed   product, add_rmsnorm_mod
    x2  = x1 + cross_attention(n2, text); n3 = rmsnorm(x2) ..., packed
    x3  = x2 + gate_f * (pack(act(n3 @ Wup^T)) @ Wdown^T)

so every activation a linear reads is written packed by the operator before it, and each
residual addition rides in the norm that follows it. Embeddings, modulation, time and text
projections and the output head stay in bf16: they are small, and precision-sensitive.

The blocks keep their own weights (checkpoints, adapters and training are not touched);
:func:`restore_model` drops the packed ones. A quantised block has no gradient and refuses
to run while gradients are recorded, and under context or head-parallel tensor parallelism,
which leave a rank with part of the tokens or heads, whether they were applied before or
after packing. On the CPU the same code runs the operators' PyTorch
restatement. The reference framework has no counterpart: its only low-precision option is
a third-party package's fp8 training (avgen/parallel/precision.py:212-284).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch import nn

from avgen_b200.models.attention import attention
from avgen_b200.models.rope import RotaryTables, apply_rotary
from avgen_b200.ops import microscale as mx

_NVFP4_RANGE = 6.0 * 448.0  # largest e2m1 times largest e4m3

__all__ = ["QuantizedBlock", "quantize_model", "quantized_block_forward", "restore_model"]


@dataclass(frozen=True)
class QuantizedBlock:
    """The packed weights of one DiT block (``up`` holds gate and up rows for SwiGLU)."""

    fmt: str
    qkv: mx.MXTensor
    out: mx.MXTensor
    up: mx.MXTensor
    down: mx.MXTensor
    cross_q: mx.MXTensor | None = None
    cross_kv: mx.MXTensor | None = None
    cross_out: mx.MXTensor | None = None
    # nvfp4: tensor scales that hold the whole range of the norms' output, [2] before modulation
    # (self-attention's and the MLP's) and [1] of cross-attention's; None for the other formats
    norm_scales: torch.Tensor | None = None
    cross_scale: torch.Tensor | None = None

    @property
    def nbytes(self) -> int:
        parts = (self.qkv, self.out, self.up, self.down, self.cross_q, self.cross_kv, self.cross_out)
        return sum(p.nbytes for p in parts if p is not None)


def _split_by(block: nn.Module) -> str | None:
    """The parallelism that spreads the block's heads or tokens over ranks, if any."""
    if block.attention_impl is not None or block.attention.cp_mesh is not None:
        return "context parallelism"
    parts = (block, block.attention, block.cross_attention, block.feed_forward)
    if any(getattr(m, "tp", None) is not None for m in parts):
        return "head-parallel tensor parallelism"
    return None


def _check(block: nn.Module, name: str) -> None:
    from torch.distributed.tensor import DTensor

    linears = {n: m for n, m in block.named_modules() if isinstance(m, nn.Linear)}
    split = _split_by(block)
    if split is not None:
        raise ValueError(f"{name}: a quantised block takes whole heads and sequences, it does not run under {split}")
    if any(isinstance(m.weight, DTensor) for m in linears.values()):
        raise ValueError(f"{name}: sharded weights cannot be quantised; quantise before sharding or gather first")
    biased = [n for n, m in linears.items() if m.bias is not None]
    if biased:
        raise ValueError(f"{name}: quantised linears have no bias; found {', '.join(biased)}")


def _weight(layer: nn.Linear) -> torch.Tensor:
    """The layer's weight, adapters included."""
    adapted = getattr(layer, "adapted_weight", None)
    return (adapted() if callable(adapted) else layer.weight).detach()


def _norm_scale(norm: nn.Module, width: int, device: torch.device) -> torch.Tensor:
    """The nvfp4 tensor scale of a norm's output before modulation: no normalised value is
    above sqrt(width), and the largest a tensor scale g can hold is 2688 g."""
    w = _norm_weight(norm)
    gain = torch.ones(1, device=device) if w is None else w.abs().amax().reshape(1)
    return (gain * (math.sqrt(width) / _NVFP4_RANGE)).clamp(min=2.0 ** -100)


def _modulated_scales(combined: torch.Tensor, p: QuantizedBlock) -> tuple[torch.Tensor, torch.Tensor]:
    """Tensor scales of the two modulated norms, from the largest shift and 1 + |scale| of the
    call: |y| <= 2688 g (1 + |scale|) + |shift|, so nothing saturates, and blocks down to
    1 / 28000 of that bound keep normal scales. A modulation that is not finite (its rows are
    NaN in any case) counts as 2, so that other rows stay what they are."""
    if len(combined) == 0:
        return p.norm_scales[:1], p.norm_scales[1:]
    peak = torch.linalg.vector_norm(combined, float("inf"), dim=(0, 2)).nan_to_num(nan=2.0, posinf=2.0)  # [6]
    g = torch.addcmul(p.norm_scales, p.norm_scales, peak[1::3]).add_(peak[0::3], alpha=1.0 / _NVFP4_RANGE)
    return g[:1], g[1:]


def _pack(fmt: str, *layers: nn.Linear) -> mx.MXTensor:
    w = [_weight(layer) for layer in layers]
    return mx.quantize(w[0] if len(w) == 1 else torch.cat(w, 0), fmt)


def quantize_model(model: nn.Module, fmt: str = "mxfp8") -> int:
    """Pack the linears of every DiT block of ``model`` in ``fmt`` (``mxfp8``, ``mxfp4`` or
    ``nvfp4``), on the device they are on; returns how many blocks. Call it again after the
    weights change or move."""
    from avgen_b200.models.blocks import DiTBlock

    mx.block_size(fmt)  # raises on an unknown format
    blocks = {n: m for n, m in model.named_modules() if isinstance(m, DiTBlock)}
    for name, block in blocks.items():
        _check(block, name or type(block).__name__)
    with torch.no_grad():
        for block in blocks.values():
            att, ff, ca = block.attention, block.feed_forward, block.cross_attention
            up = (ff.gate_proj, ff.up_proj) if hasattr(ff, "gate_proj") else (ff.up_proj,)
            more = {}
            if ca is not None:
                more = {"cross_q": _pack(fmt, ca.q_proj), "cross_kv": _pack(fmt, ca.k_proj, ca.v_proj),
                        "cross_out": _pack(fmt, ca.out_proj)}
            if fmt == "nvfp4":
                device = att.q_proj.weight.device
                more["norm_scales"] = torch.cat([_norm_scale(n, block.width, device)
                                                 for n in (block.attention_norm, block.ffn_norm)])
                if ca is not None:
                    more["cross_scale"] = _norm_scale(block.cross_norm, block.width, device)
            block.quantized = QuantizedBlock(fmt, qkv=_pack(fmt, att.q_proj, att.k_proj, att.v_proj),
                                             out=_pack(fmt, att.out_proj), up=_pack(fmt, *up),
                                             down=_pack(fmt, ff.down_proj), **more)
    return len(blocks)


def restore_model(model: nn.Module) -> int:
    """Drop the packed weights: blocks run their own again. Returns how many had them."""
    from avgen_b200.models.blocks import DiTBlock

    found = [m for m in model.modules() if isinstance(m, DiTBlock) and m.quantized is not None]
    for block in found:
        block.quantized = None
    return len(found)


def _norm_weight(norm: nn.Module) -> torch.Tensor | None:
    w = getattr(norm, "weight", None)
    return None if w is None else w.detach().float().contiguous()


def _on_kernels(t: torch.Tensor, head_dim: int) -> bool:
    """Whether heads run on the fused block's kernels; any other head dim takes what the plain
    block's layers take, which on a GPU is :func:`attention`'s refusal."""
    return t.is_cuda and head_dim == 128


def _heads(rows: torch.Tensor, batch: int, heads: int, norm: nn.Module) -> torch.Tensor:
    """``[B*L, H*D]`` rows -> ``[B, H, L, D]``, normalised per head."""
    return norm(rows.view(batch, -1, heads, rows.shape[-1] // heads).transpose(1, 2))


def _split_heads(module: nn.Module, rows: torch.Tensor, batch: int, heads: int, kv_heads: int, rope,  # noqa: ANN001
                 eps: float) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Query, key and value heads ``[B, H, L, D]`` of packed projection rows (either may have none)."""
    coords = freq = axis = tables = None
    kernels = _on_kernels(rows, module.head_dim)
    if isinstance(rope, RotaryTables):
        tables = rope
    elif rope is not None:
        if kernels:  # the kernel forms the angles itself
            coords, freq, axis = rope.kernel_args()
        else:
            tables = rope.tables()
    d = module.head_dim
    if kernels:
        from avgen_b200.ops import kernels as K

        normed = isinstance(module.q_norm, nn.RMSNorm)
        q, k, v = K.qkv_rope(rows, batch=batch, length=rows.shape[0] // batch, heads=heads, kv_heads=kv_heads,
                             head_dim=d, q_weight=_norm_weight(module.q_norm) if normed and heads else None,
                             k_weight=_norm_weight(module.k_norm) if normed and kv_heads else None, coords=coords,
                             freq=freq, axis=axis, eps=eps)
    else:
        q, k, v = rows.split((heads * d, kv_heads * d, kv_heads * d), -1)
        q = _heads(q, batch, heads, module.q_norm) if heads else None
        k = _heads(k, batch, kv_heads, module.k_norm) if kv_heads else None
        v = _heads(v, batch, kv_heads, nn.Identity()) if kv_heads else None
    if tables is not None:
        q, k = apply_rotary(q, tables), apply_rotary(k, tables)
    return q, k, v


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: torch.Tensor | None) -> torch.Tensor:
    """Token-major attention output as rows ``[B*L, H*D]``."""
    if _on_kernels(q, q.shape[-1]):
        from avgen_b200.ops import kernels as K

        out, _ = K.attention_fwd(q, k, v, kmask=K.pack_key_mask(mask), scale=1.0 / math.sqrt(q.shape[-1]),
                                 want_lse=False)
    else:
        out = attention(q, k, v, key_mask=mask, layout="blhd")
    return out.reshape(-1, out.shape[-2] * out.shape[-1])


def quantized_block_forward(block: nn.Module, hidden: torch.Tensor, combined: torch.Tensor, *, rope,  # noqa: ANN001
                            key_mask: torch.Tensor | None, context: torch.Tensor | None,
                            context_mask: torch.Tensor | None, mod_index: torch.Tensor | None) -> torch.Tensor:
    """One block on its packed weights; arguments as the fused block takes them (``combined``:
    modulation rows with the block's table added, picked per token by ``mod_index``)."""
    if torch.is_grad_enabled():
        raise RuntimeError("a quantised block has no gradient; run it under torch.no_grad() or call restore_model "
                           "first")
    split = _split_by(block)
    if split is not None:  # set after packing: this rank's share alone would be attended to
        raise RuntimeError(f"a quantised block does not run under {split}; call restore_model first")
    p = block.quantized
    if p.qkv.device != hidden.device:
        raise RuntimeError(f"packed weights are on {p.qkv.device}, the input on {hidden.device}: call quantize_model "
                           "after moving the model")
    b, length, w = hidden.shape
    fmt, eps = p.fmt, block.attention_norm.eps or 1e-6
    groups, per = None, length
    if mod_index is not None:
        groups = mod_index.expand(b, length).reshape(-1).to(torch.int32).contiguous()
    elif combined.ndim == 4:
        combined, per = combined.expand(b, length, *combined.shape[2:]).reshape(b * length, *combined.shape[2:]), 1
    else:
        combined = combined.expand(b, *combined.shape[1:])
    rows = {"rows_per_batch": per, "groups": groups}
    combined = combined.float().contiguous()
    shift_a, scale_a, gate_a, shift_f, scale_f, gate_f = combined.unbind(1)
    g_a = g_f = None
    if p.norm_scales is not None:
        g_a, g_f = _modulated_scales(combined, p)
    x = hidden.reshape(b * length, w)
    if x.is_cuda:
        x = x.to(torch.bfloat16)  # the fused block's residual stream, whatever type comes in
    att, ca = block.attention, block.cross_attention

    _, n = mx.add_rmsnorm_mod(x, None, _norm_weight(block.attention_norm), scale_a, shift_a, **rows, eps=eps, fmt=fmt,
                             global_scale=g_a)
    q, k, v = _split_heads(att, mx.matmul(n, p.qkv, out_dtype=x.dtype), b, att.num_heads, att.num_kv_heads, rope, eps)
    update = mx.matmul(mx.quantize(_attend(q, k, v, key_mask), fmt), p.out, out_dtype=x.dtype)
    gate = gate_a
    if ca is not None and context is not None and context.shape[1] > 0:
        x, n = mx.add_rmsnorm_mod(x, update, _norm_weight(block.cross_norm), gate=gate_a, **rows,
                                  eps=block.cross_norm.eps or eps, fmt=fmt, global_scale=p.cross_scale)
        text = mx.quantize(context.to(x.dtype).reshape(-1, context.shape[-1]), fmt)
        q, _, _ = _split_heads(ca, mx.matmul(n, p.cross_q, out_dtype=x.dtype), b, ca.num_heads, 0, None, eps)
        _, k, v = _split_heads(ca, mx.matmul(text, p.cross_kv, out_dtype=x.dtype), b, 0, ca.num_kv_heads, None, eps)
        update = mx.matmul(mx.quantize(_attend(q, k, v, context_mask), fmt), p.cross_out, out_dtype=x.dtype)
        gate = None
    x, n = mx.add_rmsnorm_mod(x, update, _norm_weight(block.ffn_norm), scale_f, shift_f, gate=gate, **rows,
                              eps=block.ffn_norm.eps or eps, fmt=fmt, global_scale=g_f)
    h = mx.matmul(n, p.up, out_dtype=x.dtype)
    if hasattr(block.feed_forward, "gate_proj"):
        gated, up = h.chunk(2, -1)
        h = F.silu(gated) * up
    else:
        h = F.gelu(h, approximate="tanh")
    update = mx.matmul(mx.quantize(h, fmt), p.down, out_dtype=x.dtype).float()
    if groups is not None:
        out = torch.addcmul(x.float(), gate_f[groups.long()], update)
    else:
        out = torch.addcmul(x.float().view(-1, per, w), gate_f[:, None], update.view(-1, per, w))
    return out.to(x.dtype).to(hidden.dtype).view(b, length, w)
