"""Quantised DiT blocks: against the same block with each linear's operands rounded to the
format, and against the unquantised block; what quantising refuses and leaves alone."""
from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

import microscale_oracle as oracle
from avgen_b200.models import DiTBlock, RopeInputs, RotaryEmbedding, quantize_model, restore_model
from avgen_b200.ops import microscale as mx

# The error a format may add to a block's output, relative to its norm. An element is off by
# at most half a spacing: a relative 2^-4 in e4m3 (rms about 2^-4 / sqrt(3) = 0.036 / 2) and
# 2^-2 in e2m1 (rms 0.14 / 2); seven products in a row, each with two rounded operands whose
# errors add as squares, and a residual stream that carries most of the output.
BOUND = {"mxfp8": 0.036 / 2 * 14 ** 0.5, "mxfp4": 0.14 * 14 ** 0.5 / 2, "nvfp4": 0.14 * 14 ** 0.5 / 2}


def _block(width: int = 256, heads: int = 2, **more: object) -> DiTBlock:
    block = DiTBlock(width, heads, hidden=2 * width, **more)
    block.init_weights(depth=2)
    with torch.no_grad():
        for p in block.parameters():
            p.add_(0.02 * torch.randn_like(p))
    return block


def _inputs(form: str, device: str = "cpu", dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, dict]:
    b, length, width = 2, 160, 256
    rope = RopeInputs((torch.rand(b, length, 3) * 8).to(device), RotaryEmbedding(128))
    index = None
    if form == "grouped":
        mod = 0.1 * torch.randn(2 * b, 6, width)
        index = (torch.arange(b)[:, None] * 2 + (torch.arange(length) < 40).long()[None]).int().to(device)
    elif form == "token":
        mod = 0.1 * torch.randn(b, length, 6, width)
    else:
        mod = 0.1 * torch.randn(b, 6, width)
    key = torch.ones(b, length, dtype=torch.bool)
    key[0, 120:] = False
    text = torch.ones(b, 24, dtype=torch.bool)
    text[1, 20:] = False
    kwargs = {"modulation": mod.to(device), "rope": rope, "key_mask": key.to(device), "modulation_index": index,
              "context": torch.randn(b, 24, width).to(device, dtype), "context_mask": text.to(device)}
    return torch.randn(b, length, width).to(device, dtype), kwargs


def _rounded_block(block: DiTBlock, fmt: str, monkeypatch: pytest.MonkeyPatch) -> None:
    """Every linear of the eager block multiplies rounded operands (mxfp8 and mxfp4: no tensor scale to share)."""
    from avgen_b200.models import layers

    def rounded(x: torch.Tensor, layer: nn.Linear) -> torch.Tensor:
        w = mx.dequantize(mx.quantize(layer.weight.detach(), fmt), torch.float32)
        xq = mx.dequantize(mx.quantize(x.reshape(-1, x.shape[-1]), fmt), torch.float32)
        return (xq @ w.t()).view(*x.shape[:-1], -1)

    monkeypatch.setattr(layers, "linear", rounded)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("ffn,form", [("swiglu", "sample"), ("gelu", "grouped"), ("swiglu", "token")])
def test_block_is_the_eager_block_on_rounded_operands(fmt: str, ffn: str, form: str,
                                                      monkeypatch: pytest.MonkeyPatch) -> None:
    torch.manual_seed(0)
    block = _block(ffn=ffn)
    hidden, kwargs = _inputs(form)
    with torch.no_grad():
        assert quantize_model(block, fmt) == 1
        got = block(hidden, **kwargs)
        restore_model(block)
        _rounded_block(block, fmt, monkeypatch)
        want = block(hidden, **kwargs)
    # the same rounding at every linear; fp32 sums in another order move single elements across
    # a rounding boundary, a spacing each, in few places
    assert float((got - want).norm() / want.norm()) < 2e-3


@pytest.mark.parametrize("fmt", mx.FORMATS)
def test_block_stays_near_the_unquantised_block(fmt: str) -> None:
    torch.manual_seed(1)
    block = _block()
    hidden, kwargs = _inputs("grouped")
    with torch.no_grad():
        want = block(hidden, **kwargs)
        quantize_model(block, fmt)
        got = block(hidden, **kwargs)
        assert 0 < float((got - want).norm() / want.norm()) < BOUND[fmt]
        assert restore_model(block) == 1 and restore_model(block) == 0
        assert torch.equal(block(hidden, **kwargs), want)


def test_without_cross_attention_and_with_adapters() -> None:
    from avgen_b200.finetune import LoRAConfig, apply_lora

    torch.manual_seed(2)
    block = _block(cross_attention=False)
    hidden, kwargs = _inputs("sample")
    kwargs["context"] = None
    with torch.no_grad():
        quantize_model(block, "mxfp8")
        block(hidden, **kwargs)
    apply_lora(block, LoRAConfig(rank=4, target_modules=("q_proj", "up_proj")))
    with torch.no_grad():
        for name, p in block.named_parameters():
            if name.endswith("lora_b"):
                p.normal_(std=0.1)
        restore_model(block)
        want = block(hidden, **kwargs)
        quantize_model(block, "mxfp8")
        assert float((block(hidden, **kwargs) - want).norm() / want.norm()) < BOUND["mxfp8"]


def test_state_and_refusals() -> None:
    block = _block()
    keys = set(block.state_dict())
    hidden, kwargs = _inputs("sample")
    quantize_model(block, "nvfp4")
    assert set(block.state_dict()) == keys
    packed = block.quantized
    plain = sum(p.numel() for n, p in block.named_parameters() if "proj" in n)
    assert plain * 9 / 16 <= packed.nbytes <= plain * 9 / 16 * 1.01
    with pytest.raises(RuntimeError, match="no gradient"):
        block(hidden, **kwargs)
    assert copy.deepcopy(block).quantized.fmt == "nvfp4"
    with pytest.raises(ValueError, match="format must be"):
        quantize_model(block, "int4")
    other = _block()
    other.attention_impl = object()
    with pytest.raises(ValueError, match="context parallelism"):
        quantize_model(other, "mxfp8")
    biased = _block()
    biased.attention.q_proj = nn.Linear(256, 256)
    with pytest.raises(ValueError, match="no bias"):
        quantize_model(nn.ModuleList([_block(), biased]), "mxfp8")


def _only(block: DiTBlock, branch: str) -> None:
    """Silence the branches of ``block`` but one."""
    last = {"attention": block.attention.out_proj, "cross": block.cross_attention.out_proj,
            "mlp": block.feed_forward.down_proj}
    with torch.no_grad():
        for name, layer in last.items():
            if name != branch:
                layer.weight.zero_()


# What nvfp4 may add to one branch, relative to it: an element of a block whose scale is exact
# to e4m3's bits is off by an rms of 0.1 of the block's values; two products in a row (three in
# the gated MLP, whose activation doubles its input's part) with two rounded operands each
# make sqrt(6) * 0.1, and a fifth of it for what attention's weights add.
NVFP4_BRANCH = 0.1 * 6 ** 0.5 * 1.2


@pytest.mark.parametrize("branch", ["attention", "cross", "mlp"])
@pytest.mark.parametrize("gain", [1.0, 0.03, 0.002])
def test_nvfp4_norms_keep_small_gains(branch: str, gain: float) -> None:
    """Normalised rows far below 1 keep their bits, whether the norm's weight or the modulation makes them small."""
    torch.manual_seed(5)
    block = _block()
    _only(block, branch)
    hidden, kwargs = _inputs("sample")
    norm = {"attention": block.attention_norm, "cross": block.cross_norm, "mlp": block.ffn_norm}[branch]
    table = block.scale_shift_table.detach().clone()
    kwargs["modulation"][:, [0, 3]] = -table[[0, 3]]  # no shift
    kwargs["modulation"][:, [1, 4]] = -table[[1, 4]]  # 1 + scale = 1
    kwargs["modulation"][:, [2, 5]] = 1e4  # the branch well above the residual stream's own rounding
    with torch.no_grad():
        norm.weight.mul_(gain)
        small = dict(kwargs, modulation=kwargs["modulation"].clone())
        want = block(hidden, **kwargs) - hidden
        quantize_model(block, "nvfp4")
        got = block(hidden, **kwargs) - hidden
        assert float((got - want).norm() / want.norm()) < NVFP4_BRANCH
        if branch == "cross":
            return
        restore_model(block)
        norm.weight.div_(gain)
        small["modulation"][:, [1, 4]] += gain - 1
        want = block(hidden, **small) - hidden
        quantize_model(block, "nvfp4")
        got = block(hidden, **small) - hidden
        assert float((got - want).norm() / want.norm()) < NVFP4_BRANCH


@pytest.mark.parametrize("form", ["sample", "grouped", "token"])
def test_nvfp4_norms_hold_their_largest_values(form: str) -> None:
    """A channel that carries its whole row, times a large 1 + scale, plus a large shift, does not saturate."""
    torch.manual_seed(6)
    block = _block()
    _only(block, "mlp")
    hidden, kwargs = _inputs(form)
    hidden[..., 7] += 1000.0
    kwargs["modulation"][..., 4, :] += 400.0
    kwargs["modulation"][..., 3, :] += 900.0
    with torch.no_grad():
        want = block(hidden, **kwargs) - hidden
        quantize_model(block, "nvfp4")
        got = block(hidden, **kwargs) - hidden
    assert float((got - want).norm() / want.norm()) < NVFP4_BRANCH


def test_nvfp4_norm_scales_outlive_a_sample_that_is_not_finite() -> None:
    torch.manual_seed(7)
    block = _block()
    hidden, kwargs = _inputs("sample")
    quantize_model(block, "nvfp4")
    with torch.no_grad():
        for bad in (float("nan"), float("inf")):
            kwargs["modulation"][1, 1, 3] = bad
            out = block(hidden, **kwargs)
            assert torch.isfinite(out[0]).all() and not torch.isfinite(out[1]).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rotary_tables_do_what_their_coordinates_do(device: str) -> None:
    torch.manual_seed(8)
    block = _block()
    _only(block, "attention")
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    hidden, kwargs = _inputs("sample", device, dtype)
    kwargs["rope"].coords.mul_(4.0)
    kwargs["modulation"][:, 2] = 1e2
    block.to(device)
    quantize_model(block, "mxfp8")
    with torch.no_grad():
        want = (block(hidden, **kwargs) - hidden).float()
        got = (block(hidden, **dict(kwargs, rope=kwargs["rope"].tables())) - hidden).float()
        none = (block(hidden, **dict(kwargs, rope=None)) - hidden).float()
    off = float((got - want).norm() / want.norm())
    # the same numbers on the CPU; on a GPU the heads are rounded to bf16 once more before they are rotated
    assert off == 0 if device == "cpu" else off < 2 ** -5
    assert float((none - want).norm() / want.norm()) > 2 ** -2


@pytest.mark.parametrize("form", ["sample", "grouped", "token", "frame"])
def test_modulation_shared_by_the_batch(form: str) -> None:
    """Modulation (or its row numbers) of one sample stands for all, as in the plain block."""
    torch.manual_seed(11)
    block = _block()
    hidden, kwargs = _inputs("token" if form == "frame" else form)
    full = dict(kwargs)
    if form == "grouped":
        kwargs["modulation_index"] = kwargs["modulation_index"][:1]
        full["modulation_index"] = kwargs["modulation_index"].expand(2, 160).contiguous()
    else:
        one = kwargs["modulation"][:, :1] if form == "frame" else kwargs["modulation"][:1]
        full["modulation"] = one.expand_as(kwargs["modulation"]).contiguous()
        kwargs["modulation"] = one
    with torch.no_grad():
        assert torch.equal(block(hidden, **kwargs), block(hidden, **full))
        for fmt in ("mxfp8", "nvfp4"):
            quantize_model(block, fmt)
            assert torch.equal(block(hidden, **kwargs), block(hidden, **full))


# ----------------------------------------------------------------------------- every part of a block
def _marked_block(ffn: str) -> DiTBlock:
    """A block whose every part has a large share in its output."""
    block = _block(ffn=ffn)
    with torch.no_grad():
        for m in block.modules():
            if isinstance(m, nn.Linear):
                m.weight.normal_(std=m.in_features ** -0.5)
        for norm in (block.attention_norm, block.cross_norm, block.ffn_norm):
            norm.weight.uniform_(0.5, 1.5)
        for att in (block.attention, block.cross_attention):
            att.q_norm.weight.uniform_(2.0, 3.0)  # attention that looks at a few keys
            att.k_norm.weight.uniform_(0.5, 1.5)
            att.out_proj.weight.mul_(2.0)
        block.scale_shift_table.normal_(std=0.5)
    return block


class _Reference:
    """The parts of a block in 64 bits, each from the packed operands and stored rows the block itself had."""

    def __init__(self, block: DiTBlock, kwargs: dict) -> None:
        self.block, self.kwargs = block, kwargs
        mod = (kwargs["modulation"] + block.scale_shift_table.detach()).double()
        if kwargs["modulation_index"] is not None:
            mod = mod[kwargs["modulation_index"].long()]
        elif mod.ndim == 3:
            mod = mod[:, None].expand(-1, 160, -1, -1)
        self.mod = mod.reshape(320, 6, 256).unbind(1)

    def norm(self, x: torch.Tensor, norm: nn.Module, chunk: int | None) -> torch.Tensor:
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * norm.weight.detach().double()
        return y if chunk is None else y * (1 + self.mod[chunk + 1]) + self.mod[chunk]

    def attention(self, att: nn.Module, q: torch.Tensor, kv: torch.Tensor, *, rope: bool,
                  mask: torch.Tensor | None) -> torch.Tensor:
        def heads(rows: torch.Tensor, norm: nn.Module | None) -> torch.Tensor:
            t = rows.view(2, -1, 2, 128).transpose(1, 2)
            if norm is None:
                return t
            return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * norm.weight.detach().double()

        def turn(t: torch.Tensor) -> torch.Tensor:
            tables = self.kwargs["rope"].tables()
            z = torch.view_as_complex(t.reshape(*t.shape[:-1], 64, 2))
            return torch.view_as_real(z * torch.complex(tables.cos.double(), tables.sin.double())).flatten(-2)

        q, k, v = heads(q, att.q_norm), heads(kv[:, :256], att.k_norm), heads(kv[:, 256:], None)
        if rope:
            q, k = turn(q), turn(k)
        s = q @ k.transpose(-1, -2) / 128 ** 0.5
        if mask is not None:
            s = s.masked_fill(~mask[:, None, None], float("-inf"))
        return (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(320, 256)

    def activation(self, h: torch.Tensor) -> torch.Tensor:
        if hasattr(self.block.feed_forward, "gate_proj"):
            gate, up = h.chunk(2, -1)
            return nn.functional.silu(gate) * up
        return nn.functional.gelu(h, approximate="tanh")


def _tape(monkeypatch: pytest.MonkeyPatch) -> list:
    """The operators' calls of a quantised block, in order: (arguments, result)."""
    import types

    from avgen_b200.models import quantized

    calls: list = []

    def kept(name: str):  # noqa: ANN202
        def call(*args: object, **more: object) -> object:
            out = getattr(mx, name)(*args, **more)
            calls.append((args, out))
            return out

        return call

    names = ("quantize", "matmul", "add_rmsnorm_mod")
    monkeypatch.setattr(quantized, "mx", types.SimpleNamespace(**{name: kept(name) for name in names}))
    return calls


def _off(got: torch.Tensor, want: torch.Tensor) -> float:
    got = got.detach().double().cpu().reshape(want.shape)
    return float((got - want).norm() / want.norm())


# What a stage may be off, relative to its norm, from the 64-bit one on the same operands. On the
# CPU: sums of up to 512 fp32 products and their functions. On a GPU: up to five roundings to
# bf16 of 2^-9 / sqrt(3) each, of which those of q and k reach attention's scores times their
# size (2.5) and come out averaged; rows that are stored are rounded once or twice.
STAGE = {"cpu": 1e-5, "cuda": 2.0 ** -6}
STORED = {"cpu": 1e-5, "cuda": 2.0 ** -8}
# Packed values beside the packed 64-bit ones: an element that crosses a rounding boundary is a
# spacing off; fp32 arithmetic moves at most one in 10^4 there.
PACKED = 1e-2


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("ffn,form", [("swiglu", "sample"), ("gelu", "grouped"), ("swiglu", "token")])
def test_every_part_of_a_block(fmt: str, ffn: str, form: str, device: str, monkeypatch: pytest.MonkeyPatch) -> None:
    """Each stage of the block against 64 bits, within far less than any part of it (rotation, masks, each
    modulation, residuals) adds."""
    torch.manual_seed(12)
    block = _marked_block(ffn)
    hidden, kwargs = _inputs(form)
    kwargs["modulation"] = 0.5 * torch.randn_like(kwargs["modulation"])
    kwargs["modulation"][..., [2, 5], :] += 1.0
    hidden, kwargs["context"] = hidden.bfloat16().float(), kwargs["context"].bfloat16().float()
    ref = _Reference(copy.deepcopy(block), kwargs)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    block.to(device)
    quantize_model(block, fmt)
    calls = _tape(monkeypatch)
    given = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in kwargs.items()}
    given["rope"] = RopeInputs(kwargs["rope"].coords.to(device), kwargs["rope"].rope)
    given["context"] = given["context"].to(dtype)
    with torch.no_grad():
        out = block(hidden.to(device, dtype), **given)

    norm1, qkv, pack1, out1, norm2, text, cq, ckv, pack2, out2, norm3, up, pack3, down = calls
    p, ca = block.quantized, ref.block.cross_attention
    weight = {n: oracle.decode(getattr(p, n)) for n in ("qkv", "out", "cross_q", "cross_kv", "cross_out", "up", "down")}
    x = [hidden.double().view(320, 256)] + [call[1][0].double().cpu() for call in (norm2, norm3)]
    tight, stored = STAGE[device], STORED[device]

    # the packed norms
    for i, (call, norm, chunk) in enumerate(((norm1, ref.block.attention_norm, 0), (norm2, ref.block.cross_norm, None),
                                             (norm3, ref.block.ffn_norm, 3))):
        y, t = ref.norm(x[i], norm, chunk), call[1][1]
        if i > 0 and device == "cuda":  # they take the fp32 sum, of which x holds the rounding to bf16
            y = ref.norm(call[0][0].double().cpu() + call[0][1].double().cpu() * (ref.mod[2] if i == 1 else 1.0), norm,
                         chunk)
        g = None if t.global_scale is None else t.global_scale.cpu()
        assert _off(oracle.decode(t), oracle.decode(mx.quantize(y.float(), fmt, global_scale=g))) < PACKED
        if chunk is not None:
            for part in (0, 1):
                assert _off(y - ref.mod[chunk] if part == 0 else ref.norm(x[i], norm, None), y) > 0.1
    # self-attention
    rows = oracle.decode(norm1[1][1]) @ weight["qkv"].t()
    want = ref.attention(ref.block.attention, rows[:, :256], rows[:, 256:], rope=True, mask=kwargs["key_mask"])
    assert _off(pack1[0][0], want) < tight
    for rope, mask in ((False, kwargs["key_mask"]), (True, None)):
        assert _off(ref.attention(ref.block.attention, rows[:, :256], rows[:, 256:], rope=rope, mask=mask), want) > 0.1
    # its projection and gated residual
    update = oracle.decode(pack1[1]) @ weight["out"].t()
    assert _off(out1[1], update) < stored and _off(x[1], x[0] + ref.mod[2] * update) < stored
    assert _off(x[0] + update, x[1]) > 0.1
    # cross-attention, its projection and residual
    assert _off(oracle.decode(text[1]), oracle.decode(mx.quantize(kwargs["context"].view(-1, 256), fmt))) == 0
    q = oracle.decode(norm2[1][1]) @ weight["cross_q"].t()
    kv = oracle.decode(text[1]) @ weight["cross_kv"].t()
    want = ref.attention(ca, q, kv, rope=False, mask=kwargs["context_mask"])
    assert _off(pack2[0][0], want) < tight
    assert _off(ref.attention(ca, q, kv, rope=False, mask=None), want) > 0.05
    update = oracle.decode(pack2[1]) @ weight["cross_out"].t()
    assert _off(out2[1], update) < stored and _off(x[2], x[1] + update) < stored
    # the MLP and its gated residual
    assert _off(pack3[0][0], ref.activation(oracle.decode(norm3[1][1]) @ weight["up"].t())) < tight
    update = oracle.decode(pack3[1]) @ weight["down"].t()
    assert _off(down[1], update) < stored and _off(out, x[2] + ref.mod[5] * update) < stored
    assert _off(x[2] + update, out.double().cpu().view(320, 256)) > 0.1
    # nothing between the stages: each reads what the one before wrote
    for a, b in ((norm1[1][1], qkv[0][0]), (pack1[1], out1[0][0]), (out1[1], norm2[0][1]), (norm2[1][1], cq[0][0]),
                 (text[1], ckv[0][0]), (pack2[1], out2[0][0]), (out2[1], norm3[0][1]), (norm2[1][0], norm3[0][0]),
                 (norm3[1][1], up[0][0]), (pack3[1], down[0][0])):
        assert a is b


def _parallelise(block: DiTBlock, where: str) -> None:
    if where == "cp fused":
        block.attention_impl = object()
    elif where == "cp eager":
        block.attention.cp_mesh = object()
    else:
        {"tp": block, "tp attention": block.attention, "tp cross": block.cross_attention,
         "tp mlp": block.feed_forward}[where].tp = object()


@pytest.mark.parametrize("where,kind", [("cp fused", "context"), ("cp eager", "context"), ("tp", "tensor"),
                                        ("tp attention", "tensor"), ("tp cross", "tensor"), ("tp mlp", "tensor")])
def test_parallelism_applied_after_packing_is_refused(where: str, kind: str) -> None:
    """A block that holds part of the tokens or heads must not attend to that part alone."""
    block = _block()
    hidden, kwargs = _inputs("sample")
    quantize_model(block, "mxfp8")
    _parallelise(block, where)
    with torch.no_grad(), pytest.raises(RuntimeError, match=f"{kind} parallelism"):
        block(hidden, **kwargs)
    restore_model(block)
    with pytest.raises(ValueError, match=f"{kind} parallelism"):
        quantize_model(block, "mxfp8")


def test_context_parallelism_over_packed_blocks_is_refused() -> None:
    from avgen_b200.parallel.context import apply_context_parallel

    class Mesh:  # what context parallelism asks of a mesh before its first collective
        def size(self) -> int:
            return 2

        def get_group(self) -> None:
            return None

    model = nn.ModuleList([_block()])
    hidden, kwargs = _inputs("sample")
    quantize_model(model, "mxfp8")
    apply_context_parallel(model, Mesh(), ring=False)
    with torch.no_grad(), pytest.raises(RuntimeError, match="context parallelism"):
        model[0](hidden, **kwargs)


def _two_ranks(rank: int, port: int) -> None:
    import os

    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.fsdp import fully_shard

    from avgen_b200.parallel.context import apply_context_parallel
    from avgen_b200.parallel.tensor import apply_tensor_parallel

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    mesh = init_device_mesh("cpu", (2,), mesh_dim_names=("tp",))

    def packed() -> tuple[nn.Module, torch.Tensor, dict]:
        torch.manual_seed(13)
        model = nn.Module()
        model.blocks = nn.ModuleList([_block()])
        hidden, kwargs = _inputs("sample")
        quantize_model(model, "mxfp8")
        return model, hidden, kwargs

    with torch.no_grad():
        model, hidden, kwargs = packed()
        want = model.blocks[0](hidden, **kwargs)
        for apply in (lambda m: apply_tensor_parallel(m, mesh, style="dtensor"),
                      lambda m: fully_shard(m.blocks[0], mesh=mesh)):
            model = packed()[0]
            apply(model)
            with pytest.raises(ValueError, match="sharded weights"):
                quantize_model(model, "mxfp8")
            assert torch.equal(model.blocks[0](hidden, **kwargs), want)
        for apply, kind in ((lambda m: apply_tensor_parallel(m, mesh, style="heads"), "tensor"),
                            (lambda m: apply_tensor_parallel(m, mesh, style="heads", sequence_parallel=True), "tensor"),
                            (lambda m: apply_context_parallel(m, mesh), "context")):
            model = packed()[0]
            apply(model)
            with pytest.raises(RuntimeError, match=f"{kind} parallelism"):
                model.blocks[0](hidden, **kwargs)
    dist.destroy_process_group()


def test_packed_blocks_on_two_ranks() -> None:
    """What leaves a block's call whole (DTensor plans, FSDP2) gives its result; what splits it is refused."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_two_ranks, args=(port,), nprocs=2, join=True)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", mx.FORMATS)
@pytest.mark.parametrize("ffn,form", [("swiglu", "sample"), ("gelu", "grouped"), ("swiglu", "token")])
def test_gpu_block_stays_near_the_fp32_block(fmt: str, ffn: str, form: str) -> None:
    from avgen_b200.ops._ext import check_errors

    torch.manual_seed(3)
    block = _block(ffn=ffn)
    hidden, kwargs = _inputs(form)
    with torch.no_grad():
        want = block(hidden, **kwargs)
        block.cuda()
        quantize_model(block, fmt)
        kwargs = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kwargs.items()}
        kwargs["rope"] = RopeInputs(kwargs["rope"].coords.cuda(), kwargs["rope"].rope)
        kwargs["context"] = kwargs["context"].bfloat16()
        got = block(hidden.cuda().bfloat16(), **kwargs)
    assert got.dtype is torch.bfloat16
    assert float((got.float().cpu() - want).norm() / want.norm()) < BOUND[fmt] + 2e-2  # the bf16 residual stream
    assert check_errors() == 0


@pytest.mark.gpu
def test_gpu_block_refuses_weights_packed_elsewhere() -> None:
    block = _block()
    hidden, kwargs = _inputs("sample", "cuda", torch.bfloat16)
    quantize_model(block, "mxfp8")
    block.cuda()
    with torch.no_grad(), pytest.raises(RuntimeError, match="after moving the model"):
        block(hidden, **kwargs)


@pytest.mark.gpu
def test_gpu_model_samples_quantised() -> None:
    from dataclasses import asdict

    from avgen_b200.codecs import ReferenceTextEncoder, ReferenceVideoCodec
    from avgen_b200.infer import GenerationConfig, GenerationPipeline, ScheduleConfig
    from avgen_b200.models import build_model, preset

    torch.manual_seed(4)
    cfg = {k: v for k, v in asdict(preset("tiny_gpu")).items() if k != "rope_scaling"}
    model = build_model("video_dit", cfg).cuda().eval()
    model.init_weights()
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.02 * torch.randn_like(p))
    video = ReferenceVideoCodec(channels=cfg["in_channels"], temporal_compression=1, spatial_compression=1)
    text = ReferenceTextEncoder(width=cfg["text_width"], max_length=16)
    settings = GenerationConfig(steps=2, height=32, width=32, num_frames=4, schedule=ScheduleConfig(steps=2))
    pipe = GenerationPipeline(model, video_codec=video, text_encoder=text, config=settings, device=torch.device("cuda"))
    full = pipe(["a kite"], seed=1).video.float()
    assert quantize_model(model, "mxfp8") == cfg["depth"]
    packed = pipe(["a kite"], seed=1).video.float()
    assert torch.isfinite(packed).all()
    assert float((packed - full).norm() / full.norm()) < 0.2


@pytest.mark.gpu
def test_gpu_model_quantises_beside_blocks_of_other_head_dims() -> None:
    """A joint model whose audio tower has heads the kernels do not take: video alone samples, as unquantised."""
    from dataclasses import asdict

    from avgen_b200.codecs import ReferenceTextEncoder, ReferenceVideoCodec
    from avgen_b200.infer import GenerationConfig, GenerationPipeline, ScheduleConfig
    from avgen_b200.models import build_model, preset

    torch.manual_seed(9)
    cfg = {k: v for k, v in asdict(preset("tiny_gpu")).items() if k != "rope_scaling"}
    cfg.update(audio_width=128, audio_num_heads=2, audio_in_channels=4, audio_ffn_hidden=256)
    model = build_model("av_dit", cfg).cuda().eval()
    model.init_weights()
    video = ReferenceVideoCodec(channels=cfg["in_channels"], temporal_compression=1, spatial_compression=1)
    text = ReferenceTextEncoder(width=cfg["text_width"], max_length=16)
    settings = GenerationConfig(steps=2, height=32, width=32, num_frames=4, schedule=ScheduleConfig(steps=2),
                                generate_audio=False)
    pipe = GenerationPipeline(model, video_codec=video, text_encoder=text, config=settings, device=torch.device("cuda"))
    assert torch.isfinite(pipe(["a kite"], seed=1).video).all()
    assert quantize_model(model, "mxfp8") == 2 * cfg["depth"]
    assert torch.isfinite(pipe(["a kite"], seed=1).video).all()


@pytest.mark.gpu
def test_gpu_block_of_another_head_dim_refuses_when_it_runs() -> None:
    block = DiTBlock(256, 4, hidden=512).cuda()
    hidden, kwargs = _inputs("sample", "cuda", torch.bfloat16)
    kwargs["rope"] = None
    for pack in (False, True):
        if pack:
            quantize_model(block, "mxfp8")
        with torch.no_grad(), pytest.raises(NotImplementedError, match="head_dim 128"):
            block(hidden, **kwargs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gpu_block_takes_other_types_as_the_plain_block_does(dtype: torch.dtype) -> None:
    torch.manual_seed(10)
    block = _block().cuda()
    hidden, kwargs = _inputs("sample", "cuda", torch.bfloat16)
    hidden, kwargs["context"] = hidden.to(dtype), kwargs["context"].to(dtype)
    with torch.no_grad():
        for pack in (False, True):
            if pack:
                quantize_model(block, "nvfp4")
            out = block(hidden, **kwargs)
            assert out.dtype is dtype
            assert torch.equal(out, block(hidden.bfloat16(), **kwargs).to(dtype))
