"""Run a DiT's linears in 8 or 4 bits: pack its blocks, compare outputs, restore it.

`quantize_model` packs every block's weights once in a block-scaled format; each forward
then normalises straight into packed rows and multiplies packed operands (on a B200 in the
tensor cores' block-scaled modes, on a CPU in their PyTorch restatement). The same
operators are there to be called one by one.

    python examples/06_quantized_sampling.py
"""
from __future__ import annotations

import torch

from avgen_b200.models import DiTBlock, RopeInputs, RotaryEmbedding, quantize_model, restore_model
from avgen_b200.ops import microscale as mx


def main() -> None:
    torch.manual_seed(0)
    device = "cuda" if torch.cuda.is_available() else "cpu"
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    model = torch.nn.ModuleList(DiTBlock(256, 2, hidden=512) for _ in range(2)).to(device).eval()
    for block in model:
        block.init_weights(depth=2)
        with torch.no_grad():  # gates and tables as after some training
            for p in block.parameters():
                p.add_(0.02 * torch.randn_like(p))
    hidden = torch.randn(2, 192, 256, device=device, dtype=dtype)
    inputs = {"modulation": 0.1 * torch.randn(2, 6, 256, device=device),
              "rope": RopeInputs(torch.rand(2, 192, 3, device=device) * 8, RotaryEmbedding(128)),
              "context": torch.randn(2, 24, 256, device=device, dtype=dtype)}

    def run() -> torch.Tensor:
        out = hidden
        for block in model:
            out = block(out, **inputs)
        return out.float()

    with torch.no_grad():
        full = run()
        for fmt in mx.FORMATS:
            quantize_model(model, fmt)
            error = float((run() - full).norm() / full.norm())
            packed = sum(block.quantized.nbytes for block in model)
            print(f"{fmt}: output off by {error:.3f}, blocks packed in {packed / 1e6:.2f} MB")
        restore_model(model)

        # the operators themselves: a residual update, its norm in 8 bits, the next linear layer
        x, update = torch.randn(192, 256, device=device, dtype=dtype), torch.randn(192, 256, device=device, dtype=dtype)
        weight = mx.quantize(torch.randn(512, 256, device=device) / 16, "mxfp8")
        x, normed = mx.add_rmsnorm_mod(x, update, None)
        y = mx.matmul(normed, weight)
        plain = torch.nn.functional.rms_norm(x.float(), (256,), eps=1e-6) @ mx.dequantize(weight, torch.float32).t()
        print(f"norm in 8 bits and product: off by {float((y.float() - plain).norm() / plain.norm()):.4f}")


if __name__ == "__main__":
    main()
