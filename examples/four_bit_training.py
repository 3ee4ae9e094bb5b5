"""Train a small language model with 4-bit products in its blocks, then serve it from kept 4-bit weights.

The blocks' norms are ``LayerNorm`` and their linear layers ``Float4Linear``: weights and activations
are quantized to 4 bits in blocks of 32 where a product reads them, gradients too, rounded up or down
by chance. The layers at both ends, which see tokens one by one, keep 8 bits. All weights stay
float32 for the optimizer: Dion moves the matrices, AdamW the embedding, the norms and the biases.
After training, each layer's weight is quantized once and kept. A prompt's norms are quantized as they
are made, for the product behind them; a single token's go through ``float4_linear``, which quantizes
it itself.

    python examples/four_bit_training.py [--steps 200]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor, nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import dionw_amd as dionw  # noqa: E402
from examples.eight_bit_training import CONTEXT, VOCAB, sequence  # noqa: E402

WIDTH, LAYERS = 256, 2


class Block(nn.Module):
    """A norm and a gated MLP."""

    def __init__(self) -> None:
        super().__init__()
        self.norm = dionw.LayerNorm(WIDTH)
        self.up = dionw.Float4Linear(WIDTH, 4 * WIDTH)
        self.down = dionw.Float4Linear(2 * WIDTH, WIDTH)

    def forward(self, x: Tensor) -> Tensor:
        gate, value = self.up(self.norm(x)).chunk(2, -1)
        return x + self.down(nn.functional.silu(gate) * value)


class Model(nn.Module):
    """Predicts a token from the CONTEXT tokens before it."""

    def __init__(self) -> None:
        super().__init__()
        self.embed = nn.Embedding(VOCAB, WIDTH)
        self.mix = dionw.Float8Linear(CONTEXT * WIDTH, WIDTH)
        self.blocks = nn.ModuleList(Block() for _ in range(LAYERS))
        self.norm = dionw.LayerNorm(WIDTH)
        self.head = dionw.Float8Linear(WIDTH, VOCAB, bias=False)

    def forward(self, tokens: Tensor) -> Tensor:
        x = self.mix(self.embed(tokens).flatten(1))
        for block in self.blocks:
            x = block(x)
        return self.head(self.norm(x))


def train(steps: int) -> tuple[Model, list[float]]:
    """The trained model and the loss of every step."""
    torch.manual_seed(0)
    model = Model().cuda()
    groups, _ = dionw.param_groups(model)
    optimizer = dionw.Dion(groups, lr=3e-3, weight_decay=0.01)
    generator = torch.Generator().manual_seed(1)
    losses = []
    for _ in range(steps):
        tokens, following = sequence(1024, generator)
        loss = nn.functional.cross_entropy(model(tokens), following)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return model, torch.stack(losses).tolist()


class Server:
    """The model from kept 4-bit and 8-bit weights."""

    def __init__(self, model: Model) -> None:
        self.model = model
        layers = (dionw.Float4Linear, dionw.Float8Linear)
        self.kept = {m: m.quantized_weight() for m in model.modules() if isinstance(m, layers)}

    def _up(self, block: Block, x: Tensor) -> Tensor:
        norm, up = block.norm, block.up
        if x.shape[0] > 16:
            q = dionw.float4_layer_norm(x, norm.weight, norm.bias, norm.eps)
            return dionw.float4_matmul(q, self.kept[up], up.bias, dtype=x.dtype)
        return dionw.float4_linear(norm(x), self.kept[up], up.bias)

    @torch.no_grad()
    def __call__(self, tokens: Tensor) -> Tensor:
        model = self.model
        x = dionw.float8_linear(model.embed(tokens).flatten(1), self.kept[model.mix], model.mix.bias)
        for block in model.blocks:
            gate, value = self._up(block, x).chunk(2, -1)
            x = x + dionw.float4_linear(nn.functional.silu(gate) * value, self.kept[block.down], block.down.bias)
        return dionw.float8_linear(model.norm(x), self.kept[model.head])


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    model, losses = train(parser.parse_args().steps)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}")
    server = Server(model)
    tokens, following = sequence(64, torch.Generator().manual_seed(2))
    right = int((server(tokens).argmax(1) == following).sum())
    print(f"64 contexts at once from kept weights: {right} tokens right")
    right = sum(int(server(tokens[i:i + 1]).argmax()) == int(following[i]) for i in range(16))
    print(f"one at a time: {right} of 16 tokens right")


if __name__ == "__main__":
    main()
