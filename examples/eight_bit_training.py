"""Train a small language model with 8-bit products and 8-bit AdamW state, then decode from 8-bit weights.

The model's linear layers are ``Float8Linear``: products run on weights, activations and
gradients quantized in blocks of 128. Its weights stay float32 for the optimizer: Dion moves the
matrices, AdamW the embedding, the norms and the biases, with moments held in 8 bits. After
training, each layer's weight is quantized once and kept; a token then reads one byte a weight.

    python examples/eight_bit_training.py [--steps 200]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor, nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import dionw_amd as dionw  # noqa: E402

VOCAB, WIDTH, LAYERS, CONTEXT = 211, 256, 2, 8


class Block(nn.Module):
    """A norm and a gated MLP."""

    def __init__(self) -> None:
        super().__init__()
        self.norm = nn.LayerNorm(WIDTH)
        self.up = dionw.Float8Linear(WIDTH, 4 * WIDTH)
        self.down = dionw.Float8Linear(2 * WIDTH, WIDTH)

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
        self.head = dionw.Float8Linear(WIDTH, VOCAB, bias=False)

    def forward(self, tokens: Tensor) -> Tensor:
        x = self.mix(self.embed(tokens).flatten(1))
        for block in self.blocks:
            x = block(x)
        return self.head(x)


def sequence(count: int, generator: torch.Generator) -> tuple[Tensor, Tensor]:
    """Contexts of a rule (each token a function of two before it), and the tokens that follow."""
    tokens = torch.randint(VOCAB, (count, CONTEXT + 1), generator=generator)
    for i in range(2, CONTEXT + 1):
        tokens[:, i] = (3 * tokens[:, i - 1] + tokens[:, i - 2] + 7) % VOCAB
    return tokens[:, :-1].cuda(), tokens[:, -1].cuda()


def train(steps: int, eight_bit: bool = True) -> tuple[Model, list[float]]:
    """The trained model and the loss of every step."""
    torch.manual_seed(0)
    model = Model().cuda()
    if not eight_bit:
        for module in model.modules():
            if isinstance(module, dionw.Float8Linear):
                module.forward = lambda x, m=module: nn.functional.linear(x, m.weight, m.bias)
    groups, _ = dionw.param_groups(model)
    state = dionw.AdamWState.EIGHT_BIT if eight_bit else dionw.AdamWState.FLOAT32
    optimizer = dionw.Dion(groups, lr=3e-3, weight_decay=0.01, adamw_state=state)
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


class Decoder:
    """The model from kept 8-bit weights: what a server holds."""

    def __init__(self, model: Model) -> None:
        self.model = model
        self.kept = {m: m.quantized_weight() for m in model.modules() if isinstance(m, dionw.Float8Linear)}

    def _linear(self, layer: dionw.Float8Linear, x: Tensor) -> Tensor:
        return dionw.float8_linear(x, self.kept[layer], layer.bias)

    @torch.no_grad()
    def __call__(self, tokens: Tensor) -> Tensor:
        model = self.model
        x = self._linear(model.mix, model.embed(tokens).flatten(1))
        for block in model.blocks:
            gate, value = self._linear(block.up, block.norm(x)).chunk(2, -1)
            x = x + self._linear(block.down, nn.functional.silu(gate) * value)
        return self._linear(model.head, x)


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    steps = parser.parse_args().steps
    for name, eight_bit in (("float32", False), ("8 bits", True)):
        model, losses = train(steps, eight_bit)
        print(f"{name}: loss {losses[0]:.3f} -> {losses[-1]:.3f}")
    decoder = Decoder(model)
    tokens, following = sequence(16, torch.Generator().manual_seed(2))
    right = sum(int(decoder(tokens[i:i + 1]).argmax()) == int(following[i]) for i in range(16))
    print(f"decoding one at a time from 8-bit weights: {right} of 16 tokens right")


if __name__ == "__main__":
    main()
