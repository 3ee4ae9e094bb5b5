"""The 4-bit example runs, its gradients are those of its operators, and the server's layers
give the model's outputs (GPU)."""

from __future__ import annotations

import copy

import pytest
import torch

from dionw_amd import Float4Linear, Float8Linear, float4_linear, float4_quantize, float8_linear, layer_norm
from examples import four_bit_training as example

pytestmark = pytest.mark.gpu


def test_it_trains_a_few_steps() -> None:
    model, losses = example.train(3)
    assert len(losses) == 3 and all(loss == loss and loss < 1e3 for loss in losses)
    assert all(p.isfinite().all() for p in model.parameters())


def _by_hand(model: example.Model, tokens: torch.Tensor, seeds: list[int]) -> torch.Tensor:
    seeds = list(seeds)
    x = float8_linear(model.embed(tokens).flatten(1), model.mix.weight, model.mix.bias)
    for block in model.blocks:
        h = layer_norm(x, block.norm.weight, block.norm.bias, block.norm.eps)
        gate, value = float4_linear(h, block.up.weight, block.up.bias, seed=seeds.pop(0)).chunk(2, -1)
        h = torch.nn.functional.silu(gate) * value
        x = x + float4_linear(h, block.down.weight, block.down.bias, seed=seeds.pop(0))
    return float8_linear(layer_norm(x, model.norm.weight, model.norm.bias, model.norm.eps), model.head.weight)


def test_its_gradients_are_those_of_its_operators() -> None:
    """With the seeds that the layers draw, every parameter's gradient bit for bit."""
    torch.manual_seed(0)
    model = example.Model().cuda()
    twin = copy.deepcopy(model)
    tokens, following = example.sequence(100, torch.Generator().manual_seed(1))
    torch.manual_seed(5)
    torch.nn.functional.cross_entropy(model(tokens), following).backward()
    torch.manual_seed(5)
    seeds = [int(torch.empty((), dtype=torch.int64).random_()) for _ in range(2 * example.LAYERS)]
    torch.nn.functional.cross_entropy(_by_hand(twin, tokens, seeds), following).backward()
    for (name, p), q in zip(model.named_parameters(), twin.parameters()):
        assert p.grad is not None and bool(p.grad.any()), name
        assert torch.equal(p.grad, q.grad), name


@pytest.mark.parametrize("rows", [1, 16, 17, 100])
def test_the_server_gives_every_layers_output(rows) -> None:
    """Kept weights hold the values that the layers multiply by, and a float32 norm quantized as it is
    made those of the norm quantized later, so that on one input both sum the same products: each is off
    by ``(depth + 1) x 2^-23 x sum |a| |b|`` at most, whatever its order, and by a rounding."""
    torch.manual_seed(0)
    model = example.Model().cuda()
    server = example.Server(model)
    tokens, _ = example.sequence(rows, torch.Generator().manual_seed(1))
    seen = {}
    for module in model.modules():
        if isinstance(module, (example.Block, Float4Linear)):
            module.register_forward_hook(lambda m, args, out: seen.__setitem__(m, args[0]))
    with torch.no_grad():
        want = model(tokens)

        def check(got, layer, x):
            q, w = float4_quantize(x).values().double(), float4_quantize(layer.weight, tiles=True).values().double()
            size = q.abs() @ w.abs().T + layer.bias.double().abs()
            exact = q @ w.T + layer.bias.double()
            bound = (x.shape[1] + 1) * 2.0 ** -23 * size + 2.0 ** -24 * exact.abs()
            for y in (got, layer(x)):
                assert bool(((y.double() - exact).abs() <= bound).all())

        for block in model.blocks:
            check(server._up(block, seen[block]), block.up, block.norm(seen[block]))
            check(float4_linear(seen[block.down], server.kept[block.down], block.down.bias), block.down,
                  seen[block.down])
    got = server(tokens)
    assert got.shape == want.shape and bool(got.isfinite().all())


def test_which_layers_take_which_bits() -> None:
    model = example.Model()
    kinds = [type(m) for m in model.modules() if isinstance(m, (Float4Linear, Float8Linear))]
    assert kinds.count(Float4Linear) == 2 * example.LAYERS and kinds.count(Float8Linear) == 2
