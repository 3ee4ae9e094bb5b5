"""The example that trains with 8-bit products and 8-bit AdamW state and decodes from 8-bit weights (GPU)."""

from __future__ import annotations

import pytest
import torch

from examples import eight_bit_training as example

pytestmark = pytest.mark.gpu


def test_training_follows_float32_and_decoding_the_model() -> None:
    """100 steps: quantizing must cost less than a tenth of what training gains, and 16 kept-weight
    decodings must rank the model's own next token first wherever it leads by more than 8-bit
    noise can move (both read the same quantized weights; activations differ by accumulation only)."""
    _, plain = example.train(100, eight_bit=False)
    model, losses = example.train(100)
    gain = plain[0] - sum(plain[-10:]) / 10
    assert gain > 1.0
    assert losses[0] - sum(losses[-10:]) / 10 > 0.9 * gain
    decoder = example.Decoder(model)
    tokens, _ = example.sequence(16, torch.Generator().manual_seed(2))
    with torch.no_grad():
        together = model(tokens)
    for i in range(16):
        alone = decoder(tokens[i:i + 1])
        assert torch.allclose(alone[0], together[i], rtol=0, atol=0.05 * float(together.abs().max()))
