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


def test_decoding_ranks_the_models_token_first() -> None:
    """Where the model's first token leads by more than twice what the test above lets a logit
    move, decoding from kept weights must rank it first; after 200 steps it does so somewhere."""
    model, _ = example.train(200)
    decoder = example.Decoder(model)
    tokens, _ = example.sequence(64, torch.Generator().manual_seed(3))
    with torch.no_grad():
        together = model(tokens)
    first, second = together.topk(2, -1).values.unbind(-1)
    clear = first - second > 2 * 0.05 * together.abs().amax()
    assert clear.any()
    for i in clear.nonzero().flatten().tolist():
        assert decoder(tokens[i:i + 1]).argmax() == together[i].argmax()
