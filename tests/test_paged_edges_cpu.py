"""Edges of the paged operators and of the decoder's paged_step without a GPU."""

import pytest
import torch

from selective_attention import paged
from selective_attention.model import ModelConfig, SelectiveLM


def small_model(attention="selective", **kw):
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=97, n_layers=2, d_model=64, n_heads=4, context_length=64, attention=attention)
    return SelectiveLM(cfg).eval()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("precision", [None, "bf16", "ieee"])
def test_step_paged_passes_the_slots_precision_on(monkeypatch, precision):
    model = small_model()
    for block in model.transformer.h:
        block.attn.dot_precision = precision
    seen, plain = [], paged.selective_attention_paged_reference
    monkeypatch.setattr(paged, "selective_attention_paged_reference",
                        lambda *args, dot_precision="not passed", **kw: seen.append(dot_precision) or plain(*args, **kw))
    with torch.no_grad():
        model.paged_step(torch.arange(5), ints(3, 2), model.new_paged_cache(2, 4, 16))
    assert seen == [precision] * 2


def test_an_unknown_precision_is_refused():
    model = small_model()
    model.transformer.h[0].attn.dot_precision = "fp8"
    with pytest.raises(ValueError, match="dot_precision"), torch.no_grad():
        model.paged_step(torch.arange(5), ints(3, 2), model.new_paged_cache(2, 4, 16))
