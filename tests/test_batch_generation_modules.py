"""What a batch of requests runs itself instead of the model's modules: adapters it cannot add are refused, not dropped."""
import pytest
import torch

from alpaca_lora_4bit_amd import inference, models

from test_batch_generation import PROMPTS, Plain, _adapters, _model


@pytest.mark.parametrize("targets", [("lm_head",), ("q_proj", "lm_head")])
def test_adapters_of_layers_that_a_batch_does_not_add(monkeypatch, targets):
    Plain(monkeypatch)
    model = _model()
    bank = models.AdapterBank(model, _adapters(model, [targets], (8,), 1), device="cpu")
    with pytest.raises(ValueError, match="lm_head"):
        inference.generate_batch(model, PROMPTS, 2, bank, [0] * len(PROMPTS), use_graph=False)
    both = models.AdapterBank(model, _adapters(model, [("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")], (8,), 1), device="cpu")
    assert len(inference.generate_batch(model, PROMPTS, 2, both, [0] * len(PROMPTS), use_graph=False)) == len(PROMPTS)
