"""The factor of a saved adapter's update: lora_alpha / r and the fields of adapter_config.json that change it."""
import json
import math

import pytest
import torch

from alpaca_lora_4bit_amd import models
from alpaca_lora_4bit_amd.model_attn_mlp_patch import adapter_factor

CONFIGS = [
    # the fields, then the factors of layer 0's q_proj, layer 0's v_proj and layer 1's q_proj
    (dict(), (2.0, 2.0, 2.0)),
    (dict(use_rslora=False, alpha_pattern={}, rank_pattern=None), (2.0, 2.0, 2.0)),
    (dict(use_rslora=True), (16 / math.sqrt(8),) * 3),
    (dict(alpha_pattern={"v_proj": 4}), (2.0, 0.5, 2.0)),
    (dict(rank_pattern={"v_proj": 4}), (2.0, 4.0, 2.0)),
    (dict(rank_pattern={"model.layers.0.self_attn.q_proj": 2}, alpha_pattern={"q_proj": 6}), (3.0, 2.0, 0.75)),
    (dict(rank_pattern={r"layers\.0\..*": 4}, use_rslora=True), (8.0, 8.0, 16 / math.sqrt(8))),
    (dict(alpha_pattern={"proj": 100, "_proj": 100, "elf_attn.q_proj": 100}), (2.0, 2.0, 2.0)),
]
PATHS = [f"model.layers.{i}.self_attn.{n}_proj" for i, n in ((0, "q"), (0, "v"), (1, "q"))]


@pytest.mark.parametrize("fields,want", CONFIGS)
def test_factor_of_a_layer(fields, want):
    assert [adapter_factor(dict(r=8, lora_alpha=16, **fields), p) for p in PATHS] == pytest.approx(list(want))


class _Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        block = lambda: torch.nn.ModuleDict({"self_attn": torch.nn.ModuleDict({n: torch.nn.Linear(64, 64, bias=False) for n in ("q_proj", "v_proj")})})
        self.model = torch.nn.ModuleDict({"layers": torch.nn.ModuleList([block(), block()])})


@pytest.mark.parametrize("fields,want", CONFIGS)
def test_a_bank_takes_each_layers_factor(tmp_path, fields, want):
    from safetensors.torch import save_file
    model = _Model()
    state = {f"base_model.model.{p}.lora_{m}.weight": torch.ones((8, 64) if m == "A" else (64, 8)) for p in PATHS for m in "AB"}
    save_file(state, str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps(dict(r=8, lora_alpha=16, **fields)))
    bank = models.AdapterBank(model, [(state, 0.25), str(tmp_path)], device="cpu")
    layers = dict(model.named_modules())
    assert [bank._layers[layers[p]][2].tolist() for p in PATHS] == [pytest.approx([0.25, w]) for w in want]
