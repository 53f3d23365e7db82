"""A saved adapter whose layers have factors of their own, on projections that stand by themselves and on concatenated ones."""
import json
import os

import pytest
import torch

from tiny_llama import GROUPSIZE, build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("concatenate", [False, True])
@pytest.mark.parametrize("fields,q,v", [(dict(), 2.0, 2.0), (dict(use_rslora=True), 16 / 8 ** 0.5, 16 / 8 ** 0.5), (dict(alpha_pattern={"v_proj": 48}), 2.0, 6.0),
                                        (dict(rank_pattern={"q_proj": 2}), 8.0, 2.0)])
def test_injected_layers_have_the_factors_of_their_configuration(tmp_path, oracle, concatenate, fields, q, v):
    """scaling * B @ A of what was injected is factor * B @ A of the file.  A and B round to fp16 once each (half a step, 2^-11, and of both
    2^-22; 2^-25 below the normal numbers, times 8 products with factors up to 0.3)."""
    from safetensors.torch import save_file
    from alpaca_lora_4bit_amd import autograd_4bit as ag
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import inject_lora_layers, make_quant_attn
    ckpt, folder = str(tmp_path / "ckpt"), tmp_path / "lora"
    build(ckpt, oracle, seed=6, with_tokenizer=True)
    folder.mkdir()
    gen = torch.Generator().manual_seed(3)
    state = {f"base_model.model.model.layers.{i}.self_attn.{n}.lora_{m}.weight": torch.randn((8, 256) if m == "A" else (256, 8), generator=gen) * 0.05
             for i in range(2) for n in ("q_proj", "v_proj") for m in "AB"}
    save_file(state, str(folder / "adapter_model.safetensors"))
    (folder / "adapter_config.json").write_text(json.dumps(dict(r=8, lora_alpha=16, **fields)))
    model, _ = ag.load_llama_model_4bit_low_ram(ckpt, os.path.join(ckpt, "model.safetensors"), groupsize=GROUPSIZE, half=True, device_map={"": 0})
    make_quant_attn(model, concatenate=concatenate)
    layers = inject_lora_layers(model, str(folder))
    assert len(layers) == (2 if concatenate else 4)
    for i, block in enumerate(model.model.layers):
        for n, factor, first in (("q_proj", q, 0), ("v_proj", v, 512)):
            layer = block.self_attn.qkv_proj if concatenate else getattr(block.self_attn, n)
            a, b = (getattr(layer, m)["default"].weight.detach().double().cpu() for m in ("lora_A", "lora_B"))
            got = layer.scaling["default"] * (b @ a)
            got = got[first:first + 256] if concatenate else got
            fa, fb = (state[f"base_model.model.model.layers.{i}.self_attn.{n}.lora_{m}.weight"].double() for m in "AB")
            bound = factor * ((fb.abs() @ fa.abs()) * (2 * 2.0 ** -11 + 2.0 ** -22) + 8 * 2 * 0.3 * 2.0 ** -25)
            assert ((got - factor * fb @ fa).abs() <= bound).all()
    with torch.no_grad():
        assert torch.isfinite(model(torch.tensor([[1, 5, 9, 20]]).cuda()).logits).all()
