"""Steps of whole 4-bit models that keep 8 bits: one group a column (the script's default), adapters on every projection, few rows and many."""
import json
import os

import pytest
import torch

from tiny_llama import GROUPSIZE, build

pytestmark = pytest.mark.gpu


class _Columns:
    """The oracle, with layers of one group a column whatever size is asked for."""

    def __init__(self, oracle):
        self._oracle = oracle

    def __getattr__(self, name):
        return getattr(self._oracle, name)

    def make_layer(self, K, N, groupsize, **kw):
        return self._oracle.make_layer(K, N, K, **kw)


def test_the_script_on_a_checkpoint_of_one_group_a_column(tmp_path, oracle, monkeypatch, capsys):
    from alpaca_lora_4bit_amd import finetune, quant_hip
    ckpt = str(tmp_path / "ckpt")
    build(ckpt, _Columns(oracle), seed=7)
    data = str(tmp_path / "pairs.json")
    with open(data, "w") as fh:
        json.dump([{"instruction": "alpha beta", "input": "the lora", "chosen": "gamma " * (1 + i % 3), "rejected": "delta token"} for i in range(8)], fh)
    kept, real = [], quant_hip.silu_mul_act8
    monkeypatch.setattr(quant_hip, "silu_mul_act8", lambda gate, up, **kw: (kept.append(kw.get("keep", True)), real(gate, up, **kw))[1])
    model, _, trainer = finetune.main([data, "--ds_type", "preference", "--llama_q4_config_dir", ckpt, "--llama_q4_model", os.path.join(ckpt, "model.safetensors"), "--lora_out_dir",
                                       str(tmp_path / "out"), "--mbatch_size", "2", "--batch_size", "2", "--epochs", "1", "--cutoff_len", "64", "--logging_steps", "1", "--val_set_size", "0", "--act_bits", "8"])
    assert "2 MLP blocks keep their activations in 8 bits" in capsys.readouterr().out
    assert kept.count(True) == kept.count(False) == 2 * 4      # two blocks, four steps: the policy's passes and the reference's
    assert all(torch.isfinite(m.lora_B["default"].weight).all() for m in model.modules() if "Linear4bitLt" in str(type(m)))


class _Plain(torch.autograd.Function):
    """silu(gate) * up and its gradients at the values that 8 bits hold, as elementary operations in fp32."""

    @staticmethod
    def forward(ctx, gate, up):
        from alpaca_lora_4bit_amd import quant_hip
        ctx.save_for_backward(*(quant_hip.act8_unpack(*quant_hip.act8_pack(t), torch.float32) for t in (gate, up)))
        g = gate.float()
        return (g / (1 + torch.exp(-g)) * up.float()).to(gate.dtype)

    @staticmethod
    def backward(ctx, dout):
        g, u = ctx.saved_tensors
        s = 1 / (1 + torch.exp(-g))
        return (dout.float() * u * s * (1 + g * (1 - s))).to(dout.dtype), (dout.float() * g * s).to(dout.dtype)


@pytest.mark.parametrize("checkpoints", [False, True])
@pytest.mark.parametrize("places", [2, 40])
def test_adapters_on_every_projection(tmp_path, oracle, monkeypatch, places, checkpoints):
    """Adapter gradients against those of the same step with the gated activation's formula at the values held.  The two differ where a rounding to fp16 goes the other way, 2^-11 of a
    value, in some 14 products one behind the other: 2 * 14 * 2^-11 < 2e-2 of what flows.  With two places, of which the first attends to itself alone and the second has no label, the gradients
    of q and k are zero but for such roundings: half a unit of the largest."""
    from alpaca_lora_4bit_amd import autograd_4bit as ag, model_attn_mlp_patch as patch, models, preference
    from alpaca_lora_4bit_amd.gradient_checkpointing import apply_gradient_checkpointing
    ckpt = str(tmp_path / "ckpt")
    build(ckpt, oracle, seed=5)
    ids = torch.randint(3, 300, (4, places), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    labels = preference.shifted_labels(ids)
    model, _ = ag.load_llama_model_4bit_low_ram(ckpt, os.path.join(ckpt, "model.safetensors"), groupsize=GROUPSIZE, half=True, device_map={"": 0})
    torch.manual_seed(3)
    layers = models.inject_lora_layers(model, target_modules=("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"), r=8, lora_alpha=16)
    gen = torch.Generator(device="cuda").manual_seed(3)
    with torch.no_grad():
        for layer in layers.values():
            layer.lora_B["default"].weight.normal_(0, 0.05, generator=gen)
    patch.make_quant_attn(model)
    assert patch.make_fused_mlp(model, act_bits=8) == 2
    if checkpoints:
        apply_gradient_checkpointing(model, bits=8)
    model.train()

    def step():
        model.zero_grad()
        with torch.amp.autocast("cuda", dtype=torch.float16):
            with torch.no_grad(), preference.adapters_off(model):
                ref = preference.token_logps(model(input_ids=ids, use_cache=False).logits, labels)
            logits = model(input_ids=ids, use_cache=False).logits
        loss, _ = preference.preference_loss(logits, labels, ref, beta=0.5)
        (loss * 1024).backward()
        return ref, [w.grad.double() for layer in layers.values() for w in (layer.lora_A["default"].weight, layer.lora_B["default"].weight)]
    ref, grads = step()
    monkeypatch.setattr(patch, "_SiluMulAct8", _Plain)
    again, want = step()
    assert torch.equal(ref, again) and len(want) == 28
    largest = max(float(w.norm()) for w in want)
    for a, b in zip(grads, want):
        assert float((a - b).norm()) <= 2e-2 * float(b.norm()) + 2.0 ** -11 * largest


def test_a_reference_pass_in_inference_mode(tmp_path, oracle):
    from alpaca_lora_4bit_amd import autograd_4bit as ag, models, preference
    ckpt = str(tmp_path / "ckpt")
    build(ckpt, oracle, seed=5)
    model, _ = ag.load_llama_model_4bit_low_ram(ckpt, os.path.join(ckpt, "model.safetensors"), groupsize=GROUPSIZE, half=True, device_map={"": 0})
    layers = models.inject_lora_layers(model, target_modules=("q_proj", "v_proj"), r=8, lora_alpha=16)
    for attn in (b.self_attn for b in model.model.layers):
        attn.attention_dropout = 0.5
    model.train()
    ids = torch.randint(3, 300, (2, 20), device="cuda")
    passes = []
    for mode in (torch.inference_mode, torch.no_grad, torch.no_grad):
        with mode(), preference.adapters_off(model), torch.amp.autocast("cuda", dtype=torch.float16):
            passes.append(model(input_ids=ids, use_cache=False).logits.float())
    assert torch.equal(passes[0], passes[1]) and torch.equal(passes[1], passes[2])       # no dropout of the host model's
    assert model.training and all(w.requires_grad for layer in layers.values() for w in (layer.lora_A["default"].weight, layer.lora_B["default"].weight))
