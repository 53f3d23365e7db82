"""Training on pairs with what a step keeps in 8 bits: checkpoints, gated blocks, a whole step of a 4-bit model with adapters, and the finetune script."""
import json
import math
import os
import random

import pytest
import torch

from tiny_llama import GROUPSIZE, build

pytestmark = pytest.mark.gpu

WORDS = ["alpha", "beta", "gamma", "delta", "lora", "quant", "weight", "matrix", "token", "layer", "the", "of"]


def _counted(monkeypatch, name):
    from alpaca_lora_4bit_amd import quant_hip
    seen, real = [], getattr(quant_hip, name)

    def call(*a, **kw):
        seen.append(tuple(a[0].shape) if kw.get("keep", True) else None)
        return real(*a, **kw)
    monkeypatch.setattr(quant_hip, name, call)
    return seen


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_checkpoints_in_8_bits_give_the_gradients_at_the_values_held(monkeypatch, kind):
    """Block by block the gradients are those of the block at its input as 8 bits hold it (the first block's input is a leaf and kept as it is)."""
    from transformers import LlamaConfig, LlamaForCausalLM
    from alpaca_lora_4bit_amd import quant_hip
    from alpaca_lora_4bit_amd.gradient_checkpointing import apply_gradient_checkpointing
    torch.manual_seed(1)
    cfg = LlamaConfig(vocab_size=97, hidden_size=72, intermediate_size=128, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=4, attn_implementation="eager")
    model = LlamaForCausalLM(cfg).to("cuda", getattr(torch, kind)).train()
    for p in model.model.embed_tokens.parameters():
        p.requires_grad_(False)
    apply_gradient_checkpointing(model, bits=8)
    ids = torch.randint(0, 97, (3, 19), device="cuda")
    inputs = {}
    for i, block in enumerate(model.model.layers):
        def spy(*args, _i=i, _inner=block.old_forward_for_cp, **kwargs):
            inputs.setdefault(_i, (args[0].detach().clone(), kwargs))
            return _inner(*args, **kwargs)
        block.old_forward_for_cp = spy
    packed = _counted(monkeypatch, "act8_pack")
    model(input_ids=ids, labels=ids, use_cache=False).loss.backward()
    assert packed == [(3, 19, 72)] * 3
    got = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}

    model.zero_grad()
    last = inputs[3][0]
    with torch.no_grad():
        end = model.model.layers[3].old_forward_for_cp(last, **inputs[3][1])
    end = (end[0] if isinstance(end, tuple) else end).requires_grad_()
    logits = model.lm_head(model.model.norm(end))
    loss = model.loss_function(logits=logits, labels=ids, vocab_size=97)
    (g,) = torch.autograd.grad(loss, end)
    for i in (3, 2, 1, 0):
        h, kwargs = inputs[i]
        if i:
            h = quant_hip.act8_unpack(*quant_hip.act8_pack(h), h.dtype)
        h = h.requires_grad_()
        out = model.model.layers[i].old_forward_for_cp(h, **kwargs)
        (out[0] if isinstance(out, tuple) else out).backward(g)
        g = h.grad
    for n, p in model.named_parameters():
        if "layers" in n:                                      # the same operations on the same values
            assert torch.allclose(got[n], p.grad, rtol=1e-5 if kind == "float32" else 2.0 ** -6, atol=1e-3 * float(p.grad.abs().max())), n


def test_checkpoints_in_8_bits_take_less_memory_and_keep_no_input_alive():
    from transformers import LlamaConfig, LlamaForCausalLM
    from alpaca_lora_4bit_amd.gradient_checkpointing import apply_gradient_checkpointing
    held = {}
    for bits in (16, 8):
        torch.manual_seed(1)
        cfg = LlamaConfig(vocab_size=97, hidden_size=256, intermediate_size=128, num_hidden_layers=6, num_attention_heads=4, num_key_value_heads=4)
        model = LlamaForCausalLM(cfg).cuda().half().train()
        apply_gradient_checkpointing(model, bits=bits)
        ids = torch.randint(0, 97, (4, 512), device="cuda")
        before = torch.cuda.memory_allocated()
        h = model.model(input_ids=ids, use_cache=False)[0]
        held[bits] = torch.cuda.memory_allocated() - before
        h.float().sum().backward()
        assert all(torch.isfinite(p.grad).all() for n, p in model.named_parameters() if "layers" in n)
        del h, model
    one = 4 * 512 * 256
    assert held[16] - held[8] > 0.9 * 5 * one * (2 - 1.0625)


def test_gated_block_that_keeps_8_bits(oracle, monkeypatch):
    """Outputs of the block's own forward, gradients from the values held; and what it keeps is half."""
    import torch.nn as nn
    from conftest import rel_err, to_cuda_layer
    from alpaca_lora_4bit_amd import quant_hip
    from alpaca_lora_4bit_amd.autograd_4bit import Autograd4bitQuantLinear
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp, ungroup

    class Gated(nn.Module):
        def __init__(self):
            super().__init__()
            self.act_fn = nn.SiLU()

        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))
    H, I, gs, M = 256, 512, 128, 640
    own, fused = Gated(), Gated()
    for m in (own, fused):
        for i, (name, k, n) in enumerate((("gate_proj", H, I), ("up_proj", H, I), ("down_proj", I, H))):
            lin = Autograd4bitQuantLinear(k, n, groupsize=gs)
            for key, v in to_cuda_layer(oracle.make_layer(k, n, gs, seed=40 + i)).items():
                if isinstance(v, torch.Tensor):
                    setattr(lin, key, v)
            lin.bias = torch.zeros(n, dtype=torch.float16, device="cuda")
            setattr(m, name, lin)
    assert make_fused_mlp(fused, act_bits=8) == 1
    calls, backs = _counted(monkeypatch, "silu_mul_act8"), _counted(monkeypatch, "silu_mul_act8_bwd")
    xh = torch.from_numpy(oracle.make_activations(M, H, seed=4)).cuda()
    dy = torch.from_numpy(oracle.make_activations(M, H, seed=5)).cuda()

    def run(block):
        x = xh.clone().requires_grad_(True)
        before = torch.cuda.memory_allocated()
        with torch.amp.autocast("cuda", dtype=torch.float16):
            y = block(x)
        kept = torch.cuda.memory_allocated() - before
        y.backward(dy)
        return y.detach(), x.grad, kept
    run(own), run(fused)                                       # allocations of the first calls
    calls.clear(), backs.clear()
    want, got = run(own), run(fused)
    assert calls == [(M, I)] and backs == [(M, I)]
    # sums over 256 and 512 products of intermediates one fp16 rounding apart
    assert rel_err(got[0].cpu().numpy(), want[0].double().cpu().numpy()) <= 3e-3
    x = xh.clone().requires_grad_(True)
    with torch.amp.autocast("cuda", dtype=torch.float16):
        gate, up = own.gate_proj(x), own.up_proj(x)
        out = quant_hip.silu_mul_act8(gate.detach(), up.detach())
        act = out[0].requires_grad_(True)
        (dact,) = torch.autograd.grad(own.down_proj(act), act, dy)
    dgate, dup = quant_hip.silu_mul_act8_bwd(dact, out[1])
    torch.autograd.backward([gate, up], [dgate, dup])
    assert rel_err(got[1].cpu().numpy(), x.grad.double().cpu().numpy()) <= 3e-3
    assert want[2] - got[2] > 0.9 * M * I * (2 * 2 - 2 * 1.0625)      # at least gate and up of 16 bits less their 8 bits
    with torch.no_grad():
        calls.clear()
        assert torch.equal(fused(xh), got[0]) and calls == [None]      # the same product, nothing kept where nothing is differentiated
        calls.clear()
    with torch.amp.autocast("cuda", dtype=torch.float16):
        assert torch.equal(fused(xh), got[0]) and calls == [None]
    calls.clear()
    ungroup(fused)
    assert "_q4_act_bits" not in fused.__dict__ and run(fused)[2] == want[2] and not calls
    assert make_fused_mlp(fused) == 1 and run(fused)[0].shape == (M, H) and not calls
    assert make_fused_mlp(fused, act_bits=8) == 1 and torch.equal(run(fused)[0], got[0]) and calls == [(M, I)]       # a block that is fused already


def _model(tmp_path, oracle, seed=5):
    from alpaca_lora_4bit_amd import autograd_4bit as ag, models
    ckpt = str(tmp_path / "ckpt")
    build(ckpt, oracle, seed=seed, with_tokenizer=True)
    model, tok = ag.load_llama_model_4bit_low_ram(ckpt, os.path.join(ckpt, "model.safetensors"), groupsize=GROUPSIZE, half=True, device_map={"": 0})
    layers = models.inject_lora_layers(model, target_modules=("q_proj", "v_proj"), r=8, lora_alpha=16)
    gen = torch.Generator(device="cuda").manual_seed(3)
    with torch.no_grad():
        for layer in layers.values():
            layer.lora_B["default"].weight.normal_(0, 0.1, generator=gen)
    return ckpt, model, tok, layers


@pytest.mark.parametrize("ragged", [False, True])
def test_a_step_on_pairs(tmp_path, oracle, ragged):
    """Reference without adapters, loss and adapter gradients of a 4-bit model against the same from elementary operations on its logits."""
    from alpaca_lora_4bit_amd import preference
    _, model, _, layers = _model(tmp_path, oracle)
    model.train()
    ids = torch.randint(3, 300, (6, 21), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    mask, labels = torch.ones_like(ids), ids.clone()
    labels[:, :5] = -100
    if ragged:
        for i, n in enumerate((21, 9, 5, 12, 21, 6)):
            mask[i, n:] = 0
            labels[i, n:] = -100
    labels = preference.shifted_labels(labels)
    params = [w for layer in layers.values() for w in (layer.lora_A["default"].weight, layer.lora_B["default"].weight)]

    def forward():
        with torch.amp.autocast("cuda", dtype=torch.float16):
            return model(input_ids=ids, attention_mask=mask, use_cache=False).logits
    with torch.no_grad(), preference.adapters_off(model):
        plain = forward()
        ref = preference.token_logps(plain, labels)
    assert not any(layer.disable_adapters for layer in layers.values())
    loss, rewards = preference.preference_loss(forward(), labels, ref, beta=0.5, label_smoothing=0.1)
    grads = torch.autograd.grad(loss * 1024, params)

    def sums(logits):
        lp = torch.log_softmax(logits.double(), -1).gather(-1, labels.clamp(min=0)[..., None])[..., 0]
        return torch.where(labels >= 0, lp, torch.zeros_like(lp)).sum(1)
    logits = forward()
    r = sums(logits) - sums(plain)
    z = 0.5 * (r[:3] - r[3:])
    want = -(0.9 * torch.nn.functional.logsigmoid(z) + 0.1 * torch.nn.functional.logsigmoid(-z)).mean()
    assert abs(float(loss) - float(want)) < 1e-4 and torch.allclose(rewards.double(), 0.5 * r, atol=1e-4) and float(z.abs().max()) > 1e-3
    # the same model runs backward from logit gradients that agree to one fp16 rounding
    for a, b in zip(grads, torch.autograd.grad(want * 1024, params)):
        assert float((a - b).abs().max()) <= 1e-2 * float(b.abs().max())


@pytest.mark.parametrize("chckpt,bits", [(False, 16), (True, 8), (False, 8)])
def test_finetune_module_on_pairs(tmp_path, oracle, monkeypatch, chckpt, bits):
    from safetensors.torch import load_file
    from alpaca_lora_4bit_amd import finetune
    ckpt = str(tmp_path / "ckpt")
    build(ckpt, oracle, seed=7, with_tokenizer=True)
    rnd = random.Random(4)
    say = lambda n: " ".join(rnd.choice(WORDS) for _ in range(n))
    data = str(tmp_path / "pairs.json")
    with open(data, "w") as fh:
        json.dump([{"prompt": say(3), "chosen": say(rnd.randint(1, 6)), "rejected": "the " * rnd.randint(2, 6)} for _ in range(30)], fh)
    out = str(tmp_path / "lora_out")
    packs, gated = _counted(monkeypatch, "act8_pack"), _counted(monkeypatch, "silu_mul_act8")
    model, _, trainer = finetune.main(
        [data, "--ds_type", "preference", "--llama_q4_config_dir", ckpt, "--llama_q4_model", os.path.join(ckpt, "model.safetensors"), "--groupsize", str(GROUPSIZE),
         "--lora_out_dir", out, "--mbatch_size", "4", "--batch_size", "8", "--epochs", "3", "--lr", "1e-3", "--cutoff_len", "48", "--warmup_steps", "1", "--logging_steps", "1",
         "--val_set_size", "6", "--beta", "0.2"] + (["--grad_chckpt"] if chckpt else []) + (["--act_bits", "8"] if bits == 8 else []))
    logs = [h for h in trainer.state.log_history if "loss" in h]
    evals = [h for h in trainer.state.log_history if "eval_loss" in h]
    assert len(logs) >= 6 and all(math.isfinite(h["loss"]) for h in logs + [{"loss": h["eval_loss"]} for h in evals]) and evals
    assert abs(logs[0]["loss"] - math.log(2)) < 1e-3           # adapters that add nothing yet: policy and reference are one; two micro-batches are averaged
    assert all("accuracy" in h and "margin" in h for h in logs) and all("eval_accuracy" in h for h in evals)
    lora = [m for m in model.modules() if "Linear4bitLt" in str(type(m))]
    assert len(lora) == 4 and all(float(m.lora_B["default"].weight.detach().abs().max()) > 0 and not m.disable_adapters for m in lora)
    assert bool(packs) == chckpt and bool(gated) == (bits == 8) and (None in gated) == (bits == 8)
    assert len(load_file(os.path.join(out, "adapter_model.safetensors"))) == 8
