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


def _parts(model):
    return {"root": model, "net": model.model, "block": model.model.layers[1], "attn": model.model.layers[0].self_attn, "mlp": model.model.layers[1].mlp}


@pytest.mark.parametrize("where", ["root", "net", "block", "attn", "mlp"])
@pytest.mark.parametrize("how", ["hook", "pre_hook", "forward", "class"])
def test_hooks_and_forwards_that_a_batch_would_leave_out(monkeypatch, where, how):
    """A hook or another forward on a module whose parts are run in its place is an error; on the MLP only where its parts have adapters, for it is called else."""
    Plain(monkeypatch)
    model = _model()
    module, called = _parts(model)[where], []
    if how == "hook":
        module.register_forward_hook(lambda m, a, out: called.append(1))
    elif how == "pre_hook":
        module.register_forward_pre_hook(lambda m, a: called.append(1))
    elif how == "forward":
        own = module.forward
        module.forward = lambda *a, **kw: (called.append(1), own(*a, **kw))[1]
    else:
        stock = type(module).forward
        monkeypatch.setattr(type(module), "forward", lambda self, *a, **kw: (called.append(1), stock(self, *a, **kw))[1])
    run = lambda *bank: inference.generate_batch(model, PROMPTS[:2], 3, *bank, use_graph=False)
    if where == "mlp":
        assert len(run()) == 2 and called
        bank = models.AdapterBank(model, _adapters(model, [("down_proj",)], (8,), 1), device="cpu")
        with pytest.raises(ValueError, match="mlp"):
            run(bank, [0, 0])
    else:
        with pytest.raises(ValueError, match="model"):
            run()
    assert called or where != "mlp"


def test_hooks_on_what_a_batch_calls_are_called(monkeypatch):
    Plain(monkeypatch)
    model, called = _model(), []
    net = model.model
    for m in (net.embed_tokens, net.layers[0].input_layernorm, net.layers[0].self_attn.q_proj, net.layers[1].mlp.up_proj, net.norm, model.lm_head):
        m.register_forward_hook(lambda m, a, out: called.append(m))
    inference.generate_batch(model, PROMPTS[:1], 1, use_graph=False)
    assert len(called) == 6


def test_the_packages_own_wrappers_are_taken(monkeypatch):
    from alpaca_lora_4bit_amd.amp_wrapper import AMPWrapper
    from alpaca_lora_4bit_amd.gradient_checkpointing import apply_gradient_checkpointing
    Plain(monkeypatch)
    model = _model()
    want = [t.tolist() for t in inference.generate_batch(model, PROMPTS, 3, use_graph=False)]
    AMPWrapper(model).apply_forward()
    AMPWrapper(model).apply_generate()
    apply_gradient_checkpointing(model)
    assert [t.tolist() for t in inference.generate_batch(model, PROMPTS, 3, use_graph=False)] == want
    own = model.forward
    model.forward = lambda *a, **kw: own(*a, **kw)           # somebody else's around the package's
    with pytest.raises(ValueError, match="replaced"):
        inference.generate_batch(model, PROMPTS, 3, use_graph=False)
    model.forward = own
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, out: None)
    try:
        with pytest.raises(ValueError, match="global"):
            inference.generate_batch(model, PROMPTS, 3, use_graph=False)
    finally:
        handle.remove()
