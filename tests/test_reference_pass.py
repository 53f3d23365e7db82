"""The pass of the reference model: the model without its adapters, as in evaluation, and everything as it was afterwards (CPU)."""
import pytest
import torch
import torch.nn as nn


def _lora(**kw):
    from alpaca_lora_4bit_amd.models import Linear4bitLt
    return Linear4bitLt("default", 128, 128, 128, False, r=8, lora_alpha=16, **kw)


def test_the_reference_has_no_dropout():
    """Dropout of the host model would make each pass of the reference another one."""
    from alpaca_lora_4bit_amd.preference import adapters_off

    class Host(nn.Module):
        def __init__(self):
            super().__init__()
            self.q_proj, self.drop, self.still = _lora(lora_dropout=0.1), nn.Dropout(0.5), nn.Dropout(0.5)

        def forward(self, x):
            return nn.functional.dropout(self.drop(x), 0.5, self.training)
    model = Host().train()
    model.still.eval()
    modes = [m.training for m in model.modules()]
    x = torch.ones(4096)
    with pytest.raises(KeyError), adapters_off(model) as same:
        assert same is model and torch.equal(model(x), x) and not any(m.training for m in model.modules())
        raise KeyError
    assert [m.training for m in model.modules()] == modes and not model.still.training and not torch.equal(model(x), x)
    model.eval()
    with adapters_off(model):
        pass
    assert not any(m.training for m in model.modules())


def test_a_model_without_adapters_is_refused():
    """Policy and reference would be one and the same, and the loss log 2 for good."""
    from alpaca_lora_4bit_amd.preference import adapters_off
    for model in (nn.Sequential(nn.Linear(3, 3)), nn.Linear(3, 3)):
        with pytest.raises(ValueError, match="adapter"), adapters_off(model):
            raise KeyError
    layer = _lora()                                            # the model may be one layer
    with adapters_off(layer):
        assert layer.disable_adapters


def test_frozen_adapters_stay_frozen():
    """Layers whose switch also decides what is trained: off freezes the adapters, on makes the active ones trainable."""
    from alpaca_lora_4bit_amd.preference import adapters_off

    class Switched(nn.Module):
        def __init__(self):
            super().__init__()
            self.lora_A, self.lora_B = nn.ModuleDict({"a": nn.Linear(4, 2), "b": nn.Linear(4, 2)}), nn.ModuleDict({"a": nn.Linear(2, 4), "b": nn.Linear(2, 4)})
            self.disable_adapters = False

        def enable_adapters(self, enabled):
            self.disable_adapters = not enabled
            for part in (self.lora_A, self.lora_B):
                for name, layer in part.items():
                    layer.requires_grad_(enabled and name == "a")
    frozen, other, trained = Switched(), Switched(), Switched()
    for p in frozen.parameters():
        p.requires_grad_(False)
    other.enable_adapters(False)
    other.lora_B["b"].weight.requires_grad_(True)
    model = nn.ModuleList([frozen, other, trained])
    before = [p.requires_grad for p in model.parameters()]
    with pytest.raises(KeyError), adapters_off(model):
        assert all(m.disable_adapters for m in model)
        raise KeyError
    assert [p.requires_grad for p in model.parameters()] == before
    assert [m.disable_adapters for m in model] == [False, True, False]


def test_labels_of_no_place_stay_of_no_place():
    from alpaca_lora_4bit_amd.preference import shifted_labels
    for shape in ((3, 0), (0, 4), (2, 0, 0), (0,)):
        moved = shifted_labels(torch.zeros(shape, dtype=torch.long))
        assert moved.shape == shape and moved.dtype == torch.long
    base = torch.arange(24).view(2, 3, 4)
    assert shifted_labels(base).tolist() == [[[*row[1:], -100] for row in part] for part in base.tolist()]
    assert torch.equal(shifted_labels(base.transpose(1, 2))[..., :2], base.transpose(1, 2)[..., 1:])
