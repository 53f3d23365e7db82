"""Which MLP blocks `make_fused_mlp(act_bits=8)` marks, counts and names (CPU: nothing runs)."""
import pytest
import torch
import torch.nn as nn


class Block(nn.Module):
    def __init__(self, groupsize=-1, act=None, sizes=(128, 128), bits=4):
        from alpaca_lora_4bit_amd.autograd_4bit import Autograd4bitQuantLinear
        super().__init__()
        H, I = 256, 512
        self.act_fn = nn.SiLU() if act is None else act
        self.gate_proj, self.up_proj = (Autograd4bitQuantLinear(H, I, groupsize=groupsize, bits=bits) for _ in range(2))
        self.down_proj = Autograd4bitQuantLinear(I, H, groupsize=groupsize, bits=bits)

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Doubled(Block):
    def forward(self, x):
        return 2 * self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


def _marked(block):
    return block.__dict__.get("_q4_act_bits") == 8


@pytest.mark.parametrize("groupsize", [-1, 64, 128])
def test_blocks_of_any_group_size_are_marked(groupsize):
    """-1 is a group of each layer's own width: gate's and down's differ."""
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp, ungroup
    model = nn.ModuleList([Block(groupsize) for _ in range(3)])
    assert make_fused_mlp(model, act_bits=8) == 3 and all(_marked(b) for b in model)
    assert make_fused_mlp(model, act_bits=8) == 3              # what is marked, not what this call has changed
    ungroup(model)
    assert not any("forward" in b.__dict__ or _marked(b) for b in model)


def test_blocks_that_keep_their_operands_are_not_counted_and_are_named():
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    replaced, mixed = Block(128), Block(128)
    inner = replaced.forward
    replaced.forward = lambda x: inner(x)                      # as where something else has put its own forward in place
    mixed.up_proj = nn.Linear(256, 512)
    model = nn.ModuleDict({"gelu": Block(128, act=nn.GELU()), "doubled": Doubled(128), "replaced": replaced, "mixed": mixed, "two_bits": Block(128, bits=2), "fine": Block(128)})
    with pytest.warns(UserWarning) as said:
        assert make_fused_mlp(model, act_bits=8) == 1
    assert [n for n, b in model.items() if _marked(b)] == ["fine"]
    text = str(said[0].message)
    assert len(said) == 1 and "5 MLP blocks" in text and all(n in text for n in ("gelu", "doubled", "replaced", "mixed", "two_bits")) and "fine" not in text


def test_a_block_that_an_earlier_call_has_grouped():
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    for first in (dict(), dict(fuse_decode_step=False)):
        for groupsize in (128, -1):
            block = Block(groupsize)
            assert make_fused_mlp(block, **first) == 1 and not _marked(block)
            assert make_fused_mlp(block, act_bits=8) == 1 and _marked(block)


def test_a_group_size_of_its_own_leaves_the_decode_step_out():
    """The one-launch step takes one group size for the three layers; a block marked in spite of that does not get it."""
    from alpaca_lora_4bit_amd import model_attn_mlp_patch as patch
    same, own = Block(128), Block(-1)
    patch.make_fused_mlp(nn.ModuleList([same, own]), act_bits=8)
    assert same.forward.__func__ is patch._mlp_decode_forward and own.forward.__func__ is not patch._mlp_decode_forward


def test_without_the_option_nothing_has_changed():
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    model = nn.ModuleList([Block(128), Block(-1), Block(128, act=nn.GELU())])
    assert make_fused_mlp(model) == 3 and make_fused_mlp(model) == 0
    assert ["forward" in b.__dict__ for b in model] == [True, False, False]


def test_16_bits_can_be_asked_for_again():
    from alpaca_lora_4bit_amd import model_attn_mlp_patch as patch
    model = nn.ModuleList([Block(128), Block(-1)])
    assert patch.make_fused_mlp(model, act_bits=8) == 2
    assert patch.make_fused_mlp(model, act_bits=16) == 2 and not any(_marked(b) for b in model)
    assert model[0].forward.__func__ is patch._mlp_decode_forward and "forward" not in model[1].__dict__          # as without the option
    assert patch.make_fused_mlp(model) == 0
    assert patch.make_fused_mlp(model, act_bits=8) == 2 and all(_marked(b) for b in model)


@pytest.mark.parametrize("groupsize", [-1, 128])
def test_a_batch_of_requests_takes_marked_blocks_apart(groupsize):
    """Their forward in place of the block's own changes nothing that a batch would leave out."""
    from transformers import LlamaConfig, LlamaForCausalLM
    from alpaca_lora_4bit_amd.autograd_4bit import find_layers, make_quant_for_4bit_autograd
    from alpaca_lora_4bit_amd.inference import _passed_by
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    model = LlamaForCausalLM(LlamaConfig(vocab_size=97, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=4))
    layers = find_layers(model)
    del layers["lm_head"]
    make_quant_for_4bit_autograd(model, layers, groupsize=groupsize)
    for bits in (8, 16, 8):
        assert make_fused_mlp(model, act_bits=bits) == 2
        assert all(_marked(b.mlp) == (bits == 8) and _passed_by(b.mlp, "LlamaMLP") is None for b in model.model.layers)
    mlp = model.model.layers[0].mlp
    mlp.forward = lambda x, inner=mlp.forward: inner(x)
    assert _passed_by(mlp, "LlamaMLP") == "a replaced forward"
