"""MLP blocks that keep 8 bits, on the GPU: layers of any group sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H, I = 256, 512


def _block(oracle, groupsize, seed=40):
    import torch.nn as nn
    from conftest import to_cuda_layer
    from alpaca_lora_4bit_amd.autograd_4bit import Autograd4bitQuantLinear

    class Gated(nn.Module):
        def __init__(self):
            super().__init__()
            self.act_fn = nn.SiLU()

        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))
    block = Gated()
    for i, (name, k, n) in enumerate((("gate_proj", H, I), ("up_proj", H, I), ("down_proj", I, H))):
        lin = Autograd4bitQuantLinear(k, n, groupsize=groupsize)
        for key, v in to_cuda_layer(oracle.make_layer(k, n, lin.groupsize, seed=seed + i)).items():
            if isinstance(v, torch.Tensor):
                setattr(lin, key, v)
        lin.bias = torch.zeros(n, dtype=torch.float16, device="cuda")
        setattr(block, name, lin)
    return block


def _counted(monkeypatch, name):
    from alpaca_lora_4bit_amd import quant_hip
    seen, real = [], getattr(quant_hip, name)

    def call(*a, **kw):
        seen.append(tuple(a[0].shape) if kw.get("keep", True) else None)
        return real(*a, **kw)
    monkeypatch.setattr(quant_hip, name, call)
    return seen


def _x(oracle, rows, seed=4):
    return torch.from_numpy(oracle.make_activations(rows, H, seed=seed)).cuda()


@pytest.mark.parametrize("groupsize", [-1, 128])
def test_a_block_keeps_8_bits_whatever_its_groups(oracle, monkeypatch, groupsize):
    """Layers of one group a column too (gate's as wide as its input, down's as its own): outputs of the block's own forward to fp16's roundings, half as much kept."""
    from conftest import rel_err
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    rows = 640
    own, marked = _block(oracle, groupsize), _block(oracle, groupsize)
    assert make_fused_mlp(marked, act_bits=8) == 1
    kept, backs = _counted(monkeypatch, "silu_mul_act8"), _counted(monkeypatch, "silu_mul_act8_bwd")
    xh, dy = _x(oracle, rows), _x(oracle, rows, 5)

    def run(block):
        x = xh.clone().requires_grad_(True)
        before = torch.cuda.memory_allocated()
        with torch.amp.autocast("cuda", dtype=torch.float16):
            y = block(x)
        held = torch.cuda.memory_allocated() - before
        y.backward(dy)
        return y.detach(), x.grad, held
    run(own), run(marked)                                      # allocations of the first calls
    kept.clear(), backs.clear()
    want, got = run(own), run(marked)
    assert kept == backs == [(rows, I)]
    # sums over 512 products of intermediates one fp16 rounding apart
    assert rel_err(got[0].cpu().numpy(), want[0].double().cpu().numpy()) <= 3e-3
    assert torch.isfinite(got[1]).all() and want[2] - got[2] > 0.9 * rows * I * (2 * 2 - 2 * 1.0625)
    with torch.no_grad():
        kept.clear()
        assert marked(xh[:1]).shape == (1, H) and marked(xh[:12]).shape == (12, H)
        assert rel_err(marked(xh[:1]).cpu().numpy(), want[0][:1].double().cpu().numpy()) <= 3e-3


def _then(block, change):
    """gate's and up's outputs go through `change`."""
    for lin in (block.gate_proj, block.up_proj):
        lin.forward = lambda x, own=lin.forward: change(own(x))


@pytest.mark.parametrize("kind", ["bfloat16", "columns"])
def test_operands_of_bfloat16_and_cut_out_of_others_are_kept_in_8_bits(oracle, monkeypatch, kind):
    """Layers whose outputs are bfloat16, or columns of a wider tensor: the block's gradient is that of the operators by themselves."""
    from alpaca_lora_4bit_amd import quant_hip
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    block = _block(oracle, 128)
    _then(block, lambda y: y.bfloat16() if kind == "bfloat16" else torch.cat([y, y], -1)[..., :I])
    down = block.down_proj.forward
    block.down_proj.forward = lambda act: down(act.half())
    assert make_fused_mlp(block, act_bits=8) == 1
    kept = _counted(monkeypatch, "silu_mul_act8")
    x = _x(oracle, 200).requires_grad_(True)
    dy = _x(oracle, 200, 5)
    y = block(x)
    assert kept == [(200, I)]
    (got,) = torch.autograd.grad(y, x, dy.to(y.dtype))
    gate, up = block.gate_proj(x), block.up_proj(x)
    out, held = quant_hip.silu_mul_act8(gate.detach(), up.detach())
    act = out.requires_grad_(True)
    again = block.down_proj(act)
    assert torch.equal(y, again)
    (dact,) = torch.autograd.grad(again, act, dy.to(y.dtype))
    (want,) = torch.autograd.grad([gate, up], x, list(quant_hip.silu_mul_act8_bwd(dact, held)))
    assert torch.equal(got, want)
    kept.clear()
    with torch.no_grad():
        assert torch.equal(block(x), y) and kept == [None]


def test_operands_of_float32_are_kept_as_they_are_and_said_so(oracle, monkeypatch):
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    block = _block(oracle, 128)
    _then(block, torch.Tensor.float)
    assert make_fused_mlp(block, act_bits=8) == 1
    kept = _counted(monkeypatch, "silu_mul_act8")
    x = _x(oracle, 200).requires_grad_(True)
    with pytest.warns(UserWarning, match="float32"), torch.amp.autocast("cuda", dtype=torch.float16):
        y = block(x)
    y.float().sum().backward()
    assert not kept and torch.isfinite(x.grad).all()


@pytest.mark.parametrize("rows", [1, 3, 12])
@pytest.mark.parametrize("groupsize", [-1, 128])
def test_a_few_rows_take_the_same_product_with_and_without_gradients(oracle, monkeypatch, rows, groupsize):
    """The policy's pass runs with gradients, the reference's without: gate's and up's product is the same at the sizes of the one-launch decode step too."""
    from conftest import rel_err
    from alpaca_lora_4bit_amd import quant_hip
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    block = _block(oracle, groupsize)
    make_fused_mlp(block, act_bits=8)
    kept, products = _counted(monkeypatch, "silu_mul_act8"), []
    block.down_proj.register_forward_pre_hook(lambda m, args: products.append(args[0].detach()))
    x = _x(oracle, rows)
    for training in (True, False):
        block.train(training)
        kept.clear(), products.clear()
        with torch.amp.autocast("cuda", dtype=torch.float16):
            y = block(x.clone().requires_grad_(True))
        with torch.no_grad():
            again = block(x)
        assert kept == [(rows, I), None]
        gate, up = block.gate_proj(x), block.up_proj(x)
        want = quant_hip.silu_mul_act8(gate.detach(), up.detach(), keep=False)[0]
        # sums over 256 products in another order: gate and up a step (2^-10) apart at most, and the product half a step more
        assert rel_err(products[1].cpu().numpy(), want.double().cpu().numpy()) <= 3e-3 and rel_err(products[0].cpu().numpy(), want.double().cpu().numpy()) <= 3e-3
        assert rel_err(again.cpu().numpy(), y.detach().double().cpu().numpy()) <= 3e-3
    make_fused_mlp(block, act_bits=16)
    kept.clear()
    block.down_proj._forward_pre_hooks.clear()
    with torch.no_grad():
        assert rel_err(block(x).cpu().numpy(), y.detach().double().cpu().numpy()) <= 3e-3 and not kept
