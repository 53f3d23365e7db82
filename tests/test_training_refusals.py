"""What the training operators' C entries refuse, without a GPU, and the oracle they are tested with against elementary formulas."""
import ctypes

import numpy as np
import pytest

FAKE, ODD = 0x1000, 0x1004                       # aligned and not; never dereferenced


def _kept(codes=FAKE, scales=FAKE):
    from alpaca_lora_4bit_amd import _lib
    return ctypes.byref(_lib.Act8(codes=codes, scales=scales))


def test_packing_arguments():
    from alpaca_lora_4bit_amd import _lib
    L = _lib.lib()
    for f in (lambda x=FAKE, t=0, c=FAKE, s=FAKE, n=64: L.q4_act8_pack(x, t, c, s, n, None), lambda x=FAKE, t=0, c=FAKE, s=FAKE, n=64: L.q4_act8_unpack(c, s, x, t, n, None)):
        assert f(x=None) == f(c=None) == f(s=None) == -1
        assert f(t=3) == f(t=-1) == f(n=0) == f(n=-5) == f(n=1 << 35) == -2
        assert f(x=ODD) == f(c=ODD) == f(s=ODD) == -5


def test_gated_activation_arguments():
    from alpaca_lora_4bit_amd import _lib
    L = _lib.lib()
    for f in (lambda a=FAKE, b=FAKE, t=0, o=FAKE, g=_kept(), u=_kept(), n=64: L.q4_silu_mul_act8(a, b, t, o, g, u, n, None),
              lambda a=FAKE, b=FAKE, t=0, o=FAKE, g=_kept(), u=_kept(), n=64: L.q4_silu_mul_act8_bwd(a, t, g, u, b, o, n, None)):
        assert f(a=None) == f(b=None) == f(o=None) == f(g=None) == f(u=None) == f(g=_kept(codes=None)) == f(u=_kept(scales=None)) == -1
        assert f(t=2) == f(t=7) == f(n=0) == f(n=1 << 36) == -2
        assert f(a=ODD) == f(b=ODD) == f(o=ODD) == f(g=_kept(scales=ODD)) == f(u=_kept(codes=ODD)) == -5


def test_answers_arguments():
    from alpaca_lora_4bit_amd import _lib
    L = _lib.lib()

    def fwd(x=FAKE, t=0, sb=100, st=10, B=2, S=10, V=10, lab=FAKE, lp=FAKE, stats=FAKE):
        return L.q4_token_logps(x, t, sb, st, B, S, V, lab, lp, stats, None)

    def bwd(x=FAKE, t=0, sb=100, st=10, B=2, S=10, V=10, lab=FAKE, stats=FAKE, coef=FAKE, per=10, factor=None, dx=FAKE):
        return L.q4_token_logps_bwd(x, t, sb, st, B, S, V, lab, stats, coef, per, factor, dx, None)

    def loss(x=FAKE, t=0, sb=100, st=10, P=2, S=10, V=10, lab=FAKE, ref=FAKE, beta=0.1, eps=0.0, out=FAKE, rew=FAKE, coef=FAKE, stats=FAKE, ws=FAKE, nb=1 << 20):
        return L.q4_preference_loss(x, t, sb, st, P, S, V, lab, ref, beta, eps, out, rew, coef, stats, ws, nb, None)
    for f in (fwd, bwd, loss):
        assert f(x=None) == f(lab=None) == f(stats=None) == -1
        assert f(t=3) == f(S=0) == f(V=0) == f(V=1 << 30) == f(sb=-1) == f(st=-1) == f(S=2 ** 31 - 1) == -2
        assert f(x=0x1001) == f(lab=ODD) == f(stats=ODD) == -5
    assert fwd(lp=None) == bwd(coef=None) == bwd(dx=None) == -1 and fwd(B=0) == bwd(per=0) == bwd(per=3) == -2
    assert bwd(dx=ODD) == bwd(factor=0x1002) == fwd(lp=0x1001) == -5
    assert loss(ref=None) == loss(out=None) == loss(rew=None) == loss(coef=None) == -1
    assert loss(P=0) == loss(P=2 ** 30) == loss(beta=0.0) == loss(beta=float("nan")) == loss(beta=float("inf")) == loss(eps=-0.1) == loss(eps=0.51) == -2
    need = L.q4_preference_loss_workspace_bytes(2, 10)
    assert need == 16 * (2 + 20) and loss(ws=None) == loss(nb=need - 1) == -3 and loss(ws=ODD) == -5
    assert L.q4_preference_loss_workspace_bytes(0, 4) == L.q4_preference_loss_workspace_bytes(2, 2 ** 30) == 0


def test_calls_on_the_cpu_are_refused():
    import torch
    from alpaca_lora_4bit_amd import preference, quant_hip
    z, lab = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long)
    for f in (lambda: quant_hip.act8_pack(z), lambda: quant_hip.silu_mul_act8(z.half(), z.half()), lambda: preference.token_logps(z, lab),
              lambda: preference.preference_loss(z, lab, torch.zeros(2, 3))):
        with pytest.raises(ValueError):
            f()


def test_the_oracle():
    import torch
    from oracle import training_oracle as o
    for k in range(-140, 100, 7):                              # the scale's definition, by walking over neighbouring bfloat16 values
        for m in (1.0, 1.3, 127 / 128, 1.9921875, 127 / 64):
            top = float(np.float32(m * 2.0 ** k))
            s = float(o.least_scale(top))
            bits = torch.tensor(s, dtype=torch.float64).to(torch.bfloat16).view(torch.int16)
            assert float(bits.view(torch.bfloat16)) == s and 127 * s >= top and 127 * float((bits - 1).view(torch.bfloat16)) < top
    x = np.random.RandomState(0).randn(3, 50)
    q, s = o.act8(x)
    assert np.abs(q).max() <= 127 and (np.abs(o.held(x) - x) <= np.repeat(s, 32)[:150].reshape(3, 50) / 2).all()
    t = torch.randn(4, 6, 9, dtype=torch.float64, requires_grad=True)
    lab = torch.randint(0, 9, (4, 6))
    lab[0, 2:] = -100
    logps = torch.where(lab >= 0, torch.log_softmax(t, -1).gather(-1, lab.clamp(min=0)[..., None])[..., 0], torch.zeros(()).double())
    ref = torch.randn(4, 6, dtype=torch.float64)
    r = torch.where(lab >= 0, logps - ref, torch.zeros(()).double()).sum(-1)
    z = 0.3 * (r[:2] - r[2:])
    loss = -(0.9 * torch.nn.functional.logsigmoid(z) + 0.1 * torch.nn.functional.logsigmoid(-z)).mean()
    loss.backward()
    lp, soft = o.token_logps(t.detach().numpy(), lab.numpy())
    mine, rewards, coef = o.preference(lp, ref.numpy(), lab.numpy(), 9, 0.3, 0.1)
    assert np.allclose(lp, logps.detach().numpy(), atol=1e-13) and np.isclose(mine, float(loss.detach()), atol=1e-13) and np.allclose(rewards, 0.3 * r.detach().numpy(), atol=1e-12)
    assert np.allclose(o.logits_grad(soft, lab.numpy(), np.repeat(coef[:, None], 6, 1)), t.grad.numpy(), atol=1e-13)
    g = torch.randn(5, 7, dtype=torch.float64, requires_grad=True)
    u = torch.randn(5, 7, dtype=torch.float64, requires_grad=True)
    d = torch.randn(5, 7, dtype=torch.float64)
    (torch.nn.functional.silu(g) * u).backward(d)
    dg, du = o.silu_mul_bwd(d.numpy(), g.detach().numpy(), u.detach().numpy())
    assert np.allclose(dg, g.grad.numpy(), atol=1e-13) and np.allclose(du, u.grad.numpy(), atol=1e-13)
