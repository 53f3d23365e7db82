"""The serving operators have no forward mode: tangents are refused, with gradients enabled or not, and so are gradients of what only scales."""
import pytest

from test_gpu_serving_refusals import _batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_and_gradients_are_refused(grad):
    import torch
    import torch.autograd.forward_ad as fw
    from alpaca_lora_4bit_amd import quant_hip as qh
    cache, table, lengths, q, k, v = _batch()
    rope = torch.zeros(64, 32, 2, device="cuda")
    x, index = torch.zeros(4, 64, dtype=torch.float16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    a, b = torch.zeros(2, 8, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 64, 8, dtype=torch.float16, device="cuda")
    s, y = torch.ones(2, device="cuda"), torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    append = lambda q=q, k=k, v=v, rope=rope, cache=cache: qh.kv4_append(k, v, cache, table, lengths, q=q, rope=rope)
    attend = lambda q=q, cache=cache: qh.kv4_attention(q, cache, table, lengths)
    rows = lambda x=x, a=a, b=b, s=s, y=y: qh.lora_rows(x, index, [(a, b, s, y)])
    with_scales = lambda t: (cache[0], cache[1], cache[2], t)
    calls = [lambda d: append(q=d(q)), lambda d: append(k=d(k)), lambda d: append(v=d(v)), lambda d: append(rope=d(rope)), lambda d: append(cache=with_scales(d(cache[3]))),
             lambda d: attend(q=d(q)), lambda d: attend(cache=with_scales(d(cache[3]))), lambda d: rows(x=d(x)), lambda d: rows(a=d(a)), lambda d: rows(b=d(b)),
             lambda d: rows(s=d(s)), lambda d: rows(y=d(y.clone()))]
    with torch.set_grad_enabled(grad), fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        for i, call in enumerate(calls):
            with pytest.raises(ValueError, match="tangent"):
                call(dual)
                pytest.fail(f"call {i} was taken")
        with fw._set_fwd_grad_enabled(False):                 # tangents are not asked for: taken
            attend(q=dual(q))
    for i, call in enumerate(calls):
        if grad:
            with pytest.raises(ValueError, match="requires grad"):
                call(lambda t: t.detach().clone().requires_grad_())
                pytest.fail(f"call {i} was taken with a gradient")
    append(), attend(), rows()
