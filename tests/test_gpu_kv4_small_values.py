"""One token over a long cache of small values: what rounding the weights (2^10 * p * scale, to fp16) costs, with a bound that does not grow by the number of keys."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("spread", [1.0, 3.0])
def test_small_values_keep_the_accuracy_of_the_result(size, spread):
    """Values of a mean and a deviation of `size`, scores of a deviation of `spread`, 50000 keys.  Every weight is off by half a step of its fp16 number at most, one
    way or the other: their sum by six times the root of the sum of their squares (2e-9 of all elements lie outside 6 deviations of a normal sum, and half a step is
    more than a deviation, which is 0.58 of it).  To it the output's own half step (2^-11, 2^-25 below the normal numbers) and the float32 terms of scores and sums, as in the oracle."""
    import torch
    from alpaca_lora_4bit_amd import kv4_cache, quant_hip
    from oracle import kv4_oracle as o
    L, D, heads, page, u = 50000, 64, 2, 256, 2.0 ** -24
    gen = torch.Generator(device="cuda").manual_seed(int(spread) + int(-math.log10(size)))
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    cache = kv4_cache.new_layer(-(-L // page), heads, D, page, D)
    table = torch.arange(-(-L // page), dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([L], dtype=torch.int32, device="cuda")
    quant_hip.kv4_append(normal(L, heads, D).half(), ((normal(L, heads, D) + 1) * size).half(), cache, table, lengths)
    q = (normal(1, heads, D) * spread).half()
    got = quant_hip.kv4_attention(q, cache, table, lengths)[0].double().cpu().numpy()
    host, at = [c.cpu().numpy() for c in cache], np.arange(L)
    for h in range(heads):
        k, v = o.get(host, at // page, h, at % page)
        scale = host[3][at // page, h, 0, at % page].astype(np.float64)
        x = q[0, h].double().cpu().numpy()
        s = (k @ x) / math.sqrt(D)
        p = np.exp(s - s.max())
        weight, total = 2.0 ** 10 * p * scale, 2.0 ** 10 * p.sum()
        half_step = np.maximum(2.0 ** (np.floor(np.log2(np.maximum(weight, 2.0 ** -40))) - 11), 2.0 ** -25)
        codes = v / scale[:, None]
        want = (weight @ codes) / total
        mag = (np.abs(k) @ np.abs(x)).max() / math.sqrt(D)
        eps = mag * (D + 8) * u + 4 * np.abs(s).max() * u + 4 * u
        tol = (2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 6 * np.sqrt((half_step ** 2) @ (codes ** 2)) / total
               + (np.expm1(2 * eps) + (L / 32 + 64) * 2 * u) * (p @ np.abs(v)) / p.sum())
        assert (np.abs(got[h] - want) <= tol).all()
