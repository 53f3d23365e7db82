"""Values and keys at the top of fp16's range and beyond it: what append makes of the largest numbers, scales that a cache of the caller's own holds, keys that a rotation took
above fp16, and that no finite number of a later token reaches the rows before it."""
import math

import numpy as np
import pytest

from test_gpu_kv4 import _check, _cuda, _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,group", [(128, 128), (128, 32), (64, 64)])
def test_the_largest_numbers_come_back_finite(D, group):
    """Groups whose largest magnitude is fp16's largest number or one of the next below it: what is stored stays inside fp16's range, off by a 4-bit step at most, and
    attention over it is finite for one row and for many."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(D + group)
    n, tops = 70, [65504.0, -65504.0, 65472.0, -65440.0, 65408.0]
    k, v = (rng.standard_normal((n, 1, D)).astype(np.float16) * np.float16(1000) for _ in range(2))
    for i in range(n):
        for x in (k, v):
            x[i, 0, rng.integers(group):: group] = tops[i % 5]
    want = o.new_cache(5, 1, 16, D, group)
    table = np.arange(5, dtype=np.int32)[None]
    for i in range(n):
        (kq, ks), (vq, vs) = o.quantize(k[i, 0].astype(np.float32), group), o.quantize(v[i, 0].astype(np.float32), group)
        assert max(ks.max(), vs.max()) <= 10912
        o.put(want, i // 16, 0, i % 16, kq, ks, vq, vs)
    cache = tuple(_cuda(x) for x in o.new_cache(5, 1, 16, D, group))
    args = (cache, _cuda(table), torch.tensor([n], dtype=torch.int32).cuda())
    quant_hip.kv4_append(_cuda(k), _cuda(v), *args)
    for got, w in zip(cache, want):
        assert np.array_equal(got.cpu().numpy(), w, equal_nan=w.dtype == np.float16)
    for got, x in zip(quant_hip.kv4_read(*args, n), (k, v)):
        got = got.float().cpu().numpy()
        # half a step between 4 and 6 of a scale of 10912; the largest number itself is 32 off
        assert np.isfinite(got).all() and np.abs(got - x.astype(np.float32)).max() <= 10912
        assert (np.abs(got - x.astype(np.float32))[np.abs(x.astype(np.float32)) > 60000] <= 32).all()
    for rows in (1, n):
        q = (rng.standard_normal((rows, 1, D)) * 1e-4).astype(np.float16)
        ref, tol = o.attention(q, want, table, np.array([n]), None, 1 / math.sqrt(D), rows > 64)
        _check(quant_hip.kv4_attention(_cuda(q), *args), ref, tol, rows)



@pytest.mark.parametrize("scale", [10920.0, 20000.0, -65504.0])
@pytest.mark.parametrize("D,group,length,new", [(128, 128, 200, 200), (128, 32, 300, 130), (64, 64, 1300, 150), (64, 32, 150, 150), (128, 64, 80, 2)])
def test_finite_values_of_any_scale_count_for_the_rows_that_see_them_only(D, group, length, new, scale):
    """A value of code 6 at these scales passes fp16.  Rows that see it get it, those before it are as the formula has them."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(length + new)
    cache, table = _filled(o, [length], 1, D, group, 48, rng)
    at = length - new + new // 2
    cache[3][table[0, at // 48], 0, -1, at % 48] = scale
    q = (rng.standard_normal((new, 1, D)) * 0.3).astype(np.float16)
    want, tol = o.attention(q, cache, table, np.array([length]), None, 1 / math.sqrt(D), new > 64)
    assert np.abs(want).max() < 60000
    args = (tuple(_cuda(x) for x in cache), _cuda(table), torch.tensor([length], dtype=torch.int32).cuda())
    for bounds in (dict(max_length=64), dict(max_tokens=new, max_length=5000)):
        _check(quant_hip.kv4_attention(_cuda(q), *args, **bounds), want, tol, bounds)


@pytest.mark.parametrize("scale", [11784.0, 15448.0, -65504.0])
@pytest.mark.parametrize("D,group,length,new", [(128, 128, 1100, 100), (64, 32, 1300, 400), (128, 32, 300, 100), (64, 64, 1100, 1)])
def test_keys_of_any_finite_scale_give_finite_scores(D, group, length, new, scale):
    """Two coordinates of 50000 that a rotation turns into one of 70711: finite scores whether a row sees few keys or more than a thousand."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(length + new)
    cache, table = _filled(o, [length], 1, D, group, 48, rng)
    for at in (3, length - new // 2 - 1):
        cache[2][table[0, at // 48], 0, 0, at % 48] = scale
    q = (rng.standard_normal((new, 1, D)) / abs(scale)).astype(np.float16)
    want, tol = o.attention(q, cache, table, np.array([length]), None, 1 / math.sqrt(D), new > 64)
    args = (tuple(_cuda(x) for x in cache), _cuda(table), torch.tensor([length], dtype=torch.int32).cuda())
    for bounds in (dict(max_length=64), dict(max_tokens=new, max_length=5000)):
        _check(quant_hip.kv4_attention(_cuda(q), *args, **bounds), want, tol, bounds)


@pytest.mark.parametrize("new", [1, 40, 150])
def test_lengths_at_the_ends_of_32_bits(new):
    """Far below zero: no key is seen and nothing is stored.  Far beyond the table: it ends with the table."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(new)
    claimed = np.array([-2 ** 31, -2 ** 31 + new - 1, 2 ** 31 - 1, 2 ** 31 - 1 - new, 90], np.int64)
    cache, table = _filled(o, [90] * 5, 1, 64, 64, 16, rng)
    q = rng.standard_normal((5 * new, 1, 64)).astype(np.float16)
    want, tol = o.attention(q, cache, table, claimed, None, 0.125, new > 64)
    assert (want[:2 * new] == 0).all() and (want[2 * new:] != 0).any()
    args = (tuple(_cuda(x) for x in cache), _cuda(table), torch.from_numpy(claimed.astype(np.int32)).cuda())
    for bounds in (dict(), dict(max_tokens=new, max_length=5000)):
        _check(quant_hip.kv4_attention(_cuda(q), *args, **bounds), want, tol, bounds)
    k = torch.ones(5 * new, 1, 64, dtype=torch.float16, device="cuda")
    before = [c.clone() for c in args[0]]
    rope = torch.ones(8, 16, 2, device="cuda")
    got = quant_hip.kv4_append(k[:4 * new], k[:4 * new], args[0], args[1][:4].contiguous(), args[2][:4].contiguous(), q=k[:4 * new], rope=rope)
    assert bool((got == 0).all()) and all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip(before, args[0]))
    assert not any(bool(t.any()) for t in quant_hip.kv4_read(args[0], args[1][:4].contiguous(), args[2][:4].contiguous(), 4 * new))


def test_keys_below_the_normal_numbers_in_long_prompts():
    """Keys of some 1e-5 and queries that make scores of order one of them: rounded as eighths, a half step of 2^-22 each."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(5)
    length, new, D = 1200, 100, 64
    cache, table = _filled(o, [length], 1, D, 64, 48, rng)
    cache[2][:] = np.where(np.isnan(cache[2]), cache[2], np.float16(1e-5))
    q = (rng.standard_normal((new, 1, D)) * 2000).astype(np.float16)
    want, tol = o.attention(q, cache, table, np.array([length]), None, 1 / math.sqrt(D), True)
    got = quant_hip.kv4_attention(_cuda(q), tuple(_cuda(x) for x in cache), _cuda(table), torch.tensor([length], dtype=torch.int32).cuda())
    _check(got, want, tol)
