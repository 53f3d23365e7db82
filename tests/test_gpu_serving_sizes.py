"""The serving operators at the ends of their sizes: the smallest, the widest, banks and results beyond four gigabytes, many query heads on one key head."""
import math

import numpy as np
import pytest

from test_gpu_kv4 import _check, _cuda, _filled
from test_gpu_lora_rows import _bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N,R,n,per", [(1, 32, 64, 8, 1, 1), (5, 64, 64, 8, 2, 3), (2, 1 << 20, 64, 8, 1, 1), (3, 32, 1 << 20, 16, 2, 1), (257, 32, 64, 64, 3, 1)])
def test_smallest_and_widest_layers(M, K, N, R, n, per):
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    rng = np.random.default_rng(M + K + N)
    x = rng.standard_normal((M, K), dtype=np.float32).astype(np.float16)
    a = (rng.standard_normal((n, R, K), dtype=np.float32) / np.sqrt(K)).astype(np.float16)
    b, s = rng.standard_normal((n, N, R), dtype=np.float32).astype(np.float16), np.ones(n, np.float32)
    y, index = np.zeros((M, N), np.float16), rng.integers(0, n, -(-M // per)).astype(np.int32)
    want, tol = _bound(x, a, b, s, y, np.repeat(index, per)[:M])
    got = _cuda(y)
    quant_hip.lora_rows(_cuda(x), _cuda(index), [(_cuda(a), _cuda(b), _cuda(s), got)], per)
    assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol).all()


def test_banks_beyond_four_gigabytes():
    """The last of forty adapters of rank 64 on a layer of 2^20 -> 64, and on one of 64 -> 2^20."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    n, R, wide = 40, 64, 1 << 20
    rng = np.random.default_rng(0)
    for K, N in ((wide, 64), (64, wide)):
        x = rng.standard_normal((2, K), dtype=np.float32).astype(np.float16)
        a = (rng.standard_normal((1, R, K), dtype=np.float32) / np.sqrt(K)).astype(np.float16)
        b, s, y = rng.standard_normal((1, N, R), dtype=np.float32).astype(np.float16), np.ones(n, np.float32), np.zeros((2, N), np.float16)
        bank_a, bank_b = torch.zeros(n, R, K, dtype=torch.float16, device="cuda"), torch.zeros(n, N, R, dtype=torch.float16, device="cuda")
        bank_a[-1], bank_b[-1] = _cuda(a[0]), _cuda(b[0])
        want, tol = _bound(x, a, b, s, y, [0, -1])
        got = _cuda(y)
        quant_hip.lora_rows(_cuda(x), torch.tensor([n - 1, -1], dtype=torch.int32).cuda(), [(bank_a, bank_b, _cuda(s), got)])
        assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol).all()
        del bank_a, bank_b


def test_results_beyond_four_gigabytes():
    """Rows of a batch whose k, v, q and result pass 2^32 bytes: the last ones against the restatement, the ones before them belong to nobody and stay."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    T, hq, D = (1 << 17) + 40, 128, 128
    rng = np.random.default_rng(1)
    cache, table = _filled(o, [90], 1, D, 64, 16, rng)
    last = rng.standard_normal((70, hq, D)).astype(np.float16)
    q = torch.zeros(T, hq, D, dtype=torch.float16, device="cuda")
    q[-70:] = _cuda(last)
    starts = torch.tensor([T - 70, T], dtype=torch.int32).cuda()
    args = (tuple(_cuda(c) for c in cache), _cuda(table), torch.tensor([90], dtype=torch.int32).cuda())
    want, tol = o.attention(last, cache, table, np.array([90]), None, 1 / math.sqrt(D), True)
    out = torch.full_like(q, 3.0)
    for bounds in (dict(max_tokens=70, max_length=90), dict(max_tokens=70, max_length=2000)):
        got = quant_hip.kv4_attention(q, *args, starts=starts, out=out, **bounds)
        _check(got[-70:], want, tol, bounds)
        assert bool((got[:2] == 3.0).all()) and bool((got[-72:-70] == 3.0).all())
    out.fill_(3.0)
    rope = torch.zeros(128, 64, 2, device="cuda")
    rope[..., 0] = 1.0                                       # no turn: q comes out as it is
    k = torch.zeros(T, 1, D, dtype=torch.float16, device="cuda")
    k[-70:] = 6.0
    quant_hip.kv4_append(k, k, *args, q=q, rope=rope, starts=starts, q_out=out)
    assert torch.equal(out[-70:], q[-70:]) and bool((out[-72:-70] == 3.0).all())
    kk, vv = quant_hip.kv4_read(*args, T, starts=starts)
    assert torch.equal(kk, k) and torch.equal(vv, k)


@pytest.mark.parametrize("new", [1, 2])
def test_many_query_heads_on_one_key_head(new):
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(new)
    cache, table = _filled(o, [130, 5], 1, 64, 32, 64, rng)
    q = rng.standard_normal((2 * new, 48, 64)).astype(np.float16)
    want, tol = o.attention(q, cache, table, np.array([130, 5]), None, 0.125, new * 48 > 64)
    got = quant_hip.kv4_attention(_cuda(q), tuple(_cuda(c) for c in cache), _cuda(table), torch.tensor([130, 5], dtype=torch.int32).cuda())
    _check(got, want, tol)


def test_more_blocks_of_rows_than_a_launch_has_workgroups():
    """Twenty thousand sequences of one row each without a bound on their rows: the launch is sized for all rows in one sequence and has to take them in turns."""
    import torch
    from alpaca_lora_4bit_amd import kv4_cache, quant_hip
    B = 20000
    gen = torch.Generator(device="cuda").manual_seed(0)
    half = lambda *s: torch.randn(*s, generator=gen, device="cuda").half()
    cache = kv4_cache.new_layer(B, 4, 64, 16, 64)
    table = torch.randperm(B, generator=gen, device="cuda").int().view(B, 1)
    for n in (1, 2):
        quant_hip.kv4_append(half(B, 4, 64), half(B, 4, 64), cache, table, torch.full((B,), n, dtype=torch.int32, device="cuda"))
    lengths, starts = torch.full((B,), 2, dtype=torch.int32, device="cuda"), torch.arange(B + 1, dtype=torch.int32, device="cuda")
    q = half(B, 8, 64)
    want = quant_hip.kv4_attention(q, cache, table, lengths, starts=starts, max_tokens=1)
    got = quant_hip.kv4_attention(q, cache, table, lengths, starts=starts)
    # two weights and two values, each rounded once more (2^-11 of values up to 6), and the results (2^-11)
    assert float((got.float() - want.float()).abs().max()) <= 4 * 6 * 2 ** -11
