"""Prompts over the 4-bit cache where their kernel takes another way: rows that see few keys and rows that see many, more sequences than are sorted by length, shares of
the keys, values that are no numbers in both."""
import math

import numpy as np
import pytest

from test_gpu_kv4 import _check, _cuda, _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
def test_rows_on_either_side_of_a_thousand_keys(D, group):
    """Blocks of rows below 1024 keys, across it and above it, of a long sequence and a short one, whole and in shares."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(D + group)
    lengths, new = [1250, 300], [400, 130]
    cache, table = _filled(o, lengths, 1, D, group, 48, rng)
    starts = np.cumsum([0] + new).astype(np.int32)
    q = (rng.standard_normal((int(starts[-1]), 1, D)) * 2).astype(np.float16)
    want, tol = o.attention(q, cache, table, np.array(lengths), starts, 1 / math.sqrt(D), True)
    args = (tuple(_cuda(x) for x in cache), _cuda(table), torch.tensor(lengths, dtype=torch.int32).cuda())
    for bounds in (dict(max_tokens=400, max_length=1250), dict(max_tokens=400, max_length=64), dict(max_tokens=130, max_length=5000)):
        got = quant_hip.kv4_attention(_cuda(q), *args, starts=_cuda(starts), **bounds)
        _check(got, want, tol, bounds)
        assert torch.equal(got, quant_hip.kv4_attention(_cuda(q), *args, starts=_cuda(starts), **bounds))


@pytest.mark.parametrize("count", [64, 66])
def test_many_short_prompts(count):
    """Up to 64 sequences are taken by their length, more in turns; some of no rows, some of no keys."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(count)
    new = [int(n) for n in rng.integers(0, 12, count)]
    new[3], new[10] = 12, 0
    lengths = [n + int(x) for n, x in zip(new, rng.integers(0, 40, count))]
    lengths[5] = 0
    cache, table = _filled(o, lengths, 1, 64, 64, 16, rng)
    starts = np.cumsum([0] + new).astype(np.int32)
    q = rng.standard_normal((int(starts[-1]), 6, 64)).astype(np.float16)
    want, tol = o.attention(q, cache, table, np.array(lengths), starts, 0.125, True)
    args = (tuple(_cuda(x) for x in cache), _cuda(table), torch.tensor(lengths, dtype=torch.int32).cuda())
    _check(quant_hip.kv4_attention(_cuda(q), *args, starts=_cuda(starts), max_tokens=12, max_length=52), want, tol)


@pytest.mark.parametrize("length", [900, 1500])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(length):
    """A key's or a value's scale that is infinite or NaN makes every row that sees it no number and leaves the rows before it as they were."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(length)
    cache, table = _filled(o, [length], 1, 128, 32, 16, rng)
    q = rng.standard_normal((200, 1, 128)).astype(np.float16)
    lengths = torch.tensor([length], dtype=torch.int32).cuda()
    clean = quant_hip.kv4_attention(_cuda(q), tuple(_cuda(x) for x in cache), _cuda(table), lengths)
    assert torch.isfinite(clean).all()
    at = length - 200 + 70                                   # seen by row 70 and those behind it
    for which, value in ((2, np.nan), (3, np.nan), (3, np.inf), (3, -np.inf)):
        bad = [c.copy() for c in cache]
        bad[which][table[0, at // 16], 0, 1, at % 16] = value
        got = quant_hip.kv4_attention(_cuda(q), tuple(_cuda(x) for x in bad), _cuda(table), lengths)
        assert torch.equal(got[:70], clean[:70])
        assert not torch.isfinite(got[70:]).all(dim=-1).any()
