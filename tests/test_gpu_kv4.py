"""The 4-bit key/value cache on the GPU: append, read back and attention against the CPU restatement (oracle/kv4_oracle.py)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _cuda(a):
    import torch
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _table(lengths, page, pages, width, rng):
    """A page table in random order, -1 where a sequence ends."""
    order, at = rng.permutation(pages), 0
    table = np.full((len(lengths), width), -1, np.int32)
    for b, n in enumerate(lengths):
        need = -(-n // page)
        table[b, :need] = order[at:at + need]
        at += need
    return table


def _filled(o, lengths, heads, D, group, page, rng, spread=1.0):
    """A cache whose sequences hold random values, NaN scales and all-ones codes everywhere else."""
    pages = sum(-(-n // page) for n in lengths) + 2
    width = max(1, max(-(-n // page) for n in lengths))
    table = _table(lengths, page, pages, width, rng)
    cache = o.new_cache(pages, heads, page, D, group, fill=-1)
    for b, n in enumerate(lengths):
        for j in range(n):
            for h in range(heads):
                k, v = (rng.standard_normal(D).astype(np.float32) * spread + 0.3 for _ in range(2))
                (kq, ks), (vq, vs) = o.quantize(k, group), o.quantize(v, group)
                o.put(cache, table[b, j // page], h, j % page, kq, ks, vq, vs)
    return cache, table


PROMPT_ROWS = 64            # more rows a key head and sequence (tokens times the heads that share it) go to the kernel that rounds keys and values too


def _check(got, want, tol, what=""):
    got = got.float().cpu().numpy().astype(np.float64)
    mine = ~np.isnan(want)
    err = np.abs(got - want)[mine]
    worst = float((err - tol[mine]).max()) if err.size else 0.0
    assert np.isfinite(got[mine]).all() and worst <= 0.0, f"{what}: off by {err.max()}, over the bound by {worst}"


# lengths of 0 and 1, ends of tiles of 64 and of pages on either side, several tiles per wavefront, more than one share of the keys
ATTENTION = [
    # heads, share, D, group, page, lengths, new
    (1, 1, 128, 128, 16, [1], 1),
    (2, 1, 128, 32, 16, [0, 1, 15, 16, 17], 1),
    (1, 4, 128, 64, 48, [47, 48, 49, 63, 64, 65], 1),
    (2, 3, 64, 64, 32, [255, 256, 257, 0, 300], 1),
    (1, 16, 64, 32, 256, [513, 31], 1),
    (1, 5, 128, 128, 64, [1023], 1),
    (1, 17, 128, 64, 16, [100], 1),
    (1, 2, 128, 32, 64, [2100], 2),
    (2, 2, 64, 32, 16, [40, 9], 9),
    (1, 4, 128, 64, 32, [70, 131], 33),
    (1, 1, 128, 128, 16, [129], 129),
    (1, 8, 64, 64, 128, [200, 64], 64),
    (1, 3, 128, 32, 112, [350], 77),
]


@pytest.mark.parametrize("heads,share,D,group,page,lengths,new", ATTENTION)
def test_attention_matches_float64(heads, share, D, group, page, lengths, new):
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng = np.random.default_rng(sum(lengths) + new + D + group)
    cache, table = _filled(o, lengths, heads, D, group, page, rng)
    q = (rng.standard_normal((len(lengths) * new, heads * share, D)) * 2).astype(np.float16)
    want, tol = o.attention(q, cache, table, np.array(lengths), None, 1 / math.sqrt(D), new * share > PROMPT_ROWS)
    dev, tb, ln = [_cuda(x) for x in cache], _cuda(table), torch.tensor(lengths, dtype=torch.int32).cuda()
    got = quant_hip.kv4_attention(_cuda(q), tuple(dev), tb, ln)
    _check(got, want, tol)
    # the bounds that size the launch do not change what comes out beyond the order of the sums
    for most_new, most in ((1, 1), (new, 64), (new, 100000)):
        _check(quant_hip.kv4_attention(_cuda(q), tuple(dev), tb, ln, max_tokens=most_new, max_length=most), want, tol, (most_new, most))
    assert torch.equal(got, quant_hip.kv4_attention(_cuda(q), tuple(dev), tb, ln))


@pytest.mark.parametrize("new", [[1, 3, 0, 2], [1, 40, 17, 0], [150, 1, 1, 30]])
def test_attention_of_ragged_rows_views_and_padding(new):
    """Runs of different lengths, rows before the first and behind the last sequence left as they were, queries inside a wider product."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    heads, share, D, group, page = 2, 4, 128, 64, 16
    rng = np.random.default_rng(7)
    lengths = [n + extra for n, extra in zip(new, (5, 60, 0, 33))]
    cache, table = _filled(o, lengths, heads, D, group, page, rng)
    starts = np.cumsum([2] + new).astype(np.int32)                     # two rows in front belong to nobody
    T = int(starts[-1]) + 5
    qkv = rng.standard_normal((T, heads * share * D + 24)).astype(np.float16)
    q = _cuda(qkv)[:, 8:8 + heads * share * D].unflatten(-1, (heads * share, D))
    want, tol = o.attention(q.cpu().numpy(), cache, table, np.array(lengths), starts, 0.11, True)
    out = torch.full((T, heads * share, D), 7.0, dtype=torch.float16, device="cuda")
    args = (tuple(_cuda(x) for x in cache), _cuda(table), torch.tensor(lengths, dtype=torch.int32).cuda())
    for bounds in ({}, {"max_tokens": max(new), "max_length": max(lengths)}, {"max_tokens": max(new), "max_length": 5000}):
        out.fill_(7.0)
        got = quant_hip.kv4_attention(q, *args, scale=0.11, starts=_cuda(starts), out=out, **bounds)
        assert got.data_ptr() == out.data_ptr()
        _check(got, want, tol, bounds)
        outside = np.isnan(want[:, 0, 0])
        assert outside.sum() == 7 and bool((got[torch.from_numpy(outside).cuda()] == 7.0).all())
    # odd addresses and strides: through a copy
    wide = _cuda(np.pad(qkv, ((0, 0), (1, 0))))
    got = quant_hip.kv4_attention(wide[:, 9:9 + heads * share * D].unflatten(-1, (heads * share, D)), *args, scale=0.11, starts=_cuda(starts))
    _check(got, want, tol, "odd")
    got = quant_hip.kv4_attention(q.transpose(0, 1).contiguous().transpose(0, 1), *args, scale=0.11, starts=_cuda(starts))
    _check(got, want, tol, "heads first")


@pytest.mark.parametrize("new", [1, 20, 60])
def test_attention_with_bad_pages_and_poison_in_places_that_are_not_seen(new):
    """Pages that do not exist hide their keys; later tokens of the same prompt may hold infinities and NaN; a length beyond the table ends with it."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    heads, share, D, group, page = 1, 2, 128, 64, 16
    rng = np.random.default_rng(new)
    lengths = [150, 90, 64]
    cache, table = _filled(o, lengths, heads, D, group, page, rng)
    table[0, 2], table[0, 5], table[1, 0], table[2, :] = cache[0].shape[0], -7, 2 ** 30, -1
    claimed = np.array([150, 90, 64 + 10 ** 6], np.int32)
    q = rng.standard_normal((3 * new, heads * share, D)).astype(np.float16)
    want, tol = o.attention(q, cache, table, claimed, None, 0.1, new * share > PROMPT_ROWS)
    args = (tuple(_cuda(x) for x in cache), _cuda(table), _cuda(claimed))
    _check(quant_hip.kv4_attention(_cuda(q), *args, scale=0.1), want, tol)
    assert np.all(want[2 * new:] == 0)
    # the last token of sequence 1 turns to NaN: only the row at its own position sees it
    j = 89
    for name in (2, 3):
        cache[name][table[1, j // page], 0, :, j % page] = np.nan if name == 2 else np.inf
    got = quant_hip.kv4_attention(_cuda(q), tuple(_cuda(x) for x in cache), *args[1:], scale=0.1).float().cpu().numpy()
    assert np.isnan(got[2 * new - 1]).all()
    keep = np.arange(3 * new) != 2 * new - 1
    assert (np.abs(got - want)[keep] <= tol[keep]).all()


def test_attention_with_large_and_small_scales():
    """Scales of the values far above and below one, scores of hundreds, one key that outweighs the rest."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    heads, D, group, page = 1, 128, 32, 32
    rng = np.random.default_rng(3)
    for spread, n in ((1e-4, 1), (3000.0, 1), (1e-4, 70), (3000.0, 70)):
        lengths = [333]
        cache, table = _filled(o, lengths, heads, D, group, page, rng, spread)
        cache[2][:] = np.where(np.isnan(cache[2]), cache[2], np.float16(0.2))          # keys of ordinary size
        if spread > 1:
            cache[3][table[0, 3], 0, 1] = np.float16(10000.0)
        q = (rng.standard_normal((n, 1, D)) * 20).astype(np.float16)
        want, tol = o.attention(q, cache, table, np.array(lengths), None, 1 / math.sqrt(D), n > PROMPT_ROWS)
        got = quant_hip.kv4_attention(_cuda(q), tuple(_cuda(x) for x in cache), _cuda(table), torch.tensor(lengths, dtype=torch.int32).cuda())
        _check(got, want, tol, (spread, n))


APPEND = [
    # heads, q heads, D, group, page, rot, interleaved, lengths, new
    (2, 2, 128, 128, 16, 128, False, [1, 16, 17, 40], [1, 1, 1, 1]),
    (1, 3, 128, 32, 48, 64, True, [50, 9], [5, 9]),
    (3, 6, 64, 64, 16, 64, True, [33], [33]),
    (2, 8, 64, 32, 32, 16, False, [70, 0, 31], [7, 1, 31]),
    (8, 8, 128, 64, 64, 32, False, [3, 130, 64], [1, 66, 0]),
    (1, 1, 128, 64, 16, 0, False, [20], [20]),
]


def _append_case(o, heads, hq, D, group, page, rot, lengths, new, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    T = sum(new)
    q, k, v = ((rng.standard_normal((T, h, D)) * scale).astype(np.float16) for h in (hq, heads, heads))
    pages = sum(-(-n // page) for n in lengths) + 2
    table = _table(lengths, page, pages, max(1, max(-(-n // page) for n in lengths)), rng)
    rope = None
    if rot:
        ang = np.arange(max(lengths) + 1)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
        rope = np.stack((np.cos(ang), np.sin(ang)), -1).astype(np.float32)
    starts = None if len(set(new)) == 1 else np.cumsum([0] + new).astype(np.int32)
    return rng, q, k, v, pages, table, rope, starts


def _append_oracle(o, cache, q, k, v, table, lengths, starts, rope, interleaved, group):
    T = len(k)
    qo = np.zeros(q.shape, np.float16)
    for t, (b, pos, pg, off) in enumerate(o.places(table, lengths, starts, T, cache[0].shape[0], cache[0].shape[2])):
        if b < 0:
            qo[t] = 7.0
            continue
        if pg < 0 or (rope is not None and pos >= len(rope)):
            continue
        turn = (lambda x: o.rotate(x, rope[pos], interleaved)) if rope is not None else (lambda x: x)
        qo[t] = turn(q[t].astype(np.float32)).astype(np.float16)
        kr = turn(k[t].astype(np.float32))
        for h in range(k.shape[1]):
            (kq, ks), (vq, vs) = o.quantize(kr[h], group), o.quantize(v[t, h].astype(np.float32), group)
            o.put(cache, pg, h, off, kq, ks, vq, vs)
    return qo


def _same(got, want):
    got = got.cpu().numpy()
    if want.dtype == np.float16:
        assert np.array_equal(np.isnan(got), np.isnan(want))
        got, want = np.nan_to_num(got), np.nan_to_num(want)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("heads,hq,D,group,page,rot,interleaved,lengths,new", APPEND)
def test_append_stores_the_codes_of_the_definition_and_reads_them_back(heads, hq, D, group, page, rot, interleaved, lengths, new):
    """Codes, scales and rotated queries are equal to the last bit: every step is one correctly rounded float32 operation on either side."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    rng, q, k, v, pages, table, rope, starts = _append_case(o, heads, hq, D, group, page, rot, lengths, new, sum(lengths) + D)
    k[0, 0, :] = 0                                                         # a group of zeros has scale zero
    v[-1, -1, 3] = -60000.0
    want = o.new_cache(pages, heads, page, D, group)
    qo = _append_oracle(o, want, q, k, v, table, lengths, starts, rope, interleaved, group)
    cache = tuple(_cuda(x) for x in o.new_cache(pages, heads, page, D, group))
    args = (cache, _cuda(table), torch.tensor(lengths, dtype=torch.int32).cuda())
    # keys, values and queries as parts of one product, at an odd place: strides and addresses that no 16-byte load fits
    for shift in (0, 3):
        flat = np.concatenate([x.reshape(len(k), -1) for x in (q, k, v)], 1)
        wide = _cuda(np.pad(flat, ((0, 0), (shift, 8 - shift))))
        parts = [x.unflatten(-1, (-1, D)) for x in wide[:, shift:shift + flat.shape[1]].split([hq * D, heads * D, heads * D], -1)]
        got = quant_hip.kv4_append(parts[1], parts[2], *args, q=parts[0], rope=_cuda(rope), interleaved=interleaved, starts=_cuda(starts))
        _same(got, qo)
        for g, w in zip(cache, want):
            _same(g, w)
    assert quant_hip.kv4_append(_cuda(k), _cuda(v), *args, starts=_cuda(starts), rope=_cuda(rope), interleaved=interleaved) is None
    for g, w in zip(cache, want):
        _same(g, w)
    kr, vr = quant_hip.kv4_read(*args, len(k), starts=_cuda(starts))
    for t, (b, pos, pg, off) in enumerate(o.places(table, lengths, starts, len(k), pages, page)):
        for h in range(heads):
            ek, ev = (x[0].astype(np.float16) for x in o.get(want, [pg], h, [off])) if pg >= 0 else (np.zeros(D, np.float16),) * 2
            assert np.array_equal(kr[t, h].cpu().numpy(), ek) and np.array_equal(vr[t, h].cpu().numpy(), ev)


def test_append_of_rows_without_a_place():
    """Positions before the first, behind the table or the rotations, pages that do not exist: not stored, q zero.  Rows of no sequence: nothing written."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    heads, hq, D, group, page = 2, 4, 128, 32, 16
    lengths, new = [40, 20, 2, 64, 30], [3, 3, 4, 2, 6]
    rng, q, k, v, pages, table, rope, starts = _append_case(o, heads, hq, D, group, page, 128, lengths, new, 1)
    starts = starts + 2
    q, k, v = (np.concatenate([x[:2], x, x[:3]]) for x in (q, k, v))
    table[0, 2], table[1, 1] = pages, -3
    claimed = np.array([40, 20, 2, 10 ** 6, 30], np.int32)                 # sequence 2 has fewer tokens than rows, 3 more than its table
    rope = np.ascontiguousarray(rope[:28])                                 # positions 28 and 29 of sequence 4 have no rotation
    want = o.new_cache(pages, heads, page, D, group)
    qo = _append_oracle(o, want, q, k, v, table, claimed, starts, rope, False, group)
    cache = tuple(_cuda(x) for x in o.new_cache(pages, heads, page, D, group))
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    got = quant_hip.kv4_append(_cuda(k), _cuda(v), cache, _cuda(table), _cuda(claimed), q=_cuda(q), rope=_cuda(rope), starts=_cuda(starts), q_out=out)
    assert got.data_ptr() == out.data_ptr()
    _same(got, qo)
    for g, w in zip(cache, want):
        _same(g, w)
    assert (qo == 0).reshape(len(q), -1).all(1).sum() == 3 + 3 + 2 + 2 + 2


def test_nan_and_infinity_reach_the_values():
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    D, group = 128, 64
    k = torch.randn(3, 1, D).half()
    v = torch.randn(3, 1, D).half()
    k[0, 0, 5], v[1, 0, 70], v[2, 0, 1] = float("nan"), float("inf"), float("nan")
    cache = tuple(_cuda(x) for x in o.new_cache(1, 1, 16, D, group))
    args = (cache, torch.zeros((1, 1), dtype=torch.int32).cuda(), torch.tensor([3], dtype=torch.int32).cuda())
    quant_hip.kv4_append(k.cuda(), v.cuda(), *args)
    kr, vr = (x.cpu() for x in quant_hip.kv4_read(*args, 3))
    assert torch.isnan(kr[0, 0, :64]).all() and torch.isfinite(kr[0, 0, 64:]).all() and torch.isfinite(kr[1:]).all()
    assert not torch.isfinite(vr[1, 0, 64:]).any() and torch.isnan(vr[2, 0, :64]).all() and torch.isfinite(vr[0]).all()


def test_cache_of_more_than_two_gigabytes_and_far_pages():
    """Places behind 2^31 bytes of codes and 2^31 codes: the last page of a large cache."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    from oracle import kv4_oracle as o
    heads, D, group, page, pages = 8, 128, 32, 256, 20000               # 20000 * 8 * 256 * 64 bytes = 2.6 GB of codes each
    dev = dict(device="cuda")
    cache = (torch.empty((pages, heads, page, D // 8), dtype=torch.int32, **dev), torch.empty((pages, heads, page // 4, D // 8, 4), dtype=torch.int32, **dev),
             torch.empty((pages, heads, D // group, page), dtype=torch.float16, **dev), torch.empty((pages, heads, D // group, page), dtype=torch.float16, **dev))
    rng = np.random.default_rng(0)
    n = 300
    q, k, v = (rng.standard_normal((n, h, D)).astype(np.float16) for h in (heads, heads, heads))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32).cuda()
    ln = torch.tensor([n], dtype=torch.int32).cuda()
    quant_hip.kv4_append(_cuda(k), _cuda(v), cache, table, ln)
    small = o.new_cache(2, heads, page, D, group)
    for i, x in enumerate(cache):
        small[i][:] = x[pages - 2:].flip(0).cpu().numpy()
    got = quant_hip.kv4_attention(_cuda(q[-1:]), cache, table, ln)
    want, tol = o.attention(q[-1:], small, np.array([[0, 1]]), np.array([n]), None, 1 / math.sqrt(D))
    _check(got, want, tol)
