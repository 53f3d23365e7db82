"""The serving operators' calls that are refused or allowed on the GPU's own tensors: wrong shapes and types, gradients, overlapping memory, empty batches, rows of no
sequence, bounds that are wrong."""
import pytest

pytestmark = pytest.mark.gpu


def _batch(B=2, heads=2, share=2, D=64, page=16, width=4, new=1, length=20, group=32, pages=8):
    import torch
    from alpaca_lora_4bit_amd import kv4_cache, quant_hip
    gen = torch.Generator(device="cuda").manual_seed(3)
    half = lambda *s: torch.randn(*s, generator=gen, device="cuda").half()
    cache = kv4_cache.new_layer(pages, heads, D, page, group)
    table = torch.arange(B * width, dtype=torch.int32, device="cuda").view(B, width) % pages
    lengths = torch.full((B,), length, dtype=torch.int32, device="cuda")
    full = torch.full((B,), width * page, dtype=torch.int32, device="cuda")
    quant_hip.kv4_append(half(B * width * page, heads, D), half(B * width * page, heads, D), cache, table, full)
    return cache, table, lengths, half(B * new, heads * share, D), half(B * new, heads, D), half(B * new, heads, D)


def test_calls_that_are_refused():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    cache, table, lengths, q, k, v = _batch()
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    rope = torch.zeros(64, 32, 2, device="cuda")
    ok = [c.clone() for c in cache]
    wide = torch.zeros(2, 8, 64, dtype=torch.float16, device="cuda")
    bad = [
        lambda: qh.kv4_attention(q.float(), cache, table, lengths), lambda: qh.kv4_attention(q[0], cache, table, lengths),
        lambda: qh.kv4_attention(q[:, :3], cache, table, lengths), lambda: qh.kv4_attention(q[..., :32], cache, table, lengths),
        lambda: qh.kv4_attention(q[:1], cache, table, lengths), lambda: qh.kv4_attention(q, cache, table.long(), lengths),
        lambda: qh.kv4_attention(q, cache, table, lengths.long()), lambda: qh.kv4_attention(q, cache, table, lengths[:1]),
        lambda: qh.kv4_attention(q, cache, table.cpu(), lengths), lambda: qh.kv4_attention(q, cache, table.t(), lengths),
        lambda: qh.kv4_attention(q, cache, table, lengths, starts=starts[:2]), lambda: qh.kv4_attention(q, cache, table, lengths, starts=starts.long()),
        lambda: qh.kv4_attention(q, cache, table, lengths, scale=float("nan")), lambda: qh.kv4_attention(q, cache, table, lengths, scale=float("inf")),
        lambda: qh.kv4_attention(q, cache, table, lengths, scale=0.0), lambda: qh.kv4_attention(q, cache, table, lengths, max_tokens=0),
        lambda: qh.kv4_attention(q, cache, table, lengths, max_length=0), lambda: qh.kv4_attention(q, cache, table, lengths, out=q.float()),
        lambda: qh.kv4_attention(wide[:, 1:5], cache, table, lengths, out=wide.view(-1)[:q.numel()].view(q.shape)),
        lambda: qh.kv4_attention(q.clone().requires_grad_(), cache, table, lengths),
        lambda: qh.kv4_attention(q, (cache[0], cache[1], cache[2], cache[3][:4]), table, lengths),
        lambda: qh.kv4_attention(q, (cache[0], cache[1][..., :2], cache[2], cache[3]), table, lengths),
        lambda: qh.kv4_append(k, v, cache, table, lengths, rope=rope.half()), lambda: qh.kv4_append(k, v, cache, table, lengths, rope=rope[:, :20]),
        lambda: qh.kv4_append(k, v, cache, table, lengths, rope=torch.zeros(64, 40, 2, device="cuda")), lambda: qh.kv4_append(k, v[:1], cache, table, lengths),
        lambda: qh.kv4_append(k[:, :1], v[:, :1], cache, table, lengths), lambda: qh.kv4_append(k, v, cache, table, lengths, q_out=q),
        lambda: qh.kv4_append(k, v, cache, table, lengths, q=q[:, :2], q_out=k), lambda: qh.kv4_append(k.clone().requires_grad_(), v, cache, table, lengths),
        lambda: qh.kv4_read(cache, table, lengths, -1), lambda: qh.kv4_read(cache, table, lengths, 3),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    assert all(torch.equal(a, b) for a, b in zip(ok, cache))
    x, index = torch.zeros(4, 64, dtype=torch.float16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    a, b = torch.zeros(2, 8, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 64, 8, dtype=torch.float16, device="cuda")
    s, y = torch.ones(2, device="cuda"), torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    whole = torch.zeros(6, 64, dtype=torch.float16, device="cuda")
    for i, call in enumerate([
            lambda: qh.lora_rows(x, index, []), lambda: qh.lora_rows(x, index, [(a, b, s, y)] * 5), lambda: qh.lora_rows(x, index, [(a, b, s, y), (a, b, s, y)]),
            lambda: qh.lora_rows(x, index, [(a, b, s, whole[:4]), (a, b, s, whole[2:])]), lambda: qh.lora_rows(x, index, [(a, b, s, x)]),
            lambda: qh.lora_rows(x, index, [(a, b, s, a.view(-1, 64)[:4])]), lambda: qh.lora_rows(x, index.long(), [(a, b, s, y)]),
            lambda: qh.lora_rows(x, index[:3], [(a, b, s, y)]), lambda: qh.lora_rows(x, index, [(a, b, s, y)], 2), lambda: qh.lora_rows(x, index, [(a, b, s, y)], 0),
            lambda: qh.lora_rows(x, index, [(a[:, :4], b[..., :4], s, y)]), lambda: qh.lora_rows(x, index, [(a, b[:, :32], s, y[:, :32])]),
            lambda: qh.lora_rows(x, index, [(a, b, s.half(), y)]), lambda: qh.lora_rows(x, index, [(a, b, s[:1], y)]), lambda: qh.lora_rows(x, index, [(a, b, s, y.float())]),
            lambda: qh.lora_rows(x, index, [(a.clone().requires_grad_(), b, s, y)]), lambda: qh.lora_rows(x, index, [(a, b, s.clone().requires_grad_(), y)]),
            lambda: qh.lora_rows(x.t().contiguous().t(), index, [(a, b, s, y)])]):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"lora_rows call {i} was taken")
    with torch.no_grad():                                    # no gradient is asked for: taken
        qh.lora_rows(x, index, [(a.clone().requires_grad_(), b, s, y)])
        qh.kv4_attention(q.clone().requires_grad_(), cache, table, lengths)


def test_empty_batches_and_rows_of_no_sequence():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    cache, table, lengths, q, k, v = _batch()
    before = [c.clone() for c in cache]
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert qh.kv4_attention(q[:0], cache, table, lengths, starts=none).shape == (0, 4, 64)
    assert qh.kv4_append(k[:0], v[:0], cache, table, lengths, q=q[:0], starts=none).shape == (0, 4, 64)
    assert qh.kv4_read(cache, table, lengths, 0)[0].shape == (0, 2, 64)
    x = torch.zeros(0, 64, dtype=torch.float16, device="cuda")
    qh.lora_rows(x, none[:0], [(torch.zeros(1, 8, 64, dtype=torch.float16, device="cuda"), torch.zeros(1, 64, 8, dtype=torch.float16, device="cuda"),
                                torch.ones(1, device="cuda"), torch.zeros(0, 64, dtype=torch.float16, device="cuda"))])
    # all rows belong to no sequence: nothing is written but what read returns, which is zero
    out = torch.full_like(q, 5.0)
    assert bool((qh.kv4_attention(q, cache, table, lengths, starts=none, out=out) == 5.0).all())
    assert bool((qh.kv4_append(k, v, cache, table, lengths, q=q, starts=none, q_out=out) == 5.0).all())
    torch.empty(1 << 20, device="cuda").fill_(float("nan"))
    for starts, zero in ((none, [True] * 6), (torch.tensor([1, 3, 5], dtype=torch.int32, device="cuda"), [True, False, False, False, False, True])):
        got = qh.kv4_read(cache, table, lengths, 6, starts=starts)
        for t in got:
            assert [bool((r == 0).all()) for r in t] == zero
    assert all(torch.equal(a, b) for a, b in zip(before, cache))


@pytest.mark.parametrize("new", [1, 40])
def test_results_in_place_and_bounds_that_are_wrong(new):
    """`out` and `q_out` may be the queries; bounds far too small or large change neither the result beyond the order of its sums nor the memory that is asked for."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    cache, table, lengths, q, k, v = _batch(B=3, share=4, new=new, width=40, pages=120, length=600)
    rope = torch.randn(640, 32, 2, device="cuda")
    want = qh.kv4_append(k, v, cache, table, lengths, q=q, rope=rope)
    mine = q.clone()
    assert qh.kv4_append(k, v, cache, table, lengths, q=mine, rope=rope, q_out=mine) is not None and torch.equal(mine, want)
    out = qh.kv4_attention(want, cache, table, lengths)
    assert torch.equal(qh.kv4_attention(mine, cache, table, lengths, out=mine), out)
    # weights and sums in another order, and keys rounded or not: a few half steps of the results
    for bounds in (dict(max_tokens=1), dict(max_length=1), dict(max_tokens=1, max_length=10 ** 9), dict(max_tokens=10 ** 9, max_length=10 ** 9)):
        got = qh.kv4_attention(want, cache, table, lengths, **bounds)
        assert float((got.float() - out.float()).abs().max()) < 2 ** -7 * max(1.0, float(out.float().abs().max()))
    many = torch.zeros(1 << 15, 8, 64, dtype=torch.float16, device="cuda")
    starts = torch.tensor([0, 3, 3, 3], dtype=torch.int32, device="cuda")
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    qh.kv4_attention(many, cache, table, lengths, starts=starts, max_tokens=1, max_length=640)
    assert torch.cuda.max_memory_allocated() - base <= (1 << 30) + 2 * many.numel() * 2
