"""Results over memory that the same call reads are refused, whichever tensor it is."""
import pytest

from test_gpu_serving_refusals import _batch

pytestmark = pytest.mark.gpu


def test_results_over_the_cache_or_the_batch():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    cache, table, lengths, q, k, v = _batch(pages=16)
    n = q.numel()                                            # 2 rows of 4 heads of 64: one kilobyte
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    rope = torch.zeros(64, 32, 2, device="cuda")
    half = lambda t: t.view(-1).view(torch.float16)
    wide = lambda t: torch.zeros(1024, dtype=torch.int32, device="cuda")[:t.numel()].copy_(t.view(-1)).view(t.shape)     # with room behind it in its memory
    inside = lambda t: half(torch.as_strided(t, (512,), (1,)))[:n].view(q.shape)
    table, lengths, starts = wide(table), wide(lengths), wide(starts)
    assert qh.kv4_attention(q, cache, table, lengths, starts=starts).shape == q.shape                          # as they are they fit
    for i, over in enumerate([half(c)[8 * j:][:n].view(q.shape) for c in cache for j in (0, 3)] + [inside(t) for t in (table, lengths, starts)]):
        for call in (lambda: qh.kv4_attention(q, cache, table, lengths, starts=starts, out=over),
                     lambda: qh.kv4_append(k, v, cache, table, lengths, q=q, rope=rope, starts=starts, q_out=over)):
            with pytest.raises(ValueError, match="overlaps"):
                call()
                pytest.fail(f"result {i} was taken")
    with pytest.raises(ValueError, match="overlaps"):
        qh.kv4_append(k, v, cache, table, lengths, q=q, rope=rope, q_out=half(rope)[-n:].view(q.shape))


def test_updates_over_their_index_or_factors():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    x, store = torch.zeros(4, 64, dtype=torch.float16, device="cuda"), torch.zeros(4096, dtype=torch.float16, device="cuda")
    bank = lambda: (torch.zeros(2, 8, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 64, 8, dtype=torch.float16, device="cuda"))
    y, other = store[1024:1280].view(4, 64), torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    s, index = torch.ones(2, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for first in (1024, 1272, 1022):
        over_s, over_index = store[first:first + 4].view(torch.float32), store[first:first + 8].view(torch.int32)
        for call in (lambda: qh.lora_rows(x, index, [bank() + (over_s, y)]), lambda: qh.lora_rows(x, over_index, [bank() + (s, y)]),
                     lambda: qh.lora_rows(x, index, [bank() + (s, y), bank() + (over_s, other)]), lambda: qh.lora_rows(x, index, [bank() + (over_s, other), bank() + (s, y)])):
            with pytest.raises(ValueError, match="overlaps"):
                call()
    qh.lora_rows(x, store[1280:1288].view(torch.int32), [bank() + (store[1020:1024].view(torch.float32), y), bank() + (s, other)])      # side by side: taken
