"""What the serving operators refuse, without a GPU: the C ABI's codes before anything is launched, and the binding's errors."""
import ctypes

import pytest

FAKE, ODD = 0x1000, 0x1004                       # aligned and not; never dereferenced


def _args(**over):
    from alpaca_lora_4bit_amd import _lib
    v = dict(k_codes=FAKE, v_codes=FAKE, k_scales=FAKE, v_scales=FAKE, pages=10, page=16, heads=2, D=128, group=64,
             table=FAKE, width=4, lengths=FAKE, starts=None, B=2, T=4)
    v.update(over)
    cache = _lib.Kv4Cache(**{k: v[k] for k in ("k_codes", "v_codes", "k_scales", "v_scales", "pages", "page", "heads", "D", "group")})
    batch = _lib.Kv4Batch(**{k: v[k] for k in ("table", "width", "lengths", "starts", "B", "T")})
    return ctypes.byref(cache), ctypes.byref(batch)


BAD = [(dict(k_codes=None), -1), (dict(v_scales=None), -1), (dict(table=None), -1), (dict(lengths=None), -1),
       (dict(D=96), -2), (dict(D=256), -2), (dict(group=16), -2), (dict(D=64, group=128), -2), (dict(page=8), -2), (dict(page=24), -2),
       (dict(page=2048), -2), (dict(pages=0), -2), (dict(heads=0), -2), (dict(heads=5000), -2), (dict(pages=2 ** 30), -2), (dict(width=0), -2),
       (dict(width=2 ** 23), -2), (dict(B=0), -2), (dict(T=0), -2), (dict(T=5), -2), (dict(k_codes=ODD), -5), (dict(v_scales=ODD), -5)]


@pytest.mark.parametrize("over,code", BAD)
def test_a_cache_or_batch_that_does_not_fit_is_refused_by_every_entry_point(over, code):
    from alpaca_lora_4bit_amd import _lib
    L = _lib.lib()
    assert L.q4_kv4_append_f16(*_args(**over), FAKE, 256, 128, FAKE, 256, 128, None, 0, 0, None, 0, None, 0, 0, 0, None) == code
    assert L.q4_kv4_read_f16(*_args(**over), FAKE, FAKE, None) == code
    assert L.q4_kv4_attention_f16(*_args(**over), FAKE, 256, 128, 2, 1.0, FAKE, 2, 64, FAKE, 1 << 30, None) == code
    assert L.q4_kv4_attention_workspace_bytes(*_args(**over), 2, 2, 64) == 0


def test_append_read_and_attention_arguments():
    from alpaca_lora_4bit_amd import _lib
    L = _lib.lib()

    def append(k=FAKE, v=FAKE, k_t=256, q=None, q_out=None, hq=0, rope=None, rows=0, rot=0):
        return L.q4_kv4_append_f16(*_args(), k, k_t, 128, v, 256, 128, q, 256, 128, q_out, hq, rope, rows, rot, 0, None)
    assert append(k=None) == append(v=None) == append(q=FAKE, hq=2) == append(rot=64) == -1
    assert append(q=FAKE, q_out=FAKE, hq=3) == append(q=FAKE, q_out=FAKE, hq=0) == -2
    assert append(rope=FAKE, rows=4, rot=24) == append(rope=FAKE, rows=4, rot=144) == append(rope=FAKE, rows=0, rot=64) == append(k_t=-1) == -2
    assert append(rope=ODD, rows=4, rot=64) == append(q=FAKE, q_out=ODD, hq=2) == -5
    assert L.q4_kv4_read_f16(*_args(), None, FAKE, None) == -1 and L.q4_kv4_read_f16(*_args(), FAKE, ODD, None) == -5

    def attend(q=FAKE, q_t=256, hq=2, scale=1.0, out=FAKE, mt=2, ml=64, ws=FAKE, nb=1 << 30, **over):
        return L.q4_kv4_attention_f16(*_args(**over), q, q_t, 128, hq, scale, out, mt, ml, ws, nb, None)
    assert attend(q=None) == attend(out=None) == -1
    assert attend(hq=3) == attend(hq=0) == attend(mt=0) == attend(ml=0) == attend(q_t=-8) == -2
    assert attend(scale=0.0) == attend(scale=-1.0) == attend(scale=float("nan")) == attend(scale=float("inf")) == -2
    assert attend(q=ODD) == attend(out=ODD) == attend(q_t=252) == -5
    long = dict(width=4096, B=1, T=1)
    need = L.q4_kv4_attention_workspace_bytes(*_args(**long), 2, 1, 65536)
    assert need > 0 and need % (2 * (128 + 2) * 4) == 0 and L.q4_kv4_attention_workspace_bytes(*_args(), 2, 2, 64) == 0
    assert attend(mt=1, ml=65536, ws=None, nb=0, **long) == attend(mt=1, ml=65536, nb=need - 1, **long) == -3
    assert attend(mt=1, ml=65536, ws=FAKE + 16, nb=need, **long) == -5


def test_adapter_rows_arguments():
    from alpaca_lora_4bit_amd import _lib
    L = _lib.lib()

    def rows(count=1, x=FAKE, index=FAKE, per=1, M=4, K=256, R=8, n=2, ws=FAKE, nb=1 << 20, **over):
        p = (_lib.LoraRows * 4)()
        for d in p:
            d.a = d.b = d.scaling = d.y = FAKE
            d.N = 128
        for k, v in over.items():
            setattr(p[count - 1], k, v)
        return L.q4_lora_rows_f16(p, count, x, index, per, M, K, R, n, ws, nb, None)
    assert L.q4_lora_rows_f16(None, 1, FAKE, FAKE, 1, 4, 256, 8, 2, FAKE, 1 << 20, None) == -1
    assert rows(x=None) == rows(index=None) == rows(a=None) == rows(count=2, scaling=None) == rows(y=None) == -1
    assert rows(per=0) == rows(M=0) == rows(K=250) == rows(K=0) == rows(R=4) == rows(R=12) == rows(R=72) == rows(n=0) == rows(N=96) == rows(N=0) == -2
    assert rows(x=ODD) == rows(count=3, b=ODD) == -5
    need = L.q4_lora_rows_workspace_bytes(2, 4, 256, 8)
    assert need >= 2 * 4 * 8 * 4 and L.q4_lora_rows_workspace_bytes(5, 4, 256, 8) == L.q4_lora_rows_workspace_bytes(1, 4, 256, 12) == 0
    assert rows(count=2, ws=None) == rows(count=2, nb=need - 1) == -3 and rows(ws=FAKE + 16) == -5


def test_the_binding_refuses_tensors_off_the_gpu():
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    cache = (torch.zeros((2, 1, 16, 16), dtype=torch.int32), torch.zeros((2, 1, 4, 16, 4), dtype=torch.int32),
             torch.zeros((2, 1, 1, 16), dtype=torch.float16), torch.zeros((2, 1, 1, 16), dtype=torch.float16))
    t, n, q = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros((1, 1, 128), dtype=torch.float16)
    for call in (lambda: quant_hip.kv4_attention(q, cache, t, n), lambda: quant_hip.kv4_append(q, q, cache, t, n),
                 lambda: quant_hip.kv4_read(cache, t, n, 1), lambda: quant_hip.lora_rows(q[0], n, [(q, q, q, q)])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        quant_hip.kv4_attention(q, cache, t, n, scale=-1.0)


def test_sizes_beyond_what_a_launch_can_cover():
    from alpaca_lora_4bit_amd import _lib
    L = _lib.lib()
    over = dict(T=2 ** 24 + 2)
    assert L.q4_kv4_append_f16(*_args(**over), FAKE, 256, 128, FAKE, 256, 128, None, 0, 0, None, 0, None, 0, 0, 0, None) == -2
    assert L.q4_kv4_read_f16(*_args(**over), FAKE, FAKE, None) == -2
    assert L.q4_kv4_attention_f16(*_args(**over), FAKE, 256, 128, 2, 1.0, FAKE, 2, 64, FAKE, 1 << 30, None) == -2
    assert L.q4_lora_rows_workspace_bytes(1, 2 ** 24 + 1, 256, 8) == 0 and L.q4_lora_rows_workspace_bytes(1, 2 ** 24, 256, 8) > 0
    # bounds that are far too small for the rows do not ask for more than a gigabyte
    for T, D in ((2 ** 20, 128), (2 ** 24, 64), (64, 128)):
        assert L.q4_kv4_attention_workspace_bytes(*_args(T=T, D=D, width=2 ** 22), 64, 1, 2 ** 26) <= 2 ** 30
    many = dict(B=2 ** 12, T=2 ** 12, heads=2048, pages=4)
    assert L.q4_kv4_attention_f16(*_args(**many), FAKE, 2 ** 19, 128, 2048, 1.0, FAKE, 1, 64, FAKE, 1 << 30, None) == -2
    p = (_lib.LoraRows * 4)()
    p[0].a = p[0].b = p[0].scaling = p[0].y = FAKE
    p[0].N = 2 ** 13 + 64
    assert L.q4_lora_rows_f16(p, 1, FAKE, FAKE, 1, 2 ** 24, 32, 8, 1, FAKE, 1 << 40, None) == -2
