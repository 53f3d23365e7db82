"""inference.generate_batch's decoder loop, the page pool and models.AdapterBank on the CPU: the three operators stand as plain float64 code, so that
the loop (packed prompts, parts, page tables, adapters by request, ended requests) can be held against the dense model in 64 bits."""
import json

import pytest
import torch

from alpaca_lora_4bit_amd import inference, kv4_cache, models, quant_hip

HIDDEN, INTER, HEADS, KV, VOCAB = 256, 320, 4, 2, 97


class Plain:
    """The operators over a dense store: what the cache holds is kept by the place (layer, page, offset) that the table gives."""

    def __init__(self, monkeypatch):
        self.store, self.calls = {}, []
        for name in ("kv4_append", "kv4_attention", "lora_rows"):
            monkeypatch.setattr(quant_hip, name, getattr(self, name))

    def _rows(self, table, lengths, starts, rows, page):
        B = table.shape[0]
        starts = [b * (rows // B) for b in range(B + 1)] if starts is None else starts.tolist()
        for b in range(B):
            for t in range(starts[b], starts[b + 1]):
                pos = int(lengths[b]) - starts[b + 1] + t
                yield t, b, pos, int(table[b, pos // page]) if 0 <= pos < table.shape[1] * page else -1

    def kv4_append(self, k, v, cache, table, lengths, q=None, rope=None, interleaved=False, starts=None, q_out=None):
        page, out = cache[0].shape[2], torch.zeros_like(q)
        turn = lambda x, cs: torch.cat((x[:, :32] * cs[:, 0] - x[:, 32:] * cs[:, 1], x[:, 32:] * cs[:, 0] + x[:, :32] * cs[:, 1]), -1)
        for t, b, pos, pg in self._rows(table, lengths, starts, len(k), page):
            if pg >= 0:
                cs = rope[pos].to(k.dtype)
                self.store[cache[0].data_ptr(), pg, pos % page] = (turn(k[t], cs), v[t].clone())
                out[t] = turn(q[t], cs)
        return out

    def kv4_attention(self, q, cache, table, lengths, scale=None, starts=None, max_tokens=None, max_length=None, out=None):
        page, out = cache[0].shape[2], torch.zeros_like(q)
        most = {}
        for t, b, pos, pg in self._rows(table, lengths, starts, len(q), page):
            most[b] = most.get(b, 0) + 1
            assert int(lengths[b]) <= max_length
            if pos < 0:
                continue
            kv = [self.store[cache[0].data_ptr(), int(table[b, j // page]), j % page] for j in range(pos + 1)]
            k, v = (torch.stack([x[i] for x in kv]).repeat_interleave(q.shape[1] // kv[0][0].shape[0], 1) for i in (0, 1))
            w = torch.softmax((k * q[t]).sum(-1) / 8.0, 0)
            out[t] = (w[..., None] * v).sum(0)
        assert max(most.values()) <= max_tokens
        self.calls.append(len(q))
        return out

    def lora_rows(self, x, index, specs, rows_per_index=1):
        assert len({s[0].shape[1] for s in specs}) == 1 and len(specs) <= 4
        for a, b, scaling, y in specs:
            for m, i in enumerate(index.tolist()):
                if 0 <= i < len(a):
                    y[m] += scaling[i].to(y.dtype) * (b[i].to(y.dtype) @ (a[i].to(y.dtype) @ x[m]))


def _model(seed=0, heads=HEADS, kv=KV):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(seed)
    cfg = LlamaConfig(vocab_size=VOCAB, hidden_size=HIDDEN, intermediate_size=INTER, num_hidden_layers=2, num_attention_heads=heads,
                      num_key_value_heads=kv, max_position_embeddings=64, tie_word_embeddings=False, bos_token_id=1, eos_token_id=2,
                      attn_implementation="eager")
    return LlamaForCausalLM(cfg).double().eval()


def _adapters(model, targets, ranks, seed):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for number, r in enumerate(ranks):
        state = {}
        for name, m in model.named_modules():
            if name.rsplit(".", 1)[-1] in targets[number]:
                state[f"base_model.model.{name}.lora_A.weight"] = torch.randn(r, m.in_features, generator=gen).div(16).half()
                state[f"base_model.model.{name}.lora_B.weight"] = torch.randn(m.out_features, r, generator=gen).div(4).half()
        out.append((state, 0.5 + number))
    return out


def _merged(model, adapter):
    """A copy of the model with one adapter added to its weights."""
    import copy
    other = copy.deepcopy(model)
    mods = dict(other.named_modules())
    state, scaling = adapter
    for key in state:
        if key.endswith("lora_A.weight"):
            layer = mods[key[len("base_model.model."):-len(".lora_A.weight")]]
            with torch.no_grad():
                layer.weight += scaling * state[key.replace("lora_A", "lora_B")].double() @ state[key].double()
    return other


PROMPTS = [torch.tensor(p) for p in ([5, 9, 33, 12, 80, 41, 7], [3], [60 + i for i in range(19)], [11, 12], [90, 4, 17, 8, 8, 2, 1, 55, 54])]


@pytest.mark.parametrize("prefill_rows", [8192, 16, 5])
@pytest.mark.parametrize("page", [16, 32])
def test_batch_gives_the_tokens_of_each_request_alone(monkeypatch, prefill_rows, page):
    """Greedy tokens of every request equal those of the dense model on that request (float64: no near ties), with its own adapter merged."""
    plain, model = Plain(monkeypatch), _model()
    targets = [("q_proj", "v_proj"), ("q_proj", "k_proj", "v_proj", "o_proj"), ("gate_proj", "up_proj", "down_proj", "v_proj")]
    adapters = _adapters(model, targets, (8, 3, 16), seed=4)
    bank = models.AdapterBank(model, adapters, device="cpu")
    which = [0, 2, -1, 1, 2]
    new = 9
    with torch.no_grad():
        got = inference.generate_batch(model, PROMPTS, new, bank, which, use_graph=False, page=page, prefill_rows=prefill_rows)
        for prompt, a, ids in zip(PROMPTS, which, got):
            alone = model if a < 0 else _merged(model, adapters[a])
            want = alone.generate(input_ids=prompt[None], max_new_tokens=new, min_new_tokens=new, do_sample=False,
                                  attention_mask=torch.ones_like(prompt[None]), eos_token_id=None, pad_token_id=0)
            assert ids.tolist() == want[0].tolist()
    assert max(plain.calls) <= max(prefill_rows, len(PROMPTS))


def test_requests_end_by_themselves(monkeypatch):
    """An ended request stops growing, the others go on as before; all ended: the loop stops."""
    plain, model = Plain(monkeypatch), _model(1)
    free = inference.generate_batch(model, PROMPTS, 12, use_graph=False)
    eos = free[0][len(PROMPTS[0]) + 4].item()
    ended = inference.generate_batch(model, PROMPTS, 12, eos_token_id=eos, use_graph=False)
    for prompt, a, b in zip(PROMPTS, free, ended):
        answer = a[len(prompt):].tolist()
        stop = answer.index(eos) + 1 if eos in answer else 12
        assert b.tolist() == a[:len(prompt) + stop].tolist()
    before = len(plain.calls)
    first = inference.generate_batch(model, [PROMPTS[0]], 1, use_graph=False)[0]
    assert len(first) == len(PROMPTS[0]) + 1 and len(plain.calls) == before + 2                # one prompt, one call a layer
    torch.manual_seed(0)
    sampled = inference.generate_batch(model, PROMPTS, 4, sampling={"temperature": 0.9, "top_k": 5, "repetition_penalty": 1.1}, use_graph=False)
    assert [len(s) for s in sampled] == [len(p) + 4 for p in PROMPTS]
    assert inference.generate_batch(model, [], 4) == []
    assert torch.equal(inference.generate_batch(model, [PROMPTS[0]], 0)[0], PROMPTS[0])


def test_generate_batch_refuses(monkeypatch):
    Plain(monkeypatch)
    model = _model()
    bank = models.AdapterBank(model, _adapters(model, [("q_proj",)], (8,), 1), device="cpu")
    for kw in (dict(bank=bank), dict(adapters=[0]), dict(bank=bank, adapters=[0, 0]), dict(bank=bank, adapters=[1]), dict(bank=bank, adapters=[-2]),
               dict(prefill_rows=0), dict(page=0), dict(page=24), dict(group=128), dict(group=16)):
        with pytest.raises(ValueError):
            inference.generate_batch(model, [PROMPTS[0]], 2, use_graph=False, **kw)
    for prompts in ([PROMPTS[0][None]], [PROMPTS[0][:0]]):
        with pytest.raises(ValueError):
            inference.generate_batch(model, prompts, 2, use_graph=False)
    with pytest.raises(ValueError, match="head_dim"):
        inference.generate_batch(_model(heads=8, kv=8), [PROMPTS[0]], 2, use_graph=False)
    model.config.model_type = "other"
    with pytest.raises(ValueError, match="LLaMA"):
        inference.generate_batch(model, [PROMPTS[0]], 2, use_graph=False)


def test_pages_are_taken_and_given_back():
    cache = kv4_cache.PagedKv4Cache(2, 3, 64, pages=7, page=16, group=64, device="cpu")
    assert [tuple(t.shape) for t in cache.layers[1]] == [(7, 3, 16, 8), (7, 3, 4, 8, 4), (7, 3, 1, 16), (7, 3, 1, 16)]
    a, b, c = cache.open(33), cache.open(16), cache.open(0)
    assert (len(a), len(b), len(c), cache.free_pages) == (3, 1, 0, 3) and not set(a) & set(b)
    with pytest.raises(RuntimeError):
        cache.open(49)
    assert cache.free_pages == 3
    assert cache.table([a, b, c]).tolist() == [a, b + [-1, -1], [-1, -1, -1]] and cache.table([c]).shape == (1, 1)
    gone = list(a)
    cache.close(a)
    cache.close(a)
    assert a == [] and cache.free_pages == 6
    d = cache.open(6 * 16)
    assert sorted(d + b) == list(range(7)) and set(gone) <= set(d)
    with pytest.raises(ValueError):
        cache.read(0, b, 17)
    for bad in (dict(head_dim=96), dict(group=16), dict(group=128), dict(page=8), dict(page=24), dict(page=2048), dict(pages=0), dict(heads=0)):
        with pytest.raises(ValueError):
            kv4_cache.new_layer(**dict(dict(pages=2, heads=1, head_dim=64, device="cpu"), **bad))


def test_rope_table_holds_the_angles():
    """float32 cosines of positions * inv_freq; an angle of up to 63 rounds by 2^-24 * 63 and inv_freq itself by as much."""
    table = kv4_cache.rope_table(_model().model.rotary_emb, 64, device="cpu")
    angle = torch.arange(64, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    want = torch.stack((angle.cos(), angle.sin()), -1)
    assert table.dtype == torch.float32 and (table - want).abs().max() < 64 * 4 * 2.0 ** -24

    class Dynamic(torch.nn.Module):
        rope_type = "dynamic"
    with pytest.raises(ValueError, match="dynamic"):
        kv4_cache.rope_table(Dynamic(), 8, device="cpu")


def test_bank_reads_directories_and_refuses(tmp_path):
    from safetensors.torch import save_file
    model = _model()
    (state, _), = _adapters(model, [("q_proj", "v_proj")], (5,), 3)
    save_file(state, str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 5, "lora_alpha": 10}))
    bank = models.AdapterBank(model, [str(tmp_path), (state, 0.25)], device="cpu")
    attn = model.model.layers[1].self_attn
    a, b, scaling = bank._layers[attn.q_proj]
    name = "base_model.model.model.layers.1.self_attn.q_proj.lora_"
    assert a.shape == (2, 8, HIDDEN) and b.shape == (2, HIDDEN, 8) and scaling.tolist() == [2.0, 0.25]
    assert torch.equal(a[1, :5], state[name + "A.weight"]) and not a[:, 5:].any() and torch.equal(b[0, :, :5], state[name + "B.weight"]) and not b[:, :, 5:].any()
    assert bank.holds(attn.q_proj) and not bank.holds(attn.k_proj, attn.o_proj) and bank.count == 2
    assert models.AdapterBank(model, [], device="cpu").count == 0
    ok = {k: v for k, v in state.items() if "layers.0.self_attn.q_proj" in k}
    key = next(iter(ok))
    for bad in ({"nothing.lora_A.weight": torch.zeros(2, 2)}, {key: torch.zeros(8, 3)}, {key: ok[key]}, {"model.norm.weight": torch.zeros(3)},
                {k: torch.zeros((65, HIDDEN) if "lora_A" in k else (HIDDEN, 65)) for k in ok},
                {k: v[:2] if "lora_A" in k else v for k, v in ok.items()}):
        with pytest.raises(ValueError):
            models.AdapterBank(model, [(bad, 1.0)], device="cpu")
