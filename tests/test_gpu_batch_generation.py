"""The serving operators together: generation of a batch of requests (4-bit paged cache, adapters by request) on the synthetic 4-bit LLaMA, every
operator call of the run against the 64-bit restatements, captured steps against eager ones, and captured runs of the three operators beside
other work."""
import json
import math
import os

import numpy as np
import pytest
import torch

from tiny_llama import GROUPSIZE, build

pytestmark = pytest.mark.gpu


def _loaded(path):
    from alpaca_lora_4bit_amd import autograd_4bit as ag, inference
    model, tokenizer = ag.load_llama_model_4bit_low_ram(path, os.path.join(path, "model.safetensors"), groupsize=GROUPSIZE, half=True, device_map={"": 0})
    return inference.prepare_model(model).eval(), tokenizer


def _bank(model):
    """Three adapters: q and v, all of attention, the MLP."""
    from alpaca_lora_4bit_amd import models
    gen = torch.Generator().manual_seed(5)
    adapters = []
    for number, (targets, r) in enumerate(((("q_proj", "v_proj"), 8), (("q_proj", "k_proj", "v_proj", "o_proj"), 12), (("gate_proj", "up_proj", "down_proj"), 16))):
        state = {}
        for name, m in model.named_modules():
            if name.rsplit(".", 1)[-1] in targets:
                state[f"{name}.lora_A.weight"] = torch.randn(r, m.in_features, generator=gen).div(16)
                state[f"{name}.lora_B.weight"] = torch.randn(m.out_features, r, generator=gen).div(8)
        adapters.append((state, 1.0))
    return models.AdapterBank(model, adapters)


def _prompts():
    return [torch.tensor([1] + [7 + (13 * i + 5 * n) % 180 for i in range(n)]).cuda() for n in (9, 0, 33, 70, 4)]


@pytest.mark.parametrize("fuse", [False, True])
def test_every_call_of_a_batch_matches_its_formula(tmp_path, oracle, monkeypatch, fuse):
    """Prompts in parts of 40 rows and six tokens of five requests; every append's codes, every attention and every adapter update is checked with
    the tensors it really got."""
    from alpaca_lora_4bit_amd import inference, quant_hip
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp, make_quant_attn
    from oracle import kv4_oracle as o
    from test_gpu_kv4 import PROMPT_ROWS
    from test_gpu_lora_rows import _bound
    build(str(tmp_path), oracle, seed=8)
    model, _ = _loaded(str(tmp_path))
    if fuse:
        assert make_quant_attn(model) == 2 and make_fused_mlp(model) == 2
    bank = _bank(model)
    real = {n: getattr(quant_hip, n) for n in ("kv4_append", "kv4_attention", "lora_rows")}
    seen = {n: 0 for n in real}
    host = lambda t: None if t is None else t.cpu().numpy()

    def append(k, v, cache, table, lengths, q=None, rope=None, interleaved=False, starts=None, q_out=None):
        want = [host(c).copy() for c in cache]
        out = real["kv4_append"](k, v, cache, table, lengths, q, rope, interleaved, starts, q_out)
        cs, tb, ln = host(rope), host(table), host(lengths)
        qs = np.zeros(q.shape, np.float32)
        for t, (b, pos, pg, off) in enumerate(o.places(tb, ln, host(starts), len(k), len(want[0]), want[0].shape[2])):
            if pg < 0:
                continue
            kq, ks = o.quantize(o.rotate(host(k)[t].astype(np.float32), cs[pos], False), 32)
            vq, vs = o.quantize(host(v)[t].astype(np.float32), 32)
            qs[t] = o.rotate(host(q)[t].astype(np.float32), cs[pos], False)
            for h in range(k.shape[1]):
                o.put(want, pg, h, off, kq[h], ks[h], vq[h], vs[h])
        assert all(np.array_equal(w, host(c)) for w, c in zip(want, cache))
        # the turned q, from float32 products and one difference of them: half a step of fp16 and three of float32
        bound = np.abs(qs) * 2.0 ** -11 + 2.0 ** -25 + 3 * 2.0 ** -24 * 2 * np.abs(host(q)).max()
        assert (np.abs(host(out).astype(np.float64) - qs) <= bound).all()
        seen["kv4_append"] += 1
        return out

    def attention(q, cache, table, lengths, scale=None, starts=None, max_tokens=None, max_length=None, out=None):
        got = real["kv4_attention"](q, cache, table, lengths, scale, starts, max_tokens, max_length, out)
        want, tol = o.attention(host(q), [host(c) for c in cache], host(table), host(lengths), host(starts), 1 / math.sqrt(q.shape[-1]),
                                max_tokens * q.shape[1] // cache[0].shape[1] > PROMPT_ROWS)
        assert (np.abs(host(got) - want) <= tol).all()
        seen["kv4_attention"] += 1
        return got

    def rows(x, index, specs, rows_per_index=1):
        before = [host(s[3]).copy() for s in specs]
        real["lora_rows"](x, index, specs, rows_per_index)
        for (a, b, s, y), was in zip(specs, before):
            want, tol = _bound(host(x), host(a), host(b), host(s), was, host(index))
            assert (np.abs(host(y) - want) <= tol).all()
        seen["lora_rows"] += 1

    for name, f in (("kv4_append", append), ("kv4_attention", attention), ("lora_rows", rows)):
        monkeypatch.setattr(quant_hip, name, f)
    got = inference.generate_batch(model, _prompts(), 7, bank, [0, 1, -1, 2, 1], use_graph=False, page=16, prefill_rows=40)
    assert [len(g) for g in got] == [len(p) + 7 for p in _prompts()]
    steps = -(-sum(len(p) for p in _prompts()) // 40) + 6
    assert seen["kv4_append"] == seen["kv4_attention"] == 2 * steps and seen["lora_rows"] >= 4 * 2 * steps


@pytest.mark.parametrize("adapters", [None, [0, 1, -1, 2, 1]])
def test_captured_steps_give_the_eager_tokens(tmp_path, oracle, adapters):
    from alpaca_lora_4bit_amd import inference
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp, make_quant_attn
    build(str(tmp_path), oracle, seed=8)
    model, tokenizer = _loaded(str(tmp_path))
    make_quant_attn(model), make_fused_mlp(model)
    bank = None if adapters is None else _bank(model)
    want = [t.tolist() for t in inference.generate_batch(model, _prompts(), 24, bank, adapters, use_graph=False)]
    # an id that never comes makes the loop read every token on the host between two replays
    for eos in (None, -1):
        got = inference.generate_batch(model, _prompts(), 24, bank, adapters, eos_token_id=eos)
        assert [t.tolist() for t in got] == want
    # a request that ends early leaves the others as they were
    n = len(_prompts()[2])
    eos = want[2][n + 3]
    got = inference.generate_batch(model, _prompts(), 24, bank, adapters, eos_token_id=eos)
    for p, w, g in zip(_prompts(), want, got):
        answer = w[len(p):]
        assert g.tolist() == w[:len(p) + (answer.index(eos) + 1 if eos in answer else 24)]
    if adapters is not None:
        base = [t.tolist() for t in inference.generate_batch(model, _prompts(), 24)]
        assert base != want


def test_prompts_in_small_parts(tmp_path, oracle):
    """Parts in which no prompt ends, one row at a time at the least; the same parts give the same tokens."""
    from alpaca_lora_4bit_amd import inference
    build(str(tmp_path), oracle, seed=8)
    model, _ = _loaded(str(tmp_path))
    for rows in (1, 7):
        got = [[t.tolist() for t in inference.generate_batch(model, _prompts()[:3], 3, prefill_rows=rows, page=32, group=64)] for _ in range(2)]
        assert got[0] == got[1] and [len(g) for g in got[0]] == [len(p) + 3 for p in _prompts()[:3]]


def test_requests_from_the_command_line(tmp_path, oracle):
    from safetensors.torch import save_file
    from alpaca_lora_4bit_amd import inference
    ckpt = str(tmp_path / "ckpt")
    build(ckpt, oracle, seed=8, with_tokenizer=True)
    model, _ = _loaded(ckpt)
    gen = torch.Generator().manual_seed(2)
    lora = tmp_path / "lora"
    lora.mkdir()
    state = {}
    for name, m in model.named_modules():
        if name.endswith(("q_proj", "v_proj")):
            state[f"base_model.model.{name}.lora_A.weight"] = torch.randn(8, m.in_features, generator=gen).div(16)
            state[f"base_model.model.{name}.lora_B.weight"] = torch.randn(m.out_features, 8, generator=gen)
    save_file(state, str(lora / "adapter_model.safetensors"))
    (lora / "adapter_config.json").write_text(json.dumps({"r": 8, "lora_alpha": 16}))
    requests = tmp_path / "requests.jsonl"
    requests.write_text("\n".join(json.dumps(r) for r in ({"prompt": "alpha beta gamma"}, {"prompt": "alpha beta gamma", "lora": str(lora)},
                                                          {"prompt": "the layer of weight and matrix", "lora": None})) + "\n\n")
    args = [ckpt, os.path.join(ckpt, "model.safetensors"), "--groupsize", str(GROUPSIZE), "--max_new_tokens", "12", "--requests", str(requests)]
    texts, _ = inference.main(args + ["--greedy"])
    assert len(texts) == 3 and texts[0].startswith("alpha beta gamma") and texts[1].startswith("alpha beta gamma") and texts[0] != texts[1]
    assert inference.main(args + ["--greedy", "--fuse", "--hip_graph"])[0] == texts
    sampled, _ = inference.main(args + ["--hip_graph"])
    assert all(isinstance(t, str) for t in sampled)


def _step(B=6, heads=2, share=4, D=128, page=16, width=8, rows_of=2, seed=0):
    """The tensors of one decode step of B requests and a function that runs append, attention and adapters on them."""
    from alpaca_lora_4bit_amd import kv4_cache, quant_hip
    gen = torch.Generator(device="cuda").manual_seed(seed)
    half = lambda *s: torch.randn(*s, generator=gen, device="cuda").half()
    cache = kv4_cache.new_layer(B * width, heads, D, page, 64)
    rope = torch.randn(width * page, D // 2, 2, generator=gen, device="cuda")
    table = torch.randperm(B * width, generator=gen, device="cuda").int().view(B, width)
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    index = torch.tensor([0, 1, -1, 2, 1, 0][:B], dtype=torch.int32, device="cuda")
    K = heads * share * D
    x, k, v = half(B, K), half(B, heads, D), half(B, heads, D)
    bank = (half(3, 16, K) / 32, half(3, 256, 16), torch.rand(3, generator=gen, device="cuda"))

    def run():
        lengths.add_(1)
        q = quant_hip.kv4_append(k, v, cache, table, lengths, q=x.view(B, heads * share, D), rope=rope)
        o = quant_hip.kv4_attention(q, cache, table, lengths, max_tokens=1, max_length=width * page)
        y = torch.zeros(B, 256, dtype=torch.float16, device="cuda")
        quant_hip.lora_rows(o.view(B, -1), index, [bank + (y,)])
        return o, y
    return run, (x, k, v), lengths, cache


def test_captured_operators_follow_lengths_and_inputs():
    """Two graphs over two sets of tensors, replayed in turns with eager runs and synchronizations between them, on a stream of their own: every replay
    equals the eager run."""
    eager, graphs = [_step(seed=s) for s in (1, 2)], []
    side = torch.cuda.Stream()
    for s in (1, 2):
        run, inputs, lengths, cache = _step(seed=s)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        lengths.zero_()
        for c in cache:
            c.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out, inputs, lengths, cache, run))                # run holds the tensors that the graph reads
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i in range(40):
        which = i % 3 % 2
        run, inputs, lengths, cache = eager[which]
        graph, out, ginputs, glengths, gcache, _ = graphs[which]
        for t, g in zip(inputs, ginputs):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
            g.copy_(t)
        if i == 12:                                          # a request ends and another takes its place
            lengths[3] = -1
            glengths[3] = -1
        want = run()
        if i % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graph.replay()
        if i % 4 == 0:
            torch.cuda.synchronize()
            torch.zeros(1 << 20, device="cuda").sum().item()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), i
        assert torch.equal(lengths, glengths) and all(torch.equal(a, b) for a, b in zip(cache[:2], gcache[:2]))


def test_runs_on_two_streams_at_once():
    """Two independent runs on two streams give what each gives alone."""
    want = []
    for s in (3, 4):
        run = _step(seed=s)[0]
        want.append([tuple(t.clone() for t in run()) for _ in range(20)])
    torch.cuda.synchronize()
    steps, streams = [_step(seed=s)[0] for s in (3, 4)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(20):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                got[n].append(tuple(t.clone() for t in steps[n]()))
    torch.cuda.synchronize()
    for n in (0, 1):
        for a, b in zip(want[n], got[n]):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_pool_reads_what_a_request_holds():
    from alpaca_lora_4bit_amd import kv4_cache, quant_hip
    cache = kv4_cache.PagedKv4Cache(1, 2, 64, pages=5, page=16, group=32)
    a, b = cache.open(30), cache.open(40)
    gen = torch.Generator(device="cuda").manual_seed(1)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -1, -6], device="cuda").half()
    pick = lambda: grid[torch.randint(0, 10, (70, 2, 64), generator=gen, device="cuda")]
    k, v = pick(), pick()
    for t in (k, v):
        t[..., ::32] = 6.0                                   # the largest value of each group: its scale is 1 and every value is held exactly
    lengths, starts = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([30, 40], [0, 30, 70]))
    assert quant_hip.kv4_append(k, v, cache.layers[0], cache.table([a, b]), lengths, starts=starts) is None
    for handle, first, n in ((a, 0, 30), (b, 30, 40), (b, 30, 17), (a, 0, 0)):
        got = cache.read(0, handle, n)
        assert torch.equal(got[0], k[first:first + n]) and torch.equal(got[1], v[first:first + n])
