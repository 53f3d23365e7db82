"""Text generation with a 4-bit GPTQ LLaMA: the flow of the reference's top-level inference.py:1-49 as a module,

    python -m alpaca_lora_4bit_amd.inference ./llama-7b-4bit/ ./llama-7b-4bit/model.safetensors --groupsize 128 \\
        --prompt "I think the meaning of life is"

Steps as in the reference: load the packed model, `model.half()` and halve `scales` / `bias` (v1: `zeros`) of every
4-bit layer (`:15-22`), wrap `generate` in autocast (`:24-27`), sample with the reference's settings (`:33-44`:
temperature 0.9, top-p 0.95, top-k 40, repetition penalty 1.1, 20 new tokens), print the text and the seconds taken.
`--lora` applies an adapter directory written by `alpaca_lora_4bit_amd.finetune` (or by peft) first.

Two additions for decode speed, both off by default: `--fuse` gives q/k/v one grouped launch on their own tensors and
runs the MLP decode step (gate, up, silu * up, down) as one launch, adapters included
(model_attn_mlp_patch.make_quant_attn / make_fused_mlp, which the reference's model server calls, server/server.py:100-113),
and `--hip_graph` captures the one-token step once as a HIP graph and replays it per token, which removes the host
time of the ~1000 small launches a decoder step consists of; the choice of the next token (argmax with `--greedy`,
otherwise the reference's sampling settings) runs eagerly between two replays.

`--requests FILE` answers many prompts together, each with the adapter of its own choice: a JSON object per line,
`{"prompt": ..., "lora": directory}` ("lora" may be left out).  Their keys and values are held in 4 bits in a paged cache
(kv4_cache.py) and their adapters beside each other (models.AdapterBank); see `generate_batch`.
"""
import argparse
import contextlib
import json
import time

import torch

SAMPLING = dict(do_sample=True, use_cache=True, repetition_penalty=1.1, temperature=0.9, top_p=0.95, top_k=40,
                return_dict_in_generate=True, output_attentions=False, output_hidden_states=False,
                output_scores=False)


def _parse(argv):
    p = argparse.ArgumentParser(description="Generate text with a 4-bit GPTQ LLaMA")
    p.add_argument("config_path", nargs="?", default="./llama-13b-4bit/")
    p.add_argument("model_path", nargs="?", default="./llama-13b-4bit.pt")
    p.add_argument("--groupsize", type=int, default=-1)
    p.add_argument("--v1", action="store_true")
    p.add_argument("--lora", default=None, help="adapter directory to apply")
    p.add_argument("--lora_r", type=int, default=8)
    p.add_argument("--lora_alpha", type=int, default=16)
    p.add_argument("--prompt", default="I think the meaning of life is")
    p.add_argument("--max_new_tokens", type=int, default=20)
    p.add_argument("--greedy", action="store_true", help="argmax decoding instead of sampling")
    p.add_argument("--fuse", action="store_true", help="one launch for q+k+v and one for gate+up")
    p.add_argument("--hip_graph", action="store_true", help="decode with the token step replayed as a HIP graph")
    p.add_argument("--requests", default=None, help="file with a JSON object per line, {\"prompt\": ..., \"lora\": directory}: answer them as one batch")
    return p.parse_args(argv)


def prepare_model(model):
    """fp16 everywhere the reference puts it (inference.py:15-22)."""
    from .autograd_4bit import Autograd4bitQuantLinear
    model.half()
    for _, m in model.named_modules():
        if isinstance(m, Autograd4bitQuantLinear):
            if m.is_v1_model:
                m.zeros = m.zeros.half()
            m.scales = m.scales.half()
            m.bias = m.bias.half()
    return model


def _token_picker(sampling):
    """Returns pick(ids_so_far, logits) -> next token [1, 1].  `sampling` None: argmax.  Otherwise a dict with the
    reference's settings (inference.py:33-44: repetition_penalty, temperature, top_k, top_p) applied through
    transformers' own logits processors in the order `generate` applies them, then one multinomial draw."""
    if sampling is None:
        return lambda ids, logits: logits.argmax(-1, keepdim=True)
    from transformers import (LogitsProcessorList, RepetitionPenaltyLogitsProcessor, TemperatureLogitsWarper,
                              TopKLogitsWarper, TopPLogitsWarper)
    procs = LogitsProcessorList()
    if sampling.get("repetition_penalty", 1.0) != 1.0:
        procs.append(RepetitionPenaltyLogitsProcessor(penalty=sampling["repetition_penalty"]))
    if sampling.get("temperature", 1.0) != 1.0:
        procs.append(TemperatureLogitsWarper(sampling["temperature"]))
    if sampling.get("top_k"):
        procs.append(TopKLogitsWarper(top_k=sampling["top_k"]))
    if sampling.get("top_p", 1.0) < 1.0:
        procs.append(TopPLogitsWarper(top_p=sampling["top_p"]))

    def pick(ids, logits):
        scores = procs(ids, logits.float())
        return torch.multinomial(torch.softmax(scores, dim=-1), num_samples=1)
    return pick


def generate_graph(model, input_ids, max_new_tokens, eos_token_id=None, sampling=None, use_graph=True):
    """Decoding of one sequence with the model's one-token forward captured once as a HIP graph and replayed for
    every further token: eager prefill into a static KV cache, the second token from one eager step (the warm-up
    that graph capture wants: every lazy allocation and per-layer check of the kernels' host side happens there),
    then replays.  Token id and position live in device buffers that the replays read; the choice of the next
    token (argmax, or the logits processors + multinomial of `sampling`) runs eagerly between two replays.
    `use_graph=False` runs the same loop without capture.  Returns the ids [1, prompt + new] like `generate`;
    stops early at `eos_token_id`."""
    from transformers import StaticCache
    dev = input_ids.device
    prompt = input_ids.shape[1]
    pick = _token_picker(sampling)
    with torch.no_grad():
        cache = StaticCache(config=model.config, max_cache_len=prompt + max_new_tokens)
        out = model(input_ids=input_ids, past_key_values=cache, use_cache=True,
                    cache_position=torch.arange(prompt, device=dev))
        ids = input_ids
        tok_buf = torch.empty((1, 1), dtype=input_ids.dtype, device=dev)
        pos_buf = torch.tensor([prompt - 1], device=dev)

        def advance(logits):
            nonlocal ids
            nxt = pick(ids, logits)
            tok_buf.copy_(nxt)
            pos_buf.add_(1)
            ids = torch.cat([ids, nxt], dim=1)
            return eos_token_id is not None and int(nxt[0, 0]) == eos_token_id

        def step():
            o = model(input_ids=tok_buf, past_key_values=cache, use_cache=True, cache_position=pos_buf)
            return o.logits[:, -1]

        done = advance(out.logits[:, -1])
        if not done and max_new_tokens > 1:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                logits = step()
            torch.cuda.current_stream().wait_stream(side)
            done = advance(logits)
            remaining = max_new_tokens - 2
            if not done and remaining > 0:
                if use_graph:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        logits = step()
                for _ in range(remaining):
                    if use_graph:
                        graph.replay()
                    else:
                        logits = step()
                    if advance(logits):
                        break
    return ids


def greedy_generate_graph(model, input_ids, max_new_tokens, eos_token_id=None):
    """`generate_graph` with argmax decoding."""
    return generate_graph(model, input_ids, max_new_tokens, eos_token_id=eos_token_id)


def _passed_by(module, cls):
    """What would be left out if `module`, in whose place a batch runs its parts, were not called: a hook, or a forward that is not the one of
    transformers' LLaMA class `cls`.  None where there is no such thing: this package's groups and its wrappers of a forward (autocast,
    checkpointing, the fused MLP step) are known to change nothing here."""
    from .gradient_checkpointing import _ForwardPatch
    from .model_attn_mlp_patch import _FusedGroup, _MemberGroup, _mlp_decode_forward, _mlp_gated_forward
    for hooks in (module._forward_hooks, module._forward_pre_hooks, module._backward_hooks, module._backward_pre_hooks):
        if any(not isinstance(getattr(h, "__self__", None), (_FusedGroup, _MemberGroup)) for h in hooks.values()):
            return "a hook"
    own = module.__dict__
    forward = own.get("forward")
    if "_q4_mlp_forward" in own and getattr(forward, "__func__", None) in (_mlp_decode_forward, _mlp_gated_forward):
        forward = own["_q4_mlp_forward"]
    elif "non_autocast_forward" in own and getattr(forward, "__wrapped__", None) is own["non_autocast_forward"]:
        forward = own["non_autocast_forward"]
    elif "old_forward_for_cp" in own and isinstance(getattr(forward, "__self__", None), _ForwardPatch):
        forward = own["old_forward_for_cp"]
    if forward is not None and getattr(forward, "__func__", None) is not type(module).forward:
        return "a replaced forward"
    stock = type(module).forward
    if (stock.__module__, stock.__qualname__) != ("transformers.models.llama.modeling_llama", f"{cls}.forward"):
        return "a forward that is not LLaMA's"
    return None


def _check_blocks(model, bank):
    """Everything that a batch takes apart is as it knows it (ValueError otherwise)."""
    if torch.nn.modules.module._has_any_global_hook():
        raise ValueError("batches of requests do not call every module: a global module hook would miss some")
    net = model.model
    parts = [("the model", model, "LlamaForCausalLM"), ("model", net, "LlamaModel")]
    for i, block in enumerate(net.layers):
        parts += [(f"model.layers.{i}", block, "LlamaDecoderLayer"), (f"model.layers.{i}.self_attn", block.self_attn, "LlamaAttention")]
        if bank is not None and bank.holds(*(getattr(block.mlp, n, None) for n in ("gate_proj", "up_proj", "down_proj"))):
            parts.append((f"model.layers.{i}.mlp", block.mlp, "LlamaMLP"))
    for name, module, cls in parts:
        what = _passed_by(module, cls)
        if what is not None:
            raise ValueError(f"batches of requests take {name} apart, which has {what} that they would leave out")


class _BatchModel:
    """A LLaMA's blocks over rows of many sequences: the modules of the loaded model do the products and norms, the keys and values go through
    the 4-bit paged cache and every row's own adapter is added to the products."""

    def __init__(self, model, cache, bank, positions):
        from .kv4_cache import rope_table
        cfg = model.config
        self.model, self.cache, self.bank = model, cache, bank
        _check_blocks(model, bank)
        if bank is not None:
            taken = {getattr(part, n, None) for block in model.model.layers for part, names in ((block.self_attn, "qkvo"), (block.mlp, ("gate", "up", "down")))
                     for n in (f"{x}_proj" for x in names)}
            for layer, name in bank.names.items():
                if layer not in taken:
                    raise ValueError(f"the bank has an adapter of {name or 'a layer'}, which a batch of requests does not add")
        self.heads, self.kv_heads, self.head_dim = _attention_shape(cfg)
        self.rope = rope_table(model.model.rotary_emb, positions, cache.device)

    def _add(self, x, index, *pairs):
        if self.bank is not None and index is not None:
            self.bank.apply(x, index, pairs)

    def _mlp(self, mlp, x, index):
        if index is None or self.bank is None or not self.bank.holds(mlp.gate_proj, mlp.up_proj, mlp.down_proj):
            return mlp(x)
        gate, up = mlp.gate_proj(x), mlp.up_proj(x)
        self._add(x, index, (mlp.gate_proj, gate), (mlp.up_proj, up))
        act = (mlp.act_fn(gate) * up).contiguous()
        out = mlp.down_proj(act)
        self._add(act, index, (mlp.down_proj, out))
        return out

    def __call__(self, ids, table, lengths, starts, index, max_tokens, max_length, wanted=None):
        """Logits [rows, vocabulary] of the rows `ids` (`wanted`: of these rows only); see quant_hip.kv4_attention for the batch's tensors."""
        from . import quant_hip
        net = self.model.model
        h = net.embed_tokens(ids)
        for block, layer in zip(net.layers, self.cache.layers):
            attn = block.self_attn
            x = block.input_layernorm(h).contiguous()
            q, k, v = attn.q_proj(x), attn.k_proj(x), attn.v_proj(x)
            self._add(x, index, (attn.q_proj, q), (attn.k_proj, k), (attn.v_proj, v))
            k, v = (t.view(-1, self.kv_heads, self.head_dim) for t in (k, v))
            q = quant_hip.kv4_append(k, v, layer, table, lengths, q=q.view(-1, self.heads, self.head_dim), rope=self.rope, starts=starts)
            o = quant_hip.kv4_attention(q, layer, table, lengths, starts=starts, max_tokens=max_tokens, max_length=max_length)
            o = o.view(-1, self.heads * self.head_dim)
            out = attn.o_proj(o)
            self._add(o, index, (attn.o_proj, out))
            h = h + out
            h = h + self._mlp(block.mlp, block.post_attention_layernorm(h).contiguous(), index)
        if wanted is not None:
            h = h[wanted]
        return self.model.lm_head(net.norm(h))


def _attention_shape(cfg):
    if getattr(cfg, "model_type", None) != "llama":
        raise ValueError(f"batches of requests are built for LLaMA models, not for {getattr(cfg, 'model_type', None)!r}")
    heads = cfg.num_attention_heads
    return heads, getattr(cfg, "num_key_value_heads", None) or heads, getattr(cfg, "head_dim", None) or cfg.hidden_size // heads


_capture_streams = {}                                        # by device: torch's own is one for all, on the device that captured first


def _capture_stream(dev):
    if dev.index not in _capture_streams:
        _capture_streams[dev.index] = torch.cuda.Stream(dev)
    return _capture_streams[dev.index]


def generate_batch(model, prompts, max_new_tokens, bank=None, adapters=None, eos_token_id=None, sampling=None, use_graph=True,
                   page=64, group=32, prefill_rows=8192):
    """Continues many prompts together.  `prompts`: 1-D id tensors, of any lengths; `adapters`: for each of them the number of its adapter in
    `bank` (a models.AdapterBank), or -1.  The prompts run without padding, their rows one after another, in parts of at most `prefill_rows`
    rows; then every step answers one token of every request, its forward captured once as a HIP graph (`use_graph`) as in
    `generate_graph`.  Keys and values are held in 4 bits with a scale per `group` dimensions, in pages of `page` tokens.  Returns a list of id
    tensors, prompt and answer, each ended by `eos_token_id` or after `max_new_tokens`."""
    from .kv4_cache import PagedKv4Cache
    count = len(prompts)
    if count == 0 or max_new_tokens < 1:
        return [p.clone() for p in prompts]
    if any(p.dim() != 1 or p.numel() == 0 for p in prompts):
        raise ValueError("prompts must be 1-D tensors of at least one id")
    if (bank is None) != (adapters is None) or (adapters is not None and len(adapters) != count):
        raise ValueError("`bank` and `adapters` (one number for each prompt) go together")
    if adapters is not None and any(not -1 <= a < bank.count for a in adapters):
        raise ValueError(f"adapters must be -1 .. {bank.count - 1}")
    if prefill_rows < 1 or page < 1:
        raise ValueError("prefill_rows and page must be positive")
    heads, kv_heads, head_dim = _attention_shape(model.config)
    dev = prompts[0].device
    totals = [p.numel() + max_new_tokens for p in prompts]
    longest = max(totals)
    pages = sum(-(-t // page) for t in totals)
    pick = _token_picker(sampling)
    ints = dict(dtype=torch.int32)
    with torch.no_grad(), torch.cuda.device(dev) if dev.type == "cuda" else contextlib.nullcontext():
        cache = PagedKv4Cache(len(model.model.layers), kv_heads, head_dim, pages, page, group, dev)
        run = _BatchModel(model, cache, bank, longest)
        handles = [cache.open(t) for t in totals]
        index = None if adapters is None else torch.tensor(list(adapters), **ints).to(dev)

        # the prompts, in parts of at most prefill_rows rows: each part is runs of tokens of some requests
        parts, part, room = [], [], prefill_rows
        for b, p in enumerate(prompts):
            done = 0
            while done < p.numel():
                take = min(room, p.numel() - done)
                part.append((b, done, done + take))
                done += take
                room -= take
                if room == 0:
                    parts.append(part)
                    part, room = [], prefill_rows
        if part:
            parts.append(part)
        first = [None] * count
        for part in parts:
            rows = [stop - start for _, start, stop in part]
            starts = [0]
            for r in rows:
                starts.append(starts[-1] + r)
            ends = [(b, starts[i + 1] - 1) for i, (b, _, stop) in enumerate(part) if stop == prompts[b].numel()]
            logits = run(torch.cat([prompts[b][start:stop] for b, start, stop in part]), cache.table([handles[b] for b, _, _ in part]),
                         torch.tensor([stop for _, _, stop in part], **ints).to(dev), torch.tensor(starts, **ints).to(dev),
                         None if index is None else torch.repeat_interleave(index[[b for b, _, _ in part]], torch.tensor(rows, device=dev)),
                         max(rows), max(stop for _, _, stop in part), torch.tensor([row for _, row in ends], dtype=torch.long, device=dev))
            for (b, _), line in zip(ends, logits):
                first[b] = line

        table = cache.table(handles)
        lengths = torch.tensor([p.numel() for p in prompts], **ints).to(dev)
        tokens = torch.zeros(count, dtype=prompts[0].dtype, device=dev)
        alive = torch.ones(count, **ints).to(dev)
        ids = list(prompts)
        going = [True] * count

        def advance(logits):
            """The next token of every request; True when all of them have ended.  An ended request keeps its row, with a length of zero: nothing
            of it is stored and its attention reads nothing."""
            if sampling is None:
                nxt = logits.argmax(-1)
            else:
                nxt = torch.cat([pick(ids[b][None], logits[b][None])[0] if going[b] else tokens[b:b + 1] for b in range(count)])
            nxt = nxt.to(tokens.dtype)
            for b in range(count):
                if going[b]:
                    ids[b] = torch.cat([ids[b], nxt[b:b + 1]])
            tokens.copy_(nxt)
            if eos_token_id is not None:
                for b, t in enumerate(nxt.tolist()):
                    if going[b] and t == eos_token_id:
                        going[b] = False
                        alive[b] = 0
                        lengths[b] = 0
            return not any(going)

        def step():
            lengths.add_(alive)
            return run(tokens, table, lengths, None, index, 1, longest)

        left = max_new_tokens - 1
        done = advance(torch.stack(first))
        graph, warm = None, not use_graph
        while left and not done:
            if graph is not None:
                graph.replay()
            elif not warm:
                # one eager step on a side stream first: every lazy allocation and per-layer check happens there
                side = torch.cuda.Stream(dev)
                side.wait_stream(torch.cuda.current_stream(dev))
                with torch.cuda.stream(side):
                    logits = step()
                torch.cuda.current_stream(dev).wait_stream(side)
                warm = True
            elif use_graph and left > 1:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=_capture_stream(dev)):
                    logits = step()
                graph.replay()
            else:
                logits = step()
            left -= 1
            done = advance(logits)
        return ids


def _answer_requests(model, tokenizer, args):
    """--requests: (texts, seconds)."""
    from . import models
    with open(args.requests) as fh:
        requests = [json.loads(line) for line in fh if line.strip()]
    dirs = sorted({r["lora"] for r in requests if r.get("lora")})
    bank = models.AdapterBank(model, dirs) if dirs else None
    adapters = [dirs.index(r["lora"]) if r.get("lora") else -1 for r in requests] if dirs else None
    prompts = [tokenizer(r["prompt"], return_tensors="pt", add_special_tokens=False)["input_ids"][0].cuda() for r in requests]
    sampling = None if args.greedy else {k: SAMPLING[k] for k in ("repetition_penalty", "temperature", "top_k", "top_p")}
    start = time.time()
    sequences = generate_batch(model, prompts, args.max_new_tokens, bank, adapters, eos_token_id=getattr(tokenizer, "eos_token_id", None),
                               sampling=sampling, use_graph=args.hip_graph)
    texts = [tokenizer.decode(s.tolist()) for s in sequences]
    seconds = time.time() - start
    for text in texts:
        print(text)
    print(seconds)
    return texts, seconds


def main(argv=None):
    """Returns (text, seconds); with --requests (texts, seconds)."""
    args = _parse(argv)
    from . import models
    from .amp_wrapper import AMPWrapper
    from .autograd_4bit import load_llama_model_4bit_low_ram
    if models.HAVE_PEFT:
        from .monkeypatch.peft_tuners_lora_monkey_patch import replace_peft_model_with_int4_lora_model
        replace_peft_model_with_int4_lora_model()

    model, tokenizer = load_llama_model_4bit_low_ram(args.config_path, args.model_path, groupsize=args.groupsize,
                                                      is_v1_model=args.v1)
    if args.lora is not None:
        from .finetune import LORA_TARGETS, load_adapter
        models.inject_lora_layers(model, target_modules=LORA_TARGETS, r=args.lora_r, lora_alpha=args.lora_alpha)
        print(load_adapter(model, args.lora), "adapter tensors loaded from", args.lora)
    print("Fitting 4bit scales and zeros to half")
    prepare_model(model)

    if args.fuse:
        from .model_attn_mlp_patch import make_fused_mlp, make_quant_attn
        print("Fused", make_quant_attn(model), "attention blocks and", make_fused_mlp(model), "MLP blocks")

    if args.requests is not None:
        return _answer_requests(model, tokenizer, args)

    print("Apply AMP Wrapper ...")
    AMPWrapper(model).apply_generate()

    batch = tokenizer(args.prompt, return_tensors="pt", add_special_tokens=False)
    batch = {k: v.cuda() for k, v in batch.items()}
    options = dict(SAMPLING, max_new_tokens=args.max_new_tokens)
    if args.greedy:
        options.update(do_sample=False, temperature=None, top_p=None, top_k=None)
    start = time.time()
    if args.hip_graph:
        sampling = None if args.greedy else {k: SAMPLING[k] for k in ("repetition_penalty", "temperature", "top_k", "top_p")}
        with torch.amp.autocast(device_type="cuda"):
            sequences = generate_graph(model, batch["input_ids"], args.max_new_tokens,
                                       eos_token_id=getattr(tokenizer, "eos_token_id", None), sampling=sampling)
    else:
        with torch.no_grad():
            sequences = model.generate(inputs=batch["input_ids"], **options)["sequences"]
    text = tokenizer.decode(sequences.cpu().tolist()[0])
    seconds = time.time() - start
    print(text)
    print(seconds)
    return text, seconds


if __name__ == "__main__":
    main()
