"""Training adapters on pairs of answers, a preferred and a rejected one, and what such a step keeps for its backward pass.

  "checkpoint"  a block's input held in 8 bits between forward and backward: packed, and read back
  "gated"       silu(gate) * up of a gated block, keeping gate and up in 8 bits, and its gradients from what was kept
  "logps"       log-probabilities of the tokens of answers, for scoring or with the gradient of the logits
  "preference"  the loss of the pairs, from the logits and the reference's log-probabilities, and the gradient of the logits

8 bits: of every 32 neighbouring values the scale s is the least bfloat16 with 127 s >= the largest magnitude, and a value is held as the
nearest whole number of s (ties to the even one).  Logits [B, S, V] at a place are those of the token that `labels` [B, S] has there; a label
outside 0 .. V - 1 is no token of the answer.  With the first half of the B sequences preferred to the second half, sequence by sequence,

  r_b  = sum over the answer of (log-probability - the reference's)        z_p  = beta (r_p - r_{p + B/2})
  loss = mean over p of -(1 - smoothing) log sigmoid(z_p) - smoothing log sigmoid(-z_p)          rewards = beta r

Widths are those of the 7B and 13B layers (4096 and 5120 features, 11008 and 13824 between the projections of a gated block), vocabularies those of the
test models and of 32000 tokens, one more with a token for padding.
"""
import torch

own = False

_BLOCK = 32
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    c, g = {"op": "checkpoint"}, {"op": "gated"}
    s, p = {"op": "logps"}, {"op": "preference"}
    return [
        # one short sample: latency
        {"name": "checkpoint_1_sample", **c, "rows": 61, "cols": 4096, "type": "fp16"},
        # the block inputs of the script's micro-batch of four samples of 256 tokens
        {"name": "checkpoint_4x256", **c, "rows": 1024, "cols": 4096, "type": "fp16"},
        # 13B, eight pairs of long answers, the residual stream in 32 bits
        {"name": "checkpoint_16x1024_fp32", **c, "rows": 16384, "cols": 5120, "type": "fp32"},
        # a short sample through a gated block, an odd number of values
        {"name": "gated_1_sample_odd", **g, "rows": 61, "cols": 2731, "type": "fp16"},
        # the same micro-batch through the 7B gated block
        {"name": "gated_4x256", **g, "rows": 1024, "cols": 11008, "type": "fp16"},
        # pairs of long answers through the 13B gated block, in bfloat16
        {"name": "gated_8x1024_bf16", **g, "rows": 8192, "cols": 13824, "type": "bf16"},
        # scoring one short answer: latency
        {"name": "logps_1_answer", **s, "b": 1, "s": 37, "v": 32000, "type": "fp16", "prompt": 0.0, "train": False},
        # the reference's pass over four pairs of the script's 256 tokens, logits handed over in 32 bits
        {"name": "logps_8x256_fp32", **s, "b": 8, "s": 256, "v": 32000, "type": "fp32", "prompt": 0.4, "train": False},
        # token by token with a gradient; rows of an odd number of 16-bit values
        {"name": "logps_train_odd_rows", **s, "b": 5, "s": 333, "v": 32001, "type": "bf16", "prompt": 0.2, "train": True},
        # one pair of short answers: latency
        {"name": "preference_1_pair", **p, "b": 2, "s": 48, "v": 32000, "type": "fp16", "prompt": 0.3, "smoothing": 0.0},
        # four pairs as the script trains them
        {"name": "preference_4_pairs_fp32", **p, "b": 8, "s": 256, "v": 32000, "type": "fp32", "prompt": 0.4, "smoothing": 0.0},
        # sixteen pairs of long answers
        {"name": "preference_16_pairs_long", **p, "b": 32, "s": 1024, "v": 32000, "type": "fp16", "prompt": 0.3, "smoothing": 0.1},
    ]


def _log_between(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges: up to 16384 rows of a block's width, up to 32 sequences of 2048 tokens over 300 to 131072 words."""
    op = rng.choice(["checkpoint", "gated", "logps", "preference"])
    if op in ("checkpoint", "gated"):
        cols = rng.choice([4096, 5120] if op == "checkpoint" else [11008, 13824]) if rng.random() < 0.6 else _log_between(rng, 33, 13824)
        most = (16384 * 5120 if op == "checkpoint" else 8192 * 13824) // cols
        return {"op": op, "rows": _log_between(rng, 1, min(16384, most)), "cols": cols, "type": rng.choice(["fp16", "fp16", "bf16"] + ["fp32"] * (op == "checkpoint"))}
    kind = rng.choice(["fp16", "fp16", "bf16", "fp32", "fp32"])
    b = 2 * _log_between(rng, 1, 16) if op == "preference" else _log_between(rng, 1, 32)
    s = _log_between(rng, 2, 2048)
    v = rng.choice([32000, 32000, 32001, _log_between(rng, 300, 131072)])
    v = max(300, min(v, 32 * 1024 * 32000 * 2 // _SIZES[kind] // (b * s)))
    c = {"op": op, "b": b, "s": s, "v": v, "type": kind, "prompt": rng.choice([0.0, 0.2, 0.4, 0.7])}
    if op == "logps":
        c["train"] = rng.random() < 0.5
    else:
        c["smoothing"] = rng.choice([0.0, 0.0, 0.1])
    return c


def _answers(c):
    """(first, behind the last) place of every sequence's answer: a prompt before it, padding behind all but the longest."""
    out = []
    for i in range(c["b"]):
        end = c["s"] if i == 0 else max(1, int(c["s"] * (1.0 - 0.5 * ((i * 0.6180339887498949) % 1.0))))
        out.append((min(end - 1, int(c["prompt"] * end)), end))
    return out


def work(case):
    c, size = case, _SIZES[case["type"]]
    if c["op"] in ("checkpoint", "gated"):
        n = c["rows"] * c["cols"]
        held = n + 2 * -(-n // _BLOCK)
        if c["op"] == "checkpoint":
            return {"bytes": 2 * (n * size + held), "flops": 4 * n}
        return {"bytes": n * size * 6 + 4 * held, "flops": 24 * n}
    live, rows, v = sum(b - a for a, b in _answers(c)), c["b"] * c["s"], c["v"]
    graded = c["op"] == "preference" or c["train"]
    return {"bytes": live * v * size + rows * 12 + (rows * v * size if graded else 0), "flops": live * v * (8 if graded else 4)}


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c, dev, kind = case, "cuda", _TYPES[case["type"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    if c["op"] in ("checkpoint", "gated"):
        shape = (c["rows"], c["cols"])

        def normal():
            return torch.randn(shape, generator=gen, device=dev)
        if c["op"] == "gated":
            return {"op": "gated", "gate": (normal() * 2.0).to(kind), "up": normal().to(kind), "dout": (normal() * 0.02).to(kind)}
        x = normal()
        x[:, ::509] *= 60.0                                    # a residual stream has a few features far above the others
        return {"op": "checkpoint", "x": x.to(kind)}
    b, s, v = c["b"], c["s"], c["v"]
    logits = torch.empty((b, s, v), dtype=kind, device=dev)
    labels = torch.full((b, s), -100, dtype=torch.long, device=dev)
    ref = torch.full((b, s), float("nan"), device=dev)         # what a reference says about places outside the answers is not asked
    for i, (first, end) in enumerate(_answers(c)):
        x = torch.randn((s, v), generator=gen, device=dev) * 2.0
        said = torch.randint(0, v, (s,), generator=gen, device=dev)
        x.scatter_add_(1, said[:, None], 4.0 + 6.0 * torch.rand((s, 1), generator=gen, device=dev))
        logits[i] = x.to(kind)
        labels[i, first:end] = said[first:end]
        x = logits[i, first:end].float()
        top = x.amax(-1)
        mine = x.gather(1, said[first:end, None])[:, 0] - top - (x - top[:, None]).exp().sum(-1).log()
        ref[i, first:end] = mine + 0.2 * torch.randn(mine.shape, generator=gen, device=dev)
    st = {"op": c["op"], "logits": logits.requires_grad_(c["op"] == "preference" or c["train"]), "labels": labels}
    if c["op"] == "preference":
        # a loss scaled as for training in 16 bits
        return {**st, "ref": ref, "beta": 0.1, "smoothing": c["smoothing"], "grad": torch.tensor(1024.0, device=dev)}
    return {**st, "grad": torch.randn((b, s), generator=gen, device=dev) if c["train"] else None}


# ------------------------------------------------------------------------------------------------------------- the plain forms
def _held(x):
    """float32 values that 8 bits hold for x (any type), in x's shape."""
    flat = x.float().reshape(-1)
    g = torch.nn.functional.pad(flat, (0, -len(flat) % _BLOCK)).reshape(-1, _BLOCK)
    top = g.abs().amax(1)
    s = (top.double() / 127).float().bfloat16()
    s = torch.where(s.float() * 127 < top, (s.view(torch.int16) + 1).view(torch.bfloat16), s).float()[:, None]
    q = torch.round(torch.where(s > 0, g / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g)))
    return (q * s).reshape(-1)[:len(flat)].reshape(x.shape)


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _gated_plain(s):
    g, u = s["gate"].float(), s["up"].float()
    out = (g * _sigmoid(g) * u).to(s["gate"].dtype)
    g, u, d = _held(s["gate"]), _held(s["up"]), s["dout"].float()
    sig = _sigmoid(g)
    return {"out": out, "dgate": (d * u * sig * (1.0 + g * (1.0 - sig))).to(out.dtype), "dup": (d * g * sig).to(out.dtype)}


def _live(logits, labels, kind):
    """(places of the answers' tokens in a list of all, their labels, x - max, log sum exp of that), the last two in `kind`."""
    v = logits.shape[-1]
    lab = labels.reshape(-1)
    at = torch.nonzero((lab >= 0) & (lab < v))[:, 0]
    x = logits.detach().reshape(-1, v)[at].to(kind)
    x = x - x.amax(-1, keepdim=True)
    return at, lab[at], x, torch.log(torch.exp(x).sum(-1, keepdim=True))


def _grad_plain(logits, at, lab, x, total, coef):
    """coef (1[label] - softmax) at the answers' tokens, zero elsewhere."""
    g = torch.exp((x - total).float()).neg_()
    g[torch.arange(len(at), device=g.device), lab] += 1.0
    out = torch.zeros_like(logits, requires_grad=False)
    out.view(-1, out.shape[-1])[at] = g.mul_(coef[:, None]).to(out.dtype)
    return out


def _logps_plain(s):
    logits, labels = s["logits"], s["labels"]
    at, lab, x, total = _live(logits, labels, torch.float32)
    out = torch.zeros(labels.shape, device=logits.device)
    out.view(-1)[at] = (x.gather(1, lab[:, None]) - total)[:, 0]
    if s["grad"] is None:
        return out
    return {"logps": out, "dlogits": _grad_plain(logits, at, lab, x, total, s["grad"].reshape(-1)[at])}


def _preference_plain(s):
    logits, labels, beta, eps = s["logits"], s["labels"], s["beta"], s["smoothing"]
    b, n = labels.shape
    at, lab, x, total = _live(logits, labels, torch.float64)        # log ratios are small differences of long sums
    ratio = torch.zeros(b * n, dtype=torch.float64, device=logits.device)
    ratio[at] = (x.gather(1, lab[:, None]) - total)[:, 0] - s["ref"].reshape(-1)[at].double()
    r = ratio.reshape(b, n).sum(1)
    z = beta * (r[:b // 2] - r[b // 2:])
    soft = torch.log1p(torch.exp(-z.abs()))
    loss = ((1 - eps) * (soft + (-z).clamp(min=0)) + eps * (soft + z.clamp(min=0))).mean()
    dz = (eps * _sigmoid(z) - (1 - eps) * _sigmoid(-z)) * (beta / (b // 2))
    coef = (torch.cat((dz, -dz)).repeat_interleave(n)[at] * s["grad"].double()).float()
    return {"loss": loss.float(), "rewards": (beta * r).float(), "dlogits": _grad_plain(logits, at, lab, x, total, coef)}


def run(state):
    s = state
    if own:
        from alpaca_lora_4bit_amd import preference, quant_hip
        if s["op"] == "checkpoint":
            codes, scales = quant_hip.act8_pack(s["x"])
            return quant_hip.act8_unpack(codes, scales, s["x"].dtype)
        if s["op"] == "gated":
            out, kept = quant_hip.silu_mul_act8(s["gate"], s["up"])
            dgate, dup = quant_hip.silu_mul_act8_bwd(s["dout"], kept)
            return {"out": out, "dgate": dgate, "dup": dup}
        if s["op"] == "logps":
            logps = preference.token_logps(s["logits"], s["labels"])
            if s["grad"] is None:
                return logps
            return {"logps": logps, "dlogits": torch.autograd.grad(logps, s["logits"], s["grad"])[0]}
        loss, rewards = preference.preference_loss(s["logits"], s["labels"], s["ref"], beta=s["beta"], label_smoothing=s["smoothing"])
        return {"loss": loss, "rewards": rewards, "dlogits": torch.autograd.grad(loss, s["logits"], s["grad"])[0]}
    if s["op"] == "checkpoint":
        return _held(s["x"]).to(s["x"].dtype)
    if s["op"] == "gated":
        return _gated_plain(s)
    return _logps_plain(s) if s["op"] == "logps" else _preference_plain(s)


# --------------------------------------------------------------------------------------------------------- in 64 bits, one by one
def _exact_held(x):
    """Nearest whole multiples of each block's scale, from mantissas and exponents."""
    n = x.numel()
    g = x.double().flatten()
    g = torch.cat((g, g.new_zeros(-n % _BLOCK))).view(-1, _BLOCK)
    m, e = torch.frexp(g.abs().max(1).values / 127)
    s = torch.ldexp(torch.ceil(m * 256), e - 8)[:, None]        # the least number of 8 leading bits that is large enough
    y = g / torch.where(s == 0, 1.0, s)
    low = torch.floor(y)
    up = (y - low > 0.5) | ((y - low == 0.5) & (torch.remainder(low, 2) == 1))
    return ((low + up) * s).flatten()[:n].view(x.shape)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "checkpoint":
        return _exact_held(s["x"])
    if c["op"] == "gated":
        out = torch.nn.functional.silu(s["gate"].double()).mul_(s["up"].double())
        g, u, d = _exact_held(s["gate"]), _exact_held(s["up"]), s["dout"].double()
        sig = torch.sigmoid(g)
        return {"out": out, "dgate": d * u * (sig + g * sig * torch.sigmoid(-g)), "dup": d * g * sig}
    logits, labels = s["logits"].detach(), s["labels"]
    half = c["b"] // 2
    logps = torch.zeros(labels.shape, dtype=torch.float64, device=logits.device)
    probs = []
    for i, (first, end) in enumerate(_answers(c)):
        lp = torch.log_softmax(logits[i, first:end].double(), -1)
        logps[i, first:end] = lp[torch.arange(end - first, device=lp.device), labels[i, first:end]]
        probs.append(lp.exp())
    if c["op"] == "logps" and not c["train"]:
        return logps
    if c["op"] == "preference":
        r = torch.stack([(logps[i, a:e] - s["ref"][i, a:e].double()).sum() for i, (a, e) in enumerate(_answers(c))])
        z = s["beta"] * (r[:half] - r[half:])
        keep, flip = 1 - s["smoothing"], s["smoothing"]
        loss = -(keep * torch.nn.functional.logsigmoid(z) + flip * torch.nn.functional.logsigmoid(-z)).mean()
        dz = -(keep * torch.sigmoid(-z) - flip * torch.sigmoid(z)) * s["beta"] / half * float(s["grad"])
        weight = torch.cat((dz, -dz))[:, None].expand(labels.shape)
    else:
        weight = s["grad"].double()
    grad = torch.zeros(logits.shape, dtype=torch.float64, device=logits.device)
    for i, (first, end) in enumerate(_answers(c)):
        rows = torch.arange(end - first, device=logits.device)
        g = -probs[i]
        g[rows, labels[i, first:end]] += 1.0
        grad[i, first:end] = g * weight[i, first:end, None]
        probs[i] = None
    if c["op"] == "logps":
        return {"logps": logps, "dlogits": grad}
    return {"loss": loss, "rewards": s["beta"] * r, "dlogits": grad}
