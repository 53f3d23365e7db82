"""Activations in 8 bits against the oracle in 64 bits: codes and scales have to be equal, and what they are read back as to be the correctly rounded
product; silu(gate) * up over them, forward and backward.

Bounds.  u is half a step of the result's type (2^-11 fp16, 2^-8 bf16).  sigmoid is formed from exp(-x) whose exponent is rounded at 2^-24 of |x| log2(e) and a
reciprocal to 2^-23: together below 2^-15 of itself; where it would be below 2^-126 the reciprocal is zero.  What it multiplies, |gate * up| forward and |dout * gate|
backward, times 2^-126 is therefore lost at most: 2^7.9 * 2^-126 for a gate of -240, which bfloat16 still holds.  The result is one more rounding.  In the
gradient of gate, 1 + x (1 - sigmoid) may cancel: its error is up to 2^-17 whatever its size, for x (1 - s) is off by |x| 2^-23 and s < 2^-24 where |x| > 17 matters."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["float16", "bfloat16", "float32"]
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -126, "float32": 2.0 ** -126}


def _np(t):
    return t.double().cpu().numpy()


def _check(x, codes, scales, oracle8):
    q, s = oracle8.act8(_np(x))
    assert codes.shape == x.shape and np.array_equal(codes.cpu().numpy().astype(np.int64), q)
    assert np.array_equal(_np(scales), s, equal_nan=True)


def _parts(kept, x):
    """(codes, scales, codes, scales) of gate and up in what a gated activation keeps for tensors like x."""
    import torch
    n, blocks = x.numel(), -(-x.numel() // 32)
    c, s = -(-n // 16) * 16, -(-2 * blocks // 16) * 16
    assert kept.dtype == torch.uint8 and kept.shape == (2 * (c + s),)
    codes = [kept[i * c:i * c + n].view(torch.int8).view(x.shape) for i in (0, 1)]
    scales = [kept[2 * c + i * s:2 * c + i * s + 2 * blocks].view(torch.bfloat16) for i in (0, 1)]
    return codes[0], scales[0], codes[1], scales[1]


@pytest.fixture(scope="module")
def oracle8():
    from oracle import training_oracle
    return training_oracle


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (31,), (32,), (33,), (3, 5, 7), (63, 61), (2, 257), (61, 4096), (2047,), (2049,), (129, 11008)])
def test_codes_scales_and_values(kind, shape, oracle8):
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    dt = getattr(torch, kind)
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = (torch.randn(shape, device="cuda", generator=gen) * torch.exp(2 * torch.randn(shape, device="cuda", generator=gen))).to(dt)
    codes, scales = qh.act8_pack(x)
    _check(x, codes, scales, oracle8)
    want = oracle8.held(_np(x))
    assert (np.abs(want - _np(x)) <= np.repeat(_np(scales), 32)[:x.numel()].reshape(x.shape) / 2).all()
    for out in TYPES:
        y = qh.act8_unpack(codes, scales, getattr(torch, out))
        assert y.dtype == getattr(torch, out) and y.is_contiguous()
        top = torch.finfo(y.dtype).max
        assert torch.equal(y.cpu(), torch.from_numpy(np.clip(want, -top, top)).to(y.dtype))
    assert qh.act8_unpack(codes, scales).dtype == torch.float16


@pytest.mark.parametrize("kind", TYPES)
def test_ends_of_the_types_ties_and_no_numbers(kind, oracle8):
    """Blocks of zeros, of the least and the largest numbers, of halves of a step, with infinities and NaN, each beside ordinary ones."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    dt = getattr(torch, kind)
    info = torch.finfo(dt)
    rows = [torch.zeros(32), torch.full((32,), -0.0), torch.arange(32) * 1.0, torch.linspace(-3, 3, 32), torch.full((32,), float(info.max)),
            torch.linspace(-1, 1, 32) * float(info.max), torch.arange(32) * float(info.smallest_normal), torch.arange(32.0) * float(info.tiny) / 16,
            torch.arange(32) * 2.0 ** -20, torch.full((32,), -float(info.max) / 3), torch.tensor([127.0] + [k + 0.5 for k in range(31)]),
            torch.tensor([-63.5] + [k / 4 for k in range(31)]), torch.tensor([127.0 * 1.5] + [(k + 0.5) * 1.5 for k in range(31)]),
            torch.tensor([1.0, float("inf")] + [2.0] * 30), torch.tensor([float("nan")] + [2.0] * 31), torch.tensor([float("-inf")] * 32),
            torch.tensor([5.0] * 31 + [float("nan")]), torch.arange(32) * 0.125]
    if kind != "float16":
        rows += [torch.arange(32.0) * 2.0 ** -133, torch.full((32,), 2.0 ** -126), torch.arange(32.0) * 2.0 ** -120, torch.arange(32.0) * 2.0 ** 120]
    if kind == "float32":
        rows += [torch.arange(32.0) * 2.0 ** -149, torch.full((32,), 2.0 ** -149)]
    x = torch.stack([r.double() for r in rows]).to(dt).cuda()
    codes, scales = qh.act8_pack(x)
    _check(x, codes, scales, oracle8)
    assert bool((codes.int().abs() <= 127).all())
    y = qh.act8_unpack(codes, scales, dt)
    bad = ~torch.isfinite(x).all(1)
    assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all())
    want = oracle8.held(_np(x))[~bad.cpu().numpy()]
    assert torch.equal(y[~bad].cpu(), torch.from_numpy(np.clip(want, -float(info.max), float(info.max))).to(dt))


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_every_value_of_a_type(kind, oracle8):
    """All finite 16-bit values, each in a block whose largest magnitude decides, at steps of the scale that are not powers of two."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    dt = getattr(torch, kind)
    x = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dt)
    x = x[torch.isfinite(x)]
    x = x[torch.randperm(x.numel(), generator=torch.Generator().manual_seed(3))]
    near = x[x.float().abs() < 300][:20000]
    for values in (x, near, torch.sort(near.float().abs()).values.to(dt)):
        v = values.cuda()
        codes, scales = qh.act8_pack(v)
        _check(v, codes, scales, oracle8)


@pytest.mark.parametrize("view", ["odd offset", "rows", "columns", "transposed", "expanded"])
def test_inputs_that_lie_otherwise(view, oracle8):
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    gen = torch.Generator(device="cuda").manual_seed(9)
    base = torch.randn(70, 96, device="cuda", generator=gen).half()
    x = {"odd offset": base.view(-1)[1:4000], "rows": base[3:40:2], "columns": base[:, 5:70], "transposed": base.t(), "expanded": base[:1].expand(9, 96)}[view]
    codes, scales = qh.act8_pack(x)
    _check(x, codes, scales, oracle8)
    out, kept = qh.silu_mul_act8(x, x)
    again, kept2 = qh.silu_mul_act8(x.clone(memory_format=torch.contiguous_format), x.contiguous())
    parts = _parts(kept, x)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(parts, _parts(kept2, x)))
    assert torch.equal(parts[0], codes) and torch.equal(parts[3], scales)
    for a, b in zip(qh.silu_mul_act8_bwd(x, kept), qh.silu_mul_act8_bwd(x.contiguous(), kept)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", [(1,), (9,), (31,), (33,), (3, 5, 683), (64, 512), (61, 2731), (33, 11008)])
def test_gated_activation(kind, shape, oracle8):
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    dt = getattr(torch, kind)
    gen = torch.Generator(device="cuda").manual_seed(sum(shape) + 1)
    gate, up, dout = (torch.randn(shape, device="cuda", generator=gen) * s for s in (4.0, 1.0, 0.02))
    gate.view(-1)[::37] *= 20
    gate, up, dout = gate.to(dt), up.to(dt), dout.to(dt)
    u, tiny = torch.finfo(dt).eps / 2, TINY[kind]
    out, kept = qh.silu_mul_act8(gate, up)
    parts = _parts(kept, gate)
    _check(gate, *parts[:2], oracle8)
    _check(up, *parts[2:], oracle8)
    want = oracle8.silu_mul(_np(gate), _np(up))
    assert (np.abs(_np(out) - want) <= (u + 2.0 ** -15) * np.abs(want) + tiny + 2.0 ** -126 * np.abs(_np(gate) * _np(up))).all()
    dgate, dup = qh.silu_mul_act8_bwd(dout, kept)
    g, v, d = oracle8.held(_np(gate)), oracle8.held(_np(up)), _np(dout)
    wg, wu = oracle8.silu_mul_bwd(d, g, v)
    assert (np.abs(_np(dgate) - wg) <= (u + 2.0 ** -15) * np.abs(wg) + 2.0 ** -17 * np.abs(d * v) + tiny).all()
    assert (np.abs(_np(dup) - wu) <= (u + 2.0 ** -15) * np.abs(wu) + tiny + 2.0 ** -126 * np.abs(d * g)).all()
    # the gradients are the differences of the function at the values held
    h = 1e-5
    num = (oracle8.silu_mul(g + h, v) - oracle8.silu_mul(g - h, v)) / (2 * h) * d
    assert (np.abs(num - wg) <= 1e-7 * (np.abs(d * v) + np.abs(wg))).all()


def test_gated_activation_at_the_ends_of_the_types():
    """Gates of the largest magnitudes: silu is 0 or the gate itself, its slope 0 or 1; infinities and NaN come out as no numbers in the gradient."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    for dt in (torch.float16, torch.bfloat16):
        top = torch.finfo(dt).max
        gate = torch.tensor([-top, top, -100.0, 100.0] * 8 + [0.5] * 32, device="cuda", dtype=dt)
        up = torch.full_like(gate, 0.5)
        one = torch.ones_like(gate)
        out, kept = qh.silu_mul_act8(gate, up)
        assert out[:4].tolist()[:2] == [0.0, float(gate[1]) / 2] and float(out[3]) == 50.0
        dgate, dup = qh.silu_mul_act8_bwd(one, kept)
        assert dgate[:2].tolist() == [0.0, 0.5] and dup[:2].tolist() == [0.0, float(top)]
        gate[5] = float("inf")
        out, kept = qh.silu_mul_act8(gate, up)
        assert float(out[5]) == float("inf")
        dgate, dup = qh.silu_mul_act8_bwd(one, kept)
        assert bool(torch.isnan(dgate[:32]).all()) and bool(torch.isfinite(dgate[32:]).all()) and bool(torch.isfinite(dup[32:]).all())


def test_refused_and_empty_calls():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    x = torch.randn(40, 33, device="cuda").half()
    codes, scales = qh.act8_pack(x)
    out, kept = qh.silu_mul_act8(x, x)
    for bad in (lambda: qh.act8_pack(x.cpu()), lambda: qh.act8_pack(x.double()), lambda: qh.act8_pack(x.int()), lambda: qh.act8_pack(x.clone().requires_grad_()),
                lambda: qh.act8_unpack(codes, scales, torch.float64), lambda: qh.act8_unpack(codes, scales[:-1]), lambda: qh.act8_unpack(codes, scales.half()),
                lambda: qh.act8_unpack(codes.int(), scales), lambda: qh.act8_unpack(codes[:, :32], scales), lambda: qh.act8_unpack(codes.cpu(), scales.cpu()),
                lambda: qh.act8_unpack(codes.view(-1)[1:1000], scales[:32]), lambda: qh.act8_unpack(codes, scales.cpu()),
                lambda: qh.silu_mul_act8(x, x.bfloat16()), lambda: qh.silu_mul_act8(x.float(), x.float()), lambda: qh.silu_mul_act8(x, x[:20]),
                lambda: qh.silu_mul_act8(x, x.cpu()), lambda: qh.silu_mul_act8_bwd(out[:20], kept), lambda: qh.silu_mul_act8_bwd(out.float(), kept),
                lambda: qh.silu_mul_act8_bwd(out, kept[:-16]), lambda: qh.silu_mul_act8_bwd(out, kept.view(torch.int8)), lambda: qh.silu_mul_act8_bwd(out, kept.cpu()),
                lambda: qh.silu_mul_act8_bwd(out.cpu(), kept)):
        with pytest.raises(ValueError):
            bad()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError):
            qh.act8_pack(torch.autograd.forward_ad.make_dual(x.float(), x.float()))
    e = x[:0]
    codes, scales = qh.act8_pack(e)
    assert codes.shape == (0, 33) and scales.shape == (0,) and qh.act8_unpack(codes, scales).shape == (0, 33)
    out, kept = qh.silu_mul_act8(e, e)
    assert out.shape == (0, 33) and [t.shape for t in qh.silu_mul_act8_bwd(out, kept)] == [(0, 33)] * 2


def test_on_another_stream_and_in_captured_graphs():
    """The four calls captured twice on one stream, replayed in turn with new inputs and eager work between the replays."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    gen = torch.Generator(device="cuda").manual_seed(2)
    make = lambda: torch.randn(37, 515, device="cuda", generator=gen).half()

    def step(g, u, d):
        out, kept = qh.silu_mul_act8(g, u)
        codes, scales = qh.act8_pack(out)
        return [out, qh.act8_unpack(codes, scales), *qh.silu_mul_act8_bwd(d, kept)]
    side = torch.cuda.Stream()
    sets, graphs = [], []
    for _ in range(2):
        held = [make() for _ in range(3)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(*held)
        sets.append((held, outs))
        graphs.append(graph)
    for rep in range(4):
        for held, _ in sets:
            for t in held:
                t.copy_(make())
        want = [[o.clone() for o in step(*held)] for held, _ in sets]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, outs), ref in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, ref))
    with torch.cuda.stream(side):
        got = [o.clone() for o in step(*sets[0][0])]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))


def test_more_than_2_to_the_31_values(oracle8):
    """The places of the last values pass 32 bits: what lies there comes out as it does by itself."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    n, tail = 2 ** 31 + 4096 + 37, 32 * 300 + 37
    x = torch.zeros(n, dtype=torch.float16, device="cuda")
    x[-tail:] = torch.randn(tail, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    codes, scales = qh.act8_pack(x)
    want = qh.act8_pack(x[-tail:].clone())
    assert torch.equal(codes[-tail:], want[0]) and torch.equal(scales[-len(want[1]):], want[1]) and not bool(codes[:1000].any())
    y = qh.act8_unpack(codes, scales)
    assert torch.equal(y[-tail:], qh.act8_unpack(*want)) and not bool(y[:1000].any())
    del codes, scales, y
    out, kept = qh.silu_mul_act8(x, x)
    dgate, dup = qh.silu_mul_act8_bwd(x, kept)
    alone, kept_alone = qh.silu_mul_act8(x[-tail:].clone(), x[-tail:].clone())
    a, b = qh.silu_mul_act8_bwd(x[-tail:].clone(), kept_alone)
    assert torch.equal(out[-tail:], alone) and torch.equal(dgate[-tail:], a) and torch.equal(dup[-tail:], b) and not bool(dup[:1000].any())


def test_the_product_alone():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    for dt in (torch.float16, torch.bfloat16):
        g, u = (torch.randn(7, 333, device="cuda").to(dt) for _ in range(2))
        out, kept = qh.silu_mul_act8(g, u, keep=False)
        assert kept is None and torch.equal(out, qh.silu_mul_act8(g, u)[0])


def test_two_streams_at_once():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    xs = [torch.randn(513, 4099, device="cuda").half() for _ in range(2)]
    want = [(qh.act8_pack(x)[0], qh.silu_mul_act8(x, x)[0]) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, (x, s) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(s):
                got[k].append((qh.act8_pack(x)[0], qh.silu_mul_act8(x, x)[0]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for pair in got[k] for a, b in zip(pair, want[k]))
