"""Token log-probabilities and the preference loss against the oracle in 64 bits.

Bounds.  exp(x - x_l) has an exponent rounded at 2^-24 of its size and an exponential to 2^-23; a lane adds packs of 4 or 8 (three roundings) with Kahan's sum, the rest is
in 64 bits.  So log(sum) is off by at most 2^-22 (4 + D), D the largest |x - x_l| among the words that have weight, here taken as |logp| + 8 (a word e^-8 below the
sum adds its error times that), and a log-probability in fp32 by 2^-24 of itself more.  A probability exp(x - m - log sum) has three roundings of numbers of the size
of |x - m| and |log sum|, and the exponential's exponent one more: relative 2^-22 (4 + |x - m| + |log sum|) at most; the gradient is one rounding to its type beyond."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["float16", "bfloat16", "float32"]
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -126, "float32": 2.0 ** -126}


@pytest.fixture(scope="module")
def orc():
    from oracle import training_oracle
    return training_oracle


def _np(t):
    return t.detach().double().cpu().numpy()


def _logits(shape, kind, seed, spread=2.0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=gen) * spread).to(getattr(torch, kind))


def _labels(shape, v, seed, none=0.3):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lab = torch.randint(0, v, shape, device="cuda", generator=gen)
    return torch.where(torch.rand(shape, device="cuda", generator=gen) < none, torch.full_like(lab, -100), lab)


def _logp_bound(lp):
    return 2.0 ** -22 * (12 + np.abs(lp)) + 2.0 ** -24 * np.abs(lp)


def _check_grad(got, x, labels, lp, soft, coef, kind, orc):
    import torch
    want = orc.logits_grad(soft, labels, coef)
    u = torch.finfo(getattr(torch, kind)).eps / 2
    x = _np(x)
    word = (labels >= 0) & (labels < x.shape[-1])
    with np.errstate(all="ignore"):
        d = np.abs(x - np.take_along_axis(x, np.where(word, labels, 0)[..., None], -1))
    rel = 2.0 ** -22 * (4 + d + np.abs(lp)[..., None] + 8)
    bound = u * np.abs(want) + np.where(soft > 0, soft * rel, 0) * np.abs(np.asarray(coef, dtype=np.float64))[..., None] + 2.0 ** -22 * np.abs(want) + TINY[kind]
    err = np.abs(_np(got) - want)
    assert (err <= bound).all(), float((err / bound).max())
    assert not _np(got)[~word].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 2), (3, 5, 7), (2, 4, 31), (1, 9, 300), (2, 7, 320), (3, 3, 1003), (2, 5, 2049), (2, 2, 4099), (1, 600, 5000),
                                   (2, 3, 32001), (1, 3, 100003)])
def test_log_probabilities_and_gradient(kind, shape, orc):
    import torch
    from alpaca_lora_4bit_amd import preference
    b, s, v = shape
    x = _logits(shape, kind, sum(shape)).requires_grad_()
    labels = _labels((b, s), v, b + s)
    labels.view(-1)[0] = v - 1                                 # the last word, and in what follows labels that are none
    if labels.numel() > 3:
        labels.view(-1)[1], labels.view(-1)[2], labels.view(-1)[3] = v, 2 ** 40, -1
    lp = preference.token_logps(x, labels)
    assert lp.dtype == torch.float32 and lp.shape == labels.shape
    lab = labels.cpu().numpy()
    want, soft = orc.token_logps(_np(x), lab)
    assert (np.abs(_np(lp) - want) <= _logp_bound(want)).all()
    grad = torch.randn(labels.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    (dx,) = torch.autograd.grad(lp, x, grad)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    _check_grad(dx, x, lab, want, soft, _np(grad), kind, orc)


def test_the_gradient_is_the_difference_quotient(orc):
    """Of the oracle's function in 64 bits along random directions, for both operators: truncation of central differences h^2 and rounding 1e-15 / h."""
    import torch
    from alpaca_lora_4bit_amd import preference
    x = _logits((4, 6, 53), "float32", 3).requires_grad_()
    labels = _labels((4, 6), 53, 4)
    lab, ref = labels.cpu().numpy(), _np(_logits((4, 6), "float32", 5)) - 4
    weight = _np(_logits((4, 6), "float32", 6))
    direction, h = _np(_logits((4, 6, 53), "float32", 7)), 1e-4

    def loss(z):
        return orc.preference(orc.token_logps(z, lab)[0], ref.astype(np.float32).astype(np.float64), lab, 53, 0.3, 0.1)[0]

    def total(z):
        return (orc.token_logps(z, lab)[0] * weight).sum()
    (a,) = torch.autograd.grad(preference.preference_loss(x, labels, torch.from_numpy(ref).float().cuda(), beta=0.3, label_smoothing=0.1)[0], x)
    (b,) = torch.autograd.grad(preference.token_logps(x, labels), x, torch.from_numpy(weight).float().cuda())
    for f, g in ((loss, a), (total, b)):
        num = (f(_np(x) + h * direction) - f(_np(x) - h * direction)) / (2 * h)
        mine = (_np(g) * direction).sum()
        assert abs(num - mine) <= 1e-5 * np.abs(_np(g) * direction).sum() + 1e-9


@pytest.mark.parametrize("kind", TYPES)
def test_rows_with_infinities_lowest_values_and_no_numbers(kind, orc):
    """-infinity and the type's lowest value take words away; a row of the lowest value only is uniform; labels far below the row's maximum; rows of
    infinities and NaN are no numbers where they have a label and nothing where not."""
    import torch
    from alpaca_lora_4bit_amd import preference
    v, dt = 777, getattr(torch, kind)
    low, inf, nan = float(torch.finfo(dt).min), float("inf"), float("nan")
    x = _logits((1, 16, v), kind, 8)
    labels = torch.full((1, 16), 5, device="cuda", dtype=torch.long)
    x[0, 0, 7:] = -inf
    x[0, 1, 7:] = low
    x[0, 2] = low
    x[0, 3, :] = -inf
    x[0, 3, 5] = 2.0                                           # one word left: the label's
    x[0, 4, 5] = -inf                                          # the label's word taken away
    x[0, 5, 5] = -300.0                                        # far below the others
    x[0, 6, 5] = 300.0                                         # far above
    x[0, 7, 5] = low
    x[0, 8, 100:] = 200.0
    x[0, 9] = -inf                                             # nothing left
    x[0, 10, 3] = nan
    x[0, 11, 3] = inf
    x[0, 12, 5] = inf
    x[0, 13:] = nan
    labels[0, 13:] = -100
    x.requires_grad_()
    lp = preference.token_logps(x, labels)
    (dx,) = torch.autograd.grad(lp, x, torch.full_like(lp, 0.5))
    lab = labels.cpu().numpy()
    with np.errstate(all="ignore"):
        want, soft = orc.token_logps(_np(x), lab)
    fine = [0, 1, 2, 3, 5, 6, 8]
    got = _np(lp)[0]
    assert (np.abs(got - want[0])[fine] <= _logp_bound(want[0])[fine]).all(), (got[fine], want[0][fine])
    assert got[4] == -np.inf and abs(got[2] + np.log(v)) < 1e-5 and got[3] == 0.0
    assert np.abs(got[7] - want[0][7]) <= 2.0 ** -23 * np.abs(want[0][7])
    assert np.isnan(got[9:13]).all() and not got[13:].any()
    g = _np(dx)[0]
    rows = fine + [4, 7]
    u = torch.finfo(dt).eps / 2
    truth = orc.logits_grad(soft[0][rows], lab[0][rows], np.full(len(rows), 0.5))
    assert (np.abs(g[rows] - truth) <= u * np.abs(truth) + 2.0 ** -15 * soft[0][rows] + 2.0 ** -22 * np.abs(truth) + TINY[kind]).all()
    assert np.isnan(g[9:13]).any(1).all() and not g[13:].any()


@pytest.mark.parametrize("layout", ["columns", "steps", "batch first", "expanded", "odd offset", "far words", "two", "four", "row"])
def test_logits_that_lie_otherwise(layout, orc):
    """Strides, offsets and numbers of dimensions; the gradient has the logits' shape."""
    import torch
    from alpaca_lora_4bit_amd import preference
    base = _logits((6, 8, 1001), "float16", 12)
    x = {"columns": base[:, :, 3:520], "steps": base[:, ::2, :640], "batch first": base.transpose(0, 1), "expanded": base[:1].expand(6, 8, 1001),
         "odd offset": base.view(-1)[1:1 + 40 * 1000].view(5, 8, 1000), "far words": base[:, :, ::2], "two": base[0], "four": base.view(2, 3, 8, 1001),
         "row": base[0, 0]}[layout]
    v = x.shape[-1]
    labels = _labels(x.shape[:-1], v, 2) if x.dim() > 1 else torch.tensor(7, device="cuda")
    leaf = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
    a = preference.token_logps(x, labels)
    b = preference.token_logps(leaf, labels)
    assert torch.equal(a, b)                                   # where a row begins does not change the order of its sum
    view = x.detach().requires_grad_()
    assert view.stride() == x.stride()
    gout = torch.full_like(a, 0.25)
    (da,) = torch.autograd.grad(preference.token_logps(view, labels), view, gout)
    (db,) = torch.autograd.grad(b, leaf, gout.expand_as(a))
    assert da.shape == x.shape and torch.equal(da, db)
    want, soft = orc.token_logps(_np(x), labels.cpu().numpy())
    assert (np.abs(_np(a) - want) <= _logp_bound(want)).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("pairs,places,v,smoothing,beta", [(1, 1, 5, 0.0, 0.1), (1, 37, 300, 0.0, 0.1), (2, 9, 2049, 0.1, 0.5), (3, 300, 97, 0.0, 0.02), (9, 520, 64, 0.5, 0.1),
                                                           (40, 33, 320, 0.2, 1.0), (4, 64, 32000, 0.0, 0.1)])
def test_loss_rewards_and_gradient(kind, pairs, places, v, smoothing, beta, orc):
    import torch
    from alpaca_lora_4bit_amd import preference
    shape = (2 * pairs, places, v)
    x = _logits(shape, kind, pairs + places).requires_grad_()
    labels = _labels(shape[:2], v, places)
    lab = labels.cpu().numpy()
    lp, soft = orc.token_logps(_np(x), lab)
    rnd = np.random.RandomState(pairs)
    ref = (lp + 0.3 * rnd.randn(*lp.shape)).astype(np.float32)
    ref[lab < 0] = np.nan
    loss, rewards = preference.preference_loss(x, labels, torch.from_numpy(ref).cuda(), beta=beta, label_smoothing=smoothing)
    assert loss.shape == () and rewards.shape == (2 * pairs,) and loss.dtype == rewards.dtype == torch.float32
    assert loss.requires_grad and not rewards.requires_grad
    want, wr, coef = orc.preference(lp, ref.astype(np.float64), lab, v, beta, smoothing)
    off = (2.0 ** -22 * (12 + np.abs(lp)) * (lab >= 0)).sum(1) * beta                # what the log-probabilities may be off, before rounding
    assert (np.abs(_np(rewards) - wr) <= off + 2.0 ** -24 * np.abs(wr)).all()
    dz = off[:pairs] + off[pairs:]
    assert abs(float(loss) - want) <= dz.mean() + 2.0 ** -24 * want                   # |dloss / dz| <= 1
    (dx,) = torch.autograd.grad(loss, x, torch.tensor(256.0, device="cuda"))
    c = np.repeat(coef[:, None], places, 1) * 256.0
    want_dx = orc.logits_grad(soft, lab, c)
    u = torch.finfo(x.dtype).eps / 2
    # the coefficient is off by beta / P times a quarter of dz, and by its own rounding and that of the factor
    slack = np.concatenate([dz, dz])[:, None, None] * 0.25 * beta / pairs * 256.0 * np.abs(orc.logits_grad(soft, lab, np.ones_like(c)))
    bound = u * np.abs(want_dx) + 2.0 ** -22 * (24 + np.abs(lp)[..., None]) * (soft * np.abs(c)[..., None] + np.abs(want_dx)) + slack + TINY[kind]
    # words below e^-12 of the label have a larger exponent to round, of a weight that small
    assert (np.abs(_np(dx) - want_dx) <= bound + 2.0 ** -18 * soft * np.abs(c)[..., None]).all()


def test_pairs_without_a_token_and_ratios_without_end(orc):
    """An answer of no token counts as a ratio of zero; a rejected answer that the model can't say costs nothing, a preferred one everything."""
    import torch
    from alpaca_lora_4bit_amd import preference
    x = _logits((4, 5, 40), "float32", 2)
    labels = torch.full((4, 5), -100, device="cuda")
    ref = torch.zeros(4, 5, device="cuda")
    x.requires_grad_()
    loss, rewards = preference.preference_loss(x, labels, ref)
    assert abs(float(loss) - np.log(2)) < 1e-7 and not bool(rewards.any())
    (dx,) = torch.autograd.grad(loss, x)
    assert not bool(dx.any())
    y = x.detach().clone()
    labels = torch.full((4, 5), 3, device="cuda")
    y[2, 1, 3] = float("-inf")
    y.requires_grad_()
    ref = preference.token_logps(x.detach(), labels)
    loss, rewards = preference.preference_loss(y, labels, ref, beta=0.1)              # pair 0: certain; pair 1: the policy is the reference
    assert abs(float(loss) - np.log(2) / 2) < 1e-6 and float(rewards[2]) == float("-inf")
    (dx,) = torch.autograd.grad(loss, y)
    assert not bool(dx[0].any()) and not bool(dx[2].any()) and bool(dx[1].any())
    loss, _ = preference.preference_loss(torch.cat([y[2:], y[:2]]), labels, torch.cat([ref[2:], ref[:2]]), beta=0.1)
    assert float(loss) == float("inf")


def test_refused_calls():
    import torch
    from alpaca_lora_4bit_amd import preference, quant_hip as qh
    x, labels, ref = _logits((4, 5, 40), "float16", 1), torch.zeros(4, 5, device="cuda", dtype=torch.long), torch.zeros(4, 5, device="cuda")
    lp, stats = qh.token_logps(x, labels)
    for bad in (lambda: preference.token_logps(x.cpu(), labels), lambda: preference.token_logps(x.double(), labels), lambda: preference.token_logps(x, labels.int()),
                lambda: preference.token_logps(x, labels[:, :4]), lambda: preference.token_logps(x, labels.cpu()), lambda: preference.token_logps(x[..., :0], labels),
                lambda: preference.preference_loss(x[0], labels[0], ref[0]), lambda: preference.preference_loss(x[:3], labels[:3], ref[:3]),
                lambda: preference.preference_loss(x[:0], labels[:0], ref[:0]), lambda: preference.preference_loss(x[:, :0], labels[:, :0], ref[:, :0]),
                lambda: preference.preference_loss(x, labels, ref.half()), lambda: preference.preference_loss(x, labels, ref[:2]),
                lambda: preference.preference_loss(x, labels, ref.cpu()), lambda: preference.preference_loss(x, labels, ref.clone().requires_grad_()),
                lambda: preference.preference_loss(x, labels, ref, beta=0.0), lambda: preference.preference_loss(x, labels, ref, beta=float("inf")),
                lambda: preference.preference_loss(x, labels, ref, beta=float("nan")), lambda: preference.preference_loss(x, labels, ref, label_smoothing=0.6),
                lambda: preference.preference_loss(x, labels, ref, label_smoothing=-0.1),
                lambda: qh.token_logps(x.clone().requires_grad_(), labels), lambda: qh.token_logps_bwd(x, labels, stats[:2], lp),
                lambda: qh.token_logps_bwd(x, labels, stats, lp[:, :2]), lambda: qh.token_logps_bwd(x, labels, stats, lp.half()),
                lambda: qh.token_logps_bwd(x, labels, stats, lp, factor=lp)):
        with pytest.raises(ValueError):
            bad()
    assert preference.token_logps(x[:0], labels[:0]).shape == (0, 5)
    for shape in ((0, 2, 5, 40), (3, 2, 0, 40), (2, 0, 3, 40)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        lp = preference.token_logps(e, torch.zeros(shape[:-1], device="cuda", dtype=torch.long))
        assert lp.shape == shape[:-1] and torch.autograd.grad(lp.sum(), e)[0].shape == shape
    y = x.clone().requires_grad_()
    lp = preference.token_logps(y, labels)
    with pytest.raises(Exception):                             # a graph of the backward pass
        torch.autograd.grad(lp.sum(), y, create_graph=True)
    with pytest.raises(Exception), torch.autograd.forward_ad.dual_level():
        preference.token_logps(torch.autograd.forward_ad.make_dual(x.float(), x.float()), labels)


def test_on_another_stream_repeated_and_in_captured_graphs():
    """Loss and gradient in one capture, on leaves that no eager graph holds; two graphs of one stream replayed in turn with new logits."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    labels = _labels((6, 50), 1003, 3)
    ref = _logits((6, 50), "float32", 4) - 5

    def step(x, scale):
        loss, rewards, coef, stats = qh.preference_loss(x, labels, ref, 0.1, 0.05)
        lp, st = qh.token_logps(x, labels)
        return [loss, rewards, lp, qh.token_logps_bwd(x, labels, stats, coef, scale), qh.token_logps_bwd(x, labels, st, lp)]
    side = torch.cuda.Stream()
    sets, graphs = [], []
    for k in range(2):
        x, scale = _logits((6, 50, 1003), "float16", k), torch.full((), 8.0, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, scale)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(x, scale)
        sets.append((x, scale, outs))
        graphs.append(graph)
    for rep in range(4):
        for k, (x, _, _) in enumerate(sets):
            x.copy_(_logits(x.shape, "float16", 10 * rep + k))
        want = [[o.clone() for o in step(x, scale)] for x, scale, _ in sets]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, outs), w in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w))
    with torch.cuda.stream(side):
        got = [o.clone() for o in step(*sets[1][:2])]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))


def test_a_captured_training_step():
    """Forward and backward through autograd inside one capture, as a captured training step has them."""
    import torch
    from alpaca_lora_4bit_amd import preference
    labels, ref = _labels((4, 20), 515, 3), _logits((4, 20), "float32", 4) - 5
    h = _logits((4, 20, 64), "float32", 1)

    def step(w):
        loss, _ = preference.preference_loss(h @ w, labels, ref)
        return loss.detach(), torch.autograd.grad(loss, w)[0]
    w = (_logits((64, 515), "float32", 2) * 0.1).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(w.detach().clone().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss, grad = step(w)
    for rep in range(4):
        with torch.no_grad():
            w.copy_(_logits((64, 515), "float32", 20 + rep) * 0.1)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(w.detach().clone().requires_grad_())
        torch.cuda.synchronize()
        assert torch.equal(loss, eager[0]) and torch.equal(grad, eager[1])


def test_more_than_2_to_the_31_logits(orc):
    """Rows whose places pass 32 bits come out as they do by themselves, forward and backward, in log-probabilities and loss."""
    import torch
    from alpaca_lora_4bit_amd import preference, quant_hip as qh
    v = 2 ** 20 + 3
    x = torch.zeros((2, 1030, v), dtype=torch.float16, device="cuda")
    labels = torch.full((2, 1030), -100, device="cuda")
    x[:, -3:] = _logits((2, 3, v), "float16", 1)
    labels[:, -3:] = torch.tensor([[5, v - 1, v // 2], [7, 0, 9]], device="cuda")
    alone, mine = x[:, -3:].clone(), labels[:, -3:].clone()
    lp, stats = qh.token_logps(x, labels)
    want, _ = orc.token_logps(_np(alone), mine.cpu().numpy())
    assert (np.abs(_np(lp[:, -3:]) - want) <= _logp_bound(want)).all() and not bool(lp[:, :-3].any())
    ref = torch.full((2, 1030), -14.0, device="cuda")
    loss, rewards, coef, stats = qh.preference_loss(x, labels, ref, 0.1)
    loss2, rewards2, coef2, stats2 = qh.preference_loss(alone, mine, ref[:, :3], 0.1)
    assert abs(float(loss - loss2)) < 1e-6 and bool(((rewards - rewards2).abs() < 1e-5).all())
    scale = torch.tensor(4096.0, device="cuda")
    dx = qh.token_logps_bwd(x, labels, stats, coef, scale)
    dx2 = qh.token_logps_bwd(alone, mine, stats2, coef2, scale)
    # few rows are added up by more threads, in another order; the gradients are one rounding of what agrees to 2^-20
    assert bool(((dx[:, -3:] - dx2).abs().float() <= 2.0 ** -10 * dx2.abs().float() + 2.0 ** -24).all()) and not bool(dx[0, 0].any()) and not bool(dx[1, 1026].any())


def test_two_streams_at_once():
    import torch
    from alpaca_lora_4bit_amd import quant_hip as qh
    sets = [(_logits((6, 70, 2003), "float16", k), _labels((6, 70), 2003, k), _logits((6, 70), "float32", k) - 6) for k in range(2)]

    def step(x, labels, ref):
        loss, rewards, coef, stats = qh.preference_loss(x, labels, ref, 0.1)
        return loss, rewards, qh.token_logps_bwd(x, labels, stats, coef, loss)
    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(step(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for outs in got[k] for a, b in zip(outs, want[k]))
