"""What the errors of log-probabilities add up to over long answers: a log ratio is the small difference of sums of thousands of them, so an error that goes
one way counts, however small.

Bound.  v_exp_f32 is short by 3.4e-9 of itself on average, 3e-9 are put back, so a sum of exponentials is short by 0.4e-9 of what is not the label's own exact term.  The
exponent's rounding (2^-24 of |d| log2(e), d the distance from the label) goes either way; the sums are in 64 bits, whatever word has most of the weight.  On average over the
tokens an error is 1e-9 at most, and six times what an average over these answers is off by chance."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ANSWERS, PLACES = 16, 2048


def _rows(kind, v, weight, gen):
    """(logits [PLACES, v], labels) of an answer: normal logits, one word 10 to 20 above the others where one has most of the weight."""
    import torch
    x = torch.randn(PLACES, v, device="cuda", generator=gen) * (2.0 if weight == "spread" else 1.0)
    top = torch.randint(0, v, (PLACES,), device="cuda", generator=gen)
    other = (top + torch.randint(1, v, (PLACES,), device="cuda", generator=gen)) % v
    if weight != "spread":
        at = {"sure": 18.5, "nearly sure": 12.0}[weight.split(", ")[0]]
        x.scatter_(1, top[:, None], at + 1.4 * torch.rand(PLACES, 1, device="cuda", generator=gen))
    return x.to(getattr(torch, kind)), other if weight.endswith("of another") else top


@pytest.mark.parametrize("weight", ["sure, of the label", "sure, of another", "nearly sure, of the label", "nearly sure, of another"])
@pytest.mark.parametrize("kind,v", [("float16", 32000), ("float32", 32000), ("bfloat16", 1600)])
def test_the_average_error_of_a_token(kind, v, weight):
    import torch
    from alpaca_lora_4bit_amd import preference
    gen = torch.Generator(device="cuda").manual_seed(len(weight) + v)
    off = []
    for _ in range(ANSWERS // 2):
        pair = [_rows(kind, v, weight, gen) for _ in range(2)]
        logits, labels = torch.stack([x for x, _ in pair]), torch.stack([l for _, l in pair])
        true = torch.stack([(x.double().gather(1, l[:, None]) - torch.logsumexp(x.double(), 1, keepdim=True))[:, 0] for x, l in pair])
        ref = true.float()
        _, rewards = preference.preference_loss(logits, labels, ref, beta=1.0)
        off += ((rewards.double() - (true - ref.double()).sum(1)) / PLACES).tolist()
    mean, chance = np.mean(off), np.std(off, ddof=1) / np.sqrt(ANSWERS)
    print(f"{kind} {v} {weight}: {mean:.2e} a token, by chance {chance:.1e}")
    assert abs(mean) <= 1e-9 + 6 * chance
    assert chance < 5e-9                                       # or the test says nothing
