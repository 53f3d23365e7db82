"""What the errors of log-probabilities add up to over long answers: a log ratio is the small difference of sums of thousands of them, so an error that goes
one way counts, however small.

Bound.  Over all fp32 arguments of a power of two's range v_exp_f32 is short of 2^y by 1.23e-9 to 1.33e-9 of itself on average where y >= 1 and by 3.36e-9 to 3.45e-9 where y <= -1
(each of the 2^23 arguments of [2^k, 2^(k+1)) and of its negatives against fp64, k from 0 to 6 and to 5; rms 2.6e-8).  2.33e-9 are put back, so a sum of exponentials of words spread over whole units on one side of the
label is off by 3.45e-9 - 2.33e-9 < 1.13e-9 at most, on both sides by less.  bfloat16 logits of the size of 4 are whole multiples of 2^-6 apart, some 400 differences of which 150 have the weight: the
average over so few of the function's values is off by 2.6e-8 / sqrt(150) = 2.1e-9, three times that is allowed.  The exponent's own rounding (2^-24 of |d| log2(e), d the distance from the label) goes
either way; the sums are in 64 bits, whatever word has most of the weight.  Beyond that six times what an average over these answers is off by chance."""
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


@pytest.mark.parametrize("weight", ["spread", "sure, of the label", "sure, of another", "nearly sure, of the label", "nearly sure, of another"])
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
    assert abs(mean) <= 1.13e-9 + (6.3e-9 if kind == "bfloat16" else 0.0) + 6 * chance
    assert chance < 5e-9                                       # or the test says nothing
