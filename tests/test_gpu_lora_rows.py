"""The adapters of many requests beside a shared product against float64."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _bound(x, a, b, s, y, idx):
    """(result, tolerance) in float64: y rounds once (half a step, 2^-11); x @ A^T adds K products and R of them go into the update in float32, x @ A^T * scaling
    itself as two fp16 numbers (2^-22 of it, 2^-25 where the second is subnormal)."""
    out, tol = y.astype(np.float64), np.zeros(y.shape)
    K, R = x.shape[1], a.shape[1]
    for m, i in enumerate(idx):
        if 0 <= i < len(a):
            xa = s[i] * (a[i].astype(np.float64) @ x[m])
            mag = s[i] * (np.abs(a[i]).astype(np.float64) @ np.abs(x[m]))
            bb = b[i].astype(np.float64)
            out[m] += bb @ xa
            tol[m] = 2.0 ** -11 * np.abs(out[m]) + 2.0 ** -25 + np.abs(bb) @ (mag * (K + R + 64) * 2.0 ** -24 + np.abs(xa) * 2.0 ** -22 + 2.0 ** -25)
    return out, tol


CASES = [
    # rows, K, outputs, rank, adapters, rows per index
    (1, 128, [64], 8, 1, 1),
    (3, 4096, [128, 4096], 16, 3, 1),
    (16, 416, [192], 24, 5, 1),
    (17, 1056, [320, 64, 64, 128], 64, 4, 1),
    (40, 1024, [1024], 8, 40, 1),
    (64, 5120, [640, 640], 16, 7, 1),
    (130, 2048, [448], 40, 3, 13),
    (301, 11008, [256], 32, 2, 100),
    (2048, 96, [64], 48, 8, 256),
]


@pytest.mark.parametrize("M,K,outs,R,n,per", CASES)
def test_update_matches_float64(M, K, outs, R, n, per):
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    rng = np.random.default_rng(M + K + R)
    x = rng.standard_normal((M, K)).astype(np.float16)
    index = rng.integers(-2, n + 1, -(-M // per)).astype(np.int32)             # -2, -1 and n are none
    if n > 1:
        index[0] = n - 1
    specs, wants = [], []
    for N in outs:
        a = (rng.standard_normal((n, R, K)) / np.sqrt(K)).astype(np.float16)
        b = rng.standard_normal((n, N, R)).astype(np.float16)
        s, y = rng.uniform(0.2, 2.0, n).astype(np.float32), rng.standard_normal((M, N)).astype(np.float16)
        specs.append(tuple(torch.from_numpy(t).cuda() for t in (a, b, s, y)))
        wants.append(_bound(x, a, b, s, y, np.repeat(index, per)[:M]) + (y,))
    before = [t[3].clone() for t in specs]
    xd, idx = torch.from_numpy(x).cuda(), torch.from_numpy(index).cuda()
    quant_hip.lora_rows(xd, idx, specs, per)
    first = [t[3].clone() for t in specs]
    none = ~((np.repeat(index, per)[:M] >= 0) & (np.repeat(index, per)[:M] < n))
    for (want, tol, y), got in zip(wants, first):
        got = got.cpu().numpy()
        err = np.abs(got.astype(np.float64) - want) - tol
        assert err.max() <= 0, err.max()
        assert np.array_equal(got[none], y[none])
    for t, y in zip(specs, before):
        t[3].copy_(y)
    quant_hip.lora_rows(xd, idx, specs, per)
    assert all(torch.equal(t[3], f) for t, f in zip(specs, first))             # bit-reproducible


def test_infinities_and_nan_stay_in_their_rows():
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    M, K, N, R, n = 20, 256, 128, 16, 3
    g = torch.Generator().manual_seed(0)
    x, a, b = torch.randn(M, K, generator=g).half(), torch.randn(n, R, K, generator=g).half(), torch.randn(n, N, R, generator=g).half()
    y = torch.randn(M, N, generator=g).half()
    idx = (torch.arange(M) % n).int()
    want = y.clone().cuda()
    s = torch.ones(n).cuda()
    quant_hip.lora_rows(x.cuda(), idx.cuda(), [(a.cuda(), b.cuda(), s, want)])
    x[4, 7], x[5, 0] = float("nan"), float("inf")                             # two rows of adapters 1 and 2
    a[0, 0, 0] = float("nan")                                                  # and adapter 0 itself
    got = y.clone().cuda()
    quant_hip.lora_rows(x.cuda(), idx.cuda(), [(a.cuda(), b.cuda(), s, got)])
    bad = torch.zeros(M, dtype=torch.bool)
    bad[4], bad[5], bad[idx == 0] = True, True, True
    assert torch.equal(got[~bad.cuda()], want[~bad.cuda()]) and not torch.isfinite(got[bad.cuda()]).any()


@pytest.mark.parametrize("M", [3, 40, 300])
def test_an_adapter_that_is_no_number_stays_with_its_requests(M):
    """Infinities and NaN in one adapter's matrices or scaling: its rows are no numbers, all others come out as without it."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    rng = np.random.default_rng(M)
    x = torch.from_numpy(rng.standard_normal((M, 256)).astype(np.float16)).cuda()
    a = torch.from_numpy((rng.standard_normal((3, 16, 256)) / 16).astype(np.float16)).cuda()
    b = torch.from_numpy(rng.standard_normal((3, 320, 16)).astype(np.float16)).cuda()
    index = torch.from_numpy((np.arange(M) % 4 - 1).astype(np.int32)).cuda()
    s, y0 = torch.ones(3, device="cuda"), torch.ones(M, 320, dtype=torch.float16, device="cuda")
    want = y0.clone()
    quant_hip.lora_rows(x, index, [(a, b, s, want)])
    theirs = index == 1
    for what in range(3):
        for value in (float("nan"), float("inf")):
            t = [a.clone(), b.clone(), s.clone()]
            t[what].view(3, -1)[1] = value
            y = y0.clone()
            quant_hip.lora_rows(x, index, [(t[0], t[1], t[2], y)])
            assert torch.equal(y[~theirs], want[~theirs])
            assert not torch.isfinite(y[theirs]).all(dim=-1).any()
