"""The adapters of many requests where x @ A^T * scaling lies beyond fp16's range, above or below, and the update does not."""
import numpy as np
import pytest

from test_gpu_lora_rows import _bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,R", [(1, 8), (3, 64), (40, 16), (300, 24), (700, 40)])
def test_sums_beyond_the_range_of_fp16(M, R):
    """x @ A^T * scaling around 1e5 and far above, or far below fp16's smallest numbers, with B the other way round: the update is finite and within the bound."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    rng = np.random.default_rng(M + R)
    K, N, n = 512, 192, 3
    x = (rng.standard_normal((M, K)) * 100).astype(np.float16)
    x[::3] *= np.float16(1e-3)                                                  # rows of other sizes beside them
    index = rng.integers(-1, n, M).astype(np.int32)
    for size, scaling, b_size in ((1.0, 40.0, 1e-3), (50.0, 1e3, 1e-5), (1e-3, 1e-6, 1e4)):
        a = (rng.standard_normal((n, R, K)) * size).astype(np.float16)
        b = (rng.standard_normal((n, N, R)) * b_size).astype(np.float16)
        s, y = np.full(n, scaling, np.float32), rng.standard_normal((M, N)).astype(np.float16)
        want, tol = _bound(x, a, b, s, y, index)
        for m, i in enumerate(index):                                           # the term of numbers below fp16's normal ones: here 2^-39 of a row's largest sum
            if i >= 0:
                weight = np.abs(b[i].astype(np.float64)).sum(1)
                tol[m] += weight * (2.0 ** -39 * scaling * np.abs(a[i].astype(np.float64) @ x[m]).max() - 2.0 ** -25)
        fits = np.abs(want) < 60000
        got = torch.from_numpy(y).cuda()
        quant_hip.lora_rows(torch.from_numpy(x).cuda(), torch.from_numpy(index).cuda(), [tuple(torch.from_numpy(t).cuda() for t in (a, b, s)) + (got,)])
        got = got.cpu().numpy().astype(np.float64)
        assert np.isfinite(got[fits]).all() and (np.abs(got - want) <= tol)[fits].all() and fits.mean() > 0.5, (size, scaling)
