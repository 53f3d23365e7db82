"""One adapter for many rows: runs that are longer than the rows there are, up to the largest 64-bit number."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per", [37, 38, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 62, 2 ** 63 - 1])
def test_runs_longer_than_the_rows(per):
    """One entry of the index stands for all rows; what follows it in memory is not read (it would name another adapter)."""
    import torch
    from alpaca_lora_4bit_amd import quant_hip
    rng = np.random.default_rng(0)
    M, K, N, R = 37, 64, 64, 8
    x, a, b = (torch.from_numpy(rng.standard_normal(s).astype(np.float16)).cuda() for s in ((M, K), (2, R, K), (2, N, R)))
    s, y = torch.ones(2, device="cuda"), torch.zeros(M, N, dtype=torch.float16, device="cuda")
    index = torch.tensor([1] + [0] * 40, dtype=torch.int32, device="cuda")[:1]
    want = y.clone()
    quant_hip.lora_rows(x, torch.ones(M, dtype=torch.int32, device="cuda"), [(a, b, s, want)])
    quant_hip.lora_rows(x, index, [(a, b, s, y)], per)
    assert torch.equal(y, want)
