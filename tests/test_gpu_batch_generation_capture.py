"""Short answers and many requests with the captured step: the first steps meet code that the prompts did not run."""
import pytest
import torch

from test_gpu_batch_generation import _bank, _loaded
from tiny_llama import build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [2, 3, 4])
def test_short_answers_of_more_requests_than_a_prompt_part_has_rows(tmp_path, oracle, new):
    """Prompts in parts of eight rows, then steps of twenty: the tiled products are met first in a step.  Captured and eager tokens are the same."""
    from alpaca_lora_4bit_amd import inference
    build(str(tmp_path), oracle, seed=8)
    prompts = [torch.tensor([1] + [7 + (13 * i + 5 * n) % 180 for i in range(n % 5)]).cuda() for n in range(20)]
    got = []
    for use_graph in (True, False):
        model, _ = _loaded(str(tmp_path))
        bank = _bank(model)
        got.append([t.tolist() for t in inference.generate_batch(model, prompts, new, bank, [n % 4 - 1 for n in range(20)], use_graph=use_graph, prefill_rows=8)])
    assert got[0] == got[1] and [len(g) for g in got[0]] == [len(p) + new for p in prompts]
