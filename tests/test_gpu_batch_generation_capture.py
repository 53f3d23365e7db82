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


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second device")
def test_a_model_on_another_device_than_the_current_one(tmp_path, oracle):
    """Captures on both devices, one after the other, while the first is the current one."""
    from alpaca_lora_4bit_amd import autograd_4bit as ag, inference
    from tiny_llama import GROUPSIZE
    build(str(tmp_path), oracle, seed=8)
    got = []
    for i in (0, 1):
        model, _ = ag.load_llama_model_4bit_low_ram(str(tmp_path), str(tmp_path / "model.safetensors"), groupsize=GROUPSIZE, half=True, device_map={"": i})
        inference.prepare_model(model).eval()
        prompts = [torch.tensor([1, 7, 20 + n], device=f"cuda:{i}") for n in range(3)]
        got.append([t.tolist() for t in inference.generate_batch(model, prompts, 8)])
    assert got[0] == got[1]
