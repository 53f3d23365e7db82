"""What inference.generate_batch captures and when, on the CPU: streams and graphs stand as recorders, the operators as plain float64 code."""
import contextlib

import pytest
import torch

from alpaca_lora_4bit_amd import inference

from test_batch_generation import PROMPTS, Plain, _model


@pytest.fixture
def events(monkeypatch):
    """'eager' and 'capture' for every one-token step that runs, 'replay' for every replay."""
    _model()                                                 # imports what looks at torch.cuda while it is imported
    seen, inside = [], []
    plain = Plain(monkeypatch)
    append = plain.kv4_append

    def counted(k, v, cache, table, lengths, **kw):
        if kw.get("starts") is None and (not seen or seen[-1][1] != int(lengths.sum())):
            seen.append(("capture" if inside else "eager", int(lengths.sum())))
        return append(k, v, cache, table, lengths, **kw)
    from alpaca_lora_4bit_amd import quant_hip
    monkeypatch.setattr(quant_hip, "kv4_append", counted)

    class Stream:
        def __init__(self, device=None):
            assert device is not None and device.type == "cpu"           # where the prompts are

        def wait_stream(self, other):
            pass

    class Graph:
        def replay(self):
            seen.append(("replay", -1))

    @contextlib.contextmanager
    def graph(g, stream):
        assert isinstance(stream, Stream)
        inside.append(g)
        yield
        inside.pop()
    monkeypatch.setattr(inference, "_capture_streams", {})
    for name, value in (("Stream", Stream), ("current_stream", Stream), ("stream", lambda s: contextlib.nullcontext()), ("CUDAGraph", Graph), ("graph", graph)):
        monkeypatch.setattr(torch.cuda, name, value)
    return seen


@pytest.mark.parametrize("new,want", [(1, []), (2, ["eager"]), (3, ["eager", "eager"]), (4, ["eager", "capture", "replay", "replay"]),
                                      (6, ["eager", "capture"] + ["replay"] * 4)])
def test_a_step_runs_before_one_is_captured(events, new, want):
    """The first step is never captured (what is allocated and checked at a first use has to happen outside a graph), nor is one for a single replay."""
    got = inference.generate_batch(_model(), PROMPTS, new)
    assert [e for e, _ in events] == want
    assert [len(g) for g in got] == [len(p) + new for p in PROMPTS]
