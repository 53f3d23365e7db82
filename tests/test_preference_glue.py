"""Host side of training on pairs (CPU): the reader and collator of preference records, the options, switching adapters off, and what the 8-bit
options refuse."""
import json

import pytest
import torch

from test_finetune_glue import ToyTokenizer


def _records(tmp_path, records):
    path = str(tmp_path / "pairs.json")
    with open(path, "w") as fh:
        json.dump(records, fh)
    return path


def test_reader_of_preference_records(tmp_path):
    from alpaca_lora_4bit_amd.train_data import TrainPreference, collate_pairs
    tok = ToyTokenizer()
    path = _records(tmp_path, [{"prompt": "a b", "chosen": "c d", "rejected": "e"}, {"prompt": "a b a b a b a b", "chosen": "c " * 20, "rejected": "e f"}])
    data = TrainPreference(path, 0, tok, 10)
    data.prepare_data(use_eos_token=True, thd=-1)
    assert data.val_data is None and len(data.train_data) == 2 and set(data.train_data.column_names) == {"chosen_ids", "chosen_labels", "rejected_ids", "rejected_labels"}
    a, b, c, d, e, f = (tok.vocab[w] for w in "abcdef")
    first = data.train_data[0]                                 # "\n" has no word of its own here
    assert first["chosen_ids"] == [1, a, b, c, d, 2] and first["chosen_labels"] == [-100] * 3 + [c, d, 2]
    assert first["rejected_ids"] == [1, a, b, e, 2] and first["rejected_labels"] == [-100] * 3 + [e, 2]
    second = data.train_data[1]                                # the prompt takes half of the window at most, a cut answer has no end
    assert second["chosen_ids"] == [1, a, b, a, b] + [c] * 5 and second["chosen_labels"] == [-100] * 5 + [c] * 5
    assert second["rejected_ids"] == [1, a, b, a, b, e, f, 2]
    batch = collate_pairs([data.train_data[0], data.train_data[1]], 0)
    assert batch["input_ids"].tolist() == [first["chosen_ids"] + [0] * 4, second["chosen_ids"], first["rejected_ids"] + [0] * 5, second["rejected_ids"] + [0] * 2]
    assert batch["attention_mask"].sum(1).tolist() == [6, 10, 5, 8] and batch["labels"].dtype == torch.int64
    assert batch["labels"][2].tolist() == [-100] * 3 + [e, 2] + [-100] * 5
    data.prepare_data(use_eos_token=False)
    assert data.train_data[0]["rejected_ids"] == [1, a, b, e]
    assert len(collate_pairs([data.train_data[0]], 7)["input_ids"]) == 2


def test_records_with_alpaca_fields_and_a_validation_split(tmp_path):
    from alpaca_lora_4bit_amd.train_data import TrainPreference
    tok = ToyTokenizer()
    data = TrainPreference(_records(tmp_path, [{"instruction": "do it", "input": "now", "chosen": "yes", "rejected": "no"}] * 10), 0.3, tok, 128)
    data.prepare_data()
    assert len(data.train_data) == 7 and len(data.val_data) == 3
    ids = data.train_data[0]["chosen_ids"]
    assert ids[0] == 1 and ids[-1] == 2 and all(tok.vocab[w] in ids for w in ("do", "it", "now", "yes")) and tok.vocab["no"] not in ids
    assert data.train_data[0]["chosen_labels"][-2:] == [tok.vocab["yes"], 2]


def test_options():
    from alpaca_lora_4bit_amd.arg_parser import get_config, parse_commandline
    plain = get_config([])
    assert (plain.act_bits, plain.beta, plain.label_smoothing) == (16, 0.1, 0.0) and "beta" not in parse_commandline([])
    cfg = get_config(["pairs.json", "--ds_type", "preference", "--act_bits", "8", "--beta", "0.3", "--label_smoothing", "0.1"])
    assert (cfg.ds_type, cfg.act_bits, cfg.beta, cfg.label_smoothing) == ("preference", 8, 0.3, 0.1) and "act_bits=8" in str(cfg)
    with pytest.raises(SystemExit):
        parse_commandline(["--act_bits", "4"])


def test_labels_move_one_place():
    from alpaca_lora_4bit_amd.preference import shifted_labels
    assert shifted_labels(torch.tensor([[1, 2, 3], [-100, 5, -100]])).tolist() == [[2, 3, -100], [5, -100, -100]]
    assert shifted_labels(torch.tensor([[4]])).tolist() == [[-100]]


def test_adapters_are_off_and_come_back():
    import torch.nn as nn
    from alpaca_lora_4bit_amd.models import Linear4bitLt
    from alpaca_lora_4bit_amd.preference import adapters_off
    a, b = (Linear4bitLt("default", 128, 128, 128, False, r=8, lora_alpha=16) for _ in range(2))
    model = nn.ModuleList([a, nn.Linear(3, 3), b])
    b.enable_adapters(False)
    with pytest.raises(KeyError), adapters_off(model):
        assert a.disable_adapters and b.disable_adapters
        raise KeyError
    assert not a.disable_adapters and b.disable_adapters


def test_8_bit_options_that_are_refused():
    from transformers import LlamaConfig, LlamaForCausalLM
    from alpaca_lora_4bit_amd.gradient_checkpointing import apply_gradient_checkpointing
    from alpaca_lora_4bit_amd.model_attn_mlp_patch import make_fused_mlp
    model = LlamaForCausalLM(LlamaConfig(vocab_size=97, hidden_size=32, intermediate_size=64, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=4))
    for bad in (lambda: make_fused_mlp(model, act_bits=4), lambda: make_fused_mlp(model, act_bits=8, concatenate=True), lambda: make_fused_mlp(model, act_bits=8, fuse_decode_step=False),
                lambda: apply_gradient_checkpointing(model, bits=4)):
        with pytest.raises(ValueError):
            bad()
    assert not any("old_forward_for_cp" in m.__dict__ for m in model.modules())
    apply_gradient_checkpointing(model, bits=8)
    ids = torch.randint(0, 97, (2, 5))
    with pytest.raises(ValueError, match="GPU"):               # the second block's input would have to be packed
        model.train()(input_ids=ids, labels=ids, use_cache=False)
    with torch.no_grad():
        model(input_ids=ids, use_cache=False)
    model.eval()(input_ids=ids, use_cache=False)
