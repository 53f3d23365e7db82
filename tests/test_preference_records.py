"""Prompts of preference records in the Alpaca form, to the last id, with a tokenizer that knows every character (CPU)."""
import json

import pytest

TAIL = "### Response:\n"


class Characters:
    """One id a character, BOS in front; the end-of-sequence text is one id."""
    bos_token_id, eos_token_id, eos_token, pad_token_id = 1, 2, "</s>", 0

    def __call__(self, text, truncation=False, max_length=None, padding=False, **kw):
        ids = [1] + [i for part in [text.split(self.eos_token)] for k, piece in enumerate(part) for i in ([2] if k else []) + [ord(c) + 3 for c in piece]]
        ids = ids[:max_length] if truncation and max_length else ids
        return {"input_ids": ids, "attention_mask": [1] * len(ids)}


class Pieces(Characters):
    """As sentencepiece does it, a space mark in front of every text; a word that follows it is another id than one that doesn't."""

    def __call__(self, text, **kw):
        enc = super().__call__(text, **kw)
        enc["input_ids"].insert(1, ord(" ") + 3)
        enc["attention_mask"].append(1)
        return enc


def _text(ids):
    return "".join("</s>" if i == 2 else chr(i - 3) for i in ids if i != 1)


def _reader(tmp_path, tok, window, records):
    from alpaca_lora_4bit_amd.train_data import TrainPreference
    path = str(tmp_path / "pairs.json")
    with open(path, "w") as fh:
        json.dump(records, fh)
    return TrainPreference(path, 0, tok, window)


@pytest.mark.parametrize("tok", [Characters(), Pieces()])
@pytest.mark.parametrize("fields", [{"instruction": "do it"}, {"instruction": "do it", "input": "now\n\nor never"}, {"instruction": "### Response:\n?", "input": ""}])
def test_a_prompt_that_fits_is_the_template_and_nothing_else(tmp_path, tok, fields):
    """The ids are those that the reader of Alpaca records makes of the same record with this answer."""
    from alpaca_lora_4bit_amd.train_data import TrainSAD
    record = {**fields, "chosen": "yes", "rejected": "\nno"}
    data = _reader(tmp_path, tok, 1000, [record])
    data.prepare_data()
    got = data.train_data[0]
    for name in ("chosen", "rejected"):
        want = TrainSAD(None, 0, tok, 1000).generate_and_tokenize_prompt({**fields, "output": record[name]})["input_ids"]
        assert got[name + "_ids"] == want
        answer = len(record[name]) + 1
        assert got[name + "_labels"] == [-100] * (len(want) - answer) + want[-answer:] and _text(want[:-answer]).endswith(TAIL)


@pytest.mark.parametrize("tok", [Characters(), Pieces()])
@pytest.mark.parametrize("window", [120, 301])
def test_a_prompt_that_is_too_long_keeps_where_the_answer_begins(tmp_path, tok, window):
    """Half of the window, the template's last line whole in it, and the answer right behind."""
    data = _reader(tmp_path, tok, window, [{"instruction": "do it " * 50, "input": "now " * 30, "chosen": "yes", "rejected": "n" * 1000}])
    data.prepare_data()
    got = data.train_data[0]
    whole = tok("Below is an instruction that describes a task, paired with an input that provides further ")["input_ids"]
    head = got["chosen_ids"][:window // 2]
    assert head[:30] == whole[:30] and _text(head).endswith("\n\n" + TAIL)
    assert _text(got["chosen_ids"][window // 2:]) == "yes</s>" and got["chosen_labels"] == [-100] * (window // 2) + got["chosen_ids"][window // 2:]
    assert got["rejected_ids"][:window // 2] == head and len(got["rejected_ids"]) == window and _text(got["rejected_ids"][window // 2:]) == "n" * (window - window // 2)


@pytest.mark.parametrize("window", [1, 2, 3, 5, 16, 31, 32, 33, 34])
def test_windows_that_do_not_hold_the_last_line(tmp_path, window):
    tok = Characters()
    data = _reader(tmp_path, tok, window, [{"instruction": "do it", "chosen": "yes", "rejected": "no"}])
    data.prepare_data()
    got = data.train_data[0]
    for name in ("chosen", "rejected"):
        ids, labels = got[name + "_ids"], got[name + "_labels"]
        assert len(ids) == len(labels) <= window and labels[:window // 2] == [-100] * (window // 2) and labels[window // 2:] == ids[window // 2:]
        assert _text(ids[window // 2:]) == (("yes" if name == "chosen" else "no") + "</s>" * (window > 8))[:window - window // 2] or window <= 8
        assert window < 4 or ids[0] == 1 and _text(ids[:window // 2]).endswith(("\n\n" + TAIL)[-(window // 2 - 1):])


def test_a_plain_prompt_its_newline_and_the_answer_are_each_by_themselves(tmp_path):
    for tok, want in ((Characters(), "Say yes o\nyes</s>"), (Pieces(), " Say yes  \n yes</s>")):
        data = _reader(tmp_path, tok, 20, [{"prompt": "Say yes or no now.", "chosen": "yes", "rejected": "no"}])
        data.prepare_data()
        assert _text(data.train_data[0]["chosen_ids"]) == want and _text(data.train_data[0]["rejected_ids"]) == want.replace("yes</s>", "no</s>")
