"""Options of the preference loss are refused before anything is loaded (CPU)."""
import pytest


@pytest.mark.parametrize("option,values", [("--beta", ["0", "-0.1", "nan", "inf", "much"]), ("--label_smoothing", ["-0.01", "0.51", "0.7", "nan", "inf", "much"])])
def test_values_that_the_loss_refuses(option, values, monkeypatch, capsys):
    from alpaca_lora_4bit_amd import autograd_4bit, finetune

    def loaded(*a, **kw):
        raise AssertionError("the model was loaded")
    monkeypatch.setattr(autograd_4bit, "load_llama_model_4bit_low_ram", loaded, raising=False)
    for value in values:
        with pytest.raises(SystemExit) as end:
            finetune.main(["pairs.json", "--ds_type", "preference", f"{option}={value}"])
        assert end.value.code == 2 and option in capsys.readouterr().err


def test_values_at_the_ends_are_taken():
    from alpaca_lora_4bit_amd.arg_parser import get_config
    for beta, smoothing in ((1e-6, 0.0), (0.3, 0.5), (100.0, 0.1)):
        cfg = get_config(["--beta", str(beta), "--label_smoothing", str(smoothing)])
        assert (cfg.beta, cfg.label_smoothing) == (beta, smoothing)


def test_a_config_made_by_hand_is_checked_too():
    from alpaca_lora_4bit_amd.Finetune4bConfig import Finetune4bConfig
    from alpaca_lora_4bit_amd.arg_parser import parse_commandline, _RENAMED
    plain = {_RENAMED.get(k, k): v for k, v in parse_commandline([]).items()}
    assert Finetune4bConfig(**plain).beta == 0.1
    for bad in (dict(beta=0.0), dict(beta=float("nan")), dict(label_smoothing=0.6), dict(label_smoothing=-1.0), dict(act_bits=4)):
        with pytest.raises(ValueError):
            Finetune4bConfig(**plain, **bad)
