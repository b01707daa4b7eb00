"""What the generation command refuses before it looks for a device or a model."""
import pytest

from ug_b200 import generate


@pytest.mark.parametrize("option,value", [("--temperature", "-0.1"), ("--temperature", "nan"), ("--temperature", "1e21"), ("--top-k", "-1"), ("--top-p", "0"), ("--top-p", "nan"),
                                          ("--min-p", "-0.1"), ("--min-p", "1.5")])
def test_settings_outside_their_range(option, value, capsys):
    with pytest.raises(SystemExit) as e:
        generate.main(["--model", "nowhere", "--prompt", "1,2", option, value])
    assert e.value.code == 2 and option[2:] in capsys.readouterr().err


def test_prompts_of_different_lengths(capsys):
    with pytest.raises(SystemExit):
        generate.main(["--model", "nowhere", "--prompt", "1,2", "--prompt", "1"])
    assert "one length" in capsys.readouterr().err


def test_a_seed_below_zero(capsys):
    with pytest.raises(SystemExit) as e:
        generate.main(["--model", "nowhere", "--prompt", "1,2", "--seed", "-1"])
    assert e.value.code == 2 and "seed" in capsys.readouterr().err


def test_a_share_that_vanishes_in_32_bits(capsys):
    with pytest.raises(SystemExit) as e:
        generate.main(["--model", "nowhere", "--prompt", "1,2", "--top-p", "1e-60"])
    assert e.value.code == 2 and "top-p" in capsys.readouterr().err
