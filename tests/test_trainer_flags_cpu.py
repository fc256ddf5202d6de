"""Flags of grpo_train that an algorithm would pass over are refused."""
import pytest

from kharon_b200 import grpo_train


@pytest.mark.parametrize("flags", [["--inner", "2", "--clip-eps", "0.2"], ["--clip-eps", "0.2"], ["--inner", "2"]])
def test_flags_of_the_clipped_loss_are_refused_with_preferences(flags):
    with pytest.raises(SystemExit, match="--algo dpo"):
        grpo_train.main(["--layers", "1", "--d", "32", "--heads", "2", "--G", "2", "--prompts", "1", "--steps", "0", "--sft", "0", "--device", "cpu", "--algo", "dpo"] + flags)


def test_preferences_need_an_even_number_of_samples():
    """Said at once, not after the supervised steps."""
    with pytest.raises(SystemExit, match="--G"):
        grpo_train.main(["--layers", "1", "--d", "32", "--heads", "2", "--G", "3", "--prompts", "1", "--steps", "0", "--sft", "0", "--device", "cpu", "--algo", "dpo"])
