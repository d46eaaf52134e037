"""Settings of `sample` that no floating number can hold: refused like any other that is out of range."""
import pytest
import torch

from thundergbm_amd import scores as S


@pytest.mark.parametrize("name", ["p", "min_p", "temperature"])
@pytest.mark.parametrize("v", [10**400, -10**400], ids=["above", "below"])
def test_numbers_beyond_a_double(name, v):
    with pytest.raises(ValueError, match=name + " is"):
        S._one_setting(name, v, *S._FINE[name])
    with pytest.raises(ValueError, match=name + " is"):
        S._setting(torch, name, v, torch.zeros(3, 5), torch.float32, *S._FINE[name])


def test_counts_have_no_end():
    assert S._one_setting("k", 10**400, *S._FINE["k"]) == 10**400
