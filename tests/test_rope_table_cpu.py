"""CPU tests of RotaryTable's base: one without a table of finite turns is refused."""

import pytest
import torch

import flash_mlm


@pytest.mark.parametrize("base", [0.0, -10000.0, float("nan"), float("inf")])
def test_base_refusals(base):
    with pytest.raises(ValueError, match="base"):
        flash_mlm.RotaryTable(8, 16, base=base, device="cpu")


def test_base_is_not_looked_at_with_frequencies_of_ones_own():
    t = flash_mlm.RotaryTable(8, 16, base=0.0, inv_freq=torch.ones(8), device="cpu")
    assert torch.isfinite(t.table).all()
