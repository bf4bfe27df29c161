"""GPU tests of positions outside the rotary table: the nearest row is used and reported."""

import pytest
import torch

from test_gpu_rope import BF16, DEV, fm

pytestmark = pytest.mark.gpu
FAR = 2**31 - 1


@pytest.mark.parametrize("offset,row", [(FAR, 7), (FAR - 3, 7), (2**31 - 9, 7), (8, 7), (-(2**31), 0), (-6, 0)])
def test_offsets_past_either_end(offset, row):
    """Six tokens behind an offset near the ends of 32 bits: all of them past the table's end, or before its start."""
    table = fm().RotaryTable(8, 64, device=DEV)
    x = torch.randn((1, 2, 6, 64), device=DEV).to(BF16)
    offs = torch.tensor([offset], dtype=torch.int32, device=DEV)
    got, _ = fm().qk_norm_rope(x, x, table, position_offsets=offs)
    with pytest.raises(RuntimeError, match="position"):
        fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    want, _ = fm().qk_norm_rope(x, x, table, positions=torch.full((1, 6), row, dtype=torch.int32, device=DEV))
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    assert torch.equal(got, want)


def test_one_sequence_outside_leaves_the_others_alone():
    table = fm().RotaryTable(8, 64, device=DEV)
    x = torch.randn((3, 2, 4, 64), device=DEV).to(BF16)
    offs = torch.tensor([2, FAR, -FAR], dtype=torch.int32, device=DEV)
    got, _ = fm().qk_norm_rope(x, x, table, position_offsets=offs)
    with pytest.raises(RuntimeError, match="position"):
        fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    want, _ = fm().qk_norm_rope(x[:1], x[:1], table, position_offsets=offs[:1])
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    assert torch.equal(got[:1], want)
