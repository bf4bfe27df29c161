"""Forward-mode differentiation of qk_norm_rope is refused, not silently dropped."""

import pytest
import torch
from torch.autograd import forward_ad

import flash_mlm
from flash_mlm.host import rope


def refused(q, k, table, weight):
    with forward_ad.dual_level():
        for which in range(3):
            args = [q, k, weight]
            args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            for grad in (True, False):  # (no_grad turns reverse mode off only)
                with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError)):
                    flash_mlm.qk_norm_rope(*args[:2], table, q_weight=args[2])
        # without a tangent the call is as ever
        y, _ = flash_mlm.qk_norm_rope(q, k, table, q_weight=weight)
        assert forward_ad.unpack_dual(y).tangent is None
    return y


def test_refused_on_cpu_with_the_kernel_stubbed_out(monkeypatch):
    monkeypatch.setattr(rope, "_validate", lambda *a: None)
    monkeypatch.setattr(rope, "_launch", lambda *a, **k: None)
    x = torch.zeros((1, 2, 8, 64), dtype=torch.float16)
    refused(x, x.clone(), flash_mlm.RotaryTable(8, 64, device="cpu"), torch.ones(64))


@pytest.mark.gpu
def test_refused_and_values_unchanged():
    table = flash_mlm.RotaryTable(8, 64, device="cuda")
    x, w = torch.randn((1, 2, 8, 64), device="cuda").half(), torch.ones(64, device="cuda")
    y = refused(x, x.clone(), table, w)
    assert torch.equal(y, flash_mlm.qk_norm_rope(x, x, table, q_weight=w)[0])
