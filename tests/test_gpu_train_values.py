"""GPU tests of attention's gradients for values far from 1: large scores, scales
at the ends of float16's range, small gradients."""

import pytest
import torch

import train_ref
from test_gpu_train import BF16, DEV, F16, assert_within, fm, meta_of, rand
from train_ref import batch_reference

pytestmark = pytest.mark.gpu


def device():
    return torch.device(DEV, torch.cuda.current_device())


def gradients(q, k, v, do, scale, **kw):
    out, lse = fm().flash_attn_mlm_fwd(q, k, v, scale, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (out, *fm().flash_attn_mlm_bwd(do, q, k, v, out, lse, scale, **kw))))


def within(monkeypatch, r32, q, k, v, do, scale):
    """Output and gradients of a dense batch, with r32 for what 32 bits cost."""
    monkeypatch.setattr(train_ref, "R32", r32)
    val, bnd = batch_reference(q, k, v, do, scale, [q.shape[2]] * q.shape[0])
    got = gradients(q, k, v, do, scale)
    fm().check_device_errors(device())
    for name, x in got.items():
        assert_within(x, val[name], bnd[name], name)


# A score S of float32 is off by up to 2^-24 S at each rounding, and its probability by that share:
# the forward pass rounds S log2(e) - max, the maximum, lse twice; the backward pass lse log2(e),
# that over the scale, the difference's scale: eight in all where q k^T itself is exact.  Where it is not,
# its sum (one rounding per 16 columns, 16 at most, of partial sums that need not be smaller) doubles and adds.


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("lse", [163840, 196608, 262144, -262144])
def test_large_offset(monkeypatch, dtype, D, lse):
    """Scores near one large number (one column of q and k, the others in halves, so that q k^T is exact)."""
    g = torch.Generator().manual_seed(1)
    q, k = ((torch.randint(-2, 3, (1, h, 300, D), generator=g) / 2).to(dtype).to(DEV) for h in (4, 2))
    q[..., 0], k[..., 0] = 1024, lse / 128
    v, do = rand(g, (1, 2, 300, D), dtype), rand(g, (1, 4, 300, D), dtype)
    within(monkeypatch, 8 * 2.0**-24 * abs(lse), q, k, v, do, 0.125)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("magnitude", [100, 160, 300])
def test_large_rows(monkeypatch, dtype, magnitude):
    """q = k of large rows, as an unnormed projection may give them."""
    g = torch.Generator().manual_seed(2)
    q = (torch.randn((1, 2, 300, 64), generator=g) * magnitude).to(dtype).to(DEV)
    v, do = (rand(g, (1, 2, 300, 64), dtype) for _ in range(2))
    top = 0.125 * q.double().square().sum(-1).max().item()
    within(monkeypatch, 40 * 2.0**-24 * top, q, q.clone(), v, do, 0.125)


@pytest.mark.parametrize("scale,size", [(2.0**-24, 2.0**12), (2.0**-20, 2.0**10), (2.0**-16, 2.0**7), (-(2.0**-20), 2.0**10),
                                        (2.0**13, 2.0**-8), (2.0**20, 2.0**-11), (-(2.0**20), 2.0**-11)])
def test_float16_scales(monkeypatch, scale, size):
    """Small scales of large rows and large scales of small ones: scores up to a few hundred."""
    g = torch.Generator().manual_seed(3)
    q, k = ((torch.randn((1, h, 200, 64), generator=g).clamp(-3.9, 3.9) * size).to(F16).to(DEV) for h in (4, 2))
    v, do = rand(g, (1, 2, 200, 64), F16), rand(g, (1, 4, 200, 64), F16)
    top = (scale * q.double() @ k.double().repeat_interleave(2, 1).transpose(2, 3)).abs().max().item()
    within(monkeypatch, max(train_ref.R32, 40 * 2.0**-24 * top), q, k, v, do, scale)


def test_float16_scores_that_do_not_fit_are_reported():
    q = torch.zeros((1, 1, 9, 64), dtype=F16, device=DEV)
    q[..., :2] = 65504.0
    v = torch.ones_like(q)
    out, lse = fm().flash_attn_mlm_fwd(q, q, v, 2.0**-24)
    dq = fm().flash_attn_mlm_bwd(v, q, q, v, out, lse, 2.0**-24, need_dkv=False)[0]
    fm().check_device_errors(device())
    assert torch.isfinite(dq).all()
    fm().flash_attn_mlm_bwd(v, q, q, v, out, lse, 2.0**-24)
    with pytest.raises(RuntimeError, match="too large"):
        fm().check_device_errors(device())
    fm().check_device_errors(device())


def test_float16_scores_that_do_not_fit_among_others_are_reported():
    """Rows of 2^14 a column: scores of 2^33 before their scale, past the 2^31 that dk and dv can hold."""
    g = torch.Generator().manual_seed(3)
    q, k = ((torch.randn((1, h, 200, 64), generator=g).clamp(-3.9, 3.9) * 2.0**14).to(F16).to(DEV) for h in (4, 2))
    v, do = rand(g, (1, 2, 200, 64), F16), rand(g, (1, 4, 200, 64), F16)
    gradients(q, k, v, do, 2.0**-24)
    with pytest.raises(RuntimeError, match="too large"):
        fm().check_device_errors(device())


def test_float16_padding_and_other_sequences_are_not_reported():
    """What lies past a sequence has no statistics to report, whatever it holds."""
    g = torch.Generator().manual_seed(4)
    x = rand(g, (2, 2, 150, 64), F16)
    x[0, :, 20:], x[1, :, 140:] = 65504.0, float("inf")
    gradients(x, x, x, x, 0.125, q_meta=meta_of([20, 140], 150))
    fm().check_device_errors(device())


@pytest.mark.parametrize("D", [64, 128])
def test_float16_nan_reaches_the_gradients_it_enters(D):
    """A NaN in one key makes every probability of the rows that see it NaN, and with them dk and dv of all their keys."""
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (rand(g, (1, 2, 200, D), F16) for _ in range(4))
    k[0, 0, 7, 3] = float("nan")
    got = gradients(q, k, v, do, 0.125)
    fm().check_device_errors(device())
    for name, x in got.items():
        assert torch.isnan(x[0, 0]).all(), name
        assert torch.isfinite(x[0, 1]).all(), name
