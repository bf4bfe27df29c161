"""GPU tests of the forms in which tensors reach the training operators."""

import pytest
import torch

from test_gpu_train import BF16, DEV, F16, assert_within, fm, meta_of, rand
from train_ref import batch_reference

pytestmark = pytest.mark.gpu


def no_errors():
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))


def projection(x):
    """The values in a projection's layout: the heads of a row side by side."""
    return x.transpose(-2, -3).contiguous().transpose(-2, -3)


def pitched(x):
    """The values in rows of an odd pitch, of which a single one counts as contiguous."""
    wide = torch.zeros((*x.shape[:-1], x.shape[-1] + 3), dtype=x.dtype, device=x.device)
    wide[..., : x.shape[-1]] = x
    return wide[..., : x.shape[-1]]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 64, 256])
@pytest.mark.parametrize("lay", [projection, pitched])
@pytest.mark.parametrize("B,H,HK", [(3, 4, 2), (2, 1, 1), (1, 1, 1)])
def test_one_row_dense(dtype, D, lay, B, H, HK):
    g = torch.Generator().manual_seed(1)
    q, do = (lay(rand(g, (B, H, 1, D), dtype)) for _ in range(2))
    k, v = (lay(rand(g, (B, HK, 1, D), dtype)) for _ in range(2))
    val, bnd = batch_reference(q, k, v, do, 0.25, [1] * B, exact_delta=True, two_parts=True)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = fm().flash_attn_mlm_train(*leaves, 0.25)
    grads = torch.autograd.grad(out, leaves, do)
    no_errors()
    for name, x in zip(("o", "dq", "dk", "dv"), (out, *grads)):
        assert_within(x, val[name], bnd[name], name)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lay", [projection, pitched])
@pytest.mark.parametrize("H,HK", [(4, 2), (1, 1)])
def test_one_packed_row_over_a_context(dtype, lay, H, HK):
    """One new token: its gradients, and those of the context, are not trivial."""
    g = torch.Generator().manual_seed(2)
    q, do = (rand(g, (H, 1, 64), dtype) for _ in range(2))
    k, v = (rand(g, (HK, 1, 64), dtype) for _ in range(2))
    kc, vc = (rand(g, (HK, 70, 64), dtype) for _ in range(2))
    val, bnd = batch_reference(*(x[None] for x in (q, k, v, do)), 0.25, [1], kc, vc, [70], two_parts=True)
    leaves = [lay(x).detach().requires_grad_() for x in (q, k, v, kc, vc)]
    out = fm().flash_attn_mlm_train(*leaves[:3], 0.25, meta_of([1], 1), *leaves[3:], meta_of([70], 70))
    grads = torch.autograd.grad(out, leaves, lay(do))
    no_errors()
    for name, x in zip(("o", "dq", "dk", "dv", "dkc", "dvc"), (out, *grads)):
        w, e = (t[name] if name in ("dkc", "dvc") else t[name][0] for t in (val, bnd))
        assert_within(x, w, e, name)


@pytest.mark.parametrize("lay", [projection, pitched])
def test_one_row_without_autograd(lay):
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (rand(g, (2, 4, 1, 64), BF16) for _ in range(4))
    results = []
    for f in (lambda x: x, lay):
        a, b, c, d = (f(x) for x in (q, k, v, do))
        out, lse = fm().flash_attn_mlm_fwd(a, b, c, 0.125)
        results.append((out, lse, *fm().flash_attn_mlm_bwd(d, a, b, c, f(out), f(lse[..., None])[..., 0], 0.125)[:3]))
    no_errors()
    assert all(torch.equal(x, y) for x, y in zip(*results))
