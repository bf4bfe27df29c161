"""GPU tests of attention for training: output, statistics and gradients
against 64-bit math within the bounds of tests/train_ref.py, over layouts,
types, head counts and lengths from none to several tiles."""

import pytest
import torch

from train_ref import batch_reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


def fm():
    import flash_mlm

    return flash_mlm


def meta_of(lens, N, dev=DEV):
    return fm().build_pack_metadata(torch.tensor(lens, dtype=torch.int32, device=dev), N, 64)


def rand(g, shape, dtype):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def pack(x, lens):
    """[B, H, N, D] -> [H, T, D] by torch indexing."""
    return torch.cat([x[b, :, :n] for b, n in enumerate(lens)], 1)


def assert_within(got, val, bnd, what):
    got = got.detach().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert got.shape == val.shape, what
    bad = (got - val).abs() > bnd
    if bad.any():
        i = int(((got - val).abs() - bnd).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside their bounds; worst at flat index {i}: got "
                             f"{got.flatten()[i]:.6g}, want {val.flatten()[i]:.6g} within {bnd.flatten()[i]:.3g}")


def check(layout, dtype, B, H, HK, N, D, lens, ctx=None, causal=False, scale=None, seed=0, poison=True,
          exact_delta=False, two_parts=False):
    g = torch.Generator().manual_seed(seed)
    scale = D ** -0.5 if scale is None else scale
    q, do = rand(g, (B, H, N, D), dtype), rand(g, (B, H, N, D), dtype)
    k, v = rand(g, (B, HK, N, D), dtype), rand(g, (B, HK, N, D), dtype)
    kc = vc = cmeta = None
    if ctx is not None:
        kc, vc = rand(g, (HK, sum(ctx), D), dtype), rand(g, (HK, sum(ctx), D), dtype)
        cmeta = meta_of(ctx, max(ctx))
    val, bnd = batch_reference(q, k, v, do, scale, lens, kc, vc, ctx, causal, exact_delta, two_parts)
    if layout == "dense":
        meta = None
        ins = [q, k, v, do]
    elif layout == "padded":
        meta = meta_of(lens, N)
        ins = [q, k, v, do]
        if poison:  # what lies past a sequence must not matter
            ins = [x.clone() for x in ins]
            for x in ins:
                for b, n in enumerate(lens):
                    x[b, :, n:] = float("nan")
    else:
        meta = meta_of(lens, N)
        ins = [pack(x, lens).contiguous() for x in (q, k, v, do)]
    q, k, v = (x.requires_grad_() for x in ins[:3])
    leaves = [q, k, v]
    if ctx is not None:
        leaves += [kc.requires_grad_(), vc.requires_grad_()]
    out = fm().flash_attn_mlm_train(q, k, v, scale, q_meta=meta, context_k=kc, context_v=vc, context_meta=cmeta,
                                    causal_query_seq_attn=causal)
    grads = torch.autograd.grad(out, leaves, ins[3])
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    names = ["dq", "dk", "dv", "dkc", "dvc"][: len(leaves)]
    for name, got in zip(["o", *names], [out, *grads]):
        w, e = val[name], bnd[name]
        if layout == "packed" and name in ("o", "dq", "dk", "dv"):
            w, e = pack(w, lens), pack(e, lens)
        assert_within(got, w, e, f"{name}")
    return out, grads


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("N", [1, 2, 127, 128, 129, 300])
def test_dense(dtype, D, N):
    check("dense", dtype, 2, 2, 2, N, D, [N, N])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", ["padded", "packed"])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_lengths(dtype, layout, D):
    check(layout, dtype, 7, 3, 3, 290, D, [290, 0, 1, 129, 128, 64, 17])


@pytest.mark.parametrize("layout", ["dense", "padded", "packed"])
@pytest.mark.parametrize("H,HK", [(4, 1), (6, 2), (5, 5)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_grouped_heads(layout, H, HK, D):
    lens = [200, 200, 200] if layout == "dense" else [131, 200, 3]
    check(layout, BF16, 3, H, HK, 200, D, lens)


@pytest.mark.parametrize("layout", ["padded", "packed"])
@pytest.mark.parametrize("ctx", [[300], [1], [17, 0, 256, 129]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,dtype", [(32, F16), (64, BF16), (128, F16), (256, BF16)])
def test_context(layout, ctx, causal, D, dtype):
    check(layout, dtype, 4, 4, 2, 180, D, [180, 33, 0, 150], ctx=ctx, causal=causal)


@pytest.mark.parametrize("layout", ["padded", "packed"])
@pytest.mark.parametrize("D", [64, 128])
def test_causal_by_sequence(layout, D):
    check(layout, F16, 5, 2, 2, 140, D, [140, 0, 7, 128, 65], causal=True)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_scales(scale):
    check("padded", BF16, 2, 2, 2, 150, 64, [150, 77], scale=scale)


def test_many_items():
    """More items than CTAs, several of them empty, lengths that do not line up with the tiles."""
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 300, (70,), generator=g)]
    check("packed", BF16, 70, 8, 4, 300, 64, lens)
    check("padded", F16, 70, 8, 8, 300, 128, lens)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("lens,ctx,causal", [([2, 3, 1, 20, 2], None, False), ([2, 3, 1, 20, 2], [5, 1, 0, 40, 3], False),
                                             ([4, 1, 0, 7, 9], [13], True), ([64, 50, 2, 2, 2], None, False)])
def test_few_keys(dtype, D, lens, ctx, causal):
    """Rows of few keys: delta is summed in 32 bits, so its part of the bounds falls away."""
    check("packed", dtype, 5, 4, 2, 64, D, lens, ctx=ctx, causal=causal, exact_delta=True)
    if ctx is None:
        check("padded", dtype, 5, 4, 2, 64, D, lens, exact_delta=True)


def test_long():
    check("dense", BF16, 1, 2, 1, 2500, 128, [2500])
    check("packed", F16, 2, 2, 2, 2100, 64, [2100, 901], ctx=[1500])
