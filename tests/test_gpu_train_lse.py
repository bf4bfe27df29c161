"""GPU tests of the softmax statistics that flash_attn_mlm_fwd returns, against 64-bit values."""

import pytest
import torch

from test_gpu_train import BF16, DEV, F16, assert_within, fm, meta_of, pack, rand
from train_ref import batch_reference

pytestmark = pytest.mark.gpu


def check_lse(layout, dtype, B, H, HK, N, D, lens, scale, ctx=None, causal=False):
    g = torch.Generator().manual_seed(6)
    q, do = (rand(g, (B, H, N, D), dtype) for _ in range(2))
    k, v = (rand(g, (B, HK, N, D), dtype) for _ in range(2))
    kc = vc = cmeta = None
    if ctx is not None:
        kc, vc = (rand(g, (HK, sum(ctx), D), dtype) for _ in range(2))
        cmeta = meta_of(ctx, max(ctx))
    val, bnd = batch_reference(q, k, v, do, scale, lens, kc, vc, ctx, causal)
    meta = None if layout == "dense" else meta_of(lens, N)
    if layout == "packed":
        q, k, v = (pack(x, lens) for x in (q, k, v))
    out, lse = fm().flash_attn_mlm_fwd(q, k, v, scale, meta, kc, vc, cmeta, causal)
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    assert lse.dtype == torch.float32 and lse.shape == q.shape[:-1] and lse.is_contiguous()
    rows = (lambda x: x) if layout == "packed" else (lambda x: pack(x[..., None], lens)[..., 0])
    ref = lambda x: pack(x[..., None], lens)[..., 0]
    assert_within(rows(lse), ref(val["lse"]), ref(bnd["lse"]), "lse")
    o = out if layout == "packed" else pack(out, lens)
    assert_within(o, pack(val["o"], lens), pack(bnd["o"], lens), "o")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["dense", "padded", "packed"])
def test_lengths_and_grouped_heads(dtype, D, layout):
    lens = [200, 200, 200] if layout == "dense" else [200, 1, 129]
    check_lse(layout, dtype, 3, 4, 2, 200, D, lens, D ** -0.5)


@pytest.mark.parametrize("ctx", [None, [300], [17, 0, 256, 129]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,dtype", [(32, F16), (64, BF16), (128, F16), (256, BF16)])
def test_contexts_and_earlier_sequences(ctx, causal, D, dtype):
    check_lse("packed", dtype, 4, 4, 2, 180, D, [180, 33, 0, 150], D ** -0.5, ctx=ctx, causal=causal)


@pytest.mark.parametrize("scale", [-0.25, 0.0, 1.0])
@pytest.mark.parametrize("layout", ["dense", "padded", "packed"])
def test_scales(scale, layout):
    lens = [150, 150] if layout == "dense" else [150, 77]
    check_lse(layout, BF16, 2, 2, 1, 150, 64, lens, scale)
