"""GPU tests of padded batches in which most sequences are empty: a block of the
attention kernels meets partial key blocks and items without keys in turn."""

import pytest
import torch

from test_gpu_train import BF16, DEV, F16, check, fm, meta_of, rand

pytestmark = pytest.mark.gpu


def mostly_empty(seed, n, some):
    g = torch.Generator().manual_seed(seed)
    lens = [0] * n
    for i in torch.randperm(n, generator=g)[:some].tolist():
        lens[i] = int(torch.randint(1, 8, (1,), generator=g))
    return lens


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("some", [20, 90])
def test_inference_padded_output(D, some):
    """Every block has one or two partial items, then several without keys."""
    lens, H, N = mostly_empty(1, 400, some), 4, 8
    B = len(lens)
    g = torch.Generator().manual_seed(2)
    q, k, v = (rand(g, (B, H, N, D), BF16) for _ in range(3))
    args = dict(num_heads=H, q_meta=meta_of(lens, N), scale=D ** -0.5, block_n=64)
    padded = fm().flash_attn_mlm_compressed(q, k, v, out_layout="padded", **args)
    packed = fm().unpack_from_kernel(fm().flash_attn_mlm_compressed(q, k, v, **args), args["q_meta"], H)
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    assert torch.equal(padded, packed)


@pytest.mark.parametrize("D,dtype", [(32, F16), (64, BF16), (128, F16), (256, BF16)])
def test_training_padded(D, dtype):
    lens = mostly_empty(3, 300, 60)
    check("padded", dtype, len(lens), 4, 2, 8, D, lens)
