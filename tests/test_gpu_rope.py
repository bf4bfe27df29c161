"""GPU tests of qk_norm_rope against 64-bit math, values and gradients.

Bounds: every output is rounded once to its type (u, half a step relative to
the value, plus float16's half subnormal step); the 32-bit arithmetic before
it (a mean of at most 256 squares, a reciprocal root, four products and two
sums, table entries rounded to float32) stays within r = 2^-18 of the
magnitudes that enter it.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16
R32 = 2.0 ** -18


def fm():
    import flash_mlm

    return flash_mlm


def meta_of(lens, N):
    return fm().build_pack_metadata(torch.tensor(lens, dtype=torch.int32, device=DEV), N, 64)


def reference(x, w, g, pos, R, pairs, base, eps, normalize=True):
    """x, g [heads, T, D], pos [T] (float64 throughout) -> y, dx, dw and magnitudes for their bounds."""
    x, g = x.double(), g.double()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    idx0 = torch.arange(0, R, 2) if pairs == "interleaved" else torch.arange(R // 2)
    idx1 = idx0 + 1 if pairs == "interleaved" else idx0 + R // 2
    freq = base ** (-torch.arange(0, R, 2, dtype=torch.float64, device=x.device) / max(R, 1))
    ang = pos.double()[:, None] * freq

    def rotate(v, s):
        out, mag = v.clone(), v.abs()
        a, b = v[..., idx0], v[..., idx1]
        out[..., idx0] = a * ang.cos() - s * b * ang.sin()
        out[..., idx1] = b * ang.cos() + s * a * ang.sin()
        mag[..., idx0] = a.abs() + b.abs()
        mag[..., idx1] = a.abs() + b.abs()
        return out, mag

    gr, gmag = rotate(g, -1.0)
    if not normalize:
        y, ymag = rotate(x, 1.0)
        return y, ymag, gr, gmag, None, None
    rstd = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * rstd
    y, ymag = rotate(xh * w, 1.0)
    dw, dwmag = (gr * xh).sum((0, 1)), (gmag * xh.abs()).sum((0, 1))
    dx = rstd * (gr * w - xh * (gr * w * xh).mean(-1, keepdim=True))
    dxmag = rstd * (gmag * w.abs() + xh.abs() * (gmag * w.abs() * xh.abs()).mean(-1, keepdim=True))
    return y, ymag, dx, dxmag, dw, dwmag


def assert_near(got, val, mag, what):
    got = got.detach()
    u = torch.finfo(got.dtype).eps / 2
    bound = u * val.abs() + R32 * mag + (2.0 ** -25 if got.dtype == F16 else 0.0)
    got = got.double()
    assert got.shape == val.shape and torch.isfinite(got).all(), what
    bad = (got - val).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - val).abs() - bound).max():.3g}"


def check(layout, dtype, B, H, HK, N, D, R, pairs, lens=None, weights="f32", pos="index", base=10000.0, strided=True,
          normalize=True, eps=1e-6, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = [N] * B if lens is None else lens
    T = sum(lens)
    meta = meta_of(lens, N) if layout != "dense" else None

    def tensor(heads):
        shape = (T, heads, D) if layout == "packed" else (B, N, heads, D)
        x = (torch.randn(shape, generator=g) * 2).to(dtype).to(DEV).transpose(-2, -3)
        return x if strided else x.contiguous()

    q, k, gq, gk = tensor(H), tensor(HK), tensor(H), tensor(HK)
    if layout == "padded":
        for x in (q, k, gq, gk):
            for b, n in enumerate(lens):
                x[b, :, n:] = float("nan")
    wdt = {"f32": torch.float32, "same": dtype, None: None}[weights]
    qw = kw = None
    if weights:
        qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdt).to(DEV).requires_grad_() for _ in range(2))
    kwargs, max_pos = {}, N
    index = torch.cat([torch.arange(n) for n in lens])
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(lens))
    if pos == "offsets":
        offs = torch.randint(0, 100000, (B,), generator=g, dtype=torch.int32)
        kwargs["position_offsets"] = offs.to(DEV)
        position, max_pos = index + offs[seq], 100000 + N
    elif pos == "given":
        p = torch.randint(0, 5000, (T,) if layout == "packed" else (B, N), generator=g, dtype=torch.int32)
        kwargs["positions"] = p.to(DEV)
        position, max_pos = (p if layout == "packed" else p[seq, index]).long(), 5000
    else:
        position = index
    table = fm().RotaryTable(max_pos, R, base=base, pairs=pairs, device=DEV) if R else None
    if not R:
        kwargs = {}
    q.requires_grad_(), k.requires_grad_()
    oq, ok = fm().qk_norm_rope(q, k, table, q_weight=qw, k_weight=kw, normalize=normalize, eps=eps, q_meta=meta, **kwargs)
    leaves = [q, k] + ([qw, kw] if weights else [])
    grads = torch.autograd.grad([oq, ok], leaves, [gq, gk])
    with torch.no_grad():
        same = fm().qk_norm_rope(q, k, table, q_weight=qw, k_weight=kw, normalize=normalize, eps=eps, q_meta=meta, **kwargs)
    assert torch.equal(same[0], oq) and torch.equal(same[1], ok)
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))

    def rows(x):  # [heads, T, D]
        if layout == "packed":
            return x.detach()
        return torch.cat([x.detach()[b, :, :n] for b, n in enumerate(lens)], 1)

    def zeros_outside(x, what):
        if layout == "padded":
            for b, n in enumerate(lens):
                assert not x.detach()[b, :, n:].any(), what

    for i, (x, w, gr, out) in enumerate(((q, qw, gq, oq), (k, kw, gk, ok))):
        y, ym, dx, dxm, dw, dwm = reference(rows(x), w.detach() if w is not None else None, rows(gr),
                                            position.to(DEV), R, pairs, base, eps, normalize)
        assert out.is_contiguous()
        assert_near(rows(out), y, ym, f"out {i}")
        assert_near(rows(grads[i]), dx, dxm, f"dx {i}")
        zeros_outside(out, "out")
        zeros_outside(grads[i], "dx")
        if weights:
            assert_near(grads[2 + i], dw, dwm, f"dw {i}")
    return oq, ok, grads


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("D,R", [(16, 16), (32, 16), (64, 64), (64, 48), (128, 128), (128, 32), (256, 256), (256, 112)])
def test_head_dims(dtype, pairs, D, R):
    check("dense", dtype, 2, 3, 2, 37, D, R, pairs)


@pytest.mark.parametrize("layout", ["padded", "packed"])
@pytest.mark.parametrize("pos", ["index", "offsets", "given"])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths_and_positions(layout, pos, D):
    check(layout, BF16, 5, 4, 1, 70, D, D, "half", lens=[70, 0, 1, 33, 64], pos=pos, base=1e6)


@pytest.mark.parametrize("weights", ["f32", "same", None])
@pytest.mark.parametrize("strided", [True, False])
def test_weights_and_strides(weights, strided):
    check("dense", F16, 3, 5, 5, 65, 64, 64, "half", weights=weights, strided=strided, pos="given")


def test_norm_alone_and_rotation_alone():
    check("dense", BF16, 2, 4, 2, 50, 64, 0, "half")
    check("dense", BF16, 2, 4, 2, 50, 64, 64, "half", normalize=False, weights=None)
    check("padded", F16, 2, 4, 2, 50, 128, 64, "interleaved", normalize=False, weights=None, lens=[50, 7])
    check("padded", F16, 2, 4, 2, 50, 128, 64, "interleaved", eps=0.0, lens=[50, 7])


@pytest.mark.parametrize("B,H,HK,N", [(1, 1, 1, 1), (64, 16, 16, 1), (3, 40, 8, 1), (1, 7, 3, 2000), (2, 64, 64, 300)])
def test_shapes_of_the_grid(B, H, HK, N):
    check("dense", BF16, B, H, HK, N, 128, 128, "half", pos="offsets")


def test_same_bits_again():
    a = check("packed", BF16, 4, 8, 4, 700, 64, 64, "half", lens=[700, 3, 500, 650])
    b = check("packed", BF16, 4, 8, 4, 700, 64, 64, "half", lens=[700, 3, 500, 650])
    assert all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


def test_position_outside_the_table_is_reported():
    table = fm().RotaryTable(8, 64, device=DEV)
    x = torch.randn((1, 2, 9, 64), device=DEV).to(BF16)
    fm().qk_norm_rope(x, x, table)
    with pytest.raises(RuntimeError, match="position"):
        fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))
    fm().qk_norm_rope(x[:, :, :8], x[:, :, :8], table)
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))


def test_gradient_against_differences():
    """The directional derivative of a weighted sum of the outputs, taken of the
    64-bit definition by central differences, meets the kernel's gradient:
    differences are off by h^2 (1e-8 here), the gradient by its 16-bit rounding."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn((1, 2, 9, 32), generator=g).to(F16).to(DEV)
    gy = torch.randn((1, 2, 9, 32), generator=g).to(F16).to(DEV)
    direction = torch.randn((2, 9, 32), generator=g, dtype=torch.float64).to(DEV)
    table = fm().RotaryTable(9, 32, device=DEV)
    xq = x.clone().requires_grad_()
    oq, _ = fm().qk_norm_rope(xq, x, table)
    (dx,) = torch.autograd.grad(oq, [xq], gy)
    pos = torch.arange(9, device=DEV)

    def loss(v):
        return (reference(v, None, gy[0], pos, 32, "half", 10000.0, 1e-6)[0] * gy[0].double()).sum()

    h = 1e-4
    slope = (loss(x[0].double() + h * direction) - loss(x[0].double() - h * direction)) / (2 * h)
    got = (dx[0].double() * direction).sum()
    bound = (2.0 ** -11 * dx[0].double().abs() * direction.abs()).sum() + 2.0 ** -18 * direction.abs().sum() * 8 + 1e-4
    assert abs(got - slope) <= bound
