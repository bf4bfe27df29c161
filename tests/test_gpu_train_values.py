"""GPU tests of attention's gradients for values far from 1: large scores, scales
at the ends of float16's range, small gradients."""

import pytest
import torch

import train_ref
from flash_mlm import _lib
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


# --------------------------------------------------------------- small and large gradients, float16


def rms(x):
    return x.double().square().mean().sqrt().item()


def against_once_rounded(q, k, v, do, scale, got):
    """Errors of dq, dk, dv (one head) as multiples of those of gradients that are rounded only at the end."""
    a, b, c, d = (x.double() for x in (q, k, v, do))
    p = torch.softmax(scale * a @ b.T, 1)
    ds = p * (d @ c.T - (d * (p @ c)).sum(1, keepdim=True))
    want = (scale * ds @ b, scale * ds.T @ a, p.T @ d)
    return [rms(x.double() - w) / rms(w.to(F16).double() - w) for x, w in zip(got, want)]


# Many terms of either sign: rounding each by up to half a step moves their sum as much as rounding the
# sum does (a factor of sqrt(2) with both), if none is subnormal; P v's rounding in delta and the 32-bit part add little.
ONCE = 1.6


@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("n", [512, 4096])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
def test_float16_small_gradients(D, n, size):
    g = torch.Generator().manual_seed(7)
    q, k, v, do = (torch.randn((1, 1, n, D), generator=g) for _ in range(4))
    q, k, v, do = (x.to(F16).to(DEV) for x in (q, k, v, do * size))
    got = gradients(q, k, v, do, D ** -0.5)
    fm().check_device_errors(device())
    ratios = against_once_rounded(*(x[0, 0] for x in (q, k, v, do)), D ** -0.5, [got[x][0, 0] for x in ("dq", "dk", "dv")])
    assert max(ratios) <= ONCE, ratios


def test_float16_small_gradients_of_long_rows():
    g = torch.Generator(DEV).manual_seed(8)
    q, k, v, do = (torch.randn((1, 1, 16384, 64), generator=g, device=DEV) for _ in range(4))
    q, k, v, do = (x.to(F16) for x in (q, k, v, do * 1e-3))
    got = gradients(q, k, v, do, 0.125)
    fm().check_device_errors(device())
    ratios = against_once_rounded(*(x[0, 0] for x in (q, k, v, do)), 0.125, [got[x][0, 0] for x in ("dq", "dk", "dv")])
    assert max(ratios) <= ONCE, ratios


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_float16_small_gradients_of_packed_sequences(causal, shared):
    """Sequences whose gradients lie 10^4 apart, with contexts: each as near as by itself (dq, dk, dv of a sequence
    and of its context; under causal_query_seq_attn and a shared context the largest one leads)."""
    g = torch.Generator().manual_seed(9)
    lens, ctx = [700, 900], [1500] if shared else [1500, 1100]
    T, D = sum(lens), 64
    q, k, v, do = (torch.randn((1, T, D), generator=g) for _ in range(4))
    kc, vc = (torch.randn((1, sum(ctx), D), generator=g) for _ in range(2))
    do[:, :700] *= 1e-4
    q, k, v, do, kc, vc = (x.to(F16).to(DEV) for x in (q, k, v, do, kc, vc))
    kw = dict(q_meta=meta_of(lens, 900), context_k=kc, context_v=vc, context_meta=meta_of(ctx, max(ctx)),
              causal_query_seq_attn=causal)
    out, lse = fm().flash_attn_mlm_fwd(q, k, v, 0.125, **kw)
    got = fm().flash_attn_mlm_bwd(do, q, k, v, out, lse, 0.125, **kw)
    fm().check_device_errors(device())
    want = [torch.zeros(x.shape, dtype=torch.float64, device=DEV) for x in got]
    for b, (s, e) in enumerate(((0, 700), (700, 1600))):
        c0, c1 = (0, 1500) if shared or b == 0 else (1500, 2600)
        m0 = 0 if causal else s
        keys = torch.cat([kc[0, c0:c1], k[0, m0:e]]).double()
        vals = torch.cat([vc[0, c0:c1], v[0, m0:e]]).double()
        a, d = q[0, s:e].double(), do[0, s:e].double()
        p = torch.softmax(0.125 * a @ keys.T, 1)
        ds = p * (d @ vals.T - (d * (p @ vals)).sum(1, keepdim=True))
        want[0][0, s:e] = 0.125 * ds @ keys
        for i, x in ((1, 0.125 * ds.T @ a), (2, p.T @ d)):
            want[i + 2][0, c0:c1] += x[: c1 - c0]
            want[i][0, m0:e] += x[c1 - c0:]
    parts = [(i, slice(s, e)) for i in range(3) for s, e in ((0, 700), (700, 1600))] + [(i, slice(None)) for i in (3, 4)]
    if not shared:
        parts += [(i, slice(*r)) for i in (3, 4) for r in ((0, 1500), (1500, 2600))]
    for i, r in parts:
        x, w = got[i][0, r].double(), want[i][0, r]
        assert rms(x - w) <= ONCE * rms(w.to(F16).double() - w), (i, r)


def test_float16_rows_of_different_gradients():
    """Rows of one tile whose gradients lie up to 10^5 apart: dq of each is as near as its own size asks for.

    At scale 1 (scores of deviation 8) many rows have nearly one key, and dS is what P (dP - delta) leaves of two
    equal numbers: there the rounding of O inside delta counts, of which rounding the sum knows nothing.  O is off
    by at most half a step of itself and of each P (u (|O| + P |v|)), delta by e = |dO| . that, and dq by exactly
    e P k; so a row may be off by ONCE times its rounding and by e |P k|, both of them in the row's own size."""
    g = torch.Generator().manual_seed(10)
    n, D = 2048, 64
    q, k, v, do = (torch.randn((1, 1, n, D), generator=g) for _ in range(4))
    do *= 10.0 ** (-5 * torch.rand((1, 1, n, 1), generator=g))
    q, k, v, do = (x.to(F16).to(DEV) for x in (q, k, v, do))
    dq = gradients(q, k, v, do, 1.0)["dq"][0, 0].double()
    fm().check_device_errors(device())
    a, b, c, d = (x[0, 0].double() for x in (q, k, v, do))
    p = torch.softmax(a @ b.T, 1)
    o = p @ c
    w = (p * (d @ c.T - (d * o).sum(1, keepdim=True))) @ b
    e = 2.0**-11 * (d.abs() * (o.abs() + p @ c.abs())).sum(1)
    # (2^-24, half a step at the smallest: rows whose gradient is 0 in float16)
    once = (w.to(F16).double() - w).square().mean(1).sqrt() + 2.0**-24
    share = (dq - w).square().mean(1).sqrt() / (ONCE * once + e * (p @ b).square().mean(1).sqrt())
    assert share.square().mean().sqrt() <= 1.0, share.max()


@pytest.mark.parametrize("layout", ["dense", "padded"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_float16_products_past_its_range(D, layout):
    """dout of 2000, v of 4: dout v^T passes 65504 in many places, the gradients do not."""
    g = torch.Generator().manual_seed(11)
    lens = [150, 150] if layout == "dense" else [150, 77]
    q, k, v, do = (rand(g, (2, 2, 150, D), F16) for _ in range(4))
    v, do = v * 4, do * 2000
    val, bnd = batch_reference(q, k, v, do, 0.02, lens)
    assert max(val[x].abs().max() for x in ("dq", "dk", "dv")) < 60000 and (do.float() @ v.float().transpose(2, 3)).abs().max() > 65504
    got = gradients(q, k, v, do, 0.02, q_meta=None if layout == "dense" else meta_of(lens, 150))
    fm().check_device_errors(device())
    for name, x in got.items():
        assert_within(x, val[name], bnd[name], name)


@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0), (1e-4, 1.0, 1e3), (1.0, 1e4, 1e-4), (1e4, 1e-4, 1e-3)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ctx", [[300], [17, 0, 256, 129]])
def test_float16_sizes_of_values_context_and_gradients(sizes, causal, ctx):
    """v, the context's v and dout of very different sizes; short sequences, whose delta is summed anew, among them."""
    g = torch.Generator().manual_seed(12)
    lens, D = [180, 3, 0, 40], 64
    q, k, v, do = (rand(g, (4, h, 180, D), F16) for h in (4, 2, 2, 4))
    kc, vc = (rand(g, (2, sum(ctx), D), F16) for _ in range(2))
    v, vc, do = ((x.float() * s).to(F16) for x, s in zip((v, vc, do), sizes))
    val, bnd = batch_reference(q, k, v, do, 0.125, lens, kc, vc, ctx, causal)
    leaves = [x.requires_grad_() for x in (q, k, v, kc, vc)]
    out = fm().flash_attn_mlm_train(*leaves[:3], 0.125, meta_of(lens, 180), kc, vc, meta_of(ctx, max(ctx)), causal)
    grads = torch.autograd.grad(out, leaves, do)
    fm().check_device_errors(device())
    for name, x in zip(("o", "dq", "dk", "dv", "dkc", "dvc"), (out, *grads)):
        assert_within(x, val[name], bnd[name], name)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layout", ["padded", "packed"])
def test_float16_other_sequences_and_padding_leave_no_trace(D, layout):
    """The results of two sequences and their contexts, bit for bit, whatever the one between them, its context
    and the padding hold."""
    g = torch.Generator().manual_seed(13)
    lens, ctx, N = [100, 130, 40], [60, 90, 33], 150
    x = [rand(g, (3, 2, N, D), F16) for _ in range(4)]
    x[3] *= 1e-4
    xc = [rand(g, (2, sum(ctx), D), F16) for _ in range(2)]
    meta, cmeta = meta_of(lens, N), meta_of(ctx, 90)

    def run(x, xc):
        if layout == "padded":
            got = gradients(*x, 0.125, q_meta=meta)
            return [t[b, :, :n] for t in got.values() for b, n in ((0, 100), (2, 40))]
        x = [torch.cat([t[b, :, :n] for b, n in enumerate(lens)], 1).contiguous() for t in x]
        kw = dict(q_meta=meta, context_k=xc[0], context_v=xc[1], context_meta=cmeta)
        out, lse = fm().flash_attn_mlm_fwd(*x[:3], 0.125, **kw)
        grads = fm().flash_attn_mlm_bwd(x[3], *x[:3], out, lse, 0.125, **kw)
        return [t[:, r] for t in (out, *grads[:3]) for r in (slice(0, 100), slice(230, 270))] + \
               [t[:, r] for t in grads[3:] for r in (slice(0, 60), slice(150, 183))]

    want = run(x, xc)
    for what in (float("nan"), float("inf"), 65504.0, 0.0):
        bad, badc = [t.clone() for t in x], [t.clone() for t in xc]
        for t in bad:
            t[1] = what
            for b, n in enumerate(lens):
                t[b, :, n:] = what
        for t in badc:
            t[:, 60:150] = what
        assert all(torch.equal(a, b) for a, b in zip(run(bad, badc), want)), what
    _lib.error_word(device()).zero_()  # (scores of 65504 rows may be reported, which is another test's)


def test_float16_zero_gradients_and_values():
    g = torch.Generator().manual_seed(14)
    q, k, v, do = (rand(g, (1, 2, 200, 64), F16) for _ in range(4))
    for a, b in ((v, torch.zeros_like(do)), (torch.zeros_like(v), do)):
        got = gradients(q, k, a, b, 0.125)
        assert not got["dq"].any() and not got["dk"].any()
        assert bool(got["dv"].any()) == bool(b.any())
    fm().check_device_errors(device())


@pytest.mark.parametrize("n", [100, 512, 3000])
@pytest.mark.parametrize("size", [1.0, 1e-2])
def test_float16_large_values_that_nothing_attends_to(n, size):
    """One row of v near float16's end whose key no query takes (scores of -100): the gradients of the others
    are as near as without it (dS of size 1, of 1e-2 over so few keys, is in float16's normal range as it is)."""
    g = torch.Generator().manual_seed(15)
    q, k, v, do = (torch.randn((1, 1, n, 64), generator=g) for _ in range(4))
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[0, 0, 7, 0], v[0, 0, 7] = -200.0, 60000.0 * torch.sign(v[0, 0, 7])
    q, k, v, do = (x.to(F16).to(DEV) for x in (q, k, v, do * size))
    got = gradients(q, k, v, do, 0.125)
    fm().check_device_errors(device())
    ratios = against_once_rounded(*(x[0, 0] for x in (q, k, v, do)), 0.125, [got[x][0, 0] for x in ("dq", "dk", "dv")])
    # (1e-2 over 3000 keys: dS of 1e-2 / 3000 lies 2 bits below the normal range, where a step is 4 times as large)
    assert max(ratios) <= (4 * ONCE if n == 3000 and size < 1 else ONCE), ratios
