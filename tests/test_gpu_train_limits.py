"""GPU tests of the training operators at the ends of their ranges: tensors of
more than 2^31 elements, scales far from 1, two calls at the same time, a
context of many short sequences."""

import pytest
import torch

from test_gpu_train import BF16, DEV, F16, check, fm, meta_of, rand

pytestmark = pytest.mark.gpu


def no_errors():
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))


def normal(shape, dtype=BF16, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=dtype, device=DEV)


def step(q, k, v, do, meta, scale=0.125):
    out, lse = fm().flash_attn_mlm_fwd(q, k, v, scale, q_meta=meta)
    dq, dk, dv, _, _ = fm().flash_attn_mlm_bwd(do, q, k, v, out, lse, scale, q_meta=meta)
    return out, lse, dq, dk, dv


def test_packed_offsets_past_32_bits():
    """72 heads of half a million tokens (2.4e9 elements): the last sequences have the
    results that they have by themselves (tiles begin at a sequence's first row)."""
    H, lens = 72, [4096] * 127 + [3500, 301, 1, 290]
    T, tail = sum(lens), [301, 1, 290]
    n = sum(tail)
    q, do = normal((H, T, 64), seed=1), normal((H, T, 64), seed=2)
    k, v = normal((1, T, 64), seed=3), normal((1, T, 64), seed=4)
    assert q.numel() > 2**31
    short = [256] * (T // 256) + [T % 256]
    meta, rest = meta_of(short, 256), short[-2:]
    m = sum(rest)
    got = step(q, k, v, do, meta)
    alone = step(*(x[:, -m:].contiguous() for x in (q, k, v, do)), meta_of(rest, 256))
    for a, b in zip(got, alone):
        assert torch.equal(a[:, -m:], b)
    del got
    table = fm().RotaryTable(4096, 64, device=DEV)
    w = normal((64,), seed=5)
    turned = fm().qk_norm_rope(q, k, table, q_weight=w, q_meta=meta_of(lens, 4096))
    one = fm().qk_norm_rope(q[:, -n:], k[:, -n:], table, q_weight=w, q_meta=meta_of(tail, 4096))
    assert all(torch.equal(a[:, -n:], b) for a, b in zip(turned, one))
    no_errors()


def test_padded_offsets_past_32_bits():
    """A padded batch of which little is valid: the rows past each sequence are zeros in the
    gradients, and the last sequence's results are those it has by itself."""
    B, H, N, lens = 9, 8, 1 << 19, [5, 0, 1, 130, 5, 5, 5, 2, 300]
    q, do = normal((B, H, N, 64), seed=1), normal((B, H, N, 64), seed=2)
    k, v = normal((B, 1, N, 64), seed=3), normal((B, 1, N, 64), seed=4)
    assert q.numel() > 2**31
    got = step(q, k, v, do, meta_of(lens, N))
    alone = step(*(x[-1:, :, :300].contiguous() for x in (q, k, v, do)), None)
    for i, (a, b) in enumerate(zip(got, alone)):
        assert torch.equal(a[-1, :, :300], b[0]), i
        if i != 1:  # (lse is undefined at padding rows)
            assert not a[-1, :, 300:].any() and not a[3, :, 130:].any() and not a[1].any(), i
    del got, alone
    table = fm().RotaryTable(1024, 64, device=DEV)
    q1, k1 = q.requires_grad_(), k.requires_grad_()
    turned = fm().qk_norm_rope(q1, k1, table, q_meta=meta_of(lens, N))
    dq, dk = torch.autograd.grad(turned, [q1, k1], [do, v])
    qs, ks = (x[-1:, :, :300].detach().clone().requires_grad_() for x in (q, k))
    one = fm().qk_norm_rope(qs, ks, table)
    ones = torch.autograd.grad(one, [qs, ks], [x[-1:, :, :300].contiguous() for x in (do, v)])
    for a, b in zip((*turned, dq, dk), (*one, *ones)):
        assert torch.equal(a[-1:, :, :300], b) and not a[-1, :, 300:].any()
    no_errors()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_of_large_tensors_and_a_small_scale(D):
    """bfloat16 q and k 2^20 times as large and a scale of 2^-40 of the former: powers of two, so
    the same probabilities and dv to the bit, and dq, dk 2^-20 of the former."""
    q, k, v, do = (normal((1, 2, 300, D), seed=s) for s in range(4))
    out, lse, dq, dk, dv = step(q, k, v, do, None)
    out1, lse1, dq1, dk1, dv1 = step(q * 2.0**20, k * 2.0**20, v, do, None, 0.125 * 2.0**-40)
    assert torch.equal(out, out1) and torch.equal(lse, lse1) and torch.equal(dv, dv1)
    assert torch.equal(dq * 2.0**-20, dq1) and torch.equal(dk * 2.0**-20, dk1)
    no_errors()


@pytest.mark.parametrize("dtype,scale", [(F16, 2.0**-20), (F16, 2.0), (BF16, 1e-30), (BF16, -2.0)])
def test_scale_range(dtype, scale):
    check("padded", dtype, 2, 2, 1, 200, 64, [200, 131], scale=scale)


def test_two_streams_at_once():
    """Calls of two streams in flight together, each with its own workspace and counters."""
    sets = [tuple(normal((2, 4, n, 64), seed=10 * n + s) for s in range(4)) for n in (700, 450)]
    want = [step(*x, None) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*sets[i], None))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
    no_errors()


def test_many_short_contexts():
    """More sequences than a warp can look at in one step, with contexts of 0 to 4 keys of their own."""
    g = torch.Generator().manual_seed(3)
    lens = [int(x) for x in torch.randint(0, 4, (1100,), generator=g)]
    ctx = [int(x) for x in torch.randint(0, 5, (1100,), generator=g)]
    H, D = 2, 64
    T, Tc = sum(lens), sum(ctx)
    q, do, k, v = (rand(g, (H, T, D), BF16) for _ in range(4))
    kc, vc = (rand(g, (H, Tc, D), BF16) for _ in range(2))
    meta, cmeta = meta_of(lens, 4), meta_of(ctx, 4)
    out, lse = fm().flash_attn_mlm_fwd(q, k, v, 0.125, meta, kc, vc, cmeta)
    grads = fm().flash_attn_mlm_bwd(do, q, k, v, out, lse, 0.125, meta, kc, vc, cmeta)
    no_errors()
    # every sequence by itself, as a call of its own of the sequences 1000 to 1099
    a, b = sum(lens[:1000]), sum(ctx[:1000])
    part = [x[:, a:].contiguous() for x in (do, q, k, v)]
    cpart = [x[:, b:].contiguous() for x in (kc, vc)]
    m1, c1 = meta_of(lens[1000:], 4), meta_of(ctx[1000:], 4)
    out1, lse1 = fm().flash_attn_mlm_fwd(*part[1:], 0.125, m1, *cpart, c1)
    grads1 = fm().flash_attn_mlm_bwd(*part, out1, lse1, 0.125, m1, *cpart, c1)
    assert torch.equal(out[:, a:], out1) and torch.equal(lse[:, a:], lse1)
    for i, (x, y) in enumerate(zip(grads, grads1)):
        assert torch.equal(x[:, (a if i < 3 else b):], y), i


FEW = [("packed", [2, 3, 1, 20, 2], None, False, 2), ("packed", [2, 3, 1, 20, 2], [5, 1, 0, 40, 3], False, 2),
       ("packed", [4, 1, 0, 7, 9], [13], True, 2), ("packed", [64, 50, 2, 2, 2], None, False, 2),
       ("padded", [64, 30, 0, 1, 7], None, False, 2), ("dense", [64] * 5, None, False, 2), ("dense", [16] * 2, None, False, 1)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout,lens,ctx,causal,HK", FEW)
def test_gradients_of_few_terms(dtype, D, layout, lens, ctx, causal, HK):
    """At most 128 streamed rows to every tile (64 keys; two query heads of 64): P and dS in two 16-bit numbers."""
    N = max(lens) if layout == "dense" else 64
    check(layout, dtype, len(lens), 4 if HK == 2 else 8, HK, N, D, lens, ctx=ctx, causal=causal, exact_delta=True,
          two_parts=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_items_of_few_and_of_many_terms_in_turn(dtype, D):
    """Lengths on both sides of the limits, several items per block: the two forms after one another."""
    g = torch.Generator().manual_seed(9)
    lens = [int(x) for x in torch.randint(0, 3, (60,), generator=g)] + [600, 8, 9, 129, 64, 65, 300] * 3
    order = torch.randperm(len(lens), generator=g).tolist()
    lens = [lens[i] for i in order]
    check("packed", dtype, len(lens), 6, 3, 600, D, lens)
    check("packed", dtype, len(lens), 2, 1, 600, D, lens, ctx=[3])


@pytest.mark.parametrize("how", ["projection", "window", "unaligned"])
def test_padded_with_context_in_other_strides(how):
    """The layout that is packed on the way: q, k, v and the context as a program may hold them,
    and the gradient of a sum (one element, expanded)."""
    from test_gpu_train_use import relaid

    g = torch.Generator().manual_seed(4)
    lens, ctx = [70, 0, 33, 129], [20, 5, 0, 140]
    q, k, v = (rand(g, (4, h, 129, 64), BF16) for h in (4, 2, 2))
    kc, vc = (rand(g, (2, sum(ctx), 64), BF16) for _ in range(2))
    results = []
    for f in (lambda x: x, lambda x: relaid(x, how)):
        leaves = [f(x).detach().requires_grad_() for x in (q, k, v, kc, vc)]
        out = fm().flash_attn_mlm_train(*leaves[:3], 0.125, meta_of(lens, 129), *leaves[3:], meta_of(ctx, 140), True)
        results.append([out.detach(), *torch.autograd.grad(out.sum(), leaves)])
    no_errors()
    assert all(torch.equal(a, b) for a, b in zip(*results))
