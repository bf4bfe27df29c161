"""GPU tests of the training operators as programs use them: strides, shared
and broadcast inputs, streams, captured graphs, partial gradients, foreign
NaNs, and the operators one after the other."""

import pytest
import torch

from test_gpu_train import BF16, DEV, F16, assert_within, check, fm, meta_of, pack, rand
from train_ref import attention_with_gradients, batch_reference

pytestmark = pytest.mark.gpu


def no_errors():
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))


def inputs(seed, shape, kshape=None, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    kshape = kshape or shape
    return rand(g, shape, dtype), rand(g, kshape, dtype), rand(g, kshape, dtype), rand(g, shape, dtype)


# ----------------------------------------------------------------- how tensors lie


def relaid(x, how):
    """x's values in another storage: a projection's layout, a window of wider rows, unaligned rows."""
    d = x.shape[-1]
    if how == "projection":
        return x.transpose(-2, -3).contiguous().transpose(-2, -3)
    wide = torch.full((*x.shape[:-1], d + 16), 7.0, dtype=x.dtype, device=x.device)
    off = {"window": 8, "unaligned": 3}[how]
    wide[..., off:off + d] = x
    return wide[..., off:off + d]


@pytest.mark.parametrize("how", ["projection", "window", "unaligned"])
@pytest.mark.parametrize("layout", ["dense", "padded", "packed"])
def test_strides(how, layout):
    lens = [150, 150] if layout == "dense" else [150, 61]
    q, k, v, do = inputs(1, (2, 4, 150, 64), (2, 2, 150, 64))
    meta = None if layout == "dense" else meta_of(lens, 150)
    if layout == "packed":
        q, k, v, do = (pack(x, lens) for x in (q, k, v, do))
    plain = [x.contiguous() for x in (q, k, v, do)]
    laid = [relaid(x, how) for x in (q, k, v, do)]
    results = []
    for a, b, c, g in (plain, laid):
        a, b, c = (x.detach().requires_grad_() for x in (a, b, c))
        out = fm().flash_attn_mlm_train(a, b, c, 0.125, q_meta=meta)
        results.append([out.detach(), *torch.autograd.grad(out, [a, b, c], g)])
    no_errors()
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_expanded_keys_and_a_summed_loss():
    """One key head expanded to all query heads by the caller, and the expanded gradient of a sum."""
    q, k, v, _ = inputs(2, (2, 4, 140, 64), (2, 1, 140, 64))
    k1, v1, q1 = (x.clone().requires_grad_() for x in (k, v, q))
    fm().flash_attn_mlm_train(q1, k1.expand(-1, 4, -1, -1), v1.expand(-1, 4, -1, -1), 0.125).sum().backward()
    no_errors()
    val, bnd = batch_reference(q, k, v, torch.ones_like(q), 0.125, [140, 140])
    assert_within(q1.grad, val["dq"], bnd["dq"], "dq")
    # autograd adds the four heads' 16-bit gradients in 16 bits: up to four roundings of sums below the heads' total
    for name, x in (("dk", k1.grad), ("dv", v1.grad)):
        per_head = 4 * 2.0 ** -8 * 4 * val[name].abs().max()
        assert (x.double() - val[name]).abs().max() <= bnd[name].max() + per_head, name


def test_partial_gradients():
    q, k, v, do = inputs(3, (3, 2, 90, 64))
    lens = [90, 0, 33]
    meta, cmeta = meta_of(lens, 90), meta_of([70], 70)
    q, k, v, do = (pack(x, lens) for x in (q, k, v, do))
    g = torch.Generator().manual_seed(4)
    kc, vc = rand(g, (2, 70, 64), BF16), rand(g, (2, 70, 64), BF16)
    kw = dict(context_k=kc, context_v=vc, context_meta=cmeta, q_meta=meta)
    full = None
    for leaves in ("q k v kc vc", "q", "k", "v", "kc", "vc", "q vc"):
        x = {n: t.clone() for n, t in dict(q=q, k=k, v=v, kc=kc, vc=vc).items()}
        for n in leaves.split():
            x[n].requires_grad_()
        kw.update(context_k=x["kc"], context_v=x["vc"])
        out = fm().flash_attn_mlm_train(x["q"], x["k"], x["v"], 0.125, **kw)
        grads = dict(zip(leaves.split(), torch.autograd.grad(out, [x[n] for n in leaves.split()], do)))
        full = full or grads
        assert all(torch.equal(grads[n], full[n]) for n in grads), leaves
    out, lse = fm().flash_attn_mlm_fwd(q, k, v, 0.125, **kw)
    got = fm().flash_attn_mlm_bwd(do, q, k, v, out, lse, 0.125, need_dkv=False, **kw)
    assert got[1:] == (None,) * 4 and torch.equal(got[0], full["q"])
    assert fm().flash_attn_mlm_bwd(do, q, k, v, out, lse, 0.125, need_dq=False, need_dkv=False, **kw) == (None,) * 5
    no_errors()


# ----------------------------------------------------------------- values


def test_same_bits_again_and_twice_through_one_graph():
    g = torch.Generator().manual_seed(6)
    lens = [int(x) for x in torch.randint(1, 400, (40,), generator=g)]
    a = check("packed", BF16, 40, 8, 2, 400, 64, lens, ctx=[333])
    b = check("packed", BF16, 40, 8, 2, 400, 64, lens, ctx=[333])
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))
    q, k, v, do = inputs(7, (2, 2, 200, 128))
    q.requires_grad_()
    out = fm().flash_attn_mlm_train(q, k, v, 0.1)
    first = torch.autograd.grad(out, [q], do, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(out, [q], do)[0])


@pytest.mark.parametrize("D", [64, 128])
def test_nan_of_one_sequence_stays_there(D):
    lens = [100, 130, 40]
    q, k, v, do = (pack(x, lens).contiguous() for x in inputs(8, (3, 2, 130, D)))
    bad = [x.clone() for x in (q, k, v, do)]
    for x in bad:
        x[:, 100:230] = float("nan")
        x[:, 115] = float("inf")
    meta = meta_of(lens, 130)
    results = []
    for a, b, c, g in ((q, k, v, do), bad):
        a, b, c = (x.detach().requires_grad_() for x in (a, b, c))
        out = fm().flash_attn_mlm_train(a, b, c, 0.125, q_meta=meta)
        results.append([out.detach(), *torch.autograd.grad(out, [a, b, c], g)])
    no_errors()
    for x, y in zip(*results):
        assert torch.equal(x[:, :100], y[:, :100]) and torch.equal(x[:, 230:], y[:, 230:])
        assert torch.isfinite(y[:, :100]).all()


def test_large_scores():
    """Scores of several hundred: nearly one-hot rows."""
    g = torch.Generator().manual_seed(9)
    q, k, v, do = (rand(g, (1, 2, 300, 64), BF16) for _ in range(4))
    q = (q.float() * 8).to(BF16)
    val, bnd = batch_reference(q, k, v, do, 1.0, [300])
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    out = fm().flash_attn_mlm_train(q, k, v, 1.0)
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, [q, k, v], do)):
        assert_within(got, val[name], bnd[name], name)
    no_errors()


def test_gradient_against_differences():
    """The slope of a weighted sum of the outputs along a random direction, by central
    differences of the 64-bit definition (off by h^2 times third derivatives, far
    below the gradients' 16-bit bounds), meets the kernel's gradients."""
    g = torch.Generator().manual_seed(10)
    q, k, v, do = (rand(g, (1, 1, 70, 32), F16) for _ in range(4))
    dirs = [torch.randn((70, 32), generator=g, dtype=torch.float64).to(DEV) for _ in range(3)]
    x = [t[0, 0].double() for t in (q, k, v)]

    def loss(h):
        a, b, c = (t + h * d for t, d in zip(x, dirs))
        return (torch.softmax(0.2 * a @ b.T, 1) @ c * do[0, 0].double()).sum()

    h = 1e-4
    slope = (loss(h) - loss(-h)) / (2 * h)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(fm().flash_attn_mlm_train(q, k, v, 0.2), leaves, do)
    _, bnd = attention_with_gradients(*x, do[0, 0].double(), 0.2, F16)
    got = sum((gr[0, 0].double() * d).sum() for gr, d in zip(grads, dirs))
    bound = sum((bnd[n] * d.abs()).sum() for n, d in zip(("dq", "dk", "dv"), dirs)) + 1e-5
    assert abs(got - slope) <= bound


def test_empty_batches():
    g = torch.Generator().manual_seed(11)
    for shape, lens in (((0, 2, 5, 64), None), ((2, 2, 0, 64), None), ((2, 2, 5, 64), [0, 0])):
        q, k, v = (rand(g, shape, F16).requires_grad_() for _ in range(3))
        out = fm().flash_attn_mlm_train(q, k, v, 0.125, q_meta=None if lens is None else meta_of(lens, 5))
        assert out.shape == q.shape and not out.any()
        assert all(not x.any() for x in torch.autograd.grad(out, [q, k, v], torch.ones_like(out)))
    # no tokens, but a context: its gradient is zero; no context rows: as without
    q, k, v = (rand(g, (2, 0, 64), F16).requires_grad_() for _ in range(3))
    kc, vc = (rand(g, (2, 9, 64), F16).requires_grad_() for _ in range(2))
    out = fm().flash_attn_mlm_train(q, k, v, 0.125, q_meta=meta_of([0, 0], 4), context_k=kc, context_v=vc,
                                    context_meta=meta_of([9], 9))
    assert all(not x.any() for x in torch.autograd.grad(out, [kc, vc], torch.ones_like(out)))
    q, k, v = (rand(g, (2, 7, 64), F16).requires_grad_() for _ in range(3))
    kc, vc = (rand(g, (2, 0, 64), F16).requires_grad_() for _ in range(2))
    a = fm().flash_attn_mlm_train(q, k, v, 0.125, q_meta=meta_of([4, 3], 4), context_k=kc, context_v=vc,
                                  context_meta=meta_of([0], 1))
    b = fm().flash_attn_mlm_train(q, k, v, 0.125, q_meta=meta_of([4, 3], 4))
    assert torch.equal(a, b)
    assert [x.shape for x in torch.autograd.grad(a, [q, kc], torch.ones_like(a))] == [q.shape, kc.shape]
    no_errors()


def test_second_derivatives_are_refused():
    q, k, v, do = inputs(12, (1, 1, 8, 64))
    q.requires_grad_()
    (dq,) = torch.autograd.grad(fm().flash_attn_mlm_train(q, k, v, 0.1), [q], do, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()


# ----------------------------------------------------------------- streams and graphs


def test_side_stream():
    q, k, v, do = inputs(13, (2, 2, 300, 64))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(fm().flash_attn_mlm_train(q, k, v, 0.125), leaves, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(fm().flash_attn_mlm_train(q, k, v, 0.125), leaves, do)
        table = fm().RotaryTable(300, 64, device=DEV)
        turned = fm().qk_norm_rope(q.detach(), k.detach(), table)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert all(torch.equal(x, y) for x, y in zip(turned, fm().qk_norm_rope(q.detach(), k.detach(), table)))
    no_errors()


def test_captured_graphs():
    """Two captured training steps of different shapes, replayed in turn on new values, while
    an eager graph of the same tensors lives."""
    steps = []
    for seed, lens in ((14, [120, 64, 33]), (15, [300, 5])):
        N, B = max(lens), len(lens)
        meta, table = meta_of(lens, N), fm().RotaryTable(N, 64, device=DEV)
        q, k, v, do = inputs(seed, (B, 4, N, 64), (B, 2, N, 64))
        w = torch.ones(64, device=DEV)

        def step(q=q, k=k, v=v, do=do, meta=meta, table=table, w=w):
            q1, k1 = fm().qk_norm_rope(q, k, table, q_weight=w, k_weight=w, q_meta=meta)
            out, lse = fm().flash_attn_mlm_fwd(q1, k1, v, 0.125, q_meta=meta)
            return [out, *fm().flash_attn_mlm_bwd(do, q1, k1, v, out, lse, 0.125, q_meta=meta)[:3]]

        step()  # first use outside the capture (library set-up, the error word)
        eager = fm().flash_attn_mlm_train(q.clone().requires_grad_(), k, v, 0.125, q_meta=meta)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        steps.append((step, graph, outs, (q, k, v, do), eager))
    for turn in range(2):
        for i, (step, graph, outs, ins, _) in enumerate(steps):
            for x, y in zip(ins, inputs(20 + 2 * turn + i, ins[0].shape, ins[1].shape)):
                x.copy_(y)
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(outs, want)), (turn, i)
    no_errors()


# ----------------------------------------------------------------- the operators together


def test_layer_gradients_reach_projection_and_weights():
    """x -> fused projection -> norm and rotation -> attention -> loss: gradients of the
    projection and the norm weights against the same layer in 64 bits."""
    g = torch.Generator().manual_seed(30)
    B, N, H, D, lens = 3, 70, 2, 64, [70, 9, 41]
    x = rand(g, (B, N, 32), F16)
    proj = (torch.randn((32, 3 * H * D), generator=g) * 0.3).to(F16).to(DEV)
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(DEV)
    do = rand(g, (B, H, N, D), F16)
    meta, table = meta_of(lens, N), fm().RotaryTable(N, D, device=DEV)
    proj.requires_grad_(), w.requires_grad_()
    q, k, v = (x @ proj).view(B, N, 3, H, D).unbind(2)
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    q, k = fm().qk_norm_rope(q, k, table, q_weight=w, k_weight=w, q_meta=meta)
    out = fm().flash_attn_mlm_train(q, k, v, D ** -0.5, q_meta=meta)
    got = torch.autograd.grad(out, [proj, w], do)
    no_errors()

    p64, w64 = (t.detach().double().requires_grad_() for t in (proj, w))
    y = (x.double() @ p64).view(B, N, 3, H, D)
    ang = torch.arange(N, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)

    def prepared(t):
        t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w64
        a, b = t[..., : D // 2], t[..., D // 2:]
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    loss = 0.0
    for b, n in enumerate(lens):
        q1, k1, v1 = prepared(y[b, :, 0])[:n], prepared(y[b, :, 1])[:n], y[b, :n, 2]
        s = torch.einsum("ihd,jhd->hij", q1, k1) * D ** -0.5
        loss = loss + (torch.einsum("hij,jhd->hid", torch.softmax(s, -1), v1) * do[b, :, :n].double()).sum()
    want = torch.autograd.grad(loss, [p64, w64])
    # Six float16 roundings lie between (projection, q and k, P, O, dS and gradients, their product), each
    # 2^-11 of values that enter sums of signed terms: within 6 * 2^-11 of the largest gradient, and twice that in hand.
    for name, a, b in zip(("projection", "norm weight"), got, want):
        assert (a.double() - b).abs().max() <= 12 * 2.0 ** -11 * b.abs().max(), name


def test_serving_reads_what_training_computes():
    """Norm and rotation at offset positions, cache append, packed attention over the cache: the
    training call over the same context gives the same rows."""
    g = torch.Generator().manual_seed(31)
    H, D, ctx, lens, N = 2, 64, [90, 37], [1, 1], 1
    table = fm().RotaryTable(200, D, device=DEV)
    cmeta, meta = meta_of(ctx, 90), meta_of(lens, N)
    kc, vc, qc = (rand(g, (2, H, 90, D), BF16) for _ in range(3))
    q, k, v = (rand(g, (2, H, N, D), BF16) for _ in range(3))
    _, kc = fm().qk_norm_rope(qc, kc, table, q_meta=cmeta)
    offs = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    q, k = fm().qk_norm_rope(q, k, table, position_offsets=offs, q_meta=meta)
    cache = fm().InferenceCache()
    cache.reserve_kv_cache(0, capacity=200, max_entries=4, is_mla=False, num_heads=H, head_dim=D, dtype=BF16,
                           device=torch.device(DEV, torch.cuda.current_device()))
    cache.append_kv_cache(0, kc, vc, cmeta)
    served = fm().flash_attn_mlm_compressed(q, k, v, num_heads=H, q_meta=meta, scale=0.125, inference_cache=cache,
                                            layer_id=0, block_n=64)
    trained = fm().flash_attn_mlm_train(pack(q, lens), pack(k, lens), pack(v, lens), 0.125, q_meta=meta,
                                        context_k=pack(kc, ctx).contiguous(), context_v=pack(vc, ctx).contiguous(),
                                        context_meta=cmeta)
    no_errors()
    assert torch.equal(served.view(H, 2, D), trained)
