"""GPU tests of float16 training attention as programs use it, where dS's power of two is found from what a call
leaves in its workspace: partial gradients, streams at the same time, captured graphs, batches put together anew."""

import pytest
import torch

from test_gpu_train import DEV, F16, fm, meta_of, rand

pytestmark = pytest.mark.gpu


def no_errors():
    fm().check_device_errors(torch.device(DEV, torch.cuda.current_device()))


def batch(seed, lens, ctx, H=4, HK=2, D=64, size=1e-3):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q, do = rand(g, (H, T, D), F16), rand(g, (H, T, D), F16) * size
    k, v = rand(g, (HK, T, D), F16), rand(g, (HK, T, D), F16)
    kw = dict(q_meta=meta_of(lens, max(lens)))
    if ctx:
        kw.update(context_k=rand(g, (HK, sum(ctx), D), F16), context_v=rand(g, (HK, sum(ctx), D), F16),
                  context_meta=meta_of(ctx, max(ctx)))
    return (q, k, v, do), kw


def step(x, kw, **need):
    q, k, v, do = x
    out, lse = fm().flash_attn_mlm_fwd(q, k, v, 0.125, **kw)
    return [out, *fm().flash_attn_mlm_bwd(do, q, k, v, out, lse, 0.125, **kw, **need)]


def same(a, b):
    return all((x is None and y is None) or torch.equal(x, y) for x, y in zip(a, b))


FORMS = [(None, False), (None, True), ([200], False), ([200], True), ([70, 300, 0, 5], False), ([70, 300, 0, 5], True)]


@pytest.mark.parametrize("ctx,causal", FORMS)
@pytest.mark.parametrize("lens", [[300, 20, 129, 1], [2, 3, 1, 4], [0, 700, 64, 0]])
@pytest.mark.parametrize("D", [32, 128, 256])
def test_parts_alone_have_the_same_bits(ctx, causal, lens, D):
    x, kw = batch(1, lens, ctx, D=D)
    kw["causal_query_seq_attn"] = causal
    full = step(x, kw)
    assert same(full, step(x, kw))
    only_q, only_kv = step(x, kw, need_dkv=False), step(x, kw, need_dq=False)
    no_errors()
    assert torch.equal(only_q[1], full[1]) and only_q[2:] == [None] * 4
    assert only_kv[1] is None and same(only_kv[2:], full[2:])


@pytest.mark.parametrize("ctx", [None, "each"])
def test_sequences_alone_have_the_same_bits(ctx):
    """Many short sequences and some long ones, gradients and values of sizes of their own: a sequence's results
    (and its context's) are those of a call of its own."""
    g = torch.Generator().manual_seed(2)
    lens = [int(n) for n in torch.randint(0, 9, (700,), generator=g)] + [400, 0, 129, 128, 7]
    ctxs = [int(n) for n in torch.randint(0, 20, (len(lens),), generator=g)] if ctx else None
    x, kw = batch(3, lens, ctxs, H=4, HK=1)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    for t, low in ((x[2], -3), (x[3], -2)):
        sizes = (10.0 ** (low * torch.rand(len(lens), generator=g)))[seq].to(DEV)
        t.copy_((t.float() * sizes[:, None]).to(F16))
    got = step(x, kw)
    no_errors()
    for b in [0, 1, 2, 350, 698, 699, *range(700, len(lens))]:
        s, c = sum(lens[:b]), sum(ctxs[:b]) if ctx else 0
        if lens[b] == 0:
            continue
        alone_kw = dict(q_meta=meta_of([lens[b]], lens[b]))
        if ctx and ctxs[b]:
            cut = slice(c, c + ctxs[b])
            alone_kw.update(context_k=kw["context_k"][:, cut].contiguous(), context_v=kw["context_v"][:, cut].contiguous(),
                            context_meta=meta_of([ctxs[b]], ctxs[b]))
        alone = step([t[:, s:s + lens[b]].contiguous() for t in x], alone_kw)
        no_errors()
        for i in range(4):
            assert torch.equal(got[i][:, s:s + lens[b]], alone[i]), (b, i)
        for i in (4, 5):
            if alone[i] is not None:
                assert torch.equal(got[i][:, c:c + ctxs[b]], alone[i]), (b, i)


def test_streams_at_the_same_time():
    sets = [batch(10 + i, lens, ctx) for i, (lens, ctx) in enumerate((([500, 3, 260], [300]), ([90] * 40, [64] * 40), ([1000], None)))]
    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    assert all(same(r, want[i]) for i in range(len(sets)) for r in got[i])
    no_errors()


def test_captured_graphs_on_new_values():
    """Two graphs replayed in turn on gradients and values of other sizes than those they were captured with."""
    graphs = []
    for seed, lens, ctx, causal in ((20, [120, 64, 33], [50, 9, 200], False), (21, [300, 5], [128], True)):
        x, kw = batch(seed, lens, ctx)
        kw["causal_query_seq_attn"] = causal
        step(x, kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(x, kw)
        graphs.append((graph, outs, x, kw, lens, ctx))
    for turn, size in enumerate((1.0, 1e-4, 300.0)):
        for i, (graph, outs, x, kw, lens, ctx) in enumerate(graphs):
            new, _ = batch(30 + 2 * turn + i, lens, ctx, size=size)
            for a, b in zip(x, new):
                a.copy_(b)
            x[2].mul_(0.1 ** turn)
            graph.replay()
            want = step(x, kw)
            torch.cuda.synchronize()
            assert same(outs, want), (turn, i)
    no_errors()
