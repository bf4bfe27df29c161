"""The operators of a masked-LM attention layer's training step, as workloads.

Two operators, each in a plain form (``own`` false: elementary torch
operations in 32 bits) and through this package's public calls (``own`` true):

* ``attention``: bidirectional attention with its backward pass
  (``flash_mlm.flash_attn_mlm_train``) over dense, padded and packed batches,
  with shared or per-sequence context keys, the causal-by-sequence prefix and
  grouped heads;
* ``rope``: the per-head norm of queries and keys with the position rotation
  in the same pass (``flash_mlm.qk_norm_rope``), forward alone as serving runs
  it, and with its backward pass.
"""

import math
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def _package():
    """This repository's package (the tools run from the repository's root)."""
    if "flash-mlm_b200" not in sys.path:
        sys.path.insert(0, "flash-mlm_b200")
    import flash_mlm

    return flash_mlm


# --------------------------------------------------------------------------- cases


def _attn(name, layout, dtype, B, H, HK, N, D, lo, hi, lens=0, ctx="none", ctx_lo=0, ctx_hi=0, causal=False):
    case = dict(op="attention", layout=layout, dtype=dtype, B=B, H=H, HK=HK, N=N, D=D, lo=lo, hi=hi, lens=lens,
                ctx=ctx, ctx_lo=ctx_lo, ctx_hi=ctx_hi, causal=causal)
    if name:
        case["name"] = name
    return case


def _rope(name, layout, dtype, B, H, HK, N, D, R, pairs, lo, hi, lens=0, train=True, weights="f32", far=0,
          base=10000.0):
    case = dict(op="rope", layout=layout, dtype=dtype, B=B, H=H, HK=HK, N=N, D=D, R=R, pairs=pairs, lo=lo, hi=hi,
                lens=lens, train=train, weights=weights, far=far, base=base)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the smallest dense batch of this repository's benchmark: a step bound by latency
        _attn("attn_dense_small_f16", "dense", "f16", 2, 8, 8, 128, 64, 128, 128),
        # a packed batch of varying lengths over one shared 1024-token context (the benchmark's headline shapes)
        _attn("attn_packed_shared_ctx_bf16", "packed", "bf16", 32, 16, 16, 512, 64, 64, 512, lens=1, ctx="shared",
              ctx_lo=1024, ctx_hi=1024),
        # a padded batch as a data loader hands it over, head_dim 128
        _attn("attn_padded_d128_bf16", "padded", "bf16", 32, 16, 16, 512, 128, 256, 512, lens=2),
        # every sequence also sees its own context and all earlier sequences
        _attn("attn_packed_causal_ctx_f16", "packed", "f16", 64, 12, 12, 256, 64, 32, 256, lens=3, ctx="each",
              ctx_lo=256, ctx_hi=2048, causal=True),
        # four query heads to a key head, odd lengths, an empty sequence and single tokens among them
        _attn("attn_padded_grouped_odd_f16", "padded", "f16", 9, 12, 3, 777, 32, 0, 777, lens=4),
        # long documents, head_dim 128: the largest
        _attn("attn_dense_long_bf16", "dense", "bf16", 1, 16, 16, 8192, 128, 8192, 8192),
        # serving: one new token of each of 64 requests, far along
        _rope("rope_token_bf16", "dense", "bf16", 64, 16, 16, 1, 128, 128, "half", 1, 1, train=False, far=131000,
              base=1000000.0),
        # serving: a packed prefill
        _rope("rope_packed_prefill_bf16", "packed", "bf16", 32, 16, 16, 512, 64, 64, "half", 64, 512, lens=1,
              train=False),
        # training, padded, a part of each head rotated, neighbouring pairs, 16-bit weights
        _rope("rope_padded_train_f16", "padded", "f16", 24, 12, 12, 1001, 64, 32, "interleaved", 1, 1001, lens=5,
              weights="same"),
        # training on long sequences with grouped heads: the largest
        _rope("rope_dense_train_bf16", "dense", "bf16", 16, 32, 8, 4096, 128, 128, "half", 4096, 4096),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges (never more work than the largest listed one)."""
    if rng.random() < 0.55:
        limit = max(work(c)["flops"] for c in listed() if c["op"] == "attention")
        while True:
            layout = rng.choice(["dense", "padded", "packed"])
            HK = rng.choice([1, 2, 3, 4, 8, 12, 16])
            H = HK * (rng.choice([1, 1, 1, 2, 4]) if HK <= 4 else 1)
            hi = _log_int(rng, 1, 8192)
            lo = hi if layout == "dense" else rng.choice([0, hi // 8, hi // 2])
            ctx, causal = "none", False
            if layout == "packed":
                ctx = rng.choice(["none", "shared", "each"])
                causal = rng.random() < 0.3
            ctx_hi = 0 if ctx == "none" else _log_int(rng, 1, 2048)
            case = _attn("", layout, rng.choice(["f16", "bf16"]), _log_int(rng, 1, 64), H, HK, hi,
                         rng.choice([32, 64, 64, 128, 128]), lo, hi, lens=rng.randrange(1 << 30), ctx=ctx,
                         ctx_lo=0 if ctx == "none" else max(1, ctx_hi // 4), ctx_hi=ctx_hi, causal=causal)
            rows = case["B"] * hi * case["H"]
            # (a batch of lone tokens without context has nothing to learn: every score gradient is zero)
            if max(_lengths(case) + [0]) < 2 and ctx == "none":
                continue
            if work(case)["flops"] <= limit and rows <= 1 << 22 and sum(_lengths(case)) > 0:
                return case
    limit = max(work(c)["bytes"] for c in listed() if c["op"] == "rope")
    while True:
        layout = rng.choice(["dense", "padded", "packed"])
        HK = rng.choice([1, 2, 4, 8, 12, 16])
        H = HK * rng.choice([1, 1, 2, 4])
        D = rng.choice([32, 64, 64, 128, 128])
        hi = _log_int(rng, 1, 4096)
        lo = hi if layout == "dense" else rng.choice([0, hi // 2])
        case = _rope("", layout, rng.choice(["f16", "bf16"]), _log_int(rng, 1, 64), H, HK, hi, D,
                     rng.choice([D, D, D // 2]), rng.choice(["half", "interleaved"]), lo, hi,
                     lens=rng.randrange(1 << 30), train=rng.random() < 0.6, weights=rng.choice(["f32", "same"]),
                     far=rng.choice([0, 0, 100000]) if layout == "dense" else 0, base=rng.choice([10000.0, 1000000.0]))
        if work(case)["bytes"] <= limit and sum(_lengths(case)) > 0:
            return case


def _lengths(case):
    """Sequence lengths (part of the case, not of the seed)."""
    r = random.Random(case["lens"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def _ctx_lengths(case):
    if case["ctx"] == "none":
        return []
    r = random.Random(case["lens"] + 1)
    return [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(1 if case["ctx"] == "shared" else case["B"])]


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def work(case):
    lens = _lengths(case)
    T = sum(lens)
    H, HK, D = case["H"], case["HK"], case["D"]
    if case["op"] == "rope":
        rows = T * (H + HK)
        passes = 5 if case["train"] else 2  # forward: x, y; backward: x, dy, dx
        return {"bytes": 2 * D * rows * passes, "flops": (30 if case["train"] else 8) * D * rows}
    ctx = _ctx_lengths(case)
    pairs = 0
    before = 0
    for b, n in enumerate(lens):
        keys = (before if case["causal"] else 0) + n
        if ctx:
            keys += ctx[0] if case["ctx"] == "shared" else ctx[b]
        pairs += n * keys
        before += n
    # q, dO, O, dq over query heads; k, v, dk, dv over key heads (and the context's)
    moved = 4 * H * T + 4 * HK * (T + sum(ctx))
    # two products forward, five backward (scores again, dP, dV, dQ, dK), 2 D flops a pair each
    return {"bytes": 2 * D * moved, "flops": 14 * D * H * pairs}


# --------------------------------------------------------------------------- inputs


def _rand(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    lens = _lengths(case)
    B, H, HK, N, D, T = case["B"], case["H"], case["HK"], case["N"], case["D"], sum(lens)
    st = {"case": case, "lens": lens, "cu": _offsets(lens)}

    def fused(heads):
        """[.., heads, .., D] view of a projection's output, the heads of a token side by side."""
        if case["layout"] == "packed":
            return _rand(g, (T, heads, D), dt).transpose(0, 1)
        return _rand(g, (B, N, heads, D), dt).transpose(1, 2)

    if case["op"] == "rope":
        st["q"], st["k"] = fused(H), fused(HK)
        wdt = torch.float32 if case["weights"] == "f32" else dt
        st["qw"] = (1.0 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(wdt)
        st["kw"] = (1.0 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(wdt)
        st["offs"] = None
        if case["far"]:
            st["offs"] = torch.randint(0, case["far"], (B,), generator=g, device=DEV, dtype=torch.int32)
        if case["train"]:
            packed = case["layout"] == "packed"
            st["dq"] = _rand(g, (H, T, D) if packed else (B, H, N, D), dt)
            st["dk"] = _rand(g, (HK, T, D) if packed else (B, HK, N, D), dt)
        leaves = ("q", "k", "qw", "kw")
    else:
        shape = (lambda h: (h, T, D)) if case["layout"] == "packed" else (lambda h: (B, h, N, D))
        st["q"], st["k"], st["v"] = (_rand(g, shape(h), dt) for h in (H, HK, HK))
        st["do"] = _rand(g, shape(H), dt)
        st["scale"] = D ** -0.5
        cl = _ctx_lengths(case)
        st["ctx_lens"], st["ctx_cu"] = cl, _offsets(cl)
        leaves = ("q", "k", "v")
        if cl:
            st["kc"], st["vc"] = (_rand(g, (HK, sum(cl), D), dt) for _ in range(2))
            leaves += ("kc", "vc")
    if own:
        fm = _package()
        st["leaves"] = leaves
        if case["op"] == "attention" or case["train"]:
            for n in leaves:
                st[n].requires_grad_()
        st["meta"] = st["ctx_meta"] = st["table"] = None
        if case["layout"] != "dense":
            st["meta"] = fm.build_pack_metadata(torch.tensor(lens, dtype=torch.int32, device=DEV), N, 64)
        if case["op"] == "rope":
            st["table"] = fm.RotaryTable(case["far"] + N, case["R"], base=case["base"], pairs=case["pairs"], device=DEV)
        elif st["ctx_lens"]:
            st["ctx_meta"] = fm.build_pack_metadata(torch.tensor(st["ctx_lens"], dtype=torch.int32, device=DEV),
                                                    max(st["ctx_lens"]), 64)
    return st


# --------------------------------------------------------------------------- one pass


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    fm, case = _package(), st["case"]
    if case["op"] == "rope":
        q, k = fm.qk_norm_rope(st["q"], st["k"], st["table"], q_weight=st["qw"], k_weight=st["kw"], eps=EPS,
                               q_meta=st["meta"], position_offsets=st["offs"])
        if not case["train"]:
            return [q, k]
        grads = torch.autograd.grad([q, k], [st[n] for n in st["leaves"]], [st["dq"], st["dk"]])
        return [q.detach(), k.detach(), *grads]
    kw = {}
    if st["ctx_meta"] is not None:
        kw = dict(context_k=st["kc"], context_v=st["vc"], context_meta=st["ctx_meta"])
    out = fm.flash_attn_mlm_train(st["q"], st["k"], st["v"], st["scale"], q_meta=st["meta"],
                                  causal_query_seq_attn=case["causal"], **kw)
    grads = torch.autograd.grad(out, [st[n] for n in st["leaves"]], st["do"])
    return [out.detach(), *grads]


def _key_ranges(st, b):
    """(context rows, own rows) that sequence b of a packed batch attends."""
    case, cu, cc = st["case"], st["cu"], st["ctx_cu"]
    c = None
    if st["ctx_lens"]:
        j = 0 if case["ctx"] == "shared" else b
        c = (cc[j], cc[j + 1])
    return c, (0 if case["causal"] else cu[b], cu[b + 1])


def _run_plain(st):
    return _plain_rope(st) if st["case"]["op"] == "rope" else _plain_attention(st)


def _plain_attention(st):
    case, lens, scale = st["case"], st["lens"], st["scale"]
    packed = case["layout"] == "packed"
    G, HK, D = case["H"] // case["HK"], case["HK"], case["D"]
    dt = st["q"].dtype
    acc = {n: torch.zeros(st[n].shape, dtype=torch.float32, device=DEV)
           for n in ("q", "k", "v", "kc", "vc") if n in st}
    out = torch.zeros_like(acc["q"])
    for b, n in enumerate(lens):
        if n == 0:
            continue
        rows = (slice(None), slice(st["cu"][b], st["cu"][b + 1])) if packed else (b, slice(None), slice(0, n))
        c, m = _key_ranges(st, b)
        krows = (slice(None), slice(*m)) if packed else rows
        q, do = st["q"][rows].float(), st["do"][rows].float()
        k, v = st["k"][krows].float(), st["v"][krows].float()
        nc = 0
        if c is not None:
            nc = c[1] - c[0]
            k = torch.cat([st["kc"][:, c[0]:c[1]].float(), k], 1)
            v = torch.cat([st["vc"][:, c[0]:c[1]].float(), v], 1)
        q, do = q.reshape(HK, G * n, D), do.reshape(HK, G * n, D)
        p = q @ k.transpose(1, 2)
        p.mul_(scale)
        p.sub_(p.amax(-1, keepdim=True)).exp_()
        p.div_(p.sum(-1, keepdim=True))
        o = p @ v
        dv = p.transpose(1, 2) @ do
        ds = do @ v.transpose(1, 2)
        ds.sub_((o * do).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        dq = ds @ k
        dk = ds.transpose(1, 2) @ q
        out[rows] = o.reshape(HK * G, n, D)
        acc["q"][rows] = dq.reshape(HK * G, n, D)
        acc["k"][krows] += dk[:, nc:]
        acc["v"][krows] += dv[:, nc:]
        if c is not None:
            acc["kc"][:, c[0]:c[1]] += dk[:, :nc]
            acc["vc"][:, c[0]:c[1]] += dv[:, :nc]
    return [out.to(dt), *(a.to(dt) for a in acc.values())]


def _positions(st):
    """Positions of the batch's rows: [T] packed, else [B, N]."""
    case = st["case"]
    if case["layout"] == "packed":
        return torch.cat([torch.arange(n, device=DEV) for n in st["lens"]])
    pos = torch.arange(case["N"], device=DEV)[None].expand(case["B"], -1)
    return pos if st["offs"] is None else pos + st["offs"][:, None].long()


def _valid(st):
    """[B, 1, N, 1] truth of the rows inside their sequences, or None where every row is."""
    if st["case"]["layout"] != "padded":
        return None
    lens = torch.tensor(st["lens"], device=DEV)
    return (torch.arange(st["case"]["N"], device=DEV)[None] < lens[:, None])[:, None, :, None]


def _plain_rope(st):
    case = st["case"]
    R, half = case["R"], case["pairs"] == "half"
    freq = case["base"] ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    ang = _positions(st).double()[..., None] * freq
    cos, sin = ang.cos().float(), ang.sin().float()
    if case["layout"] != "packed":
        cos, sin = cos[:, None], sin[:, None]
    valid = _valid(st)

    def rotate(x, s):
        x0, x1 = (x[..., :R // 2], x[..., R // 2:R]) if half else (x[..., 0:R:2], x[..., 1:R:2])
        y0, y1 = x0 * cos - x1 * s, x1 * cos + x0 * s
        y = torch.cat([y0, y1], -1) if half else torch.stack([y0, y1], -1).flatten(-2)
        return torch.cat([y, x[..., R:]], -1)

    outs, gx, gw = [], [], []
    for n in ("q", "k"):
        x, w = st[n].float(), st[n + "w"].float()
        if valid is not None:
            x = x * valid
        rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        xh = x * rstd
        outs.append(rotate(xh * w, sin).to(st[n].dtype).contiguous())
        if case["train"]:
            g = st["d" + n].float()
            if valid is not None:
                g = g * valid
            g = rotate(g, -sin)
            gw.append((g * xh).double().sum(tuple(range(g.ndim - 1))).to(st[n + "w"].dtype))
            g = g * w
            gx.append((rstd * (g - xh * (g * xh).mean(-1, keepdim=True))).to(st[n].dtype))
    return [*outs, *gx, *gw]


# --------------------------------------------------------------------------- 64-bit values


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits (gradients by differentiating them)."""
    if case["op"] == "attention" and work(case)["flops"] > 4e12:
        return None
    st = prepare(case, seed)
    return _exact_rope(st) if case["op"] == "rope" else _exact_attention(st)


def _exact_attention(st):
    """Head by head: softmax over one sequence's keys, differentiated as it is defined."""
    case = st["case"]
    packed, G = case["layout"] == "packed", case["H"] // case["HK"]
    names = [n for n in ("q", "k", "v", "kc", "vc") if n in st]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    grads = {n: torch.zeros(st[n].shape, dtype=torch.float64, device=DEV) for n in names}
    for b, n in enumerate(st["lens"]):
        if n == 0:
            continue
        c, m = _key_ranges(st, b)
        for hk in range(case["HK"]):
            if packed:
                kw = {"k": (hk, slice(*m)), "v": (hk, slice(*m))}
            else:
                kw = {"k": (b, hk, slice(0, n)), "v": (b, hk, slice(0, n))}
            if c is not None:
                kw.update(kc=(hk, slice(*c)), vc=(hk, slice(*c)))
            x = {a: st[a][w].detach().double().requires_grad_() for a, w in kw.items()}
            for h in range(hk * G, (hk + 1) * G):
                w = (h, slice(st["cu"][b], st["cu"][b + 1])) if packed else (b, h, slice(0, n))
                with torch.enable_grad():
                    q = st["q"][w].detach().double().requires_grad_()
                    keys = torch.cat([x["kc"], x["k"]]) if c is not None else x["k"]
                    vals = torch.cat([x["vc"], x["v"]]) if c is not None else x["v"]
                    prob = torch.softmax(torch.einsum("id,jd->ij", q, keys) * st["scale"], dim=1)
                    o = torch.einsum("ij,jd->id", prob, vals)
                    gr = torch.autograd.grad(o, [q, *x.values()], st["do"][w].double())
                out[w] = o.detach()
                grads["q"][w] = gr[0]
                for a, ga in zip(x, gr[1:]):
                    grads[a][kw[a]] += ga
    return [out, *(grads[n] for n in names)]


def _exact_rope(st):
    """Pairs as complex numbers, differentiated as they are defined."""
    case = st["case"]
    R = case["R"]
    j = torch.arange(R // 2, device=DEV, dtype=torch.float64)
    turn = torch.exp(-(2.0 * j / R) * math.log(case["base"]))
    theta = _positions(st).double().unsqueeze(-1) * turn
    unit = torch.polar(torch.ones_like(theta), theta)
    if case["layout"] != "packed":
        unit = unit.unsqueeze(1)
    mask = _valid(st)
    outs, gx, gw = [], [], []
    for n in ("q", "k"):
        src = st[n].detach().double()
        if mask is not None:
            src = torch.where(mask, src, torch.zeros_like(src))
        with torch.enable_grad():
            x = src.requires_grad_()
            w = st[n + "w"].detach().double().requires_grad_()
            y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
            pr = y[..., :R]
            pr = (pr.unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["pairs"] == "half"
                  else pr.unflatten(-1, (R // 2, 2)))
            z = torch.view_as_real(torch.view_as_complex(pr.contiguous()) * unit)
            z = (z.transpose(-1, -2) if case["pairs"] == "half" else z).flatten(-2)
            y = torch.cat([z, y[..., R:]], -1)
            if mask is not None:
                y = torch.where(mask, y, torch.zeros_like(y))
            if case["train"]:
                a, bw = torch.autograd.grad(y, [x, w], st["d" + n].double())
                gx.append(a)
                gw.append(bw)
        outs.append(y.detach())
    return [*outs, *gx, *gw]
