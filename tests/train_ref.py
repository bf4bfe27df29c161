"""64-bit attention with its gradients, one (sequence, head) at a time, and the
error bounds that 16-bit tensor-core operands imply.

Bounds, with u half a step of the 16-bit type relative to the value (bf16 2^-8, f16 2^-11),
and r = 2^-14 for everything held in 32 bits
(scores of magnitude up to a hundred in float32, their exponentials, sums over
head_dim and over keys):

* O = P v: P is rounded once (u) and O once (u):  |err| <= (u + r) P|v| + u |O|
* delta = dO . O with the rounded O:  |err| <= E = sum_d |dO| ((2u + r) P|v|)
* dV = P^T dO:  |err| <= (u + r) P^T |dO| + u |dV|
* dS = P (dP - delta), rounded once:
      |err| <= e_dS = u |dS| + P E + r (|dS| + P |dO||v|^T) + t
  where t is float16's smallest half step (2^-25), 0 for bfloat16
* dQ = scale dS k:  |err| <= scale e_dS |k| + u |dQ|;  dK alike with e_dS^T |q|
* where P and dS are the sum of two 16-bit numbers, u^2 stands for the u of their
  rounding (the second number is rounded, to u of at most u of the whole);
* every float16 output may also lose t to its own subnormals.
"""

import torch

R32 = 2.0 ** -14


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def attention_with_gradients(q, k, v, do, scale, dtype, exact_delta=False, two_parts=False):
    """q, do [n, D], k, v [m, D] (float64) -> (values, bounds): dicts of o, lse, dq, dk, dv.
    ``exact_delta``: delta is summed from P dP in 32 bits (rows of few keys), E = 0.  ``two_parts``: P and dS in two 16-bit numbers (gradients of few terms)."""
    u, t = unit(dtype), tiny(dtype)
    up = u * u if two_parts else u
    s = scale * (q @ k.T)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    o = p @ v
    dp = do @ v.T
    ds = p * (dp - (do * o).sum(1, keepdim=True))
    pv = p @ v.abs()
    err_delta = (do.abs() * ((2 * u + R32) * pv)).sum(1, keepdim=True) * (0.0 if exact_delta else 1.0)
    e_ds = up * ds.abs() + p * err_delta + R32 * (ds.abs() + p * (do.abs() @ v.abs().T)) + t
    a = abs(scale)
    val = dict(o=o, lse=lse, dq=scale * ds @ k, dk=scale * ds.T @ q, dv=p.T @ do)
    bnd = dict(o=(u + R32) * pv + u * o.abs() + t, lse=R32 * (1 + lse.abs()),
               dq=a * e_ds @ k.abs() + u * val["dq"].abs() + t, dk=a * e_ds.T @ q.abs() + u * val["dk"].abs() + t,
               dv=(up + R32) * p.T @ do.abs() + u * val["dv"].abs() + t)
    return val, bnd


def batch_reference(q, k, v, do, scale, lens, kc=None, vc=None, ctx_lens=None, causal=False,
                    exact_delta=False, two_parts=False):
    """Padded [B, H, N, D] inputs (context [HK, Tc, D]) -> (values, bounds) shaped like
    out (o), lse, dq, dk, dv, dkc, dvc; a shared head's or context's gradients are summed."""
    dtype, (B, H, N, D), HK = q.dtype, q.shape, k.shape[1]
    G = H // HK
    f = [x.detach().double() for x in (q, k, v, do)]
    z = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    val = dict(o=z(q), lse=z(q[..., 0]), dq=z(q), dk=z(k), dv=z(v))
    if kc is not None:
        val.update(dkc=z(kc), dvc=z(vc))
    bnd = {n: x.clone() for n, x in val.items()}
    off = [0]
    for n in ctx_lens or []:
        off.append(off[-1] + n)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        prev = range(b + 1) if causal else [b]
        for h in range(H):
            hk = h // G
            parts = []  # (kind, index, rows) of the keys, in order
            ks, vs = [], []
            if kc is not None:
                c = 0 if len(ctx_lens) == 1 else b
                ks.append(kc[hk, off[c]:off[c + 1]].double())
                vs.append(vc[hk, off[c]:off[c + 1]].double())
                parts.append(("c", (hk, slice(off[c], off[c + 1])), ks[-1].shape[0]))
            for b2 in prev:
                ks.append(f[1][b2, hk, :lens[b2]])
                vs.append(f[2][b2, hk, :lens[b2]])
                parts.append(("m", (b2, hk, slice(0, lens[b2])), lens[b2]))
            w, e = attention_with_gradients(f[0][b, h, :n], torch.cat(ks), torch.cat(vs), f[3][b, h, :n], scale, dtype,
                                            exact_delta, two_parts)
            for dst, src in ((val, w), (bnd, e)):
                dst["o"][b, h, :n] = src["o"]
                dst["lse"][b, h, :n] = src["lse"]
                dst["dq"][b, h, :n] = src["dq"]
                r = 0
                for kind, idx, m in parts:
                    suffix = "c" if kind == "c" else ""
                    dst["dk" + suffix][idx] += src["dk"][r:r + m]
                    dst["dv" + suffix][idx] += src["dv"][r:r + m]
                    r += m
    return val, bnd
