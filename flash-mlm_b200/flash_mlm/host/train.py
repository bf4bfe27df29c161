"""Attention for training: the forward pass with its softmax statistics, the
backward pass, and a differentiable call over both.

No counterpart in the reference, whose kernels are forward only (its README
lists the backward pass as planned).  The attention pattern is that of
``flash_attn_mlm`` and ``flash_attn_mlm_compressed``: every query attends to
its context (one shared by the batch, or one per sequence), then to its own
sequence, or with ``causal_query_seq_attn`` to all sequences up to its own.
Here the context keys and values are arguments, since a training step
computes them and wants their gradients.

Three layouts:

* dense: q [B, H, N, D], no ``q_meta``: every token is valid;
* padded: q [B, H, N, D] with ``q_meta``: the first ``lengths[b]`` tokens are valid;
* packed: q [H, T, D] with ``q_meta`` of T tokens (what ``pack_for_kernel`` returns).

k and v may have fewer heads than q (a divisor): query head h attends key head
``h // (H // HK)`` and the gradients of a shared head are summed.  Inputs may
have any strides whose last one is 1; others, and tensors that the TMA unit
cannot address, are copied.  Gradients are deterministic: the same inputs give
the same bits.
"""

from __future__ import annotations

import torch

from flash_mlm import _lib
from flash_mlm.host.cache import PackMetadata
from flash_mlm.host.host_utils import pack_for_kernel, unpack_from_kernel, validate_head_dim_supported


def _tma_ready(x: torch.Tensor) -> torch.Tensor:
    """x itself if TMA can address its rows (16-byte aligned, positive strides), else a contiguous copy."""
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x
    *outer, row, last = x.stride()
    ok = last == 1 and x.data_ptr() % 16 == 0 and row >= x.shape[-1] and row % 8 == 0
    for size, stride in zip(x.shape, outer):
        ok = ok and (size == 1 or (stride > 0 and stride % 8 == 0))
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _view(x: torch.Tensor) -> tuple[int, ...]:
    """[B, H, N, D] or [H, T, D] as the fields of a [batch][heads][rows] view."""
    if x.ndim == 4:
        b, h, n, _ = x.shape
        sb, sh, sn, _ = x.stride()
        return x.data_ptr(), n, h, b, sn, sh, sb
    h, t, d = x.shape
    sh, st, _ = x.stride()
    return x.data_ptr(), t, h, 1, st, sh, h * t * d


def _validate(q, k, v, scale, q_meta, context_k, context_v, context_meta, causal):
    """Shapes, types and devices of a training call; returns the layout code."""
    if q.ndim not in (3, 4) or k.ndim != q.ndim or v.ndim != q.ndim:
        raise ValueError("q/k/v must be rank-4 tensors [B, H, N, D] or packed rank-3 tensors [H, T, D]")
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    qs, ks = q.shape, k.shape
    if qs[-2:] != ks[-2:] or (q.ndim == 4 and qs[0] != ks[0]):
        raise ValueError("q and k may differ in their number of heads only")
    h, hk = qs[-3], ks[-3]
    if hk < 1 or h < 1 or h % hk != 0:
        raise ValueError("the heads of q must be a multiple of the heads of k and v")
    validate_head_dim_supported(qs[-1])
    half = _lib.dtype_code(q.dtype) == _lib.FMLM_DTYPE_F16
    # float16: the backward pass holds lse / scale in float16 numbers, up to 2^31
    if not abs(scale) <= (2.0**20 if half else 2.0**64) or (half and abs(scale) < 2.0**-24):
        raise ValueError("scale must be finite, at most 2^64 in magnitude, for float16 in [2^-24, 2^20]")
    packed = q.ndim == 3
    if packed:
        if q_meta is None:
            raise ValueError("packed q/k/v need q_meta")
        if q_meta.total_tokens != q.shape[1]:
            raise ValueError("packed token count mismatch with PackMetadata")
    elif q_meta is not None and (q_meta.B != q.shape[0] or q_meta.N != q.shape[2]):
        raise ValueError("q_meta shape metadata does not match q/k/v padded shape")
    context = context_k is not None
    if (context_v is not None) != context or (context_meta is not None) != context:
        raise ValueError("context_k, context_v and context_meta must be provided together or all omitted")
    if (context or causal) and q_meta is None:
        raise ValueError("a context and causal_query_seq_attn need q_meta")
    tensors = [q, k, v]
    if context:
        if context_k.shape != (hk, context_meta.total_tokens, qs[-1]) or context_v.shape != context_k.shape:
            raise ValueError("context_k and context_v must be [heads of k, context_meta.total_tokens, D]")
        if context_meta.B not in (1, q_meta.B):
            raise ValueError("context_meta must describe one context, or one for every sequence")
        tensors += [context_k, context_v]
    dtype, device = q.dtype, q.device
    for x in tensors:
        if x.dtype != dtype:
            raise ValueError("q, k, v and the context must have the same dtype")
        if x.device != device:
            raise ValueError("q, k, v and the context must be on the same device")
    for m in (q_meta, context_meta):
        if m is not None:
            cu = m.cu_seqlens
            if cu.device != device:
                raise ValueError("q_meta and context_meta must be on q's device")
            if cu.dtype != torch.int32 or not cu.is_contiguous() or cu.numel() != m.B + 1:
                raise ValueError("cu_seqlens must be contiguous int32 of B + 1 elements")
    if not q.is_cuda:
        raise ValueError("All tensors must be CUDA tensors")
    if packed:
        return _lib.FMLM_BWD_PACKED
    return _lib.FMLM_BWD_DENSE if q_meta is None else _lib.FMLM_BWD_PADDED


def _require_packed(q, context_k, causal):
    if q.ndim != 3 and (context_k is not None or causal):
        raise ValueError("a context and causal_query_seq_attn need packed q/k/v [H, T, D] here "
                         "(pack_for_kernel packs; flash_attn_mlm_train does it itself)")


def _nothing_to_do(q: torch.Tensor, q_meta: PackMetadata | None) -> bool:
    return q.numel() == 0 or (q_meta is not None and q_meta.total_tokens == 0)


def flash_attn_mlm_fwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float,
    q_meta: PackMetadata | None = None,
    context_k: torch.Tensor | None = None,
    context_v: torch.Tensor | None = None,
    context_meta: PackMetadata | None = None,
    causal_query_seq_attn: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention output and softmax statistics for ``flash_attn_mlm_bwd``.

    q [B, H, N, D] (dense, or padded with ``q_meta``) or [H, T, D] (packed);
    k, v: the same with a divisor of H as heads.  ``context_k`` / ``context_v``
    [HK, Tc, D] with ``context_meta`` (of one context, or of one per sequence)
    and ``causal_query_seq_attn`` need the packed layout.

    Returns out (q's shape and dtype, contiguous; zero rows past each sequence)
    and lse (float32, q's shape without D): the natural log of each row's
    softmax denominator, undefined at padding rows.
    """
    layout = _validate(q, k, v, scale, q_meta, context_k, context_v, context_meta, causal_query_seq_attn)
    _require_packed(q, context_k, causal_query_seq_attn)
    return _forward(layout, q, k, v, scale, q_meta, context_k, context_v, context_meta, causal_query_seq_attn)


def _forward(layout, q, k, v, scale, q_meta, context_k, context_v, context_meta, causal):
    """``flash_attn_mlm_fwd`` on checked arguments."""
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
    if _nothing_to_do(q, q_meta):
        return out.zero_(), lse.fill_(float("-inf"))
    q, k, v = _tma_ready(q), _tma_ready(k), _tma_ready(v)
    h, d, hk = q.shape[-3], q.shape[-1], k.shape[-3]
    L = _lib.lib()
    code, err = _lib.dtype_code(q.dtype), _lib.error_word(q.device).data_ptr()
    views = (*_view(q), *_view(k), *_view(v))
    if layout == _lib.FMLM_BWD_DENSE:
        args = _lib.pack_dense_args(
            code, d, q.shape[0], h, q.shape[2], 0, 0, 1, 0, float(scale),  # no MLA, no prefill, no context
            *views, *_lib.NO_VIEW, *_lib.NO_VIEW, out.data_ptr(), err)
        launch = L.fmlm_attn_dense_fwd_lse
    else:
        packed = layout == _lib.FMLM_BWD_PACKED
        rows = _lib.FMLM_LAYOUT_PACKED if packed else _lib.FMLM_LAYOUT_PADDED
        ctx_bs, kc, vc, cu_kv = 1, _lib.NO_VIEW, _lib.NO_VIEW, 0
        if context_k is not None and context_meta.total_tokens > 0:
            context_k, context_v = _tma_ready(context_k), _tma_ready(context_v)
            ctx_bs, kc, vc, cu_kv = context_meta.B, _view(context_k), _view(context_v), context_meta.cu_seqlens.data_ptr()
        total = q_meta.total_tokens
        nbytes = L.fmlm_packed_workspace_bytes(q_meta.B, total, d)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        args = _lib.pack_packed_args(
            code, d, h, q_meta.B, 0, 0, int(causal), ctx_bs, float(scale),  # no MLA, no prefill
            rows, rows, 0 if packed else q.shape[2], total, *views, *kc, *vc,
            q_meta.cu_seqlens.data_ptr(), cu_kv, out.data_ptr(), total, ws.data_ptr(), nbytes, err,
            0, 0, int(not packed))  # a new schedule, no context_index, padded output
        launch = L.fmlm_attn_packed_fwd_lse
    _lib.launch(launch, q.device, "flash_attn_mlm_fwd", args, hk, lse.data_ptr())
    return out, lse


def flash_attn_mlm_bwd(
    dout: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    scale: float,
    q_meta: PackMetadata | None = None,
    context_k: torch.Tensor | None = None,
    context_v: torch.Tensor | None = None,
    context_meta: PackMetadata | None = None,
    causal_query_seq_attn: bool = False,
    need_dq: bool = True,
    need_dkv: bool = True,
) -> tuple[torch.Tensor | None, ...]:
    """Gradients (dq, dk, dv, dcontext_k, dcontext_v) of ``flash_attn_mlm_fwd``.

    ``out`` and ``lse`` are what the forward call returned for the same
    arguments, ``dout`` the gradient of ``out``.  Gradients have their
    tensors' shapes and dtypes, contiguous, with zero rows past each sequence.
    What is not needed (``need_dq``, ``need_dkv``), and the context's without
    a context, is None.

    float16: a row with |lse / scale| of 2^31 or more (scores of that size
    before they are scaled) has no valid part in dk and dv; the error word says
    so (``check_device_errors``).
    """
    layout = _validate(q, k, v, scale, q_meta, context_k, context_v, context_meta, causal_query_seq_attn)
    _require_packed(q, context_k, causal_query_seq_attn)
    for name, x in (("dout", dout), ("out", out)):
        if x.shape != q.shape or x.dtype != q.dtype or x.device != q.device:
            raise ValueError(f"{name} must have q's shape, dtype and device")
    if lse.shape != q.shape[:-1] or lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError("lse must be float32 of q's shape without the head dimension, on q's device")
    return _backward(layout, dout, q, k, v, out, lse, scale, q_meta, context_k, context_v, context_meta,
                     causal_query_seq_attn, need_dq, need_dkv)


def _backward(layout, dout, q, k, v, out, lse, scale, q_meta, context_k, context_v, context_meta, causal, need_dq,
              need_dkv):
    """``flash_attn_mlm_bwd`` on checked arguments."""
    dev = q.device

    def like(x, wanted):
        return torch.empty_like(x, memory_format=torch.contiguous_format) if wanted and x is not None else None

    dq, dk, dv = like(q, need_dq), like(k, need_dkv), like(v, need_dkv)
    dkc, dvc = like(context_k, need_dkv), like(context_v, need_dkv)
    grads = (dq, dk, dv, dkc, dvc)
    if not (need_dq or need_dkv):
        return grads
    if _nothing_to_do(q, q_meta):
        for g in grads:
            if g is not None:
                g.zero_()
        return grads
    q, k, v = _tma_ready(q), _tma_ready(k), _tma_ready(v)
    dout, out, lse = _tma_ready(dout.contiguous()), _tma_ready(out.contiguous()), lse.contiguous()
    packed = layout == _lib.FMLM_BWD_PACKED
    L = _lib.lib()
    entries, rows_c, kc, vc, cu_kv = 0, 0, _lib.NO_VIEW, _lib.NO_VIEW, 0
    if context_k is not None and context_meta.total_tokens > 0:
        context_k, context_v = _tma_ready(context_k), _tma_ready(context_v)
        entries, rows_c, cu_kv = context_meta.B, context_meta.total_tokens, context_meta.cu_seqlens.data_ptr()
        kc, vc = _view(context_k), _view(context_v)
    nbytes = L.fmlm_attn_bwd_workspace_bytes(lse.numel())
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args = _lib.pack_attn_bwd_args(
        _lib.dtype_code(q.dtype), q.shape[-1], layout, q_meta.B if packed else q.shape[0], q.shape[-3], k.shape[-3],
        0 if packed else q.shape[2], int(causal), entries, float(scale), q.shape[1] if packed else 0, rows_c,
        *_view(q), *_view(k), *_view(v), *_view(dout), *kc, *vc, out.data_ptr(), lse.data_ptr(),
        0 if q_meta is None else q_meta.cu_seqlens.data_ptr(), cu_kv,
        *[0 if g is None else g.data_ptr() for g in grads],  # dq, dk, dv and the context's
        ws.data_ptr(), nbytes, _lib.error_word(dev).data_ptr())
    _lib.launch(L.fmlm_attn_bwd, dev, "flash_attn_mlm_bwd", args)
    return grads


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, context_k, context_v, layout, scale, q_meta, context_meta, causal):
        out, lse = _forward(layout, q, k, v, scale, q_meta, context_k, context_v, context_meta, causal)
        ctx.save_for_backward(q, k, v, context_k, context_v, out, lse)
        ctx.call = (layout, scale, q_meta, context_meta, causal)
        return out

    @staticmethod
    def backward(ctx, dout):
        # (the wrapper marks the gradients as not differentiable again; without create_graph nothing could be)
        return _attention_backward_once(ctx, dout) if torch.is_grad_enabled() else _attention_backward(ctx, dout)


def _attention_backward(ctx, dout):
    q, k, v, context_k, context_v, out, lse = ctx.saved_tensors
    layout, scale, q_meta, context_meta, causal = ctx.call
    need = ctx.needs_input_grad
    grads = _backward(layout, dout, q, k, v, out, lse, scale, q_meta, context_k, context_v, context_meta, causal,
                      need[0], any(need[1:5]))
    return (*grads, None, None, None, None, None)


_attention_backward_once = torch.autograd.function.once_differentiable(_attention_backward)


class _Pack(torch.autograd.Function):
    """Padded [B, H, N, D] -> packed [H, T, D]; the gradient is unpacked."""

    @staticmethod
    def forward(ctx, x, meta):
        ctx.meta = meta
        return pack_for_kernel(x, meta)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return unpack_from_kernel(g, ctx.meta, g.shape[0]), None


class _Unpack(torch.autograd.Function):
    """Packed [H, T, D] -> padded [B, H, N, D]; the gradient is packed."""

    @staticmethod
    def forward(ctx, x, meta):
        ctx.meta = meta
        return unpack_from_kernel(x, meta, x.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return pack_for_kernel(g, ctx.meta), None


def flash_attn_mlm_train(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float,
    q_meta: PackMetadata | None = None,
    context_k: torch.Tensor | None = None,
    context_v: torch.Tensor | None = None,
    context_meta: PackMetadata | None = None,
    causal_query_seq_attn: bool = False,
) -> torch.Tensor:
    """Differentiable attention (``flash_attn_mlm_fwd``, with ``flash_attn_mlm_bwd`` as its gradient).

    The arguments of ``flash_attn_mlm_fwd``; padded q/k/v with a context or
    ``causal_query_seq_attn`` are packed first (and their gradients unpacked).
    Returns out in q's layout.  Gradients flow to q, k, v, context_k and
    context_v.  float16: the gradients have to lie in float16's range (loss
    scaling sees to that); what they are computed from need not.

    To capture the backward pass into a CUDA graph, call ``flash_attn_mlm_fwd``
    and ``flash_attn_mlm_bwd``, which involve no autograd graph.
    """
    layout = _validate(q, k, v, scale, q_meta, context_k, context_v, context_meta, causal_query_seq_attn)
    if q.ndim == 4 and (context_k is not None or causal_query_seq_attn):
        qp, kp, vp = (_Pack.apply(x, q_meta) for x in (q, k, v))
        out = _Attention.apply(qp, kp, vp, context_k, context_v, _lib.FMLM_BWD_PACKED, scale, q_meta, context_meta,
                               causal_query_seq_attn)
        return _Unpack.apply(out, q_meta)
    return _Attention.apply(q, k, v, context_k, context_v, layout, scale, q_meta, context_meta, causal_query_seq_attn)
