"""Per-head norm of queries and keys with the position rotation in the same
pass, in front of the attention (no counterpart in the reference).

``RotaryTable`` holds the cosines and sines of every position, computed in
float64 once (an angle of position 100000 has lost its low digits in float32);
``qk_norm_rope`` reads q and k once and writes them once, and is differentiable
in q, k and the norm's weights.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from flash_mlm import _lib
from flash_mlm.host.cache import PackMetadata
from flash_mlm.host.host_utils import validate_head_dim_supported

_PAIRS = {"half": _lib.FMLM_PAIRS_HALF, "interleaved": _lib.FMLM_PAIRS_INTERLEAVED}


class RotaryTable:
    """Cosines and sines [max_positions, rotary_dim / 2, 2] (float32) of the rotation angles
    ``position * base ** (-2 j / rotary_dim)``, or ``position * inv_freq[j]``.

    ``pairs``: which columns turn together: "half" (j, j + rotary_dim / 2) or
    "interleaved" (2 j, 2 j + 1).  ``rotary_dim`` is a multiple of 16; a head's
    columns past it are not rotated.
    """

    def __init__(self, max_positions: int, rotary_dim: int, *, base: float = 10000.0,
                 inv_freq: torch.Tensor | None = None, pairs: str = "half", device: torch.device | str = "cuda"):
        if max_positions < 1:
            raise ValueError("max_positions must be >= 1")
        if rotary_dim < 16 or rotary_dim % 16 != 0:
            raise ValueError("rotary_dim must be a positive multiple of 16")
        if pairs not in _PAIRS:
            raise ValueError('pairs must be "half" or "interleaved"')
        if inv_freq is None:
            if not 0.0 < float(base) < math.inf:
                raise ValueError("base must be positive and finite")
            inv_freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
        if tuple(inv_freq.shape) != (rotary_dim // 2,):
            raise ValueError("inv_freq must have rotary_dim / 2 elements")
        self.max_positions, self.rotary_dim, self.pairs = int(max_positions), int(rotary_dim), pairs
        freq = inv_freq.detach().to(device=device, dtype=torch.float64)
        angle = torch.arange(max_positions, device=device, dtype=torch.float64)[:, None] * freq
        self.table = torch.stack([angle.cos().float(), angle.sin().float()], -1).contiguous()


def _rows_ready(x: torch.Tensor) -> torch.Tensor:
    """x itself if its rows can be read in 16-byte vectors where they lie, else a contiguous copy."""
    *outer, last = x.stride()
    ok = last == 1 and x.data_ptr() % 16 == 0
    for stride in outer:
        ok = ok and stride % 8 == 0
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _view(x: torch.Tensor) -> tuple[int, ...]:
    if x.ndim == 4:
        b, h, n, _ = x.shape
        sb, sh, sn, _ = x.stride()
        return x.data_ptr(), n, h, b, sn, sh, sb
    h, t, _ = x.shape
    sh, st, _ = x.stride()
    return x.data_ptr(), t, h, 1, st, sh, 0


def _validate(q, k, rotary, q_weight, k_weight, normalize, eps, q_meta, positions, position_offsets):
    if q.ndim not in (3, 4) or k.ndim != q.ndim:
        raise ValueError("q/k must be rank-4 tensors [B, H, N, D] or packed rank-3 tensors [H, T, D]")
    qs, ks = q.shape, k.shape
    if qs[-2:] != ks[-2:] or (q.ndim == 4 and qs[0] != ks[0]):
        raise ValueError("q and k may differ in their number of heads only")
    if qs[-3] < 1 or ks[-3] < 1:
        raise ValueError("q and k must have at least one head")
    d = qs[-1]
    validate_head_dim_supported(d)
    _lib.dtype_code(q.dtype)
    if k.dtype != q.dtype:
        raise ValueError("q and k must have the same dtype")
    if q.ndim == 3:
        if q_meta is None:
            raise ValueError("packed q/k need q_meta")
        if q_meta.total_tokens != qs[1] or q_meta.token_indices.numel() != qs[1]:
            raise ValueError("packed token count mismatch with PackMetadata")
    elif q_meta is not None and (q_meta.B != qs[0] or q_meta.N != qs[2]):
        raise ValueError("q_meta shape metadata does not match q/k padded shape")
    if rotary is None and not normalize:
        raise ValueError("nothing to do: give rotary, or normalize=True")
    if rotary is not None and rotary.rotary_dim > d:
        raise ValueError("rotary_dim must be at most head_dim")
    tensors = [q, k] if rotary is None else [q, k, rotary.table]
    weights = [w for w in (q_weight, k_weight) if w is not None]
    if weights and not normalize:
        raise ValueError("weights need normalize=True")
    for w in weights:
        if tuple(w.shape) != (d,):
            raise ValueError("q_weight and k_weight must be [head_dim]")
        if (w.dtype != torch.float32 and w.dtype != q.dtype) or w.dtype != weights[0].dtype:
            raise ValueError("q_weight and k_weight must both be float32, or both of q's dtype")
    if normalize and not eps >= 0.0:
        raise ValueError("eps must be >= 0")
    tensors += weights
    if (positions is not None or position_offsets is not None) and rotary is None:
        raise ValueError("positions need rotary")
    if positions is not None and position_offsets is not None:
        raise ValueError("give positions or position_offsets, not both")
    if positions is not None:
        want = (q.shape[1],) if q.ndim == 3 else (q.shape[0], q.shape[2])
        if positions.dtype != torch.int32 or tuple(positions.shape) != want:
            raise ValueError(f"positions must be an int32 tensor of shape {list(want)}")
        tensors.append(positions)
    if position_offsets is not None:
        b = q_meta.B if q.ndim == 3 else q.shape[0]
        if position_offsets.dtype != torch.int32 or tuple(position_offsets.shape) != (b,):
            raise ValueError("position_offsets must be an int32 tensor of shape [B]")
        tensors.append(position_offsets)
    if q_meta is not None:
        tensors += [q_meta.lengths, q_meta.token_indices]
        if q_meta.lengths.dtype != torch.int32 or q_meta.token_indices.dtype != torch.int64:
            raise ValueError("q_meta must hold int32 lengths and int64 token_indices")
    if not q.is_cuda:
        raise ValueError("All tensors must be CUDA tensors")
    device = q.device
    for x in tensors:
        if x.device != device:
            raise ValueError("all tensors must be on q's device")


def _launch(fn, what, call, q, k, out_q, out_k, gq=None, gk=None, dwq=None, dwk=None):
    """One kernel call: `call` holds the arguments of ``qk_norm_rope`` behind q and k."""
    rotary, q_weight, k_weight, normalize, eps, q_meta, positions, position_offsets = call
    packed = q.ndim == 3
    keep = []  # contiguous copies, alive until the launch

    def ptr(x):
        if x is None:
            return 0
        if not x.is_contiguous():
            x = x.detach().contiguous()
            keep.append(x)
        return x.data_ptr()

    batch, seq_len = (q_meta.B, max(q_meta.N, 1)) if packed else (q.shape[0], q.shape[2])
    w = q_weight if q_weight is not None else k_weight
    weight_f32 = int(w is None or w.dtype == torch.float32)
    turn = (0, 0, 0) if rotary is None else (rotary.rotary_dim, _PAIRS[rotary.pairs], rotary.max_positions)
    lengths, tokens = (None, None) if q_meta is None else (None, q_meta.token_indices) if packed else (q_meta.lengths, None)
    ws = None
    if dwq is not None or dwk is not None:
        ws = torch.empty(_lib.lib().fmlm_qk_rope_bwd_workspace_bytes(q.shape[-1]), dtype=torch.uint8, device=q.device)
    args = _lib.pack_qk_rope_args(
        _lib.dtype_code(q.dtype), q.shape[-1], int(packed), batch, seq_len, q.shape[-3], k.shape[-3], int(normalize),
        weight_f32, *turn, float(eps), *_view(q), *_view(k),
        *(_lib.NO_VIEW if gq is None else _view(gq)), *(_lib.NO_VIEW if gk is None else _view(gk)),
        ptr(q_weight), ptr(k_weight), 0 if rotary is None else rotary.table.data_ptr(),
        ptr(positions), ptr(position_offsets), ptr(lengths), ptr(tokens), out_q.data_ptr(), out_k.data_ptr(),
        0 if dwq is None else dwq.data_ptr(), 0 if dwk is None else dwk.data_ptr(),
        0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), _lib.error_word(q.device).data_ptr())
    _lib.launch(fn, q.device, what, args)


def _outputs(q, k):
    return (torch.empty_like(q, memory_format=torch.contiguous_format),
            torch.empty_like(k, memory_format=torch.contiguous_format))


def _forward(q, k, *call):
    out_q, out_k = _outputs(q, k)
    if q.numel() and k.numel():
        _launch(_lib.lib().fmlm_qk_rope_fwd, "qk_norm_rope", call, _rows_ready(q), _rows_ready(k), out_q, out_k)
    return out_q, out_k


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, rotary, normalize, eps, q_meta, positions, position_offsets):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, position_offsets)
        ctx.call = (rotary, normalize, eps, q_meta)
        return _forward(q, k, rotary, q_weight, k_weight, normalize, eps, q_meta, positions, position_offsets)

    @staticmethod
    def backward(ctx, gq, gk):
        # (the wrapper marks the gradients as not differentiable again; without create_graph nothing could be)
        return _rope_backward_once(ctx, gq, gk) if torch.is_grad_enabled() else _rope_backward(ctx, gq, gk)


def _rope_backward(ctx, gq, gk):
    q, k, q_weight, k_weight, positions, position_offsets = ctx.saved_tensors
    rotary, normalize, eps, q_meta = ctx.call
    dq, dk = _outputs(q, k)
    dwq, dwk = (torch.empty_like(w, memory_format=torch.contiguous_format) if w is not None and need else None
                for w, need in ((q_weight, ctx.needs_input_grad[2]), (k_weight, ctx.needs_input_grad[3])))
    if not (q.numel() and k.numel()):
        for w in (dwq, dwk):
            if w is not None:
                w.zero_()
        return dq, dk, dwq, dwk, None, None, None, None, None, None
    call = (rotary, q_weight, k_weight, normalize, eps, q_meta, positions, position_offsets)
    _launch(_lib.lib().fmlm_qk_rope_bwd, "qk_norm_rope backward", call, _rows_ready(q), _rows_ready(k), dq, dk,
            _rows_ready(gq), _rows_ready(gk), dwq, dwk)
    return dq, dk, dwq, dwk, None, None, None, None, None, None


_rope_backward_once = torch.autograd.function.once_differentiable(_rope_backward)


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    rotary: RotaryTable | None = None,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    normalize: bool = True,
    eps: float = 1e-6,
    q_meta: PackMetadata | None = None,
    positions: torch.Tensor | None = None,
    position_offsets: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm each head row of q and k and rotate it by its position, in one pass.

    q [B, H, N, D] (dense, or padded with ``q_meta``: rows past a sequence come
    out as zeros, whatever they hold) or packed [H, T, D] with ``q_meta``; k the
    same with any number of heads.  Any strides, a projection's [B, N, H, D]
    transposed among them.

    ``normalize``: x / sqrt(mean(x^2) + eps) over the head dimension, times
    ``q_weight`` / ``k_weight`` [D] (float32 or q's dtype; None: ones).  The
    squares are summed in float32 (a bfloat16 row longer than 2^64 overflows it).
    ``rotary`` (None: no rotation): the token's index in its sequence is its
    position, plus ``position_offsets[b]`` (int32 [B]: tokens that came before,
    as a cached context's), or ``positions`` (int32 [B, N], packed [T]) gives
    it.  A position outside the table uses the table's nearest row and sets
    the error word (``check_device_errors``).

    Returns the new q and k, contiguous, in the layouts and dtype they came in.
    Differentiable in q, k, q_weight and k_weight, in reverse mode (forward-mode
    tangents are refused).
    """
    _validate(q, k, rotary, q_weight, k_weight, normalize, eps, q_meta, positions, position_offsets)
    # (Forward-mode tangents belong to tensors that require no gradient: the function refuses them.)
    graph = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, q_weight, k_weight))
    if graph or forward_ad._current_level >= 0:
        return _QkNormRope.apply(q, k, q_weight, k_weight, rotary, normalize, eps, q_meta, positions, position_offsets)
    return _forward(q, k, rotary, q_weight, k_weight, normalize, eps, q_meta, positions, position_offsets)
