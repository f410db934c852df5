"""RMS norm of Q and K per head with the position rotation, in one kernel.

The step between the QKV projection and the cache write: every head row is
normalised (where a weight is given), its first ``rot_dim`` elements rotated by
the row's position, and rounded once. Q and K are read in place from the fused
projection's rows through their strides.
"""

from __future__ import annotations

import torch

from . import _lib
from .runner import _ptr, _stream, dtype_code


def _rows(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> torch.Tensor:
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{name} must be (tokens, heads, head_size) with a contiguous head dim, got {tuple(t.shape)}")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} does not match {tuple(like.shape)} {like.dtype}")
    return t


def qk_norm_rope(
    q: torch.Tensor,  # (T, h_q, d) bf16 / fp16 / fp32, d contiguous, any token and head strides
    k: torch.Tensor,  # (T, h_k, d)
    positions: torch.Tensor,  # (T,) int64
    cos_sin: torch.Tensor,  # (max_positions, rot_dim) bf16 / fp16 / fp32: cos | sin halves
    q_weight: torch.Tensor | None = None,  # (d,) of any of the three types; None = no norm
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    interleaved: bool = False,  # pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)
    q_out: torch.Tensor | None = None,  # default: new tensors; q / k themselves work in place
    k_out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Normalise and rotate Q and K; returns ``(q_out, k_out)``. A position
    outside the table flags ``MJ_DEV_BAD_POSITION`` in ``status`` and leaves
    its token's output rows as they were."""
    _rows("q", q)
    _rows("k", k)
    T, h_q, d = q.shape
    if k.shape[0] != T or k.shape[2] != d or k.dtype != q.dtype or k.device != q.device:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not match q {tuple(q.shape)} {q.dtype}")
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else _rows("q_out", q_out, q)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k_out is None else _rows("k_out", k_out, k)
    if positions.dtype != torch.int64 or positions.shape != (T,) or (T > 1 and positions.stride(0) != 1):
        raise ValueError(f"positions must be a contiguous int64 ({T},), got {positions.dtype} {tuple(positions.shape)}")
    if cos_sin.dim() != 2 or (cos_sin.shape[1] > 1 and cos_sin.stride(1) != 1):
        raise ValueError(f"cos_sin must be (positions, rot_dim) with contiguous rows, got {tuple(cos_sin.shape)}")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (d,) or not w.is_contiguous() or w.dtype != weights[0].dtype:
            raise ValueError(f"norm weights must be contiguous ({d},) of one dtype, got {tuple(w.shape)} {w.dtype}")
    for t in (k, positions, cos_sin, *weights, *([] if status is None else [status])):
        if t.device != q.device:
            raise ValueError(f"every tensor must be on {q.device}, got {t.device}")
    a = _lib.QkNormRopeArgs()
    a.q, a.k, a.q_out, a.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    a.dtype, a.num_tokens, a.h_q, a.h_k = dtype_code(q.dtype), T, h_q, k.shape[1]
    a.head_size, a.rot_dim, a.interleaved = d, cos_sin.shape[1], int(interleaved)
    a.q_stride_tok, a.q_stride_head, _ = q.stride()
    a.k_stride_tok, a.k_stride_head, _ = k.stride()
    a.qo_stride_tok, a.qo_stride_head, _ = q_out.stride()
    a.ko_stride_tok, a.ko_stride_head, _ = k_out.stride()
    a.positions, a.cos_sin, a.cos_sin_dtype = positions.data_ptr(), cos_sin.data_ptr(), dtype_code(cos_sin.dtype)
    a.cos_sin_stride, a.num_positions = cos_sin.stride(0), cos_sin.shape[0]
    a.q_weight, a.k_weight = _ptr(q_weight), _ptr(k_weight)
    a.weight_dtype = dtype_code(weights[0].dtype) if weights else _lib.MJ_DT_FP32
    a.eps = float(eps)
    a.status = _ptr(status)
    with torch.cuda.device(q.device):
        _lib.qk_norm_rope(a, _stream(q.device))
    return q_out, k_out
