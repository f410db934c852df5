"""RMS norm of Q and K per head with the position rotation, in one kernel.

The step between the QKV projection and the cache write: every head row is
normalised (where a weight is given), its first ``rot_dim`` elements rotated by
the row's position, and rounded once. Q and K are read in place from the fused
projection's rows through their strides.
"""

from __future__ import annotations

import torch

from . import _lib
from .runner import _ptr, call, dtype_code


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
    shape, dtype, dev = q.shape, q.dtype, q.get_device()
    if len(shape) != 3 or len(k.shape) != 3:
        raise ValueError(f"q {tuple(shape)} and k {tuple(k.shape)} must be (tokens, heads, head_size)")
    T, h_q, d = shape
    h_k = k.shape[1]
    if k.shape[0] != T or k.shape[2] != d or k.dtype != dtype:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not match q {tuple(shape)} {dtype}")
    if q_out is None:
        q_out = torch.empty(shape, dtype=dtype, device=q.device)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=dtype, device=q.device)
    if q_out.shape != shape or q_out.dtype != dtype or k_out.shape != k.shape or k_out.dtype != dtype:
        raise ValueError(f"q_out {tuple(q_out.shape)} {q_out.dtype} / k_out {tuple(k_out.shape)} {k_out.dtype} do not match q and k")
    qs, ks, qos, kos = q.stride(), k.stride(), q_out.stride(), k_out.stride()
    if qs[2] != 1 or ks[2] != 1 or qos[2] != 1 or kos[2] != 1:
        raise ValueError("the head dim of q, k and the outputs must be contiguous")
    if positions.dtype != torch.int64 or positions.shape != (T,) or (T > 1 and positions.stride(0) != 1):
        raise ValueError(f"positions must be a contiguous int64 ({T},), got {positions.dtype} {tuple(positions.shape)}")
    if cos_sin.dim() != 2 or (cos_sin.shape[1] > 1 and cos_sin.stride(1) != 1):
        raise ValueError(f"cos_sin must be (positions, rot_dim) with contiguous rows, got {tuple(cos_sin.shape)}")
    w_dtype = torch.float32
    for w in (q_weight, k_weight):
        if w is not None:
            if w.shape != (d,) or not w.is_contiguous():
                raise ValueError(f"norm weights must be contiguous ({d},), got {tuple(w.shape)}")
            w_dtype = w.dtype
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"norm weights must share a dtype, got {q_weight.dtype} and {k_weight.dtype}")
    for t in (k, q_out, k_out, positions, cos_sin, q_weight, k_weight, status):
        if t is not None and t.get_device() != dev:
            raise ValueError(f"every tensor must be on {q.device}, got {t.device}")
    call(_lib.qk_norm_rope, _lib.QkNormRopeArgs(
        q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), dtype_code(dtype), T, h_q, h_k, d, cos_sin.shape[1],
        int(interleaved), qs[0], qs[1], ks[0], ks[1], qos[0], qos[1], kos[0], kos[1], positions.data_ptr(), cos_sin.data_ptr(),
        dtype_code(cos_sin.dtype), cos_sin.stride(0), cos_sin.shape[0], _ptr(q_weight), _ptr(k_weight), dtype_code(w_dtype),
        float(eps), _ptr(status)), dev)
    return q_out, k_out
