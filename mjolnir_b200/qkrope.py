"""RMS norm of Q and K per head with the position rotation, in one kernel.

The step between the QKV projection and the cache write: every head row is
normalised (where a weight is given), its first ``rot_dim`` elements rotated by
the row's position, and rounded once. Q and K are read in place from the fused
projection's rows through their strides. Tokens of images and video have a
position on each of several axes (time, height, width); every angle then
follows one of them (:func:`angle_axes`).
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib
from .runner import _ptr, call, dtype_code


def angle_axes(sections, alternate: bool = False) -> tuple[int, ...]:
    """The axis of each angle where axis ``x`` turns ``sections[x]`` of them:
    one section after the other, or with ``alternate`` the axes in turn (0, 1,
    2, 0, 1, 2, ...) while they last, what is left over on axis 0."""
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0:
        raise ValueError(f"sections must be numbers of angles, got {sections}")
    n, a = sum(sections), len(sections)
    if not alternate:
        return tuple(x for x, m in enumerate(sections) for _ in range(m))
    axes = tuple(i % a if i < a * sections[i % a] else 0 for i in range(n))
    if any(axes.count(x) != m for x, m in enumerate(sections)):
        raise ValueError(f"sections {sections} cannot take turns: {n} angles are too few for those after the first")
    return axes


@lru_cache(maxsize=64)
def _axes(axes: tuple[int, ...], num_axes: int, rot_dim: int):
    """The checked axes as the library takes them."""
    if not 1 <= num_axes <= _lib.ROPE_AXES:
        raise ValueError(f"positions on {num_axes} axes: 1 to {_lib.ROPE_AXES}")
    if 2 * len(axes) != rot_dim or rot_dim > 512 or any(not 0 <= x < num_axes for x in axes):
        raise ValueError(f"axes must name one of the {num_axes} axes for each of the {rot_dim // 2} angles, got {axes}")
    return (_lib.C.c_ubyte * 256)(*axes)


def qk_norm_rope(
    q: torch.Tensor,  # (T, h_q, d) bf16 / fp16 / fp32, d contiguous, any token and head strides
    k: torch.Tensor,  # (T, h_k, d)
    positions: torch.Tensor,  # (T,) int64; with axes (number of axes, T)
    cos_sin: torch.Tensor,  # (max_positions, rot_dim) bf16 / fp16 / fp32: cos | sin halves
    q_weight: torch.Tensor | None = None,  # (d,) of any of the three types; None = no norm
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    interleaved: bool = False,  # pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)
    axes: tuple[int, ...] | None = None,  # the axis of each of the rot_dim / 2 angles
    q_out: torch.Tensor | None = None,  # default: new tensors; q / k themselves work in place
    k_out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Normalise and rotate Q and K; returns ``(q_out, k_out)``. A position
    outside the table, on any axis, flags ``MJ_DEV_BAD_POSITION`` in ``status``
    and leaves its token's output rows as they were."""
    shape, k_shape, dtype, dev = q.shape, k.shape, q.dtype, q.get_device()
    if len(shape) != 3 or len(k_shape) != 3:
        raise ValueError(f"q {tuple(shape)} and k {tuple(k_shape)} must be (tokens, heads, head_size)")
    T, h_q, d = shape
    h_k = k_shape[1]
    if k_shape[0] != T or k_shape[2] != d or k.dtype != dtype:
        raise ValueError(f"k {tuple(k_shape)} {k.dtype} does not match q {tuple(shape)} {dtype}")
    if q_out is None:
        q_out = torch.empty(shape, dtype=dtype, device=q.device)
    if k_out is None:
        k_out = torch.empty(k_shape, dtype=dtype, device=q.device)
    if q_out.shape != shape or q_out.dtype != dtype or k_out.shape != k_shape or k_out.dtype != dtype:
        raise ValueError(f"q_out {tuple(q_out.shape)} {q_out.dtype} / k_out {tuple(k_out.shape)} {k_out.dtype} do not match q and k")
    qs, ks, qos, kos = q.stride(), k.stride(), q_out.stride(), k_out.stride()
    if qs[2] != 1 or ks[2] != 1 or qos[2] != 1 or kos[2] != 1:
        raise ValueError("the head dim of q, k and the outputs must be contiguous")
    ps, pst = positions.shape, positions.stride()
    if positions.dtype != torch.int64 or len(ps) != (1 if axes is None else 2) or ps[-1] != T or (T > 1 and pst[-1] != 1):
        raise ValueError(f"positions must be an int64 {f'({T},)' if axes is None else f'(axes, {T})'} with contiguous rows, got "
                         f"{positions.dtype} {tuple(positions.shape)}")
    cs, cst = cos_sin.shape, cos_sin.stride()
    if len(cs) != 2 or (cs[1] > 1 and cst[1] != 1):
        raise ValueError(f"cos_sin must be (positions, rot_dim) with contiguous rows, got {tuple(cs)}")
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
    entry, more = _lib.qk_norm_rope, None
    if axes is not None:
        n = ps[0]
        more = _lib.RopeAxes(n, pst[0] if n > 1 else 0, _axes(tuple(axes), n, cs[1]))
        entry = _lib.qk_norm_rope_axes
    a = _lib.QkNormRopeArgs(
        q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), dtype_code(dtype), T, h_q, h_k, d, cs[1],
        int(interleaved), qs[0], qs[1], ks[0], ks[1], qos[0], qos[1], kos[0], kos[1], positions.data_ptr(), cos_sin.data_ptr(),
        dtype_code(cos_sin.dtype), cst[0], cs[0], _ptr(q_weight), _ptr(k_weight), dtype_code(w_dtype),
        float(eps), _ptr(status))
    call(entry, a if more is None else (a, more), dev)
    return q_out, k_out
