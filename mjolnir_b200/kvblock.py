"""The block-scaled KV cache: e4m3 codes with one power-of-two scale per
(block of G tokens, KV head), chosen from the data as it is written.

Against the static-scale fp8 cache it needs no calibration and saturates
nothing; against a scale per token it reads 1 / G of the scale bytes. A cache
is a pair of byte tensors (:func:`alloc` makes the layout the decode kernel
streams best): codes ``(pages, h_k, page_size, K row | V row)`` and exponent
bytes ``(pages, h_k, 2, page_size / G)`` of the scales ``2^(e - 127)``. The
functions take logical views -- codes ``(pages, page_size, h_k, d)``, exponents
``(pages, page_size / G, h_k)`` -- of any strides; G is read off the shapes.

* :func:`write` -- quantise new K / V rows into the cache;
* :func:`read` -- cached tokens back as contiguous rows;
* :class:`BlockAttention` -- attention of ragged query chunks (and of single
  tokens) over the cache.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from .runner import DecodeRunner, StepPlan, _ptr, _stream, dtype_code, kv_byte_strides

HEAD_SIZES = (128, 256)
BLOCK_TOKENS = tuple(_lib.BLOCK_FORMATS)


def views(kv_cache: torch.Tensor, scales: torch.Tensor):
    """Logical ``(k, v, k_scales, v_scales)`` views of a cache as
    :func:`alloc` lays it out."""
    d = kv_cache.shape[3] // 2
    return (kv_cache[..., :d].transpose(1, 2), kv_cache[..., d:].transpose(1, 2),
            scales[:, :, 0].transpose(1, 2), scales[:, :, 1].transpose(1, 2))


def alloc(num_pages: int, page_size: int, num_kv_heads: int, head_size: int, block_tokens: int = 16,
          device: torch.device | str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """A zeroed cache: ``(codes (pages, h_k, page_size, 2 d), scales (pages,
    h_k, 2, page_size / G))``, both uint8."""
    _format(block_tokens, page_size, head_size)
    return (torch.zeros(num_pages, num_kv_heads, page_size, 2 * head_size, dtype=torch.uint8, device=device),
            torch.zeros(num_pages, num_kv_heads, 2, page_size // block_tokens, dtype=torch.uint8, device=device))


def _format(block_tokens: int, page_size: int, head_size: int) -> int:
    if block_tokens not in _lib.BLOCK_FORMATS or page_size % block_tokens:
        raise ValueError(f"blocks of {block_tokens} tokens: one of {BLOCK_TOKENS} that divides the page of {page_size}")
    if head_size not in HEAD_SIZES:
        raise ValueError(f"head_size {head_size}: the block-scaled cache holds {HEAD_SIZES}")
    return _lib.BLOCK_FORMATS[block_tokens]


def _cache_args(a, k_cache, v_cache, k_scales, v_scales, row_stride: str = "block") -> int:
    """Points an args struct at checked cache and scale views; returns the
    tokens of a block."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dim() != 4 or t.shape != k_cache.shape or t.element_size() != 1:
            raise ValueError(f"{name} must be a (pages, page_size, h_k, d) byte view, got {tuple(t.shape)} {t.dtype}")
    pages, page_size, h_k, d = k_cache.shape
    blocks = k_scales.shape[1] if k_scales.dim() == 3 else 0
    if blocks < 1 or page_size % blocks:
        raise ValueError(f"k_scales {tuple(k_scales.shape)} is not (pages, page_size / G, h_k) for pages of {page_size}")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if tuple(t.shape) != (pages, blocks, h_k) or t.element_size() != 1:
            raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} is not ({pages}, {blocks}, {h_k}) bytes")
    for t in (v_cache, k_scales, v_scales):
        if t.device != k_cache.device:
            raise ValueError(f"cache and scales must share a device, got {k_cache.device} and {t.device}")
    a.kv_format = _format(page_size // blocks, page_size, d)
    a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    a.k_stride_page, a.k_stride_row, a.k_stride_head = kv_byte_strides(k_cache)
    a.v_stride_page, a.v_stride_row, a.v_stride_head = kv_byte_strides(v_cache)
    a.k_scales, a.v_scales = k_scales.data_ptr(), v_scales.data_ptr()
    for side, t in (("ks", k_scales), ("vs", v_scales)):
        st = [0 if n == 1 else s for n, s in zip(t.shape, t.stride())]
        setattr(a, f"{side}_stride_page", st[0])
        setattr(a, f"{side}_stride_{row_stride}", st[1])
        setattr(a, f"{side}_stride_head", st[2])
    a.num_pages, a.page_size, a.h_k, a.head_size = pages, page_size, h_k, d
    return page_size // blocks


def _rows(name: str, t: torch.Tensor, h_k: int, d: int) -> None:
    if t.dim() != 3 or tuple(t.shape[1:]) != (h_k, d) or t.stride(2) != 1:
        raise ValueError(f"{name} {tuple(t.shape)} is not (rows, {h_k}, {d}) with contiguous rows")


def _on(device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"every tensor must be on {device}, got {t.device}")


def write(
    key: torch.Tensor,  # (>= T, h_k, d) bf16 / fp16 / fp32, 16-byte aligned rows
    value: torch.Tensor,
    k_cache: torch.Tensor,  # (pages, page_size, h_k, d) byte views
    v_cache: torch.Tensor,
    k_scales: torch.Tensor,  # (pages, page_size / G, h_k) uint8 views
    v_scales: torch.Tensor,
    slot_mapping: torch.Tensor,  # (T,) int64 (int32 accepted), negative = skip
    status: torch.Tensor | None = None,
) -> None:
    """Quantise T new rows into the cache. A block whose row 0 is written is
    opened with the scale its new rows need; an open block's scale only grows,
    and its earlier rows follow it. The tokens of one block stand together in
    ``slot_mapping`` (as sequences' tokens do)."""
    T = slot_mapping.shape[0]
    if T == 0:
        return
    a = _lib.CacheWriteArgs()
    _cache_args(a, k_cache, v_cache, k_scales, v_scales, row_stride="row")
    _rows("key", key, a.h_k, a.head_size)
    _rows("value", value, a.h_k, a.head_size)
    if key.shape[0] < T or value.shape[0] < T:
        raise ValueError("fewer key / value rows than slots")
    if value.dtype != key.dtype:
        raise TypeError("key and value must share a dtype")
    if slot_mapping.dim() != 1 or slot_mapping.dtype not in (torch.int64, torch.int32):
        raise TypeError("slot_mapping must be a 1-D int64")
    _on(k_cache.device, key, value, slot_mapping, status)
    slots = slot_mapping.to(torch.int64).contiguous()
    a.key, a.value, a.src_dtype, a.num_tokens = key.data_ptr(), value.data_ptr(), dtype_code(key.dtype), T
    a.key_stride_tok, a.key_stride_head = key.stride(0), key.stride(1)
    a.value_stride_tok, a.value_stride_head = value.stride(0), value.stride(1)
    a.slot_mapping, a.status = slots.data_ptr(), _ptr(status)
    with torch.cuda.device(k_cache.device):
        _lib.block_write(a, _stream(k_cache.device))


def _table(block_table: torch.Tensor, num_seqs: int) -> None:
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] < num_seqs or (
            block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 (>= {num_seqs}, blocks) with contiguous rows, got "
                         f"{block_table.dtype} {tuple(block_table.shape)}")


def read(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_table: torch.Tensor,  # (>= n, blocks) int32
    starts: torch.Tensor,  # (n,) int32: first token of each sequence to read
    offsets: torch.Tensor,  # (n + 1,) int32: its output rows, ascending from 0
    k_out: torch.Tensor,  # (rows, h_k, d) bf16 / fp16 / fp32, 16-byte aligned rows
    v_out: torch.Tensor,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Read tokens ``starts[s] ..`` of each sequence into rows ``offsets[s] ..
    offsets[s + 1] - 1`` of the outputs; returns ``(k_out, v_out)``."""
    a = _lib.BlockReadArgs()
    _cache_args(a, k_cache, v_cache, k_scales, v_scales)
    n = starts.shape[0]
    for name, t, m in (("starts", starts, n), ("offsets", offsets, n + 1)):
        if t.dtype != torch.int32 or tuple(t.shape) != (m,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 ({m},), got {t.dtype} {tuple(t.shape)}")
    _table(block_table, n)
    _rows("k_out", k_out, a.h_k, a.head_size)
    _rows("v_out", v_out, a.h_k, a.head_size)
    if v_out.shape != k_out.shape or v_out.dtype != k_out.dtype:
        raise ValueError("k_out and v_out must share a shape and dtype")
    _on(k_cache.device, block_table, starts, offsets, k_out, v_out, status)
    a.block_table, a.block_table_stride, a.block_table_cols = block_table.data_ptr(), block_table.stride(0), block_table.shape[1]
    a.starts, a.offsets, a.num_seqs, a.num_rows = starts.data_ptr(), offsets.data_ptr(), n, k_out.shape[0]
    a.k_out, a.v_out, a.out_dtype = k_out.data_ptr(), v_out.data_ptr(), dtype_code(k_out.dtype)
    a.ko_stride_tok, a.ko_stride_head = k_out.stride(0), k_out.stride(1)
    a.vo_stride_tok, a.vo_stride_head = v_out.stride(0), v_out.stride(1)
    a.status = _ptr(status)
    with torch.cuda.device(k_cache.device):
        _lib.block_read(a, _stream(k_cache.device))
    return k_out, v_out


@dataclass
class BlockPlan:
    """The plan of one step, shared by every layer."""

    query_lens: list[int]
    num_tokens: int
    block_table: torch.Tensor
    seq_lens: torch.Tensor
    q_start: torch.Tensor  # (num_seqs + 1,) int32, device
    work: torch.Tensor  # (items, 8) int32, device
    merges: torch.Tensor  # (merges, 4) int32, device
    num_slots: int
    causal: bool = True
    decode: StepPlan | None = None  # the leading sequences that the decode kernel serves


class BlockAttention:
    """Attention over a block-scaled cache for steps of any mix of lengths:
    single tokens, drafts and prompt chunks behind cached contexts.

    The leading sequences of a step that share one query length of at most
    ``max_q_len`` tokens (a batch's decodes, which schedulers put first) run on
    the decode kernel, the others on the kernel for chunks: one query token of
    a group of 4 heads fills 4 of the chunk kernel's 256 rows."""

    def __init__(self, *, num_heads: int, num_kv_heads: int, head_size: int, page_size: int, block_tokens: int = 16,
                 max_num_seqs: int = 256, max_num_tokens: int = 8192, max_q_len: int = 4, device: torch.device | str = "cuda"):
        if num_heads % num_kv_heads:
            raise ValueError("num_heads must be a multiple of num_kv_heads")
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page size {page_size} unsupported (16, 32, 64 or 128)")
        self.kv_format = _format(block_tokens, page_size, head_size)
        self.h_q, self.h_k, self.d = num_heads, num_kv_heads, head_size
        self.page_size, self.block_tokens = page_size, block_tokens
        self.max_num_seqs, self.max_num_tokens = max_num_seqs, max_num_tokens
        self.device = torch.device(device)
        _lib.load()  # fail at construction, not at the first step
        self.max_q_len = min(max_q_len, 64 // (num_heads // num_kv_heads))
        self.decode = None if self.max_q_len < 1 else DecodeRunner(
            num_heads=num_heads, num_kv_heads=num_kv_heads, head_size=head_size, page_size=page_size,
            max_num_seqs=max_num_seqs, max_q_len=self.max_q_len, kv_format=f"fp8b{block_tokens}", kernel="tc", device=device)
        self.sm_count = torch.cuda.get_device_properties(self.device).multi_processor_count
        # rows of a work item, and the partial slots that splitting for every SM can ask for
        self.rows = 128 if head_size == 256 else 256
        self.max_slots = 2 * -(-self.sm_count // num_kv_heads)
        self.max_work = max_num_tokens * (num_heads // num_kv_heads) // self.rows + max_num_seqs + self.max_slots
        # the plan: q_start | merges | work, one fixed-address buffer and one copy a step
        self._at = (-(-(max_num_seqs + 1) // 4) * 4, -(-(max_num_seqs + 1) // 4) * 4 + 4 * self.max_slots)
        self.plan_buf = torch.zeros(self._at[1] + 8 * self.max_work, dtype=torch.int32, device=self.device)
        self.o_part = torch.empty(self.max_slots * num_kv_heads * self.rows * head_size, dtype=torch.float32, device=self.device)
        self.lse_part = torch.empty(self.max_slots * num_kv_heads * self.rows, dtype=torch.float32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.one = torch.ones(1, dtype=torch.float32, device=self.device)

    def plan(self, query_lens, seq_lens_cpu, block_table: torch.Tensor, seq_lens: torch.Tensor,
             causal: bool = True) -> BlockPlan:
        """Plan a step: ``query_lens[s]`` new tokens of each sequence, which
        are the last of its ``seq_lens[s]`` tokens. The device ``seq_lens``
        (int32) are what the kernels mask with."""
        q = [int(x) for x in query_lens]
        if len(q) > self.max_num_seqs or sum(q) > self.max_num_tokens:
            raise ValueError(f"{len(q)} sequences / {sum(q)} tokens beyond the runner's capacity")
        kv = [int(x) for x in seq_lens_cpu]
        if len(q) != len(kv) or min(q, default=0) < 0 or min(kv, default=0) < 0:
            raise ValueError("query_lens and seq_lens_cpu must pair up, without negative lengths")
        _table(block_table, len(q))
        if seq_lens.dtype != torch.int32 or seq_lens.dim() != 1 or seq_lens.shape[0] < len(q) or not seq_lens.is_contiguous():
            raise ValueError("seq_lens must be a contiguous int32 tensor of every sequence")
        _on(self.status.device, block_table, seq_lens)
        decode, few = None, 0
        if q and 1 <= q[0] <= self.max_q_len:
            few = next((i for i, x in enumerate(q) if x != q[0]), len(q))
            decode = self.decode.plan(kv, few, q[0], block_table, seq_lens, causal=causal)
        if few == len(q):
            return BlockPlan(q, sum(q), block_table, seq_lens, None, None, None, 0, causal, decode)
        n, (m0, w0) = len(q), self._at
        stage = torch.empty(self.plan_buf.shape[0], dtype=torch.int32, pin_memory=True)
        host = stage.numpy()
        host[0] = 0
        np.cumsum(q, out=host[1:n + 1])
        work, merges = host[w0:].reshape(-1, 8), host[m0:w0].reshape(-1, 4)
        nw, nm, slots = _lib.block_plan([0] * few + q[few:], kv, self.h_q, self.h_k, self.d, causal, self.sm_count, self.max_slots, work, merges)
        used = w0 + 8 * nw
        self.plan_buf[:used].copy_(stage[:used], non_blocking=True)
        return BlockPlan(q, sum(q), block_table, seq_lens, self.plan_buf[:n + 1], self.plan_buf[w0:used].view(-1, 8),
                         self.plan_buf[m0:m0 + 4 * nm].view(-1, 4), slots, causal, decode)

    def run(
        self,
        plan: BlockPlan,
        query: torch.Tensor,  # (>= tokens, h_q, d) bf16 / fp16, any token and head strides
        out: torch.Tensor,  # the same dtype, written in place
        k_cache: torch.Tensor,
        v_cache: torch.Tensor,
        k_scales: torch.Tensor,
        v_scales: torch.Tensor,
        softmax_scale: float,
        lse: torch.Tensor | None = None,  # optional (tokens, h_q) fp32
    ) -> torch.Tensor:
        if plan.decode is not None:
            self.decode.run(plan.decode, query, out, k_cache, v_cache, self.one, self.one, softmax_scale, lse=lse,
                            k_scales=k_scales, v_scales=v_scales)
            if plan.work is None:
                return out
        a = _lib.BlockAttnArgs()
        g = _cache_args(a, k_cache, v_cache, k_scales, v_scales)
        if (a.page_size, g, a.h_k, a.head_size) != (self.page_size, self.block_tokens, self.h_k, self.d):
            raise ValueError(f"cache of pages {a.page_size}, blocks {g}, {a.h_k} heads of {a.head_size} is not this runner's")
        for name, t in (("query", query), ("out", out)):
            _rows(name, t, self.h_q, self.d)
            if t.shape[0] < plan.num_tokens:
                raise ValueError(f"{name} has {t.shape[0]} rows for {plan.num_tokens} tokens")
        if out.dtype != query.dtype or query.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"query and out must both be bf16 or fp16, got {query.dtype} and {out.dtype}")
        if lse is not None and (lse.dtype != torch.float32 or lse.shape[0] < plan.num_tokens or lse.shape[1:] != (self.h_q,)
                                or not lse.is_contiguous()):
            raise ValueError("lse must be a contiguous fp32 (tokens, h_q)")
        _on(self.status.device, query, out, k_cache, lse)
        a.num_seqs, a.h_q, a.num_tokens, a.dtype = len(plan.query_lens), self.h_q, plan.num_tokens, dtype_code(query.dtype)
        a.q, a.q_stride_tok, a.q_stride_head = query.data_ptr(), query.stride(0), query.stride(1)
        a.o, a.o_stride_tok, a.o_stride_head = out.data_ptr(), out.stride(0), out.stride(1)
        bt = plan.block_table
        a.block_table, a.block_table_stride, a.block_table_cols = bt.data_ptr(), bt.stride(0), bt.shape[1]
        a.seq_lens, a.q_start, a.lse = plan.seq_lens.data_ptr(), plan.q_start.data_ptr(), _ptr(lse)
        a.softmax_scale, a.causal, a.status = float(softmax_scale), int(plan.causal), self.status.data_ptr()
        a.work, a.num_work, a.merges, a.num_merges = plan.work.data_ptr(), len(plan.work), plan.merges.data_ptr(), len(plan.merges)
        a.o_part, a.lse_part, a.num_slots = self.o_part.data_ptr(), self.lse_part.data_ptr(), plan.num_slots
        with torch.cuda.device(self.status.device):
            _lib.block_attention(a, _stream(self.status.device))
        return out

    def check_status(self) -> None:
        """Raise if a kernel flagged a bad page or a wait that ran out
        (synchronizes); the status word is cleared."""
        if self.decode is not None:
            self.decode.check_status()
        code = int(self.status.item())
        if code != _lib.MJ_DEV_OK:
            self.status.zero_()
            raise _lib.MjolnirError(_lib.MJ_ERR_DEVICE, f"device status {code}")
