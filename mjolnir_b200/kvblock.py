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
from .runner import DecodeRunner, StepPlan, _ptr, call, dtype_code

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


def _cache(k_cache, v_cache, k_scales, v_scales) -> tuple:
    """Checks cache and scale views; returns (shape, kv_format, device index,
    the six code strides, the six scale strides)."""
    shape, sshape = k_cache.shape, k_scales.shape
    ks, vs, kss, vss = k_cache.stride(), v_cache.stride(), k_scales.stride(), v_scales.stride()
    if len(shape) != 4 or v_cache.shape != shape or k_cache.itemsize != 1 or v_cache.itemsize != 1 or ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"k_cache {tuple(shape)} {k_cache.dtype} and v_cache {tuple(v_cache.shape)} {v_cache.dtype} must be "
                         "(pages, page_size, h_k, d) byte views with contiguous rows")
    pages, page_size, h_k, d = shape
    if (len(sshape) != 3 or v_scales.shape != sshape or k_scales.itemsize != 1 or v_scales.itemsize != 1
            or sshape[0] != pages or sshape[2] != h_k or sshape[1] < 1 or page_size % sshape[1]):
        raise ValueError(f"k_scales {tuple(sshape)} {k_scales.dtype} and v_scales {tuple(v_scales.shape)} {v_scales.dtype} must "
                         f"be ({pages}, {page_size} / G, {h_k}) byte views")
    kv_format = _format(page_size // sshape[1], page_size, d)
    dev = k_cache.get_device()
    _on(dev, v_cache, k_scales, v_scales)
    st = (ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])
    if pages == 1 or h_k == 1:  # a dim of extent 1 may carry any stride
        st = tuple(0 if n == 1 else x for n, x in zip((*shape[:3], *shape[:3]), st))
    return shape, kv_format, dev, st, (kss[0], kss[1], kss[2], vss[0], vss[1], vss[2])


def _rows(name: str, t: torch.Tensor, h_k: int, d: int) -> tuple:
    """(token, head) strides of checked rows."""
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != h_k or shape[2] != d or st[2] != 1:
        raise ValueError(f"{name} {tuple(shape)} is not (rows, {h_k}, {d}) with contiguous rows")
    return st[0] if shape[0] > 1 else 0, st[1] if h_k > 1 else 0  # a dim of extent 1 may carry any stride


def _on(dev: int, *tensors) -> None:
    """Every tensor that is there is on the device of this index (-1: the CPU)."""
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"every tensor must be on {'cuda:%d' % dev if dev >= 0 else 'the CPU'}, got {t.device}")


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
    (pages, page_size, h_k, d), kv_format, dev, st, ss = _cache(k_cache, v_cache, k_scales, v_scales)
    kt, vt = _rows("key", key, h_k, d), _rows("value", value, h_k, d)
    if key.shape[0] < T or value.shape[0] < T:
        raise ValueError("fewer key / value rows than slots")
    if value.dtype != key.dtype:
        raise TypeError("key and value must share a dtype")
    if slot_mapping.dim() != 1 or slot_mapping.dtype not in (torch.int64, torch.int32):
        raise TypeError("slot_mapping must be a 1-D int64")
    _on(dev, key, value, slot_mapping, status)
    slots = slot_mapping
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    a = _lib.CacheWriteArgs(
        key.data_ptr(), value.data_ptr(), dtype_code(key.dtype), T, h_k, d, *kt, *vt, k_cache.data_ptr(), v_cache.data_ptr(),
        *st, pages, page_size, kv_format, slots.data_ptr(), None, 0, None, 0, _ptr(status),
        k_scales.data_ptr(), v_scales.data_ptr(), *ss)
    call(_lib.block_write, a, dev)


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
    (pages, page_size, h_k, d), kv_format, dev, st, ss = _cache(k_cache, v_cache, k_scales, v_scales)
    n = starts.shape[0]
    for name, t, m in (("starts", starts, n), ("offsets", offsets, n + 1)):
        if t.dtype != torch.int32 or t.shape != (m,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 ({m},), got {t.dtype} {tuple(t.shape)}")
    _table(block_table, n)
    ko, vo = _rows("k_out", k_out, h_k, d), _rows("v_out", v_out, h_k, d)
    if v_out.shape != k_out.shape or v_out.dtype != k_out.dtype:
        raise ValueError("k_out and v_out must share a shape and dtype")
    _on(dev, block_table, starts, offsets, k_out, v_out, status)
    a = _lib.BlockReadArgs(
        k_cache.data_ptr(), v_cache.data_ptr(), *st, k_scales.data_ptr(), v_scales.data_ptr(), *ss, pages, page_size, h_k, d,
        kv_format, block_table.data_ptr(), block_table.stride(0), block_table.shape[1], starts.data_ptr(), offsets.data_ptr(),
        n, k_out.shape[0], k_out.data_ptr(), v_out.data_ptr(), dtype_code(k_out.dtype), *ko, *vo, _ptr(status))
    call(_lib.block_read, a, dev)
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
    single tokens, drafts and prompt chunks behind cached contexts. A runner
    owns its plan buffers and split partials, so its calls belong to one
    stream at a time.

    The leading sequences of a step that share one query length of at most
    ``max_q_len`` tokens (a batch's decodes, which schedulers put first) run on
    the decode kernel while their rows per KV head fit one of its jobs: 48, or
    16 at head size 256. Beyond, and for the other sequences, the kernel for
    chunks runs, whose row tiles are 128. 16 sequences of 8K in a graph, decode
    kernel and chunk kernel: 8 KV heads of 128, 4 rows 48 and 142 us, 16 rows 66
    and 143, 48 rows 107 and 144; 4 KV heads of 128, 48 rows 65 and 101, 64 rows
    134 and 101; 4 KV heads of 256, 6 rows 51 and 117, 16 rows 72 and 118, 18 rows
    133 and 118, 48 rows 198 and 122."""

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
        self.max_q_len = min(max_q_len, (48 if head_size == 128 else 16) // (num_heads // num_kv_heads))
        # the split merge as a launch of its own: inside the decode launch it costs
        # more at every size measured (4 x 1000 tokens, 8 KV heads: 4 rows 17 us
        # against 14, 16 rows 37 against 17)
        self.decode = None if self.max_q_len < 1 else DecodeRunner(
            fused_merge=False,
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
             causal: bool = True, fixed_grid: bool = False) -> BlockPlan:
        """Plan a step: ``query_lens[s]`` new tokens of each sequence, which
        are the last of its ``seq_lens[s]`` tokens. The device ``seq_lens``
        (int32) are what the kernels mask with.

        A CUDA graph captured over :meth:`run` holds the launches of its plan:
        it replays that plan only. With ``fixed_grid`` the launches do not
        depend on the lengths, so the graph replays any later plan with
        ``fixed_grid`` of as many sequences and the same query length; only
        steps that the decode kernel serves whole have that form."""
        q = [int(x) for x in query_lens]
        if len(q) > self.max_num_seqs or sum(q) > self.max_num_tokens:
            raise ValueError(f"{len(q)} sequences / {sum(q)} tokens beyond the runner's capacity")
        kv = [int(x) for x in seq_lens_cpu]
        if len(q) != len(kv) or min(q, default=0) < 0 or min(kv, default=0) < 0:
            raise ValueError("query_lens and seq_lens_cpu must pair up, without negative lengths")
        _table(block_table, len(q))
        longest = max((x for x, n in zip(kv, q) if n), default=0)
        if longest > block_table.shape[1] * self.page_size:  # the decode kernel knows no end of a table's row
            raise ValueError(f"{longest} tokens of a sequence are more than block_table's {block_table.shape[1]} pages of {self.page_size}")
        if seq_lens.dtype != torch.int32 or seq_lens.dim() != 1 or seq_lens.shape[0] < len(q) or not seq_lens.is_contiguous():
            raise ValueError("seq_lens must be a contiguous int32 tensor of every sequence")
        _on(self.status.get_device(), block_table, seq_lens)
        decode, few = None, 0
        if q and 1 <= q[0] <= self.max_q_len:
            few = next((i for i, x in enumerate(q) if x != q[0]), len(q))
            if not fixed_grid or few == len(q):
                decode = self.decode.plan(kv, few, q[0], block_table, seq_lens, causal=causal, fixed_grid=fixed_grid)
        if fixed_grid and (few < len(q) or not q):
            raise ValueError(f"fixed_grid: a step of one query length of 1 to {self.max_q_len} tokens, got {q[:8]}")
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
        (pages, page_size, h_k, d), kv_format, dev, st, ss = _cache(k_cache, v_cache, k_scales, v_scales)
        if (page_size, kv_format, h_k, d) != (self.page_size, self.kv_format, self.h_k, self.d):
            raise ValueError(f"a cache of pages {page_size}, format {kv_format}, {h_k} heads of {d} is not this runner's")
        qs, os_ = _rows("query", query, self.h_q, d), _rows("out", out, self.h_q, d)
        tokens, dt = plan.num_tokens, dtype_code(query.dtype)
        if query.shape[0] < tokens or out.shape[0] < tokens:
            raise ValueError(f"query {tuple(query.shape)} / out {tuple(out.shape)} have fewer rows than the step's {tokens} tokens")
        if out.dtype != query.dtype or dt == _lib.MJ_DT_FP32:
            raise TypeError(f"query and out must both be bf16 or fp16, got {query.dtype} and {out.dtype}")
        if lse is not None and (lse.dtype != torch.float32 or lse.shape[0] < tokens or lse.shape[1:] != (self.h_q,)
                                or not lse.is_contiguous()):
            raise ValueError("lse must be a contiguous fp32 (tokens, h_q)")
        _on(dev, self.status, query, out, lse)
        bt, scale, causal = plan.block_table, float(softmax_scale), int(plan.causal)
        cache = (k_cache.data_ptr(), v_cache.data_ptr(), *st)
        scales = (k_scales.data_ptr(), v_scales.data_ptr())
        if plan.decode is not None:
            p, r = plan.decode, self.decode
            one = self.one.data_ptr()
            call(_lib.decode, _lib.DecodeArgs(
                p.num_seqs, p.q_len, self.h_q, h_k, d, page_size, kv_format, query.data_ptr(), dt, *qs, out.data_ptr(), dt,
                *os_, *cache, pages, bt.data_ptr(), bt.stride(0), plan.seq_lens.data_ptr(), p.work.data_ptr(), p.num_work,
                p.n_splits.data_ptr(), r.max_splits, r.o_part.data_ptr(), r.lse_part.data_ptr(), self.max_num_seqs, _ptr(lse),
                one, _lib.MJ_SCALE_TENSOR, one, _lib.MJ_SCALE_TENSOR, None, None, scale, causal, int(p.with_reduction),
                r.kernel, r.status.data_ptr(), r.merge_counters.data_ptr() if r.merges(p) else None, *scales, *ss, 0), dev)
        if plan.work is not None:
            call(_lib.block_attention, _lib.BlockAttnArgs(
                len(plan.query_lens), self.h_q, h_k, d, page_size, kv_format, dt, query.data_ptr(), *qs, out.data_ptr(), *os_,
                tokens, *cache, *scales, *ss, pages, bt.data_ptr(), bt.stride(0), bt.shape[1], plan.seq_lens.data_ptr(),
                plan.q_start.data_ptr(), _ptr(lse), scale, causal, plan.work.data_ptr(), plan.work.shape[0],
                plan.merges.data_ptr(), plan.merges.shape[0], self.o_part.data_ptr(), self.lse_part.data_ptr(),
                plan.num_slots, self.status.data_ptr()), dev)
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
