"""Refusals and layouts of the operators for long-lived contexts (no GPU needed)."""

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from mjolnir_b200 import _lib, kvblock, qkrope

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I32 = torch.int32


def test_struct_layouts_match_header():
    names = {"mj_rope_axes": (_lib.RopeAxes, "axis"), "mj_block_weigh_args": (_lib.BlockWeighArgs, "status"),
             "mj_block_evict_args": (_lib.BlockEvictArgs, "status")}
    body = "".join(f'printf("%zu %zu ", sizeof({n}), offsetof({n}, {f}));' for n, (_, f) in names.items())
    src = f'#include "mjolnir_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){{{body}return 0;}}\n'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "p.c"), "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "p.c"), "-o", os.path.join(d, "p")], check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "p")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [n for t, f in names.values() for n in (ctypes.sizeof(t), getattr(t, f).offset)]


def test_angle_axes():
    assert qkrope.angle_axes((2, 1, 1)) == (0, 0, 1, 2)
    assert qkrope.angle_axes((4, 2, 2), alternate=True) == (0, 1, 2, 0, 1, 2, 0, 0)
    assert qkrope.angle_axes((3,), alternate=True) == (0, 0, 0)
    for bad in ((), (-1, 2)):
        with pytest.raises(ValueError):
            qkrope.angle_axes(bad)
    with pytest.raises(ValueError, match="turns"):
        qkrope.angle_axes((1, 4, 4), alternate=True)


@pytest.mark.parametrize("change", [
    dict(positions=torch.zeros(4, dtype=torch.int64)),  # one axis of positions, axes named
    dict(positions=torch.zeros(3, 5, dtype=torch.int64)), dict(positions=torch.zeros(3, 4, dtype=I32)),
    dict(positions=torch.zeros(4, 3, dtype=torch.int64).t()),  # an axis' positions not contiguous
    dict(positions=torch.zeros(5, 4, dtype=torch.int64)),  # five axes
    dict(axes=(0,) * 63), dict(axes=(0,) * 63 + (3,)), dict(axes=(-1,) * 64), dict(axes=None),
])
def test_rope_axes_refuses(change):
    a = dict(q=torch.zeros(4, 3, 128), k=torch.zeros(4, 2, 128), positions=torch.zeros(3, 4, dtype=torch.int64),
             cos_sin=torch.zeros(8, 128), axes=(0, 1) * 32) | change
    with pytest.raises(ValueError):
        qkrope.qk_norm_rope(**a)


def _cache(pages=4, page=32, h_k=2, d=128, block=16):
    return kvblock.views(*kvblock.alloc(pages, page, h_k, d, block, device="cpu"))


WEIGH = dict(query=torch.zeros(5, 4, 128).half(), lse=torch.zeros(5, 4), block_table=torch.zeros(2, 3, dtype=I32),
             offsets=torch.zeros(3, dtype=I32), seq_lens=torch.zeros(2, dtype=I32), weights=torch.zeros(2, 2, 90))


@pytest.mark.parametrize("change,error", [
    (dict(query=torch.zeros(5, 3, 128).half()), ValueError), (dict(query=torch.zeros(5, 4, 64).half()), ValueError),
    (dict(query=torch.zeros(5, 4, 128)), TypeError), (dict(query=torch.zeros(5, 512).half()), ValueError),
    (dict(query=torch.zeros(5, 4, 256).half()[..., ::2]), ValueError),
    (dict(lse=torch.zeros(5, 4).half()), ValueError), (dict(lse=torch.zeros(5, 3)), ValueError), (dict(lse=torch.zeros(4, 5).t()), ValueError),
    (dict(block_table=torch.zeros(1, 3, dtype=I32)), ValueError), (dict(block_table=torch.zeros(2, 3)), ValueError),
    (dict(offsets=torch.zeros(2, dtype=I32)), ValueError), (dict(offsets=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(seq_lens=torch.zeros(2, 1, dtype=I32)), ValueError), (dict(seq_lens=torch.zeros(4, dtype=I32)[::2]), ValueError),
    (dict(weights=torch.zeros(2, 3, 90)), ValueError), (dict(weights=torch.zeros(1, 2, 90)), ValueError),
    (dict(weights=torch.zeros(2, 2, 90).half()), ValueError), (dict(weights=torch.zeros(2, 90, 2).transpose(1, 2)), ValueError),
    (dict(window=-1), ValueError), (dict(), ValueError),  # the last: tensors on the CPU
])
def test_weigh_refuses(change, error):
    a = WEIGH | dict(window=0) | change
    k, _, ks, _ = _cache()
    with pytest.raises(error):
        kvblock.weigh(a["query"], a["lse"], k, ks, a["block_table"], a["offsets"], a["seq_lens"], a["weights"], 1.0, window=a["window"])


EVICT = dict(weights=torch.zeros(2, 2, 90), block_table=torch.zeros(2, 3, dtype=I32), seq_lens=torch.zeros(2, dtype=I32),
             new_lens=torch.zeros(2, dtype=I32), kept=torch.zeros(2, 2, 40, dtype=I32), recent=4)


@pytest.mark.parametrize("change", [
    dict(weights=torch.zeros(2, 3, 90)), dict(weights=torch.zeros(2, 2, 90).double()), dict(block_table=torch.zeros(1, 3, dtype=I32)),
    dict(seq_lens=torch.zeros(2)), dict(new_lens=torch.zeros(3, dtype=I32)), dict(new_lens=torch.zeros(2, dtype=torch.int64)),
    dict(kept=torch.zeros(2, 2, 40)), dict(kept=torch.zeros(2, 3, 40, dtype=I32)), dict(kept=torch.zeros(2, 40, 2, dtype=I32).transpose(1, 2)),
    dict(recent=-1), dict(recent=41), dict(),
])
def test_evict_refuses(change):
    a = EVICT | change
    with pytest.raises(ValueError):
        kvblock.evict(a["weights"], *_cache(), a["block_table"], a["seq_lens"], a["new_lens"], a["kept"], recent=a["recent"])


def test_c_entries_refuse():
    """What the Python layer would stop first, at the C boundary: a status and a message, no launch."""
    one = ctypes.create_string_buffer(1024)
    at = (ctypes.addressof(one) + 255) // 256 * 256
    r, ax = _lib.QkNormRopeArgs(), _lib.RopeAxes()
    r.num_tokens, r.h_q, r.h_k, r.head_size, r.rot_dim = 1, 1, 1, 128, 128
    for n in (0, 5):
        ax.num_axes = n
        with pytest.raises(_lib.MjolnirError, match="axes"):
            _lib.qk_norm_rope_axes((r, ax), 0)
    ax.num_axes, ax.axis[63] = 2, 2
    with pytest.raises(_lib.MjolnirError, match="angle 63"):
        _lib.qk_norm_rope_axes((r, ax), 0)
    w = _lib.BlockWeighArgs()
    w.num_seqs, w.num_rows, w.h_q, w.h_k = 1, 1, 3, 2
    with pytest.raises(_lib.MjolnirError, match="h_q 3 h_k 2"):
        _lib.block_weigh(w, 0)
    w.h_q, w.head_size, w.page_size, w.num_pages, w.kv_format, w.k_cache, w.k_scales = 4, 128, 48, 2, _lib.BLOCK_FORMATS[16], at, at
    with pytest.raises(_lib.MjolnirError, match="page_size 48"):
        _lib.block_weigh(w, 0)
    w.page_size, w.dtype = 64, _lib.MJ_DT_FP32
    with pytest.raises(_lib.MjolnirError, match="bf16 or fp16"):
        _lib.block_weigh(w, 0)
    w.dtype = _lib.MJ_DT_BF16
    with pytest.raises(_lib.MjolnirError, match="null"):
        _lib.block_weigh(w, 0)
    w.q = w.lse = w.block_table = w.offsets = w.seq_lens = w.weights = at
    w.block_table_cols, w.weights_cols = 1, 8
    with pytest.raises(_lib.MjolnirError, match="weights stride"):
        _lib.block_weigh(w, 0)
    w.w_stride_head, w.q_stride_head = 8, 4
    with pytest.raises(_lib.MjolnirError, match="16-byte"):
        _lib.block_weigh(w, 0)
    w.q_stride_head = 128
    with pytest.raises(_lib.MjolnirError, match="cache stride of 0"):
        _lib.block_weigh(w, 0)
    e = _lib.BlockEvictArgs()
    e.num_seqs, e.budget, e.recent = 2, 4, 5
    with pytest.raises(_lib.MjolnirError, match="recent 5"):
        _lib.block_evict(e, 0)
    e.recent, e.h_k, e.head_size, e.page_size, e.num_pages, e.kv_format = 1, 1, 64, 16, 1, _lib.BLOCK_FORMATS[16]
    with pytest.raises(_lib.MjolnirError, match="head_size"):
        _lib.block_evict(e, 0)
    e.head_size, e.k_cache, e.v_cache, e.k_scales, e.v_scales = 128, at, at, at, at
    with pytest.raises(_lib.MjolnirError, match="null"):
        _lib.block_evict(e, 0)
    e.block_table = e.seq_lens = e.weights = e.kept = at
    e.new_lens, e.block_table_cols, e.weights_cols, e.w_stride_seq = at + 4, 1, 8, 8
    with pytest.raises(_lib.MjolnirError, match="overlaps"):
        _lib.block_evict(e, 0)
    e.new_lens, e.w_stride_seq = at + 64, 0
    with pytest.raises(_lib.MjolnirError, match="weights stride"):
        _lib.block_evict(e, 0)
    e.w_stride_seq = 8
    with pytest.raises(_lib.MjolnirError, match="stride of 0"):
        _lib.block_evict(e, 0)


@pytest.mark.parametrize("n,h_k,seq,head,good", [
    (3, 2, 20, 10, True), (3, 2, 10, 30, True), (3, 2, 19, 10, False), (3, 2, 10, 29, False), (3, 2, 10, 10, False),
    (3, 2, 20, 9, False), (3, 1, 10, 0, True), (3, 1, 9, 0, False), (1, 2, 0, 10, True), (1, 2, 0, 9, False), (1, 1, 0, 0, True),
    (3, 2, 2**62, 10, True), (3, 2, 2**62, 2**62 - 1, False),
])
def test_rows_of_weights_share_nothing(n, h_k, seq, head, good):
    """The strides pass, and the next check refuses; or they do not."""
    one = ctypes.create_string_buffer(1024)
    at = (ctypes.addressof(one) + 255) // 256 * 256
    e = _lib.BlockEvictArgs()
    e.num_seqs, e.budget, e.h_k, e.head_size, e.page_size, e.num_pages, e.kv_format = n, 4, h_k, 128, 16, 1, _lib.BLOCK_FORMATS[16]
    e.k_cache = e.v_cache = e.k_scales = e.v_scales = e.block_table = e.weights = e.kept = e.seq_lens = e.new_lens = at
    e.block_table_cols, e.weights_cols, e.w_stride_seq, e.w_stride_head = 1, 10, seq, head
    with pytest.raises(_lib.MjolnirError, match="new_lens overlaps" if good else "weights stride"):
        _lib.block_evict(e, 0)
