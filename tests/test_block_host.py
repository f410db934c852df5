"""Refusals and layouts of the block-scaled cache operators (no GPU needed)."""

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from mjolnir_b200 import _lib, kvblock, qkrope
from tests.block_helpers import exponent

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_header():
    names = {"mj_qk_norm_rope_args": (_lib.QkNormRopeArgs, "status"), "mj_block_read_args": (_lib.BlockReadArgs, "status"),
             "mj_block_attn_args": (_lib.BlockAttnArgs, "status")}
    body = "".join(f'printf("%zu %zu ", sizeof({n}), offsetof({n}, {f}));' for n, (_, f) in names.items())
    src = f'#include "mjolnir_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){{{body}return 0;}}\n'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "p.c"), "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "p.c"), "-o", os.path.join(d, "p")], check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "p")], check=True, capture_output=True, text=True).stdout.split()]
    want = [n for t, f in names.values() for n in (ctypes.sizeof(t), getattr(t, f).offset)]
    assert got == want


def _cache(pages=4, page=32, h_k=2, d=128, block=16):
    return kvblock.views(*kvblock.alloc(pages, page, h_k, d, block, device="cpu"))


def test_alloc_and_views():
    k, v, ks, vs = _cache(block=16)
    assert k.shape == v.shape == (4, 32, 2, 128) and ks.shape == vs.shape == (4, 2, 2)
    k[1, 5, 1, 7], vs[3, 1, 0] = 9, 8
    assert int(v.sum()) == 0 and int(ks.sum()) == 0
    for bad in (dict(block=8), dict(block=24), dict(block=64), dict(d=96), dict(page=24)):
        with pytest.raises(ValueError):
            _cache(**bad)


def test_scale_exponents():
    assert exponent(0.0) == 95 and exponent(448.0) == 127 and exponent(448.5) == 128
    assert exponent(224.0) == 126 and exponent(1e30) == 159


@pytest.mark.parametrize("change,error", [
    (dict(key=torch.zeros(3, 2, 64)), ValueError),  # head size
    (dict(key=torch.zeros(3, 3, 128)), ValueError),  # heads
    (dict(key=torch.zeros(1, 2, 128)), ValueError),  # fewer rows than slots
    (dict(key=torch.zeros(3, 2, 128).half()), TypeError),  # key and value types differ
    (dict(key=torch.zeros(3, 2, 128).double(), value=torch.zeros(3, 2, 128).double()), TypeError),
    (dict(key=torch.zeros(3, 2, 256)[..., ::2]), ValueError),  # head dim not contiguous
    (dict(slots=torch.zeros(3)), TypeError),
    (dict(slots=torch.zeros(3, 1, dtype=torch.int64)), TypeError),
    (dict(scales=torch.zeros(4, 3, 2, dtype=torch.uint8)), ValueError),  # 3 blocks in a page of 32
    (dict(scales=torch.zeros(4, 4, 2, dtype=torch.uint8)), ValueError),  # blocks of 8
    (dict(scales=torch.zeros(4, 2, 2)), ValueError),  # not bytes
    (dict(v=torch.zeros(3, 32, 2, 128, dtype=torch.uint8)), ValueError),
])
def test_write_refuses(change, error):
    k, v, ks, vs = _cache()
    x = torch.zeros(3, 2, 128)
    a = dict(key=x, value=x, slots=torch.arange(3), v=v, scales=ks) | change
    with pytest.raises(error):
        kvblock.write(a["key"], a["value"], k, a["v"], a["scales"], vs if a["scales"] is ks else a["scales"], a["slots"])


@pytest.mark.parametrize("change", [
    dict(starts=torch.zeros(2, dtype=torch.int64)), dict(offsets=torch.zeros(2, dtype=torch.int32)),
    dict(table=torch.zeros(1, 4, dtype=torch.int32)), dict(table=torch.zeros(2, 4, dtype=torch.int64)),
    dict(out=torch.zeros(5, 2, 64)), dict(out=torch.zeros(5, 2, 256)[..., ::2]),
])
def test_read_refuses(change):
    a = dict(starts=torch.zeros(2, dtype=torch.int32), offsets=torch.zeros(3, dtype=torch.int32),
             table=torch.zeros(2, 4, dtype=torch.int32), out=torch.zeros(5, 2, 128)) | change
    with pytest.raises(ValueError):
        kvblock.read(*_cache(), a["table"], a["starts"], a["offsets"], a["out"], torch.zeros_like(a["out"]))


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(4, 2, 64)), dict(k=torch.zeros(3, 2, 128)), dict(k=torch.zeros(4, 2, 128).half()),
    dict(positions=torch.zeros(4, dtype=torch.int32)), dict(positions=torch.zeros(3, dtype=torch.int64)),
    dict(cos_sin=torch.zeros(128)), dict(q_weight=torch.zeros(64)), dict(q_weight=torch.zeros(128), k_weight=torch.zeros(128).half()),
    dict(q_out=torch.zeros(4, 3, 128).half()), dict(k_out=torch.zeros(4, 3, 128)), dict(q=torch.zeros(4, 3, 256)[..., ::2]),
])
def test_rope_refuses(change):
    a = dict(q=torch.zeros(4, 3, 128), k=torch.zeros(4, 2, 128), positions=torch.zeros(4, dtype=torch.int64),
             cos_sin=torch.zeros(8, 128)) | change
    with pytest.raises(ValueError):
        qkrope.qk_norm_rope(**a)


def test_c_entries_refuse():
    """What the Python layer would stop first, at the C boundary: a status and a message, no launch."""
    r = _lib.QkNormRopeArgs()
    r.num_tokens, r.h_q, r.h_k = 1, 1, 1
    for d, rot, ok in ((120, 0, False), (528, 0, False), (128, 24, False), (128, 144, False)):
        r.head_size, r.rot_dim = d, rot
        with pytest.raises(_lib.MjolnirError) as e:
            _lib.qk_norm_rope(r, 0)
        assert e.value.code == _lib.MJ_ERR_UNSUPPORTED
    r.head_size, r.rot_dim = 128, 128
    with pytest.raises(_lib.MjolnirError, match="null"):
        _lib.qk_norm_rope(r, 0)
    w = _lib.CacheWriteArgs()
    w.num_tokens, w.h_k, w.head_size, w.page_size, w.num_pages, w.kv_format = 1, 1, 128, 16, 1, _lib.BLOCK_FORMATS[32]
    with pytest.raises(_lib.MjolnirError, match="divide the page"):
        _lib.block_write(w, 0)
    w.kv_format = _lib.MJ_KV_FP8_E4M3
    with pytest.raises(_lib.MjolnirError, match="not block-scaled"):
        _lib.block_write(w, 0)
    w.kv_format = _lib.BLOCK_FORMATS[16]
    with pytest.raises(_lib.MjolnirError, match="null"):
        _lib.block_write(w, 0)
    with pytest.raises(_lib.MjolnirError, match="mj_block_write"):
        _lib.cache_write(w, 0)
    b = _lib.BlockReadArgs()
    b.num_seqs, b.num_rows, b.h_k, b.head_size, b.page_size, b.num_pages, b.kv_format = 1, 1, 1, 64, 16, 1, _lib.BLOCK_FORMATS[16]
    with pytest.raises(_lib.MjolnirError, match="head_size"):
        _lib.block_read(b, 0)
    a = _lib.BlockAttnArgs()
    a.num_seqs, a.num_tokens, a.h_q, a.h_k = 1, 1, 3, 2
    with pytest.raises(_lib.MjolnirError, match="h_q 3 h_k 2"):
        _lib.block_attention(a, 0)
    one = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(one) + 255) // 256 * 256
    a.h_q, a.head_size, a.page_size, a.num_pages, a.kv_format, a.dtype = 4, 128, 48, 1, _lib.BLOCK_FORMATS[16], _lib.MJ_DT_BF16
    a.k_cache = a.v_cache = a.k_scales = a.v_scales = at
    with pytest.raises(_lib.MjolnirError, match="page_size 48"):
        _lib.block_attention(a, 0)
    a.page_size, a.dtype = 64, _lib.MJ_DT_FP32
    with pytest.raises(_lib.MjolnirError, match="bf16 or fp16"):
        _lib.block_attention(a, 0)
    a.dtype, a.k_stride_row = _lib.MJ_DT_BF16, 24
    with pytest.raises(_lib.MjolnirError, match="alignment"):
        _lib.block_attention(a, 0)


def test_cpu_tensors_are_refused():
    x = torch.zeros(3, 2, 128)
    with pytest.raises(ValueError, match="CUDA tensors"):
        kvblock.write(x, x, *_cache(), torch.arange(3))
    with pytest.raises(ValueError, match="CUDA tensors"):
        qkrope.qk_norm_rope(x, x, torch.zeros(3, dtype=torch.int64), torch.zeros(4, 128))


@pytest.mark.parametrize("seed", range(4))
def test_plan_covers_every_row_and_tile_once(seed):
    import random

    import numpy as np

    r = random.Random(seed)
    for _ in range(200):
        n = r.randint(0, 12)
        q = [r.choice([0, 1, 5, 70, 1500, r.randint(0, 400)]) for _ in range(n)]
        kv = [max(0, x + r.choice([-2, 0, 0, 40, 9000])) for x in q]
        h_k, h_r, d, causal = r.choice([1, 2, 8]), r.choice([1, 3, 4, 6]), r.choice([128, 256]), r.random() < 0.7
        slots = r.choice([0, 2 * -(-148 // h_k)])
        work, merges = np.zeros((20000, 8), np.int32), np.zeros((max(1, slots), 4), np.int32)
        nw, nm, ns = _lib.block_plan(q, kv, h_k * h_r, h_k, d, causal, 148, slots, work, merges)
        assert ns <= slots
        rows, items = 128 if d == 256 else 256, {}
        for s, r0, tb, te, slot, *_ in work[:nw].tolist():
            items.setdefault((s, r0), []).append((tb, te, slot))
        assert set(items) == {(s, r0) for s in range(n) for r0 in range(0, q[s] * h_r, rows)}
        used = []
        for (s, r0), pieces in items.items():
            pieces.sort()
            last = kv[s] - q[s] + (min(r0 + rows, q[s] * h_r) - 1) // h_r if causal else kv[s] - 1
            assert pieces[0][0] == 0 and pieces[-1][1] == (last // 64 + 1 if last >= 0 else 0)
            assert all(a[1] == b[0] for a, b in zip(pieces, pieces[1:]))
            got = [p[2] for p in pieces]
            if len(pieces) == 1:
                assert got == [-1]
                continue
            used += got
            assert [m[2:] for m in merges[:nm].tolist() if m[:2] == [s, r0]] == [[got[0], len(got)]]
        assert sorted(used) == list(range(ns))


def test_plan_refuses():
    import numpy as np

    work, merges = np.zeros((2, 8), np.int32), np.zeros((1, 4), np.int32)
    with pytest.raises(_lib.MjolnirError, match="capacity"):
        _lib.block_plan([1, 1, 1], [5, 5, 5], 4, 1, 128, True, 148, 0, work, merges)
    with pytest.raises(_lib.MjolnirError, match="length"):
        _lib.block_plan([1], [-5], 4, 1, 128, True, 148, 0, work, merges)
    with pytest.raises(_lib.MjolnirError, match="invalid"):
        _lib.block_plan([1], [5], 4, 3, 128, True, 148, 0, work, merges)
