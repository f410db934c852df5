"""Caches whose heads or pages share their bytes (a stride of 0, as expanded
views have): refused where a kernel could not read or write them."""

import ctypes

import pytest
import torch

from mjolnir_b200 import _lib


def _args(kind):
    """Arguments that pass every check (the call that would launch is never made)."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    a = kind()
    a.keep = buf
    a.h_k, a.head_size, a.page_size, a.num_pages, a.kv_format = 2, 128, 32, 3, _lib.BLOCK_FORMATS[16]
    a.k_cache = a.v_cache = a.k_scales = a.v_scales = at
    block = "row" if kind is not _lib.BlockAttnArgs else "block"
    for side in "kv":
        for name, n in (("page", 2 * 32 * 256), ("row", 256), ("head", 32 * 256)):
            setattr(a, f"{side}_stride_{name}", n)
        for name, n in (("page", 8), (block, 1), ("head", 2)):
            setattr(a, f"{side}s_stride_{name}", n)
    return a, at


@pytest.mark.parametrize("field", ["k_stride_page", "v_stride_row", "k_stride_head", "v_stride_head", "ks_stride_page",
                                   "vs_stride_row", "ks_stride_head"])
def test_write_refuses(field):
    a, at = _args(_lib.CacheWriteArgs)
    a.key = a.value = a.slot_mapping = at
    a.num_tokens, a.src_dtype, a.key_stride_tok, a.key_stride_head, a.value_stride_tok, a.value_stride_head = 1, 0, 256, 128, 256, 128
    setattr(a, field, 0)
    with pytest.raises(_lib.MjolnirError, match="stride of 0") as e:
        _lib.block_write(a, 0)
    assert e.value.code == _lib.MJ_ERR_UNSUPPORTED


@pytest.mark.parametrize("field", ["k_stride_page", "v_stride_row", "k_stride_head", "v_stride_head"])
def test_attention_refuses(field):
    a, at = _args(_lib.BlockAttnArgs)
    a.num_seqs, a.num_tokens, a.h_q, a.dtype = 1, 1, 2, _lib.MJ_DT_BF16
    a.q = a.o = a.block_table = a.seq_lens = a.q_start = at
    a.block_table_cols, a.q_stride_tok, a.q_stride_head, a.o_stride_tok, a.o_stride_head = 1, 256, 128, 256, 128
    setattr(a, field, 0)
    with pytest.raises(_lib.MjolnirError, match="stride of 0") as e:
        _lib.block_attention(a, 0)
    assert e.value.code == _lib.MJ_ERR_UNSUPPORTED


@pytest.mark.parametrize("field,why", [("k_stride_head", "head stride"), ("v_stride_page", "page stride"), ("v_stride_row", "row stride")])
@pytest.mark.parametrize("kv_format", [_lib.BLOCK_FORMATS[16], _lib.MJ_KV_FP8_E4M3])
def test_the_tensor_core_decode_refuses(field, why, kv_format):
    a, at = _args(_lib.DecodeArgs)
    a.kv_format, a.kernel = kv_format, _lib.MJ_KERNEL_TC
    a.num_seqs, a.q_len, a.h_q, a.num_work, a.max_splits = 1, 1, 2, 1, 1
    a.q = a.o = a.block_table = a.seq_lens = a.work = a.n_splits = at
    setattr(a, field, 0)
    with pytest.raises(_lib.MjolnirError, match=why) as e:
        _lib.decode(a, 0)
    assert e.value.code == _lib.MJ_ERR_UNSUPPORTED


@pytest.mark.gpu
def test_block_cache_with_shared_heads():
    """The read-back takes it; write and attention refuse before a launch."""
    from mjolnir_b200 import kvblock
    from tests.block_helpers import Cache

    c = Cache([40], h_k=1, split=True)
    wide = [x.expand(-1, -1, 3, *([-1] if x.dim() == 4 else [])) for x in c.args]
    table, zero = c.table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = (torch.empty(40, 3, 128, dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
    kvblock.read(*wide, table, zero, torch.tensor([0, 40], dtype=torch.int32, device="cuda"), k, v)
    torch.cuda.synchronize()
    for side, got in ((0, k), (1, v)):
        assert torch.equal(got.cpu(), c.rows(0, 0, 40, side).to(torch.bfloat16).expand(-1, 3, -1))
    with pytest.raises(_lib.MjolnirError, match="stride of 0"):
        kvblock.write(k, v, *wide, torch.arange(40, device="cuda"))
    r = kvblock.BlockAttention(num_heads=3, num_kv_heads=3, head_size=128, page_size=16, max_num_seqs=1, max_num_tokens=64)
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    for m in (1, 40):
        q = torch.zeros(m, 3, 128, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(_lib.MjolnirError, match="stride"):
            r.run(r.plan([m], [40], table, lens), q, torch.empty_like(q), *wide, 1.0)


@pytest.mark.gpu
def test_decode_with_shared_heads_runs_on_cuda_cores():
    """The other formats have a kernel that reads any strides."""
    from mjolnir_b200.runner import DecodeRunner
    from tests.block_helpers import Cache

    c = Cache([300, 41], h_k=1, split=True)
    shared = [x.expand(-1, -1, 2, -1) for x in c.kv]
    r = DecodeRunner(num_heads=8, num_kv_heads=2, head_size=128, page_size=16, max_num_seqs=2, kv_format="fp8", kernel="auto")
    plan = r.plan(c.lens, 2, 1, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda())
    q, one = torch.randn(2, 8, 128, generator=c.g).to(torch.bfloat16).cuda(), torch.full((1,), 1 / 64, device="cuda")
    outs = []
    for kv in (shared, [x.contiguous() for x in shared]):
        out = torch.empty_like(q)
        r.run(plan, q, out, *kv, one, one, 128**-0.5)
        torch.cuda.synchronize()
        r.check_status()
        outs.append(out.float())
    # two kernels of 32-bit sums, each rounded to bf16 once: within two roundings of one another
    assert ((outs[0] - outs[1]).abs() <= 2.0**-7 * outs[1].abs() + 1e-3).all()
