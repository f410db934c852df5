"""Attention over the block-scaled cache against the formula in 64 bits."""

import math

import pytest
import torch

from tests.block_helpers import Cache, assert_attention, attention_plain

pytestmark = pytest.mark.gpu


def _run(cache, q, q_lens, causal=True, lse=False, scale=None, runner=None, **kw):
    from mjolnir_b200 import kvblock

    r = runner or kvblock.BlockAttention(num_heads=q.shape[1], num_kv_heads=cache.h_k, head_size=cache.d, page_size=cache.page,
                                         block_tokens=cache.block, max_num_seqs=max(1, len(q_lens)),
                                         max_num_tokens=max(1, sum(q_lens)), **kw)
    lens = torch.tensor(cache.lens, dtype=torch.int32).cuda()
    plan = r.plan(q_lens, cache.lens, cache.table.cuda(), lens, causal=causal)
    T = q.shape[0]
    # rows inside a wider tensor: strided, with guard rows after
    qd = torch.zeros(T + 1, q.shape[1] + 2, cache.d, dtype=q.dtype, device="cuda")[:, :q.shape[1]]
    qd[:T] = q.cuda()
    od = torch.full((T + 1, q.shape[1] + 1, cache.d), 7.0, dtype=q.dtype, device="cuda")
    lse_t = torch.full((T, q.shape[1]), float("nan"), device="cuda") if lse else None
    r.run(plan, qd, od[:, :q.shape[1]], *cache.args, cache.d**-0.5 if scale is None else scale, lse=lse_t)
    torch.cuda.synchronize()
    r.check_status()
    assert (od[T:] == 7).all() and (od[:, q.shape[1]:] == 7).all(), "wrote a row it was not given"
    return od[:T, :q.shape[1]], lse_t


def _check(cache, q_lens, h_q, dtype=torch.bfloat16, causal=True, q_scale=1.0, scale=None, **kw):
    q = (torch.randn(sum(q_lens), h_q, cache.d, generator=cache.g) * q_scale).to(dtype)
    got, lse = _run(cache, q, q_lens, causal, True, scale, **kw)
    out, want_lse, mag = attention_plain(cache, q, q_lens, cache.d**-0.5 if scale is None else scale, causal)
    fine = q.isfinite().all(-1)  # a row with an infinity has no value
    got, lse, out, want_lse, mag = got.cpu()[fine], lse.double().cpu()[fine], out[fine], want_lse[fine], mag[fine]
    assert_attention(got, out, mag, f"{q_lens} / {cache.lens}")
    none = torch.isinf(want_lse)
    assert torch.equal(lse[none], want_lse[none])
    # scores of size up to ~|lse| from 32-bit sums of exact products, then a log
    assert ((lse - want_lse)[~none].abs() <= 2e-4 + 2e-5 * want_lse[~none].abs()).all()


@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("d,h_q,h_k", [(128, 8, 2), (256, 6, 1), (128, 3, 3)])
def test_ragged_chunks(page, block, d, h_q, h_k):
    q_lens = [1, 70, 5, 0, 129, 33]
    ctx = [300, 0, 17, 40, 128, 511]
    c = Cache([a + b for a, b in zip(q_lens, ctx)], h_k=h_k, d=d, page=page, block=block, seed=page + block + d)
    _check(c, q_lens, h_q, torch.bfloat16 if block != 16 else torch.float16)


@pytest.mark.parametrize("lens", [[1], [2, 1, 130, 127, 128, 129], [4000, 3], [1, 1, 1]])
@pytest.mark.parametrize("q_len", [1, 2, 3])
@pytest.mark.parametrize("d,h_q,h_k,page", [(128, 8, 2, 16), (128, 16, 1, 64), (256, 6, 2, 128)])
def test_few_tokens(lens, q_len, d, h_q, h_k, page):
    """Decode and draft steps; sequences shorter than the draft leave rows that see no key."""
    c = Cache(lens, h_k=h_k, d=d, page=page, block=16, seed=len(lens) + q_len)
    _check(c, [q_len] * len(lens), h_q)


def test_rows_that_see_nothing():
    c = Cache([0, 3, 0, 200, 1], h_k=2, seed=3)
    _check(c, [4, 9, 0, 7, 40], 4)
    _check(Cache([0], h_k=2), [1], 4)


def test_not_causal():
    _check(Cache([5, 300, 129], h_k=2, seed=4), [5, 100, 1], 8, causal=False)
    _check(Cache([50, 3000], h_k=2, seed=4), [2, 2], 8, causal=False)


@pytest.mark.parametrize("ctx", [5000, 20000])
def test_few_rows_over_a_long_context(ctx):
    """The work is split along the keys and joined."""
    _check(Cache([ctx + 17, 100], h_k=1, seed=5), [17, 3], 4)
    _check(Cache([ctx, ctx // 2 + 1], h_k=2, page=32, seed=6), [1, 1], 8)


@pytest.mark.parametrize("q_lens", [[600], [1, 1, 1]])
def test_growing_scores_and_wild_scales(q_lens):
    """Later keys raise the running maximum again and again; scales of
    neighbouring blocks differ by up to 2^20, so some values vanish beside
    others."""
    lens = [n + 900 for n in q_lens]
    _check(Cache(lens, h_k=2, seed=7, k_ramp=8.0), q_lens, 8, q_scale=4.0)
    _check(Cache(lens, h_k=2, seed=8, spread=10), q_lens, 8, q_scale=0.05)


def test_large_and_small_queries():
    c = Cache([400], h_k=1, seed=9)
    for q_scale, scale in ((3e4, 1e-6), (1e-5, 1e3), (6e4, 1e-7)):
        _check(c, [150], 4, torch.float16, q_scale=q_scale / 4, scale=scale)
        _check(c, [1], 4, torch.float16, q_scale=q_scale / 4, scale=scale)
    _check(c, [150], 4, torch.bfloat16, q_scale=1e20, scale=1e-22)


def test_separate_caches_and_head_last_scales():
    _check(Cache([333, 40], h_k=3, page=64, block=32, split=True, seed=10), [50, 40], 6)
    _check(Cache([333, 40], h_k=3, page=64, block=32, split=True, seed=11), [1, 1], 6)


def test_nan_query_stays_in_its_row():
    c = Cache([300], h_k=2, seed=12)
    q = torch.randn(200, 8, 128, generator=c.g).to(torch.bfloat16)
    q[77, 3, 5] = float("nan")
    got, _ = _run(c, q, [200])
    want, _, mag = attention_plain(c, q, [200], 128**-0.5)
    assert torch.isnan(got[77, 3]).all()
    fine = torch.ones(200, 8, dtype=torch.bool)
    fine[77, 3] = False
    assert_attention(got.cpu()[fine], want[fine], mag[fine])


@pytest.mark.parametrize("d,h_q,q_len,ctx,positions", [
    (128, 8, 150, 300, (449, 301, 420, 5)), (128, 8, 4, 300, (303, 301)), (128, 8, 3, 125, (127, 126)),
    (256, 4, 90, 0, (0, 89, 60)), (256, 4, 4, 126, (127, 129)), (128, 4, 1, 200, (200, 17)),
    (128, 8, 4, 9000, (9001, 9003)), (128, 8, 64, 5000, (5063, 5001, 4990))])
@pytest.mark.parametrize("causal", [True, False])
def test_nan_values_reach_only_the_rows_that_see_them(d, h_q, q_len, ctx, positions, causal):
    """K and V hold NaN at a few tokens: K's make the rows that see them NaN,
    V's only their own elements; rows before them are as without them."""
    c = Cache([q_len + ctx], h_k=2, d=d, seed=ctx + q_len)
    q = torch.randn(q_len, h_q, d, generator=c.g).to(torch.bfloat16)
    want, _, mag = attention_plain(c, q, [q_len], d**-0.5, causal=causal)
    nan = torch.zeros(q_len, h_q, d, dtype=torch.bool)
    limit = torch.arange(ctx, ctx + q_len) if causal else torch.full((q_len,), ctx + q_len - 1)
    for i, at in enumerate(positions):
        page, row = int(c.table[0, at // c.page]), at % c.page
        c.kv[1][page, row, 0, 3 + 31 * i] = 0x7F if i % 2 else 0xFF
        nan[limit >= at, : h_q // 2, 3 + 31 * i] = True
    key = positions[0]
    c.kv[0][int(c.table[0, key // c.page]), key % c.page, 1, 2] = 0x7F
    nan[limit >= key, h_q // 2:] = True
    got, _ = _run(c, q, [q_len], causal=causal)
    got = got.cpu()
    assert torch.equal(torch.isnan(got), nan)
    assert_attention(got[~nan], want[~nan], mag[~nan])


@pytest.mark.parametrize("q_len", [1, 40])
def test_nan_query_over_a_split_context(q_len):
    c = Cache([20000], h_k=1, seed=q_len)
    q = torch.randn(q_len, 2, 128, generator=c.g).to(torch.bfloat16)
    q[0, 1, 100] = float("nan")
    got, _ = _run(c, q, [q_len])
    want, _, mag = attention_plain(c, q, [q_len], 128**-0.5)
    assert torch.isnan(got[0, 1]).all()
    fine = torch.ones(q_len, 2, dtype=torch.bool)
    fine[0, 1] = False
    assert_attention(got.cpu()[fine], want[fine], mag[fine])


def test_bad_page_is_flagged():
    from mjolnir_b200 import _lib, kvblock

    for q_len in (1, 64):
        c = Cache([200, 100], h_k=2, seed=13)
        c.table[0, 2] = c.pages + 5
        q = torch.randn(2 * q_len, 8, 128, generator=c.g).to(torch.bfloat16)
        r = kvblock.BlockAttention(num_heads=8, num_kv_heads=2, head_size=128, page_size=16, max_num_seqs=2, max_num_tokens=128)
        with pytest.raises(_lib.MjolnirError, match="device status 1"):
            _run(c, q, [q_len, q_len], runner=r)
        c.table[0, 2] = 0
        _run(c, q, [q_len, q_len], runner=r)  # usable again


def test_plans_follow_one_another_and_replay_in_a_graph():
    """One runner, several plans; a captured step replays on another stream's order."""
    from mjolnir_b200 import kvblock

    c = Cache([500, 260], h_k=2, seed=14)
    r = kvblock.BlockAttention(num_heads=8, num_kv_heads=2, head_size=128, page_size=16, max_num_seqs=2, max_num_tokens=400)
    for q_lens in ([300, 60], [1, 1], [0, 7], [2, 2]):
        q = torch.randn(sum(q_lens), 8, 128, generator=c.g).to(torch.bfloat16)
        got, _ = _run(c, q, q_lens, runner=r)
        want, _, mag = attention_plain(c, q, q_lens, 128**-0.5)
        assert_attention(got, want, mag, str(q_lens))
    lens = torch.tensor(c.lens, dtype=torch.int32).cuda()
    for q_lens in ([40, 3], [1, 1]):
        n = sum(q_lens)
        q = torch.randn(n, 8, 128, generator=c.g).to(torch.bfloat16)
        qd, out = q.cuda(), torch.empty(n, 8, 128, dtype=torch.bfloat16, device="cuda")
        plan = r.plan(q_lens, c.lens, c.table.cuda(), lens)
        r.run(plan, qd, out, *c.args, 128**-0.5)
        torch.cuda.synchronize()
        first = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r.run(plan, qd, out, *c.args, 128**-0.5)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_the_same_call_gives_the_same_bits():
    c = Cache([9000, 41], h_k=1, seed=15)
    for q_lens in ([5, 41], [1, 1]):
        q = torch.randn(sum(q_lens), 8, 128, generator=c.g).to(torch.bfloat16)
        got = [_run(c, q, q_lens)[0].clone() for _ in range(3)]
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_pages_past_32_bit_offsets():
    from mjolnir_b200 import kvblock

    pages = (1 << 32) // (8 * 128 * 256) + 40
    views = kvblock.views(*kvblock.alloc(pages, 128, 8, 128, 16))
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.randn(300, 8, 128, device="cuda", generator=g).to(torch.bfloat16)
    y = torch.randn(300, 8, 128, device="cuda", generator=g).to(torch.bfloat16)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    pos = torch.arange(300)
    kvblock.write(x, y, *views, (table[0, pos // 128].long() * 128 + pos % 128).cuda())
    c = Cache([300], h_k=8, page=128, block=16)
    small = kvblock.views(*kvblock.alloc(c.pages, 128, 8, 128, 16))
    kvblock.write(x, y, *small, (c.table[0, pos // 128].long() * 128 + pos % 128).cuda())
    for m in (100, 1):
        q = torch.randn(m, 16, 128, device="cuda", generator=g).to(torch.bfloat16)
        outs = []
        for v, t in ((views, table), (small, c.table)):
            r = kvblock.BlockAttention(num_heads=16, num_kv_heads=8, head_size=128, page_size=128, max_num_seqs=1, max_num_tokens=100)
            plan = r.plan([m], [300], t.cuda(), torch.tensor([300], dtype=torch.int32, device="cuda"))
            outs.append(r.run(plan, q, torch.empty_like(q), *v, 128**-0.5))
            r.check_status()
        assert torch.equal(outs[0], outs[1]) and math.isfinite(outs[0].float().sum().item())


@pytest.mark.parametrize("merge", [True, False])
@pytest.mark.parametrize("d,h_q,page,block,q_len", [(128, 4, 16, 16, 1), (128, 8, 64, 64, 2), (128, 8, 128, 128, 7), (256, 6, 128, 32, 3)])
def test_decode_runner_on_block_formats(merge, d, h_q, page, block, q_len):
    """The formats through DecodeRunner itself: split merge inside the decode launch, or as a launch of its own."""
    from mjolnir_b200.runner import DecodeRunner

    c = Cache([2000, 77, 1], h_k=1, d=d, page=page, block=block, seed=q_len)
    r = DecodeRunner(num_heads=h_q, num_kv_heads=1, head_size=d, page_size=page, max_num_seqs=3, max_q_len=q_len,
                     kv_format=f"fp8b{block}", fused_merge=merge)
    q = torch.randn(3 * q_len, h_q, d, generator=c.g).to(torch.bfloat16)
    q[0, 1, 3] = float("nan")
    plan = r.plan(c.lens, 3, q_len, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda())
    assert plan.with_reduction
    out, one = torch.empty(3 * q_len, h_q, d, dtype=torch.bfloat16, device="cuda"), torch.ones(1, device="cuda")
    r.run(plan, q.cuda(), out, *c.args[:2], one, one, d**-0.5, k_scales=c.args[2], v_scales=c.args[3])
    torch.cuda.synchronize()
    r.check_status()
    want, _, mag = attention_plain(c, q, [q_len] * 3, d**-0.5)
    fine = torch.ones(3 * q_len, h_q, dtype=torch.bool)
    fine[0, 1] = False
    assert torch.isnan(out[0, 1]).all()
    assert_attention(out.cpu()[fine], want[fine], mag[fine])
    with pytest.raises(ValueError, match="needs k_scales"):
        r.run(plan, q.cuda(), out, *c.args[:2], one, one, d**-0.5)


def test_the_example_runs():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "examples", "block_cache.py")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "1942 tokens of 2 sequences" in r.stdout
