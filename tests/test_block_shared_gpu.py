"""Attention of sequences that share a cached prefix against the formula in 64 bits."""

import pytest
import torch

from tests.block_helpers import Cache, assert_attention, attention_plain

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def share(monkeypatch, request):
    """Small steps are not worth sharing: these tests share all the same."""
    from mjolnir_b200 import kvblock

    if request.node.name != "test_sharing_where_it_pays":
        monkeypatch.setattr(kvblock.BlockAttention, "_worth", lambda self, *a: True)


class Shared(Cache):
    """A cache whose groups (first, count, tokens) have their first whole pages in common."""

    def __init__(self, lens, groups, **kw):
        super().__init__(lens, **kw)
        for first, count, tokens in groups:
            pages = tokens // self.page
            for s in range(first + 1, first + count):
                self.table[s, :min(pages, -(-self.lens[s] // self.page))] = self.table[first, :min(pages, -(-self.lens[s] // self.page))]


def runner(c, h_q, q_lens, **kw):
    from mjolnir_b200 import kvblock

    return kvblock.BlockAttention(num_heads=h_q, num_kv_heads=c.h_k, head_size=c.d, page_size=c.page, block_tokens=c.block,
                                  max_num_seqs=len(q_lens), max_num_tokens=max(1, sum(q_lens)), **kw)


def check(c, q_lens, groups, h_q, dtype=torch.bfloat16, causal=True, r=None, shares=True, q=None, scale=None):
    r = r or runner(c, h_q, q_lens)
    T = sum(q_lens)
    q = (torch.randn(T, h_q, c.d, generator=c.g)).to(dtype) if q is None else q
    scale = c.d**-0.5 if scale is None else scale
    plan = r.plan(q_lens, c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda(), causal=causal, shared=groups)
    assert (plan.joins is not None) == shares
    qd = torch.zeros(T + 1, h_q + 2, c.d, dtype=dtype, device="cuda")[:, :h_q]
    qd[:T] = q.cuda()
    od = torch.full((T + 1, h_q + 1, c.d), 7.0, dtype=dtype, device="cuda")
    lse = torch.full((T, h_q), float("nan"), device="cuda")
    r.run(plan, qd, od[:, :h_q], *c.args, scale, lse=lse)
    torch.cuda.synchronize()
    r.check_status()
    assert (od[T:] == 7).all() and (od[:, h_q:] == 7).all(), "wrote a row it was not given"
    out, want_lse, mag = attention_plain(c, q, q_lens, scale, causal)
    got = od[:T, :h_q].cpu()
    assert_attention(got, out, mag, f"{q_lens} / {c.lens} / {groups}")
    none = torch.isinf(want_lse)
    lse = lse.double().cpu()
    assert torch.equal(lse[none], want_lse[none])
    # scores of size up to ~|lse| from 32-bit sums of exact products, then a log
    assert ((lse - want_lse)[~none].abs() <= 2e-4 + 2e-5 * want_lse[~none].abs()).all()
    return got


@pytest.mark.parametrize("q_len", [1, 2, 4])
@pytest.mark.parametrize("d,h_q,h_k,page,dtype", [(128, 8, 2, 16, torch.bfloat16), (128, 40, 8, 64, torch.float16), (256, 6, 2, 128, torch.bfloat16),
                                                  (256, 24, 4, 32, torch.float16), (128, 3, 3, 128, torch.bfloat16)])
def test_decode_steps(q_len, d, h_q, h_k, page, dtype):
    groups = [(0, 5, 1536)]
    c = Shared([1536 + x for x in (4, 700, 33, 128, 129)], groups, h_k=h_k, d=d, page=page, block=16, seed=page + q_len)
    check(c, [q_len] * 5, groups, h_q, dtype)


@pytest.mark.parametrize("page,block", [(16, 16), (32, 32), (64, 16), (128, 128)])
@pytest.mark.parametrize("d,h_q,h_k", [(128, 8, 2), (256, 6, 2), (128, 3, 1)])
def test_ragged_chunks(page, block, d, h_q, h_k):
    """Chunks, single tokens and sequences without queries in groups of every kind, some sequences in none."""
    q_lens = [1, 1, 1, 30, 0, 77, 5, 130, 9, 1]
    groups = [(1, 4, 640), (5, 1, 256), (6, 3, 1280)]
    lens = [300, 641, 900, 680, 640, 340, 1285, 1500, 1290, 64]
    c = Shared(lens, groups, h_k=h_k, d=d, page=page, block=block, seed=page + d)
    check(c, q_lens, groups, h_q, torch.float16 if block == 16 else torch.bfloat16)


def test_prefix_that_ends_inside_a_tile():
    """The rest of a prefix behind its last whole tile is read with each sequence."""
    groups = [(0, 3, 1500 // 16 * 16)]
    c = Shared([1500, 1501, 2000], groups, seed=1)
    check(c, [1, 1, 1], groups, 8)
    check(c, [4, 4, 400], groups, 8)


def test_no_tokens_behind_the_prefix():
    """Every cached token is shared; the queries' own ones alone are not."""
    groups = [(0, 4, 1024)]
    check(Shared([1025] * 4, groups, seed=2), [1] * 4, groups, 8)
    check(Shared([1034] * 4, groups, seed=2), [10] * 4, groups, 8)
    check(Shared([1024] * 4, groups, seed=3), [1] * 4, groups, 8, causal=False)
    check(Shared([1024] * 4, groups, seed=3), [9] * 4, groups, 8, causal=False)


@pytest.mark.parametrize("q_lens", [[1] * 70, [12] * 20, [40] * 9 + [300]])
def test_many_sequences(q_lens):
    """Several row blocks of a group; long prefixes are split along their keys."""
    groups = [(0, len(q_lens), 4096)]
    c = Shared([4096 + n + 5 * i for i, n in enumerate(q_lens)], groups, h_k=2, seed=len(q_lens))
    check(c, q_lens, groups, 16)


def test_sharing_where_it_pays():
    """The plan's own choice: many sequences behind a long prefix share, a few behind a short one do not."""
    for q_len in (1, 20):
        groups = [(0, 3, 256)]
        check(Shared([300, 290, 310], groups, seed=4), [q_len] * 3, groups, 8, shares=False)
        n = 40 if q_len == 1 else 8
        groups = [(0, n, 4096)]
        check(Shared([4096 + q_len + i for i in range(n)], groups, h_k=8, page=64, seed=5), [q_len] * n, groups, 32)


def test_not_causal():
    groups = [(0, 3, 512)]
    c = Shared([600, 515, 700], groups, seed=4)
    check(c, [2, 2, 2], groups, 8, causal=False)
    check(c, [2, 80, 600], groups, 8, causal=False)


def test_too_little_to_share():
    """Groups of one, of less than a tile, of one sequence with queries, or of tokens that a query precedes."""
    c = Shared([200, 201, 50], [], seed=5)
    for groups in ([(0, 1, 128)], [(0, 2, 127)], [(0, 3, 128)], []):
        check(c, [1, 1, 1], groups, 8, shares=False)
    check(Shared([200, 201], [(0, 2, 128)], seed=5), [100, 1], [(0, 2, 128)], 8, shares=False)
    check(Shared([200, 201], [(0, 2, 128)], seed=5), [0, 1], [(0, 2, 128)], 8, shares=False)


def test_runner_serves_plans_of_both_kinds():
    groups = [(0, 3, 768)]
    c = Shared([800, 900, 1000], groups, seed=6)
    r = runner(c, 8, [60] * 3)
    a = check(c, [1, 1, 1], groups, 8, r=r, q=torch.ones(3, 8, 128).bfloat16())
    b = check(c, [1, 1, 1], [], 8, r=r, shares=False, q=torch.ones(3, 8, 128).bfloat16())
    check(c, [50, 1, 9], groups, 8, r=r)
    check(c, [50, 1, 9], [], 8, r=r, shares=False)
    assert (a.float() - b.float()).abs().max() <= 2.0**-7 * b.float().abs().max()


@pytest.mark.parametrize("q_len", [1, 20])
def test_wild_scales_and_scores(q_len):
    groups = [(0, 4, 896)]
    for kw, scale in ((dict(k_ramp=8.0), 0.5), (dict(spread=10), 0.005)):
        c = Shared([1000 + 9 * i for i in range(4)], groups, seed=7, **kw)
        check(c, [q_len] * 4, groups, 8, scale=scale)


@pytest.mark.parametrize("q_len", [1, 30])
def test_nan_reaches_the_rows_that_see_it(q_len):
    """A NaN in the shared keys reaches every sequence; one behind them its own alone; a NaN query its row."""
    groups = [(0, 3, 512)]
    for at, who in (((0, 100), (0, 1, 2)), ((1, 530), (1,))):
        c = Shared([600, 620, 640], groups, seed=8)
        c.kv[0][int(c.table[at[0], at[1] // 16]), at[1] % 16, 0, 3] = 0x7F
        q = torch.randn(3 * q_len, 4, 128, generator=c.g).bfloat16()
        r = runner(c, 4, [q_len] * 3)
        plan = r.plan([q_len] * 3, c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda(), shared=groups)
        out = r.run(plan, q.cuda(), torch.zeros_like(q, device="cuda"), *c.args, 128**-0.5).cpu()
        want = torch.zeros(3 * q_len, 4, dtype=torch.bool)
        for s in who:
            want[s * q_len:(s + 1) * q_len, :2] = True
        assert torch.equal(torch.isnan(out).all(-1), want) and torch.equal(torch.isnan(out).any(-1), want)
    c = Shared([600, 620, 640], groups, seed=8)
    q = torch.randn(3 * q_len, 4, 128, generator=c.g).bfloat16()
    q[q_len, 2, 7] = float("nan")
    r = runner(c, 4, [q_len] * 3)
    plan = r.plan([q_len] * 3, c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda(), shared=groups)
    out = r.run(plan, q.cuda(), torch.zeros_like(q, device="cuda"), *c.args, 128**-0.5).cpu()
    want = torch.zeros(3 * q_len, 4, dtype=torch.bool)
    want[q_len, 2] = True
    assert torch.equal(torch.isnan(out).all(-1), want) and torch.equal(torch.isnan(out).any(-1), want)


def test_graph_replays_later_plans_that_share_alike():
    groups = [(1, 3, 1024)]
    a, b = ([300, 1030, 1100, 2000], [900, 4000, 1026, 1500])
    ca = Shared([max(x, y) for x, y in zip(a, b)], groups, seed=9)
    r = runner(ca, 8, [1] * 4)
    q = torch.randn(4, 8, 128, generator=ca.g).bfloat16()
    qd, out, table = q.cuda(), torch.zeros(4, 8, 128, dtype=torch.bfloat16, device="cuda"), ca.table.cuda()
    lens = torch.tensor(a, dtype=torch.int32).cuda()
    plan = r.plan([1] * 4, a, table, lens, fixed_grid=True, shared=groups)
    r.run(plan, qd, out, *ca.args, 128**-0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.run(plan, qd, out, *ca.args, 128**-0.5)
    for now in (b, a):
        lens.copy_(torch.tensor(now))
        r.plan([1] * 4, now, table, lens, fixed_grid=True, shared=groups)
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        r.check_status()
        ca.lens = now
        want, _, mag = attention_plain(ca, q, [1] * 4, 128**-0.5)
        assert_attention(out, want, mag)


def test_weights_of_a_step_behind_a_shared_prefix():
    """The lse that such a step leaves serves the weights: every row's are 1 together."""
    from mjolnir_b200 import kvblock

    groups, q_lens = [(0, 4, 640)], [1, 1, 1, 25]
    c = Shared([700, 645, 900, 680], groups, seed=10)
    r = runner(c, 8, q_lens)
    lens, table = torch.tensor(c.lens, dtype=torch.int32).cuda(), c.table.cuda()
    plan = r.plan(q_lens, c.lens, table, lens, shared=groups)
    q = torch.randn(sum(q_lens), 8, 128, generator=c.g).bfloat16().cuda()
    lse = torch.empty(sum(q_lens), 8, device="cuda")
    r.run(plan, q, torch.empty_like(q), *c.args, 128**-0.5, lse=lse)
    w = torch.zeros(4, 2, 900, device="cuda")
    offsets = torch.tensor([0, 1, 2, 3, 28], dtype=torch.int32, device="cuda")
    kvblock.weigh(q, lse, c.kv[0], c.sc[0], table, offsets, lens, w, 128**-0.5)
    want = torch.tensor(q_lens)[:, None] * 4.0
    assert ((w.double().sum(-1).cpu() - want).abs() <= 1e-4 * want).all()


def test_items_out_of_range_are_flagged():
    """Spans, slots and joins that point outside are reported, not followed."""
    from mjolnir_b200 import _lib

    groups = [(0, 3, 512)]
    c = Shared([600, 620, 640], groups, seed=11)
    r = runner(c, 8, [1] * 3)
    lens, table, q = torch.tensor(c.lens, dtype=torch.int32).cuda(), c.table.cuda(), torch.randn(3, 8, 128).bfloat16().cuda()
    for where, at, value in (("work", (0, 5), 4), ("work", (0, 5), -1), ("work", (0, 4), 10**6), ("joins", (1, 0), 3), ("joins", (0, 1), 9),
                             ("joins", (2, 4), 10**6), ("joins", (0, 5), 10**6), ("joins", (1, 6), 10**6), ("joins", (1, 7), 3000), ("joins", (1, 8), 10**8)):
        plan = r.plan([1] * 3, c.lens, table, lens, shared=groups)
        getattr(plan, where)[at] = value
        r.run(plan, q, torch.empty_like(q), *c.args, 128**-0.5)
        torch.cuda.synchronize()
        with pytest.raises(_lib.MjolnirError, match=f"status {_lib.MJ_DEV_BAD_SPLIT}"):
            r.check_status()
    check(c, [1] * 3, groups, 8, r=r)
