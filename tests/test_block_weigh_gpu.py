"""The weights that cached tokens receive, against their formula in 64 bits."""

import math

import pytest
import torch

from tests.block_helpers import Cache, attention_plain

pytestmark = pytest.mark.gpu


def weigh_plain(cache, q, lse, q_lens, old, scale, window=0):
    """(weights, bound of their error) in 64 bits, from the same lse. A score is
    a 32-bit sum of d exact products, then scaled and moved by the lse: off by at
    most d 2^-24 of the sum of its products' magnitudes and a few 2^-23 of itself
    and the lse, which is the weight's relative error; the sum of n weights adds
    n 2^-24 at most, the exponential 2^-21."""
    h_q, at, group = q.shape[1], 0, q.shape[1] // cache.h_k
    w, tol = old.double().clone(), old.double().abs() * 2.0**-23
    for s, (m, L) in enumerate(zip(q_lens, cache.lens)):
        w[s, :, max(L - m, 0):L] = 0
        k = cache.rows(s, 0, L, 0)
        first = max(m - window, 0) if window else 0
        sees = torch.arange(L)[None] <= torch.arange(L - m + first, L)[:, None]
        for h in range(h_q if m > first and L else 0):
            x, z = q[at + first:at + m, h].double(), lse[at + first:at + m, h].double()[:, None]
            sc, mag = x @ k[:, h // group].T * scale, x.abs() @ k[:, h // group].abs().T * abs(scale)
            p = torch.where(sees & (z != -math.inf), (sc - z).exp(), 0.0)
            n = (m - first) * group
            rel = cache.d * 2.0**-24 * mag + 2.0**-21 * (sc.abs() + z.abs()) + n * 2.0**-24 + 2.0**-21
            w[s, h // group, :L] += p.sum(0)
            tol[s, h // group, :L] += torch.where(p > 0, p * rel, 0.0).sum(0)
        at += m
    return w, tol + 1e-30


def offsets_of(q_lens):
    return torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")


def run(cache, q, lse, q_lens, old, scale, window=0, status=None):
    from mjolnir_b200 import kvblock

    n, most = len(q_lens), old.shape[2]
    wide = torch.full((n + 1, cache.h_k, most + 3), 5.0, device="cuda")  # strided, with guards behind
    wide[:n, :, :most] = old.cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda") if status is None else status
    got = kvblock.weigh(q, lse, cache.kv[0], cache.sc[0], cache.table.cuda(), offsets_of(q_lens),
                        torch.tensor(cache.lens, dtype=torch.int32, device="cuda"), wide[:, :, :most], scale, window=window, status=status)
    torch.cuda.synchronize()
    assert (wide[n:] == 5).all() and (wide[:, :, most:] == 5).all()
    return got[:n].cpu(), int(status)


def check(cache, q_lens, h_q, dtype=torch.bfloat16, window=0, q_scale=1.0, scale=None):
    q = (torch.randn(sum(q_lens), h_q, cache.d, generator=cache.g) * q_scale).to(dtype)
    scale = cache.d**-0.5 if scale is None else scale
    lse = attention_plain(cache, q, q_lens, scale)[1].float()
    most = max(cache.lens) + 5
    old = torch.rand(len(q_lens), cache.h_k, most, generator=cache.g) * (8 / most)
    # rows inside a wider tensor
    qd = torch.full((q.shape[0], h_q + 1, cache.d), float("nan"), dtype=dtype, device="cuda")[:, :h_q]
    qd.copy_(q)
    got, status = run(cache, qd, lse.cuda(), q_lens, old, scale, window)
    assert status == 0
    want, tol = weigh_plain(cache, q, lse, q_lens, old, scale, window)
    for s, L in enumerate(cache.lens):
        assert torch.equal(got[s, :, L:], old[s, :, L:]), "wrote behind the sequence"
        g, x = got[s, :, :L].double(), want[s, :, :L]
        assert torch.equal(torch.isnan(g), torch.isnan(x)), "a row with an infinity has weights of 0, or NaN where it is one of its scores"
        err = torch.where(torch.isnan(x), 0.0, (g - x).abs())
        assert (err <= tol[s, :, :L]).all(), (s, (err / tol[s, :, :L]).max().item())
    return got


@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("d,h_q,h_k", [(128, 8, 2), (256, 6, 1), (128, 3, 3)])
def test_ragged_chunks(page, block, d, h_q, h_k):
    q_lens = [1, 70, 5, 0, 129, 33]
    ctx = [300, 0, 17, 40, 128, 511]
    c = Cache([a + b for a, b in zip(q_lens, ctx)], h_k=h_k, d=d, page=page, block=block, seed=page + block + d)
    check(c, q_lens, h_q, torch.bfloat16 if block != 16 else torch.float16)


@pytest.mark.parametrize("lens", [[1], [2, 1, 130, 127, 128, 129], [4000, 3], [1, 1, 1]])
@pytest.mark.parametrize("q_len", [1, 2, 4])
@pytest.mark.parametrize("d,h_q,h_k,page", [(128, 8, 2, 16), (128, 40, 1, 64), (256, 6, 2, 128), (128, 8, 8, 16)])
def test_few_tokens(lens, q_len, d, h_q, h_k, page):
    """Decode and draft steps; sequences shorter than the draft leave rows that see no key."""
    check(Cache(lens, h_k=h_k, d=d, page=page, block=16, seed=len(lens) + q_len), [q_len] * len(lens), h_q)


@pytest.mark.parametrize("h_q", [80, 130, 257])
@pytest.mark.parametrize("d", [128, 256])
def test_many_heads_of_one_kv_head(h_q, d):
    check(Cache([150, 20], h_k=1, d=d, seed=h_q), [9, 1], h_q)


@pytest.mark.parametrize("window", [1, 16, 31, 400])
@pytest.mark.parametrize("d,h_q,h_k", [(128, 8, 2), (256, 6, 2), (128, 3, 1)])
def test_window(window, d, h_q, h_k):
    check(Cache([500, 40, 0, 7, 33], h_k=h_k, d=d, page=32, block=32, seed=window), [200, 40, 0, 1, 20], h_q, torch.float16, window)


def test_rows_that_see_nothing():
    check(Cache([0, 3, 0, 200, 1], h_k=2, seed=3), [4, 9, 0, 7, 40], 4)
    check(Cache([0], h_k=2), [1], 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_prompt(dtype):
    check(Cache([1500], h_k=1, seed=5), [1500], 5, dtype)
    check(Cache([20017, 100], h_k=1, seed=5), [17, 3], 4, dtype)


def test_wild_scales_and_growing_scores():
    check(Cache([900], h_k=2, seed=7, k_ramp=8.0), [600], 8, q_scale=4.0)
    check(Cache([900], h_k=2, seed=8, spread=10), [600], 8, q_scale=0.05)


def test_large_and_small_queries():
    c = Cache([400], h_k=1, seed=9)
    for q_scale, scale in ((3e4, 1e-6), (1e-5, 1e3), (6e4, 1e-7)):
        check(c, [150], 4, torch.float16, q_scale=q_scale / 4, scale=scale)
    check(c, [150], 4, torch.bfloat16, q_scale=1e20, scale=1e-22)


def test_separate_caches_and_head_last_scales():
    check(Cache([333, 40], h_k=3, page=64, block=32, split=True, seed=10), [50, 40], 6)


def test_weights_of_a_step_sum_to_its_rows():
    """After the attention itself: every row's weights are 1 together."""
    from mjolnir_b200 import kvblock

    q_lens = [1, 1, 1]
    c = Cache([700, 3, 129], h_k=2, seed=13)
    r = kvblock.BlockAttention(num_heads=8, num_kv_heads=2, head_size=128, page_size=16, max_num_seqs=3, max_num_tokens=256)
    for q_lens in ([1, 1, 1], [200, 3, 50]):
        lens, table = torch.tensor(c.lens, dtype=torch.int32).cuda(), c.table.cuda()
        plan = r.plan(q_lens, c.lens, table, lens)
        q = torch.randn(sum(q_lens), 8, 128, generator=c.g).bfloat16().cuda()
        lse = torch.empty(sum(q_lens), 8, device="cuda")
        r.run(plan, q, torch.empty_like(q), *c.args, 128**-0.5, lse=lse)
        w = torch.zeros(3, 2, 700, device="cuda")
        kvblock.weigh(q, lse, c.kv[0], c.sc[0], table, offsets_of(q_lens), lens, w, 128**-0.5)
        # P of the attention rounds, its row sum does not: the sums agree to what the lse's score arithmetic leaves
        want = torch.tensor(q_lens)[:, None] * 4.0
        assert ((w.double().sum(-1).cpu() - want).abs() <= 1e-4 * want).all()


def test_nan_and_infinite_lse():
    """A NaN lse reaches the keys its row sees, -inf none, +inf adds 0."""
    c = Cache([300], h_k=2, seed=14)
    q = torch.randn(100, 8, 128, generator=c.g).bfloat16()
    lse = attention_plain(c, q, [100], 128**-0.5)[1].float()
    lse[40, 1], lse[50, 6], lse[60, 7] = math.nan, -math.inf, math.inf
    old = torch.zeros(1, 2, 300)
    got, _ = run(c, q.cuda(), lse.cuda(), [100], old, 128**-0.5)
    lse[40, 1] = 0.0
    want, tol = weigh_plain(c, q, lse, [100], old, 128**-0.5)
    assert torch.isnan(got[0, 0, :241]).all() and not torch.isnan(got[0, 0, 241:]).any() and not torch.isnan(got[0, 1]).any()
    assert ((got[0, 1].double() - want[0, 1]).abs() <= tol[0, 1]).all()


def test_nan_rows_of_other_sequences_and_pages():
    """Q rows and pages that belong to no sequence of the call hold NaN; so do a neighbour's rows."""
    c = Cache([65, 40], h_k=1, seed=15)
    q = torch.randn(13, 4, 128, generator=c.g).bfloat16()
    q[5:] = math.nan
    lse = torch.full((13, 4), math.nan)
    lse[:5] = attention_plain(c, torch.nan_to_num(q), [5, 8], 128**-0.5)[1][:5].float()
    old = torch.zeros(2, 1, 65)
    got, _ = run(c, q.cuda(), lse.cuda(), [5, 8], old, 128**-0.5)
    want, tol = weigh_plain(c, q[:5], lse[:5], [5, 0], old, 128**-0.5)
    assert ((got[0].double() - want[0]).abs() <= tol[0]).all()
    assert torch.isnan(got[1, :, :40]).all()


def test_bad_lengths_and_pages():
    from mjolnir_b200 import _lib

    c = Cache([100, 60], h_k=2, seed=16)
    q = torch.randn(2, 4, 128, generator=c.g).bfloat16()
    lse = attention_plain(c, q, [1, 1], 128**-0.5)[1].float()
    old = torch.rand(2, 2, 90, generator=c.g)  # the first does not fit
    got, status = run(c, q.cuda(), lse.cuda(), [1, 1], old, 128**-0.5)
    want, tol = weigh_plain(c, q, lse, [1, 1], torch.cat([old, torch.zeros(2, 2, 10)], -1), 128**-0.5)
    assert status == _lib.MJ_DEV_BAD_LENGTH
    assert torch.equal(got[0], old[0]) and ((got[1].double() - want[1, :, :90]).abs() <= tol[1, :, :90]).all()
    got, status = run(c, q.cuda(), lse.cuda(), [1, 5], torch.zeros(2, 2, 100), 128**-0.5)  # rows past the end of q
    assert status == _lib.MJ_DEV_BAD_LENGTH and (got[1] == 0).all()
    for bad in (-1, c.pages):
        c.table[0, 3] = bad
        got, status = run(c, q.cuda(), lse.cuda(), [1, 1], torch.zeros(2, 2, 100), 128**-0.5)
        assert status == _lib.MJ_DEV_BAD_PAGE
        keep = [j for j in range(100) if j // 16 != 3]
        w, t = want[:, :, :100], tol[:, :, :100]
        assert ((got[0][:, keep].double() - (w[0] - torch.cat([old, torch.zeros(2, 2, 10)], -1)[0] * (torch.arange(100) < 99))[:, keep]).abs()
                <= t[0][:, keep] + 2.0**-20).all()


def test_same_result_twice_and_from_a_graph():
    """Sums in a fixed order: bit-identical; a graph replays for later lengths and offsets."""
    from mjolnir_b200 import kvblock

    c = Cache([700, 3, 1029], h_k=2, seed=17)
    q_lens = [33, 3, 70]
    q = torch.randn(sum(q_lens), 8, 128, generator=c.g).bfloat16()
    lse = attention_plain(c, q, q_lens, 128**-0.5)[1].float()
    qd, ld, table = q.cuda(), lse.cuda(), c.table.cuda()
    offsets, lens = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    w = torch.zeros(3, 2, 1029, device="cuda")
    step = lambda: kvblock.weigh(qd, ld, c.kv[0], c.sc[0], table, offsets, lens, w, 128**-0.5)  # noqa: E731
    step()
    torch.cuda.synchronize()
    assert (w == 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    offsets.copy_(offsets_of(q_lens))
    lens.copy_(torch.tensor(c.lens))
    seen = []
    for _ in range(3):
        w.zero_()
        graph.replay()
        seen.append(w.cpu())
    assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[2])
    want, tol = weigh_plain(c, q, lse, q_lens, torch.zeros(3, 2, 1029), 128**-0.5)
    assert ((seen[0].double() - want).abs() <= tol).all()


def test_on_another_stream():
    from mjolnir_b200 import kvblock

    c = Cache([5000, 700], h_k=2, seed=18)
    q = torch.randn(2, 8, 128, generator=c.g).bfloat16()
    lse = attention_plain(c, q, [1, 1], 128**-0.5)[1].float()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros(2, 2, 5000, device="cuda") for _ in range(2)]
    args = (q.cuda(), lse.cuda(), c.kv[0], c.sc[0], c.table.cuda(), offsets_of([1, 1]), torch.tensor(c.lens, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    for s, w in zip(streams, outs):  # two calls at once
        with torch.cuda.stream(s):
            for _ in range(3):
                kvblock.weigh(*args, w, 128**-0.5)
    torch.cuda.synchronize()
    want, tol = weigh_plain(c, q, lse, [1, 1], torch.zeros(2, 2, 5000), 128**-0.5)
    for w in outs:
        fresh = torch.zeros(2, 2, 5000, dtype=torch.bool)
        for s, L in enumerate(c.lens):
            fresh[s, :, L - 1] = True  # the step's own token starts anew each time
        total = torch.where(fresh, want, 3 * want)
        assert ((w.cpu().double() - total).abs() <= 4 * tol).all()


@pytest.mark.parametrize("d,h_q,h_k,page", [(128, 8, 2, 16), (256, 5, 1, 64), (128, 16, 1, 32)])
@pytest.mark.parametrize("window", [0, 3])
def test_single_tokens_beside_chunks(d, h_q, h_k, page, window):
    """A sequence of few rows and one of many go different ways in one call; more than 32 sequences."""
    q_lens = [1, 140, 1, 0, 4, 1, 17, 2] + [1] * 30 + [3, 66]
    ctx = [300, 5, 128, 12, 0, 700, 255, 40] + [9 * i for i in range(30)] + [127, 400]
    check(Cache([a + b for a, b in zip(q_lens, ctx)], h_k=h_k, d=d, page=page, seed=d + window), q_lens, h_q, window=window)


def test_no_more_tokens_than_sequences():
    """All taken for single ones, yet one has most of them."""
    check(Cache([90, 300, 0, 7] + [0] * 200, h_k=2, seed=21), [1, 150, 0, 2] + [0] * 200, 8)


def test_graph_whose_sequences_change_places():
    """Captured with a chunk and single tokens, replayed with the chunk elsewhere, grown or gone."""
    from mjolnir_b200 import kvblock

    c = Cache([400, 300, 500], h_k=2, seed=22)
    q = torch.randn(120, 8, 128, generator=c.g).bfloat16()
    qd, table, lens = q.cuda(), c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    ld, offsets, w = torch.zeros(120, 8, device="cuda"), offsets_of([1, 70, 1]), torch.zeros(3, 2, 500, device="cuda")
    graph = torch.cuda.CUDAGraph()
    kvblock.weigh(qd, ld, c.kv[0], c.sc[0], table, offsets, lens, w, 128**-0.5)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kvblock.weigh(qd, ld, c.kv[0], c.sc[0], table, offsets, lens, w, 128**-0.5)
    for q_lens in ([1, 70, 1], [70, 1, 1], [1, 1, 1], [60, 0, 60], [4, 5, 3]):
        n = sum(q_lens)
        lse = attention_plain(c, q[:n], q_lens, 128**-0.5)[1].float()
        ld[:n] = lse.cuda()
        offsets.copy_(offsets_of(q_lens))
        w.zero_()
        graph.replay()
        want, tol = weigh_plain(c, q[:n], lse, q_lens, torch.zeros(3, 2, 500), 128**-0.5)
        assert ((w.cpu().double() - want).abs() <= tol).all(), q_lens


def test_heads_outermost():
    """Weights as (heads, sequences, tokens) in memory, K's views of a cache whose heads are outermost too."""
    from mjolnir_b200 import kvblock

    c = Cache([260, 45], h_k=2, seed=23)
    q = torch.randn(31, 6, 128, generator=c.g).bfloat16()
    lse = attention_plain(c, q, [30, 1], 128**-0.5)[1].float()
    k = c.kv[0].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    e = c.sc[0].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    w = torch.zeros(2, 2, 260, device="cuda").transpose(0, 1)
    kvblock.weigh(q.cuda(), lse.cuda(), k, e, c.table.cuda(), offsets_of([30, 1]), torch.tensor(c.lens, dtype=torch.int32, device="cuda"), w, 128**-0.5)
    want, tol = weigh_plain(c, q, lse, [30, 1], torch.zeros(2, 2, 260), 128**-0.5)
    assert ((w.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("q_lens", [[1, 2, 1], [1, 90, 1]])
def test_rows_that_are_not_finite(q_lens, d):
    """A row with a NaN makes the keys it sees NaN, one with an infinity at most touches them; nothing else."""
    c = Cache([200, 200, 140], h_k=2, d=d, seed=24)
    q = torch.randn(sum(q_lens), 8, d, generator=c.g).bfloat16()
    lse = attention_plain(c, q, q_lens, d**-0.5)[1].float()
    old = torch.zeros(3, 2, 200)
    want, tol = weigh_plain(c, q, lse, q_lens, old, d**-0.5)
    q[0, 1, 7], q[1, 6, 9] = math.nan, math.inf
    got, status = run(c, q.cuda(), lse.cuda(), q_lens, old, d**-0.5)
    ok = (got.double() - want).abs() <= tol
    sees = 200 - q_lens[1] + 1  # of the row with the infinity
    assert status == 0 and torch.isnan(got[0, 0]).all() and ok[0, 1].all() and ok[1, 0].all() and ok[1, 1, sees:].all() and ok[2].all()


@pytest.mark.parametrize("lens,q_lens,d,h_q,h_k,window", [
    ([1000], [1000], 128, 6, 1, 0), ([700], [100], 128, 6, 1, 0), ([2600], [700], 128, 5, 1, 0), ([2600], [701], 256, 6, 1, 100),
    ([1200, 900, 40], [1200, 300, 40], 128, 8, 4, 0), ([1500], [1500], 256, 6, 3, 0), ([150, 300], [60, 90], 128, 257, 1, 0),
    ([3000, 1, 800], [600, 1, 800], 128, 12, 2, 0), ([900, 300, 0, 5], [900, 300, 0, 5], 128, 12, 3, 200), ([400], [399], 128, 40, 1, 0),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_jobs_of_many_rows(lens, q_lens, d, h_q, h_k, window, dtype):
    """Jobs whose rows the CTAs of a cluster share: two, four and eight, with and without a tile for each; the same bits every time."""
    c = Cache(lens, h_k=h_k, d=d, page=32, seed=sum(lens) + h_q)
    state = c.g.get_state()
    first = check(c, q_lens, h_q, dtype, window)
    c.g.set_state(state)
    again = check(c, q_lens, h_q, dtype, window)
    assert torch.equal(first, again)


def test_shared_jobs_of_two_calls_at_once():
    from mjolnir_b200 import kvblock

    c = Cache([900, 500], h_k=2, seed=25)
    q_lens = [900, 400]
    q = torch.randn(1300, 8, 128, generator=c.g).bfloat16()
    lse = attention_plain(c, q, q_lens, 128**-0.5)[1].float()
    args = (q.cuda(), lse.cuda(), c.kv[0], c.sc[0], c.table.cuda(), offsets_of(q_lens), torch.tensor(c.lens, dtype=torch.int32, device="cuda"))
    outs = [torch.zeros(2, 2, 900, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    for w in outs:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(4):
                w.zero_()
                kvblock.weigh(*args, w, 128**-0.5)
    torch.cuda.synchronize()
    want, tol = weigh_plain(c, q, lse, q_lens, torch.zeros(2, 2, 900), 128**-0.5)
    for w in outs:
        assert ((w.cpu().double() - want).abs() <= tol).all()


def test_offsets_that_fall():
    """Flagged, whichever kernel the others go to; they are done all the same."""
    from mjolnir_b200 import _lib, kvblock

    c = Cache([50, 60, 70], h_k=1, seed=26)
    q = torch.randn(40, 4, 128, generator=c.g).bfloat16()
    for offsets, ok in (([0, 1, 0, 0], 0), ([5, 0, 0, 0], None), ([0, 30, 29, 29], 0), ([0, 0, 30, 29], 1)):
        lse, status, w = torch.zeros(40, 4), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(3, 1, 70, device="cuda")
        if ok is not None:
            n = offsets[ok + 1] - offsets[ok]
            rows = [n if s == ok else 0 for s in range(3)]
            lse[offsets[ok]:offsets[ok] + n] = attention_plain(c, q[offsets[ok]:offsets[ok] + n], rows, 128**-0.5)[1].float()
        kvblock.weigh(q.cuda(), lse.cuda(), c.kv[0], c.sc[0], c.table.cuda(), torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                      torch.tensor(c.lens, dtype=torch.int32, device="cuda"), w, 128**-0.5, status=status)
        assert int(status) == _lib.MJ_DEV_BAD_LENGTH
        want, tol = torch.zeros(3, 1, 70, dtype=torch.float64), torch.zeros(3, 1, 70, dtype=torch.float64)
        if ok is not None:
            want, tol = weigh_plain(c, q[offsets[ok]:], lse[offsets[ok]:], rows, torch.zeros(3, 1, 70), 128**-0.5)
        assert ((w.cpu().double() - want).abs() <= tol).all()
