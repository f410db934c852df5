"""Eviction by weight against a plain implementation: every byte."""

import math

import numpy as np
import pytest
import torch

from oracle import quant
from tests.block_helpers import Cache, codes_of, exponent

pytestmark = pytest.mark.gpu


def kept_plain(w, L, budget, recent):
    """The tokens that one KV head keeps: float32 weights (>= L,)."""
    if L <= budget:
        return list(range(L)) + [-1] * (budget - L)
    old = w[:L - recent].tolist()
    order = sorted(range(L - recent), key=lambda t: (0 if math.isnan(old[t]) else 1, 0 if math.isnan(old[t]) else -old[t], t))
    return sorted(order[:budget - recent]) + list(range(L - recent, L))


def evict_plain(cache, weights, budget, recent):
    """(codes, exps, weights, kept) as numpy / torch copies after the eviction."""
    codes, exps = cache.codes.numpy().copy(), cache.exps.numpy().copy()
    w = weights.clone()
    kept = torch.full((len(cache.lens), cache.h_k, budget), -1, dtype=torch.int32)
    page, block = cache.page, cache.block
    for s, L in enumerate(cache.lens):
        for h in range(cache.h_k):
            keep = kept_plain(weights[s, h], L, budget, recent)
            kept[s, h] = torch.tensor(keep, dtype=torch.int32)
            if L <= budget:
                continue
            w[s, h, :budget] = weights[s, h, keep]
            pos = np.arange(L)
            pg, row = cache.table[s].numpy()[pos // page], pos % page
            for side in range(2):
                e_old = np.clip(cache.exps.numpy()[side][pg, row // block, h].astype(int), 95, 159)
                x = quant.decode_fp8(cache.codes.numpy()[side][pg, row, h]).astype(np.float64) * 2.0 ** (e_old - 127.0)[:, None]
                for b in range(0, budget, block):
                    part = x[keep[b:b + block]]
                    fine = np.abs(part[np.isfinite(part)])
                    e = exponent(fine.max() if fine.size else 0.0)
                    exps[side][pg[b], row[b] // block, h] = e
                    for i in range(len(part)):
                        codes[side][pg[b + i], row[b + i], h] = codes_of(part[i], e)
    return codes, exps, w, kept


def run(cache, weights, budget, recent, status=None):
    from mjolnir_b200 import kvblock

    n = len(cache.lens)
    wide = torch.full((n + 1, cache.h_k, weights.shape[2] + 3), 5.0, device="cuda")
    wide[:n, :, :weights.shape[2]] = weights.cuda()
    new = torch.full((n + 1,), -9, dtype=torch.int32, device="cuda")
    kept = torch.full((n + 1, cache.h_k, budget), -9, dtype=torch.int32, device="cuda")
    lens = torch.tensor(cache.lens, dtype=torch.int32, device="cuda")
    kvblock.evict(wide[:, :, :weights.shape[2]], *cache.args, cache.table.cuda(), lens, new[:n], kept[:n], recent=recent, status=status)
    torch.cuda.synchronize()
    assert (wide[n:] == 5).all() and (wide[:, :, weights.shape[2]:] == 5).all() and (kept[n:] == -9).all() and int(new[n]) == -9
    codes = [x.cpu().numpy() for x in cache.kv]
    exps = [x.cpu().numpy() for x in cache.sc]
    return codes, exps, wide[:n, :, :weights.shape[2]].cpu(), new[:n].cpu(), kept[:n].cpu()


def check(cache, budget, recent, weights=None):
    most = max([1, *cache.lens])
    if weights is None:
        weights = torch.rand(len(cache.lens), cache.h_k, most, generator=cache.g)
        weights[torch.rand(weights.shape, generator=cache.g) < 0.3] = 0.25  # ties
    codes, exps, w, new, kept = run(cache, weights, budget, recent)
    want = evict_plain(cache, weights, budget, recent)
    assert torch.equal(kept, want[3])
    assert new.tolist() == [min(L, budget) for L in cache.lens]
    assert np.array_equal(w.numpy(), want[2].numpy(), equal_nan=True)
    for side in range(2):
        assert np.array_equal(exps[side], want[1][side]), "exponents"
        assert np.array_equal(codes[side] & 0x7F, want[0][side] & 0x7F), "magnitudes"
        nan = (want[0][side] & 0x7F) == 0x7F
        assert np.array_equal(codes[side][~nan], want[0][side][~nan]), "signs"


@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (128, 32), (128, 128), (48, 16), (96, 32)])
@pytest.mark.parametrize("d,h_k", [(128, 2), (256, 1), (128, 3)])
@pytest.mark.parametrize("budget,recent", [(40, 8), (129, 0), (17, 17)])
def test_bytes(page, block, d, h_k, budget, recent):
    check(Cache([300, 17, 40, 0, 129, 130], h_k=h_k, d=d, page=page, block=block, seed=page + block + d + budget), budget, recent)


@pytest.mark.parametrize("budget", [1, 2, 31, 32, 500, 999, 1000])
@pytest.mark.parametrize("recent", [0, 1, 30])
def test_budgets(budget, recent):
    check(Cache([1000, 999, 33, 1], h_k=2, seed=budget, split=True), budget, min(recent, budget))


@pytest.mark.parametrize("L,budget", [(5000, 3000), (9000, 128), (9000, 8500)])
def test_long(L, budget):
    """Several steps of several CTAs."""
    check(Cache([L, L // 2], h_k=1, page=32, block=32, seed=L), budget, 100)


def test_order_of_weights():
    """Zeros of both signs are equal; NaN and infinities rank; negative weights too."""
    c = Cache([64], h_k=1, seed=2)
    w = torch.zeros(1, 1, 64)
    w[0, 0, ::2] = -0.0
    check(c, 20, 0, w)
    w = torch.randn(1, 1, 64, generator=c.g)
    w[0, 0, [3, 40, 41]] = math.nan
    w[0, 0, [5, 50]] = math.inf
    w[0, 0, [7, 55]] = -math.inf
    w[0, 0, 9] = 1e-42
    for budget in (1, 2, 4, 5, 6, 30, 62, 63):
        check(Cache([64], h_k=1, seed=2), budget, 0, w)


def test_everything_equal():
    check(Cache([3000], h_k=2, seed=3), 1500, 10, torch.zeros(1, 2, 3000))
    check(Cache([3000], h_k=2, seed=3), 1500, 0, torch.full((1, 2, 3000), math.nan))


def test_nan_codes_and_wild_scales():
    c = Cache([400], h_k=2, seed=4, spread=12)
    for at in (3, 77, 200, 399):
        page, row = int(c.table[0, at // 16]), at % 16
        for side in range(2):
            c.codes[side][page, row, 1, 5] = 0x7F if at % 2 else 0xFF
            c.kv[side][page, row, 1, 5] = 0x7F if at % 2 else 0xFF
    check(c, 150, 20)
    c = Cache([200], h_k=1, seed=5)  # blocks of nothing but zeros, and of nothing but NaN
    for at in range(200):
        page, row = int(c.table[0, at // 16]), at % 16
        code = 0 if at < 100 else 0x7F
        for side in range(2):
            c.codes[side][page, row] = code
            c.kv[side][page, row] = code
    check(c, 90, 10)


def test_budget_of_nothing():
    check(Cache([100, 0], h_k=2, seed=6), 0, 0)


def test_left_alone():
    """Sequences too long for their tensors, of negative length, or with a bad page."""
    from mjolnir_b200 import _lib, kvblock

    for what, code in (("page", _lib.MJ_DEV_BAD_PAGE), ("cols", _lib.MJ_DEV_BAD_LENGTH), ("negative", _lib.MJ_DEV_BAD_LENGTH)):
        c = Cache([300, 200], h_k=2, seed=7)
        w = torch.rand(2, 2, 300 if what != "cols" else 250, generator=c.g)
        if what == "page":
            c.table[0, 7] = c.pages
        lens = torch.tensor([-5 if what == "negative" else 300, 200], dtype=torch.int32, device="cuda")
        new, kept = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 50, dtype=torch.int32, device="cuda")
        status, wd = torch.zeros(1, dtype=torch.int32, device="cuda"), w.cuda()
        kvblock.evict(wd, *c.args, c.table.cuda(), lens, new, kept, recent=5, status=status)
        torch.cuda.synchronize()
        assert int(status) == code and new.tolist() == [int(lens[0]), 50] and (kept[0] == -1).all()
        assert torch.equal(wd[0].cpu(), w[0])
        c.lens[0] = 0
        want = evict_plain(c, torch.cat([w, torch.zeros(2, 2, 300 - w.shape[2])], -1), 50, 5)
        assert torch.equal(kept[1].cpu(), want[3][1])
        for side in range(2):
            assert np.array_equal(c.kv[side].cpu().numpy(), want[0][side]) and np.array_equal(c.sc[side].cpu().numpy(), want[1][side])


def test_again_and_from_a_graph():
    """A second cut of the shortened sequence, replayed from a graph that was captured for the first."""
    from mjolnir_b200 import kvblock

    c = Cache([600, 90], h_k=2, seed=8)
    w = torch.rand(2, 2, 600, generator=c.g)
    wd, lens = w.cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    new, kept = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 100, dtype=torch.int32, device="cuda")
    table = c.table.cuda()
    step = lambda: kvblock.evict(wd, *c.args, table, lens, new, kept, recent=10)  # noqa: E731
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens.copy_(torch.tensor(c.lens))
    graph.replay()
    torch.cuda.synchronize()
    codes, exps, want_w, want_k = evict_plain(c, w, 100, 10)
    assert torch.equal(kept.cpu(), want_k) and new.tolist() == [100, 90] and torch.equal(wd.cpu(), want_w)
    for side in range(2):
        assert np.array_equal(c.kv[side].cpu().numpy(), codes[side]) and np.array_equal(c.sc[side].cpu().numpy(), exps[side])


def test_twice_at_once():
    """Two calls over caches of their own, on two streams."""
    from mjolnir_b200 import kvblock

    caches = [Cache([900, 400], h_k=2, seed=s) for s in (9, 10)]
    ws = [torch.rand(2, 2, 900, generator=c.g) for c in caches]
    state = [(w.cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 300, dtype=torch.int32, device="cuda"),
              torch.tensor(c.lens, dtype=torch.int32, device="cuda"), c.table.cuda()) for c, w in zip(caches, ws)]
    torch.cuda.synchronize()
    for c, (w, new, kept, lens, table) in zip(caches, state):
        with torch.cuda.stream(torch.cuda.Stream()):
            kvblock.evict(w, *c.args, table, lens, new, kept, recent=20)
    torch.cuda.synchronize()
    for c, w, (wd, new, kept, _, _) in zip(caches, ws, state):
        codes, exps, want_w, want_k = evict_plain(c, w, 300, 20)
        assert torch.equal(kept.cpu(), want_k) and torch.equal(wd.cpu(), want_w)
        for side in range(2):
            assert np.array_equal(c.kv[side].cpu().numpy(), codes[side]) and np.array_equal(c.sc[side].cpu().numpy(), exps[side])


def test_more_heads_than_the_gpu_holds():
    lens = [40 + 3 * i for i in range(120)]
    check(Cache(lens, h_k=3, seed=11), 64, 7)


@pytest.mark.parametrize("d,n,budget", [(256, 1, 9000), (256, 2, 700), (128, 3, 1024), (128, 5, 1025)])
def test_long_of_several_sequences(d, n, budget):
    """Tokens beyond those whose keys a CTA holds, in every size of cluster."""
    check(Cache([20000 + 61 * i for i in range(n)], h_k=1 if n < 3 else 4, d=d, page=64, block=64, seed=n + d), budget, 64)


def test_weights_heads_outermost():
    from mjolnir_b200 import kvblock

    c = Cache([300, 90], h_k=2, seed=12)
    w = torch.rand(2, 2, 300, generator=c.g)
    wd = w.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    new, kept = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 100, dtype=torch.int32, device="cuda")
    kvblock.evict(wd, *c.args, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32, device="cuda"), new, kept, recent=3)
    codes, exps, want_w, want_k = evict_plain(c, w, 100, 3)
    assert torch.equal(kept.cpu(), want_k) and torch.equal(wd.cpu(), want_w)
    for side in range(2):
        assert np.array_equal(c.kv[side].cpu().numpy(), codes[side]) and np.array_equal(c.sc[side].cpu().numpy(), exps[side])
