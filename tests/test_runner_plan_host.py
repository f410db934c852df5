"""DecodeRunner.plan on the host, the device buffers on the CPU (no GPU needed)."""

import time

import pytest
import torch

from mjolnir_b200 import runner
from mjolnir_b200.plan import plan_split_kv


def planner(n):
    r = object.__new__(runner.DecodeRunner)
    r.max_q_len, r.max_num_seqs, r.h_k, r.h_r, r.sm_count, r.max_splits, r._cap, r.rebalance = 4, n, 8, 4, 148, 16, 0, True
    r.device, r.n_tiles, r.ctas = torch.device("cpu"), lambda q_len: 1, lambda q_len: 1
    r.work_buf, r.nsplit_buf = torch.zeros(0, 4, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)
    return r


def size(r, lens):
    r.work_buf = torch.zeros(plan_split_kv(lens, 8, 1, 148, ctas_per_sm=1, max_splits=16, pad_to=0, rebalance=True).work_array().shape, dtype=torch.int32)
    return r


def test_no_starts_are_starts_of_zero():
    lens = [1000 + 37 * s for s in range(40)] + [0, 1, 128]
    a, b = size(planner(len(lens)), lens), size(planner(len(lens)), lens)
    p, q = a.plan(lens, len(lens), 1, None, None), b.plan(lens, len(lens), 1, None, None, starts=[0] * len(lens))
    assert torch.equal(a.work_buf, b.work_buf) and torch.equal(a.nsplit_buf, b.nsplit_buf)
    assert (p.num_work, p.tile_jobs, p.with_reduction, p.pieces) == (q.num_work, q.tile_jobs, q.with_reduction, q.pieces)


def test_starts_are_checked():
    r = size(planner(2), [300, 300])
    for starts in ([0], [64, 0], [-128, 0], [384, 0]):
        with pytest.raises(ValueError, match="starts"):
            r.plan([300, 300], 2, 1, None, None, starts=starts)


def test_a_plan_without_starts_pays_nothing_for_them(monkeypatch):
    """Of 1024 sequences, the split left out: under four fifths of the time that checked starts of zero take (measured: half)."""
    lens = [1000 + 7 * s for s in range(1024)]
    r = size(planner(1024), lens)
    fixed = plan_split_kv(lens, 8, 1, 148, ctas_per_sm=1, max_splits=16, pad_to=0, rebalance=True)
    array = fixed.work_array()
    fixed.work_array, fixed.work = lambda: array, fixed.work[:1]
    monkeypatch.setattr(runner, "plan_split_kv", lambda *a, **kw: fixed)

    def best(**kw):
        times = []
        for _ in range(60):
            t = time.perf_counter()
            r.plan(lens, 1024, 1, None, None, **kw)
            times.append(time.perf_counter() - t)
        return min(times)

    assert best() < 0.8 * best(starts=[0] * 1024)
