"""Calls of many tokens and few heads (multi-query layouts, narrow shards)."""

import pytest
import torch

from tests.test_qk_rope_gpu import _check, _plain

pytestmark = pytest.mark.gpu


def _call(T, h_q, h_k, d, dtype):
    g = torch.Generator("cuda").manual_seed(h_q)
    x = torch.randn(T, h_q + h_k, d, generator=g, device="cuda").to(dtype)
    w = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dtype)
    table = torch.randn(4096, d, generator=g, device="cuda")
    pos = torch.randint(0, 4096, (T,), generator=g, device="cuda")
    out = [torch.empty(T, h, d, dtype=dtype, device="cuda") for h in (h_q, h_k)]
    return dict(q=x[:, :h_q], k=x[:, h_q:], positions=pos, cos_sin=table, q_weight=w, k_weight=w, q_out=out[0], k_out=out[1])


def _time(calls):
    """Of one replay of all the calls."""
    from mjolnir_b200 import qkrope

    qkrope.qk_norm_rope(**calls[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            for a in calls:
                qkrope.qk_norm_rope(**a)
    times = []
    for _ in range(9):
        e = [torch.cuda.Event(enable_timing=True) for _ in (0, 1)]
        e[0].record()
        graph.replay()
        e[1].record()
        torch.cuda.synchronize()
        times.append(e[0].elapsed_time(e[1]))
    return sorted(times)[4]


@pytest.mark.parametrize("h_q,h_k", [(1, 1), (2, 1)])
def test_a_call_costs_no_more_than_its_parts(h_q, h_k):
    """2^20 threads' rows at once, and in five calls that fill the GPU less."""
    T = (1 << 17) // (h_q + h_k)
    whole = _call(T, h_q, h_k, 128, torch.bfloat16)
    parts = []
    for i in range(5):
        at = slice(i * T // 5, (i + 1) * T // 5)
        parts.append({k: v[at] if k in ("q", "k", "positions", "q_out", "k_out") else v for k, v in whole.items()})
    a, b = _time([whole]), _time(parts)
    assert a <= b, f"{h_q} + {h_k} heads: {a * 100:.1f} us at once, {b * 100:.1f} in parts"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,h_q,h_k", [(40_000, 1, 1), (9000, 8, 1), (9000, 3, 5), (4000, 16, 4), (2100, 16, 0)])
def test_formula_on_both_sides_of_the_variants(T, h_q, h_k, dtype):
    from mjolnir_b200 import qkrope

    a = _call(T, h_q, h_k, 128, dtype)
    x = [t.clone() for t in (a["q"], a["k"])]
    got = qkrope.qk_norm_rope(**a)
    torch.cuda.synchronize()
    some = torch.cat([torch.arange(40), torch.arange(T - 40, T)])
    for i, side in enumerate("qk"):
        want = _plain(x[i][some.cuda()].cpu(), a["q_weight"].cpu(), a["cos_sin"].cpu(), a["positions"].cpu()[some], False, 1e-6)
        if got[i].numel():
            _check(got[i][some.cuda()], *want)
