"""The partials of steps that share prefixes: how much, when, and after a plan that found no memory."""

import pytest
import torch

from tests.block_helpers import Cache, assert_attention, attention_plain

pytestmark = pytest.mark.gpu


def runner(h_q, h_k, d, **kw):
    from mjolnir_b200 import kvblock

    return kvblock.BlockAttention(num_heads=h_q, num_kv_heads=h_k, head_size=d, page_size=16, max_num_seqs=64, max_num_tokens=64, **kw)


def plan(r, n=64, prefix=16384):
    table, lens = torch.zeros(n, 1100, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    return r.plan([1] * n, [prefix + 1 + s for s in range(n)], table, lens, shared=[(0, n, prefix)])


@pytest.mark.parametrize("h_q,h_k,d", [(32, 8, 128), (32, 32, 128), (64, 64, 128), (32, 32, 256), (24, 4, 256)])
def test_partials_are_bounded(h_q, h_k, d):
    r = runner(h_q, h_k, d)
    before = torch.cuda.memory_allocated()
    assert plan(r).joins is not None
    assert torch.cuda.memory_allocated() - before <= 195e6


def test_a_constructor_that_is_told_allocates_them():
    r = runner(32, 8, 128, shared_prefixes=True)
    plan(r)
    before = torch.cuda.memory_allocated()
    keep = plan(r)
    assert keep.joins is not None and torch.cuda.memory_allocated() - before < 1e6


def test_a_plan_without_memory_leaves_a_runner_that_plans(monkeypatch):
    from mjolnir_b200 import kvblock

    c = Cache([1100, 1040, 1030], h_k=2, seed=4)
    c.table[1:, :64] = c.table[0, :64]
    monkeypatch.setattr(kvblock.BlockAttention, "_worth", lambda self, *a: True)
    r = kvblock.BlockAttention(num_heads=8, num_kv_heads=2, head_size=128, page_size=16, max_num_seqs=3, max_num_tokens=3)
    args = ([1] * 3, c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda())
    empty, left = torch.empty, [0]

    def no_memory(*a, **kw):
        if "pin_memory" not in kw:
            left[0] += 1
            raise torch.OutOfMemoryError("no memory")
        return empty(*a, **kw)

    monkeypatch.setattr(torch, "empty", no_memory)
    with pytest.raises(torch.OutOfMemoryError):
        r.plan(*args, shared=[(0, 3, 1024)])
    monkeypatch.setattr(torch, "empty", empty)
    assert left[0] == 1
    q = torch.randn(3, 8, 128, generator=c.g).bfloat16()
    out = torch.empty(3, 8, 128, dtype=torch.bfloat16, device="cuda")
    p = r.plan(*args, shared=[(0, 3, 1024)])
    assert p.joins is not None
    r.run(p, q.cuda(), out, *c.args, 128**-0.5)
    torch.cuda.synchronize()
    r.check_status()
    want, _, mag = attention_plain(c, q, [1] * 3, 128**-0.5)
    assert_attention(out, want, mag)
