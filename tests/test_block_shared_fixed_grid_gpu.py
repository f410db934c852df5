"""With fixed_grid the launches of plans of the same `shared` are the same at every length."""

import pytest
import torch

from tests.block_helpers import Cache, assert_attention, attention_plain

pytestmark = pytest.mark.gpu


def launches(p):
    return (p.joins is not None, None if p.work is None else p.work.shape[0], None if p.joins is None else p.joins.shape[0], p.num_rows,
            p.num_slots, p.decode.num_work)


@pytest.mark.parametrize("n,prefix", [(16, 6272), (16, 6784), (16, 6800), (32, 4096), (4, 256)])
def test_launches_follow_from_the_arguments(n, prefix):
    """Around prefixes where a step whose own query stands inside the group's last tile plans otherwise."""
    from mjolnir_b200 import kvblock

    r = kvblock.BlockAttention(num_heads=32, num_kv_heads=8, head_size=128, page_size=16, max_num_seqs=n, max_num_tokens=4 * n)
    table = torch.zeros(n, 1000, dtype=torch.int32, device="cuda")
    lens = torch.ones(n, dtype=torch.int32, device="cuda")
    whole = prefix // 128 * 128
    for q_len in (1, 4):
        got = set()
        for more in (0, q_len - 1, q_len, q_len + 1, 127, 128, 129, 5000):
            kv = [whole + more + s * (more > q_len) for s in range(n)]
            if more < q_len:
                with pytest.raises(ValueError, match="fixed_grid"):
                    r.plan([q_len] * n, kv, table, lens, fixed_grid=True, shared=[(0, n, prefix)])
            else:
                got.add(launches(r.plan([q_len] * n, kv, table, lens, fixed_grid=True, shared=[(0, n, prefix)])))
        assert len(got) == 1, got


def test_a_graph_replays_from_the_first_token_behind_the_prefix():
    from mjolnir_b200 import kvblock

    n, prefix, h_q = 16, 6272, 8
    groups = [(0, n, prefix)]
    first, later = [prefix + 1] * n, [prefix + 2 + 37 * s for s in range(n)]
    c = Cache(later, h_k=2, seed=3)
    c.table[1:, :prefix // c.page] = c.table[0, :prefix // c.page]
    r = kvblock.BlockAttention(num_heads=h_q, num_kv_heads=2, head_size=128, page_size=c.page, block_tokens=c.block, max_num_seqs=n, max_num_tokens=n)
    q = torch.randn(n, h_q, 128, generator=c.g).bfloat16()
    qd, out, table = q.cuda(), torch.zeros(n, h_q, 128, dtype=torch.bfloat16, device="cuda"), c.table.cuda()
    lens = torch.tensor(first, dtype=torch.int32).cuda()
    plan = r.plan([1] * n, first, table, lens, fixed_grid=True, shared=groups)
    r.run(plan, qd, out, *c.args, 128**-0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.run(plan, qd, out, *c.args, 128**-0.5)
    for now in (later, first):
        lens.copy_(torch.tensor(now))
        r.plan([1] * n, now, table, lens, fixed_grid=True, shared=groups)
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        r.check_status()
        c.lens = now
        want, _, mag = attention_plain(c, q, [1] * n, 128**-0.5)
        assert_attention(out, want, mag)
