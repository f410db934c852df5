"""What BlockAttention.plan refuses and keeps."""

import pytest
import torch

from tests.block_helpers import Cache

pytestmark = pytest.mark.gpu


def _runner(c, h_q=8, seqs=2, tokens=100):
    from mjolnir_b200 import kvblock

    return kvblock.BlockAttention(num_heads=h_q, num_kv_heads=c.h_k, head_size=c.d, page_size=c.page, block_tokens=c.block,
                                  max_num_seqs=seqs, max_num_tokens=tokens)


@pytest.mark.parametrize("q_lens", [[1, 1], [1, 40], [40, 1]])
def test_sequences_longer_than_their_table_row(q_lens):
    c = Cache([64, 30])
    r = _runner(c)
    lens = torch.tensor([64, 30], dtype=torch.int32).cuda()
    r.plan(q_lens, [64, 30], c.table[:, :4].cuda(), lens)
    for long in ([65, 30], [30, 65]):
        with pytest.raises(ValueError, match="more than block_table's 4 pages"):
            r.plan(q_lens, long, c.table[:, :4].cuda(), lens)
    r.plan([q_lens[0], 0], [64, 1000], c.table[:, :4].cuda(), lens)  # not attended in this step


@pytest.mark.parametrize("d,h_q,h_k,q_len", [(128, 8, 2, 1), (128, 8, 1, 3), (256, 6, 1, 2)])
def test_a_captured_step_replays_later_plans(d, h_q, h_k, q_len):
    """Captured over short sequences, replayed over plans of other lengths:
    longer ones split, shorter ones not, one sequence empty."""
    from tests.block_helpers import assert_attention, attention_plain

    n = 3
    c = Cache([9000, 6000, 700], h_k=h_k, d=d, seed=q_len)
    r, eager = _runner(c, h_q, n, n * q_len), _runner(c, h_q, n, n * q_len)
    q = torch.randn(n * q_len, h_q, d, generator=c.g).to(torch.bfloat16)
    qd, out, want_eager = q.cuda(), torch.empty(n * q_len, h_q, d, dtype=torch.bfloat16, device="cuda"), torch.empty(n * q_len, h_q, d, dtype=torch.bfloat16, device="cuda")
    table, lens, q_lens = c.table.cuda(), torch.zeros(n, dtype=torch.int32, device="cuda"), [q_len] * n

    def step(now):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        return r.plan(q_lens, now, table, lens, fixed_grid=True)

    plan = step([40, 300, 17])
    r.run(plan, qd, out, *c.args, d**-0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.run(plan, qd, out, *c.args, d**-0.5)
    for now in ([40, 300, 17], [41, 301, 18], [9000, 6000, 700], [9000, 0, 5], [1, 5999, 128]):
        step(now)
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        r.check_status()
        eager.run(eager.plan(q_lens, now, table, lens), qd, want_eager, *c.args, d**-0.5)
        torch.cuda.synchronize()
        assert torch.equal(out, want_eager), now
        c.lens = now
        want, _, mag = attention_plain(c, q, q_lens, d**-0.5)
        assert_attention(out, want, mag, str(now))


def test_a_fixed_grid_is_for_steps_of_the_decode_kernel():
    c = Cache([64, 30])
    r = _runner(c)
    lens = torch.tensor([64, 30], dtype=torch.int32).cuda()
    for q_lens in ([40, 1], [1, 40], [1, 2], [0, 0]):
        with pytest.raises(ValueError, match="fixed_grid"):
            r.plan(q_lens, [64, 30], c.table.cuda(), lens, fixed_grid=True)
    with pytest.raises(ValueError, match="fixed_grid"):
        r.plan([], [], c.table.cuda(), lens, fixed_grid=True)
