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
