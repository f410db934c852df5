"""Plan entries that point outside the step's sequences, rows, keys or partial
slots are flagged and skipped."""

import pytest
import torch

from tests.block_helpers import Cache, assert_attention, attention_plain

pytestmark = pytest.mark.gpu

BIG = 2**31 - 1


@pytest.mark.parametrize("which,column,value", [
    ("merges", 0, -1), ("merges", 0, 2), ("merges", 0, BIG), ("merges", 1, -128), ("merges", 2, -1), ("merges", 2, BIG),
    ("merges", 3, BIG), ("work", 0, -1), ("work", 0, 2), ("work", 1, -1), ("work", 1, BIG), ("work", 2, -1), ("work", 3, BIG),
    ("work", 4, BIG)])
def test_flagged(which, column, value):
    from mjolnir_b200 import _lib, kvblock

    c = Cache([9000, 300], h_k=1, seed=1)
    q_lens = [40, 20]
    q = torch.randn(60, 4, 128, generator=c.g).to(torch.bfloat16)
    qd, out = q.cuda(), torch.zeros(60, 4, 128, dtype=torch.bfloat16, device="cuda")
    r = kvblock.BlockAttention(num_heads=4, num_kv_heads=1, head_size=128, page_size=16, max_num_seqs=2, max_num_tokens=60)
    lens = torch.tensor(c.lens, dtype=torch.int32).cuda()
    plan = r.plan(q_lens, c.lens, c.table.cuda(), lens)
    assert len(plan.merges) == 1 and plan.merges[0, 0] == 0
    r.run(plan, qd, out, *c.args, 128**-0.5)
    r.check_status()
    first = out.clone()
    getattr(plan, which)[0, column] = value
    out.fill_(7)
    r.run(plan, qd, out, *c.args, 128**-0.5)
    torch.cuda.synchronize()
    with pytest.raises(_lib.MjolnirError, match=f"device status {_lib.MJ_DEV_BAD_SPLIT}"):
        r.check_status()
    assert torch.equal(out[40:], first[40:])  # the other sequence's rows
    if which == "merges":
        assert (out[:40] == 7).all()
    plan = r.plan(q_lens, c.lens, c.table.cuda(), lens)  # usable again
    r.run(plan, qd, out, *c.args, 128**-0.5)
    r.check_status()
    want, _, mag = attention_plain(c, q, q_lens, 128**-0.5)
    assert_attention(out, want, mag)


def test_an_empty_merge_is_skipped():
    from mjolnir_b200 import kvblock

    c = Cache([9000], h_k=1, seed=2)
    q = torch.randn(40, 4, 128, generator=c.g).to(torch.bfloat16).cuda()
    out = torch.full((40, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    r = kvblock.BlockAttention(num_heads=4, num_kv_heads=1, head_size=128, page_size=16, max_num_seqs=1, max_num_tokens=40)
    plan = r.plan([40], c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda())
    plan.merges[0, 3] = 0
    r.run(plan, q, out, *c.args, 128**-0.5)
    r.check_status()
    assert (out == 7).all()
