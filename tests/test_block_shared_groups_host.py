"""Which groups of a step share their prefix (no GPU needed)."""

import pytest

from mjolnir_b200.kvblock import BlockAttention


def planner(h_q=32, h_k=8, d=128, slots=40, worth=None):
    r = object.__new__(BlockAttention)
    r.h_q, r.h_k, r.d, r.rows, r.sm_count, r.max_shared_slots = h_q, h_k, d, 128 if d == 256 else 256, 148, slots
    if worth is not None:
        r._worth = lambda *a: worth
    return r


@pytest.mark.parametrize("order", [(0, 1, 2), (2, 0, 1), (1, 2, 0)])
def test_a_group_without_room_leaves_the_others_theirs(order):
    """100 chunks of 70 tokens of 4 heads are 110 row blocks of the group and 200 of the chunks: more than 40 slots."""
    sizes = [(100, 70), (6, 40), (4, 5)]
    q, groups, want = [], [], []
    for i in order:
        count, tokens = sizes[i]
        groups.append((len(q), count, 4096))
        if i:
            want.append(groups[-1])
        q += [tokens] * count
    assert planner(worth=True)._groups(groups, q, [4096 + n for n in q], 0, True) == want


def test_room_is_what_the_kept_groups_left():
    """Groups of 8 chunks of 64 tokens of 4 heads take 8 slots each and 8 of their chunks: two fit 40 slots, a small third one too."""
    q = [64] * 24 + [1] * 2
    groups = [(0, 8, 512), (8, 8, 512), (16, 8, 512), (24, 2, 512)]
    assert planner(worth=True)._groups(groups, q, [600] * 26, 0, True) == [groups[0], groups[1], groups[3]]
