"""The plan of steps whose sequences share prefixes (no GPU needed)."""

import ctypes
import os
import random
import subprocess
import tempfile

import numpy as np
import pytest

from mjolnir_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_header():
    src = ('#include "mjolnir_b200.h"\n#include <stdio.h>\n#include <stddef.h>\n'
           'int main(){printf("%zu %zu", sizeof(mj_block_join_args), offsetof(mj_block_join_args, status));return 0;}\n')
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "p.c"), "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "p.c"), "-o", os.path.join(d, "p")], check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "p")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.BlockJoinArgs), _lib.BlockJoinArgs.status.offset]


@pytest.mark.parametrize("seed", range(4))
def test_plan_covers_every_row_and_key_once(seed):
    r = random.Random(seed)
    for _ in range(200):
        n = r.randint(0, 12)
        few = r.randint(0, n)
        q = [r.choice([1, 3])] * few + [r.choice([0, 1, 5, 70, 900, r.randint(0, 400)]) for _ in range(n - few)]
        groups, at = [], r.randint(0, 3)
        while at < n:
            count = r.randint(1, n - at)
            groups.append((at, count, 128 * r.choice([1, 5, 40])))
            at += count + r.randint(0, 3)
        member = {s: g for g, (first, count, _) in enumerate(groups) for s in range(first, first + count)}
        kv = [x + r.choice([0, 0, 40, 3000]) + (groups[member[s]][2] if s in member else 0) for s, x in enumerate(q)]
        h_k, h_r, d, causal = r.choice([1, 2, 8]), r.choice([1, 3, 4, 6]), r.choice([128, 256]), r.random() < 0.7
        rows = 128 if d == 256 else 256
        need = sum(-(-sum(q[f:f + c]) * h_r // rows) + sum(-(-x * h_r // rows) for x in q[max(f, few):max(f + c, few)]) for f, c, _ in groups)
        slots = need + r.choice([0, 40, 300])
        pieces = [r.choice([0, 2, 3]) if s not in member else r.choice([1, 2]) for s in range(few)]
        work, joins = np.zeros((20000, 8), np.int32), np.zeros((2000, 12), np.int32)
        nw, nj, nr, ns = _lib.block_shared_plan(q, kv, pieces, groups, h_k * h_r, h_k, d, causal, 148, slots, work, joins)
        assert ns <= slots
        # items: the keys of every row, once, in whole pieces
        used, items = [], {}
        for s, r0, tb, te, slot, span, *_ in work[:nw].tolist():
            items.setdefault((s, r0, span), []).append((tb, te, slot))
            used += [slot] if slot >= 0 else []
        assert sorted(used) == list(range(ns))
        want = {(f, r0, c) for f, c, _ in groups for r0 in range(0, sum(q[f:f + c]) * h_r, rows)}
        want |= {(s, r0, 0) for s in range(few, n) for r0 in range(0, q[s] * h_r, rows)}
        assert set(items) == want
        for (s, r0, span), parts in items.items():
            parts.sort(key=lambda p: (p[2], p[0]))
            if span:
                begin, end = 0, groups[member[s]][2] // 64
            else:
                last = kv[s] - q[s] + (min(r0 + rows, q[s] * h_r) - 1) // h_r if causal else kv[s] - 1
                begin = groups[member[s]][2] // 64 if s in member else 0
                end = max(begin, last // 64 + 1 if last >= 0 else 0)
            assert parts[0][0] == begin and parts[-1][1] == end and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
            assert [p[2] for p in parts] == ([-1] if parts[0][2] < 0 else list(range(parts[0][2], parts[0][2] + len(parts))))
            assert parts[0][2] >= 0 or (len(parts) == 1 and not span and s not in member)
        # joins: every row that has partials, with all of them
        total, seen = 0, {}
        for s, r0, count, before, own, m, first, shared, place, *_ in joins[:nj].tolist():
            assert before == total and count > 0
            total += count
            for x in range(r0, r0 + count):
                assert (s, x) not in seen
                seen[s, x] = True
                if s < few:
                    assert own == -1 and m == pieces[s]
                else:
                    assert sorted(p[2] for p in items[s, r0, 0]) == list(range(own, own + m))
                if s in member:
                    f, c, _ = groups[member[s]]
                    p = place + x - r0
                    assert p == sum(q[f:s]) * h_r + x
                    assert sorted(i[2] for i in items[f, p // rows * rows, c]) == list(range(first + p // rows * shared, first + (p // rows + 1) * shared))
                else:
                    assert shared == 0
        assert total == nr
        for s in range(n):
            for x in range(0, q[s] * h_r, 7):
                final = s >= few and s not in member and len(items[s, x // rows * rows, 0]) == 1
                assert ((s, x) in seen) != final


def test_plan_refuses():
    work, joins = np.zeros((2, 8), np.int32), np.zeros((1, 12), np.int32)
    plan = lambda q, kv, pieces, groups, **kw: _lib.block_shared_plan(  # noqa: E731
        q, kv, pieces, groups, 4, kw.get("h_k", 1), 128, True, 148, kw.get("slots", 10), work, joins)
    with pytest.raises(_lib.MjolnirError, match="invalid argument"):
        plan([1], [5], [], [], h_k=3)
    with pytest.raises(_lib.MjolnirError, match="invalid argument"):
        plan([1], [5], [1, 1], [])
    for groups in ([(0, 2, 128)], [(0, 0, 128)], [(0, 1, 100)], [(0, 1, 0)], [(-1, 1, 128)], [(0, 1, 128), (0, 1, 128)]):
        with pytest.raises(_lib.MjolnirError, match="a group"):
            plan([1], [200], [1], groups)
    with pytest.raises(_lib.MjolnirError, match="before the end"):
        plan([80], [200], [], [(0, 1, 128)])
    with pytest.raises(_lib.MjolnirError, match="max_slots"):
        plan([1, 1], [200, 200], [], [(0, 2, 128)], slots=2)
    with pytest.raises(_lib.MjolnirError, match="items"):
        plan([1, 1], [200, 200], [], [(0, 2, 128)])
    with pytest.raises(_lib.MjolnirError, match="joins"):
        plan([1, 1], [200, 200], [1, 1], [(0, 2, 128)])
    with pytest.raises(_lib.MjolnirError, match="length"):
        plan([-1], [200], [], [])


def test_worth():
    """Many short rows behind a long prefix: yes. Few, short prefixes, or rows that fill their tiles alone: no."""
    worth = lambda q, tokens, own=200, few=0, h_k=8, d=128: _lib.block_shared_worth(  # noqa: E731
        q, [tokens + own + x for x in q], few, [(0, len(q), tokens)], 4 * h_k, h_k, d, True, 148, 166)
    assert worth([1] * 64, 16384, few=64) and worth([24] * 16, 4096) and worth([3] * 16, 4096, d=256, h_k=4)
    assert not worth([1] * 4, 16384, few=4) and not worth([24] * 2, 1024) and not worth([500] * 8, 1024) and not worth([0, 0], 4096)
    with pytest.raises(_lib.MjolnirError, match="a group"):
        _lib.block_shared_worth([1], [200], 0, [(0, 2, 128)], 4, 1, 128, True, 148, 10)
    with pytest.raises(_lib.MjolnirError, match="invalid"):
        _lib.block_shared_worth([1], [200], 2, [(0, 1, 128)], 4, 1, 128, True, 148, 10)


def test_join_refuses():
    j = _lib.BlockJoinArgs()
    j.num_seqs, j.num_tokens, j.h_q, j.h_k = 1, 1, 3, 2
    with pytest.raises(_lib.MjolnirError, match="h_q 3 h_k 2"):
        _lib.block_join(j, 0)
    j.h_q, j.head_size = 4, 64
    with pytest.raises(_lib.MjolnirError, match="head_size"):
        _lib.block_join(j, 0)
    j.head_size, j.dtype = 128, _lib.MJ_DT_FP32
    with pytest.raises(_lib.MjolnirError, match="dtype"):
        _lib.block_join(j, 0)
    j.dtype, j.num_joins, j.num_rows = _lib.MJ_DT_BF16, 1, 1
    with pytest.raises(_lib.MjolnirError, match="buffers"):
        _lib.block_join(j, 0)


def test_groups_are_checked():
    from mjolnir_b200 import kvblock

    r = object.__new__(kvblock.BlockAttention)
    r._worth = lambda *a: True
    r.h_q, r.h_k, r.rows, r.max_shared_slots = 8, 2, 256, 40
    q, kv = [1, 1, 1, 50], [1000, 900, 1500, 800]
    ok = lambda *g: r._groups(g, q, kv, 3, True)  # noqa: E731
    assert ok((0, 4, 640)) == [(0, 4, 640)] and ok((2, 2, 700), (0, 2, 700)) == [(0, 2, 640), (2, 2, 640)]
    assert ok((0, 4, 10**6)) == [(0, 4, 640)]  # query 0 of the last sequence sees 750 tokens before it
    assert ok((0, 1, 640)) == [] and ok((0, 4, 127)) == [] and ok() == []
    for bad in (((0, 5, 128),), ((0, 0, 128),), ((-1, 2, 128),), ((0, 2, -1),), ((0, 2, 128), (1, 2, 128))):
        with pytest.raises(ValueError, match="shared"):
            ok(*bad)
    r.max_shared_slots = 1  # room for the group's rows, not for those of its chunk
    assert ok((0, 4, 640)) == [] and ok((0, 3, 640)) == [(0, 3, 640)]
