"""What a call of kvblock.weigh launches, and arguments at the ends of their ranges."""

import pytest
import torch

from tests.block_helpers import Cache

pytestmark = pytest.mark.gpu


def step(lens, q_lens, h_q=8, h_k=2, rows=None, seed=1, cols=None):
    """(arguments of weigh but the weights, weights)"""
    c = Cache(lens, h_k=h_k, seed=seed)
    rows = rows or sum(q_lens)
    q = torch.randn(rows, h_q, 128, generator=c.g).bfloat16().cuda()
    lse = (torch.randn(rows, h_q, generator=c.g) + 5).cuda()
    at = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32).cuda()
    lens = torch.tensor(lens, dtype=torch.int32).cuda()
    return (q, lse, c.kv[0], c.sc[0], c.table.cuda(), at, lens), torch.rand(len(q_lens), h_k, cols or max(c.lens), generator=c.g).cuda()


def launches(call):
    """The kernels of a call, from the graph that it is captured into."""
    from cuda.bindings import runtime

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    err, _, count = runtime.cudaGraphGetNodes(graph.raw_cuda_graph())
    assert int(err) == 0
    return count


@pytest.mark.parametrize("q_lens,window,want", [([30, 40], 0, 2), ([30, 40], 5, 2), ([30, 40], 4, 1), ([30, 40], 1, 1), ([1, 1], 0, 1), ([40], 0, 1),
                                                ([40], 4, 1), ([3], 0, 1)])
def test_a_launch_that_cannot_find_a_sequence_is_left_out(q_lens, window, want):
    """Sequences of at most 4 queries (16 rows of 4 heads) have one kernel, those of more the other."""
    from mjolnir_b200 import kvblock

    args, w = step([300 + n for n in q_lens], q_lens)
    assert launches(lambda: kvblock.weigh(*args, w, 0.1, window=window)) == want


@pytest.mark.parametrize("window", [2**31 - 1, 2**31, 2**32, 2**32 + 1, 2**40 + 3])
def test_windows_beyond_32_bits_are_every_query(window):
    from mjolnir_b200 import kvblock

    args, w = step([200, 90, 61], [40, 3, 60])
    want = kvblock.weigh(*args, w.clone(), 0.1)
    assert torch.equal(kvblock.weigh(*args, w.clone(), 0.1, window=window), want)


@pytest.mark.parametrize("rows", [40, 3])
@pytest.mark.parametrize("lens,at", [([500, 90], [0, 0, 0]), ([90, 500], [0, 0, 0]), ([90, -1], [0, 0, 0]), ([90, 90], [99, 99, 99]), ([90, 90], [0, 0, -2]),
                                     ([90, 90], [-1, -1, -1])])
def test_lengths_and_offsets_out_of_range_are_flagged_without_queries_too(lens, at, rows):
    """Whatever the call launches (rows for both kernels, or for one)."""
    from mjolnir_b200 import _lib, kvblock

    args, w = step([90, 90], [rows - 1, 1], cols=100)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = w.clone()
    kvblock.weigh(*args[:5], torch.tensor(at, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), w, 0.1, status=status)
    assert status.item() == _lib.MJ_DEV_BAD_LENGTH and torch.equal(w, before)
