"""Q/K norm with the rotation by positions of several axes, against its formula in 64 bits."""

import pytest
import torch

from tests.block_helpers import UNIT

pytestmark = pytest.mark.gpu


def _plain(x, w, table, pos, axes, interleaved, eps):
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    rot, out = table.shape[1], y.clone()
    for i, axis in enumerate(axes):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = table.double()[pos[axis], i][:, None], table.double()[pos[axis], rot // 2 + i][:, None]
        out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    # 32-bit arithmetic: the row's sum of squares and each product round at most
    # a few dozen times 2^-24 of the largest normed element
    return out, 64 * 2.0**-24 * y.abs().amax(-1, keepdim=True)


def _check(got, want, slack):
    tol = slack + UNIT[got.dtype] * (want.abs() + slack) + (2.0**-25 if got.dtype == torch.float16 else 0.0)
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), (err / tol).max().item()


def _case(T, h, d, rot, dtype, num_axes, seed=0, table_dtype=torch.float32, positions=64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, h, d, generator=g).to(dtype)
    table = torch.randn(positions, rot, generator=g).to(table_dtype)
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in (0, 1)]
    axes = tuple(torch.randint(0, num_axes, (rot // 2,), generator=g).tolist())
    return x, table, w, torch.randint(0, positions, (num_axes, T), generator=g), axes


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rot,sections", [(64, 64, (8, 12, 12)), (128, 128, (16, 24, 24)), (128, 32, (6, 5, 5)), (256, 256, (44, 42, 42)),
                                            (256, 64, (8, 8, 8, 8)), (80, 48, (24,)), (16, 16, (5, 3)), (512, 512, (64, 64, 64, 64))])
@pytest.mark.parametrize("interleaved,alternate", [(False, False), (False, True), (True, False)])
def test_formula(dtype, d, rot, sections, interleaved, alternate):
    from mjolnir_b200 import qkrope

    T, h_q, h_k = 21, 5, 2
    if alternate:  # what the smallest section leaves over goes to the first axis
        sections = [sum(sections) - (len(sections) - 1) * min(sections)] + [min(sections)] * (len(sections) - 1)
    axes = qkrope.angle_axes(sections, alternate)
    x, table, w, pos, _ = _case(T, h_q + 2 * h_k, d, rot, dtype, len(sections), seed=d + rot)
    fused = x.reshape(T, -1).cuda()
    q, k = fused.view(T, -1, d)[:, :h_q], fused.view(T, -1, d)[:, h_q:h_q + h_k]
    for wq, wk in ((w[0], w[1]), (None, None)):
        qo, ko = qkrope.qk_norm_rope(q, k, pos.cuda(), table.cuda(), None if wq is None else wq.cuda(), None if wk is None else wk.cuda(),
                                     eps=1e-5, interleaved=interleaved, axes=axes)
        torch.cuda.synchronize()
        _check(qo, *_plain(x[:, :h_q], wq, table, pos, axes, interleaved, 1e-5))
        _check(ko, *_plain(x[:, h_q:h_q + h_k], wk, table, pos, axes, interleaved, 1e-5))
    assert torch.equal(fused.cpu(), x.reshape(T, -1))


@pytest.mark.parametrize("table_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1])
def test_any_order_of_axes_and_unaligned_tables(table_dtype, offset):
    """Axes in no order at all; a table whose rows begin at odd addresses."""
    from mjolnir_b200 import qkrope

    x, table, w, pos, axes = _case(300, 12, 128, 96, torch.bfloat16, 4, seed=3, table_dtype=table_dtype)
    wide = torch.zeros(64, 96 + 3, dtype=table_dtype, device="cuda")[:, offset:offset + 96]
    wide.copy_(table.cuda())
    many = torch.full((4, 2, 300), 99, device="cuda")  # the axes' rows stand apart
    many[:, 0] = pos.cuda()
    q = x.cuda()
    qo, ko = qkrope.qk_norm_rope(q[:, :8], q[:, 8:], many[:, 0], wide, w[0].cuda(), w[1].cuda(), axes=axes)
    torch.cuda.synchronize()
    _check(qo, *_plain(x[:, :8], w[0], table, pos, axes, False, 1e-6))
    _check(ko, *_plain(x[:, 8:], w[1], table, pos, axes, False, 1e-6))


@pytest.mark.parametrize("T,h_q,h_k", [(0, 4, 4), (1, 1, 1), (1, 32, 8), (3, 0, 2), (700, 32, 8)])
def test_sizes(T, h_q, h_k):
    from mjolnir_b200 import qkrope

    x, table, w, pos, axes = _case(T, h_q + h_k, 128, 128, torch.bfloat16, 3, seed=T)
    q = x.cuda()
    qo, ko = qkrope.qk_norm_rope(q[:, :h_q], q[:, h_q:], pos.cuda(), table.cuda(), w[0].cuda(), w[1].cuda(), axes=axes)
    torch.cuda.synchronize()
    _check(qo, *_plain(x[:, :h_q], w[0], table, pos, axes, False, 1e-6))
    _check(ko, *_plain(x[:, h_q:], w[1], table, pos, axes, False, 1e-6))


@pytest.mark.parametrize("T", [40, 900])
def test_equal_positions_are_the_rotation_by_one(T):
    """Text: the same position on every axis is the rotation without axes, to the bit, in place too."""
    from mjolnir_b200 import qkrope

    x, table, w, pos, axes = _case(T, 40, 128, 128, torch.bfloat16, 3, seed=T)
    one = pos[0].cuda()
    q, k = x[:, :32].cuda(), x[:, 32:].cuda()
    want = qkrope.qk_norm_rope(q, k, one, table.cuda(), w[0].cuda(), w[1].cuda())
    qkrope.qk_norm_rope(q, k, one.expand(3, T), table.cuda(), w[0].cuda(), w[1].cuda(), axes=axes, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    single = qkrope.qk_norm_rope(x[:, :32].cuda(), x[:, 32:].cuda(), one[None], table.cuda(), w[0].cuda(), w[1].cuda(), axes=(0,) * 64)
    assert torch.equal(single[0], want[0]) and torch.equal(single[1], want[1])


def test_bad_position_on_any_axis():
    from mjolnir_b200 import _lib, qkrope

    x, table, w, pos, axes = _case(6, 10, 128, 128, torch.bfloat16, 3, seed=5)
    for t, axis, bad in ((1, 0, -1), (4, 2, 64)):
        p = pos.clone()
        p[axis, t] = bad
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        qo, ko = (torch.full((6, h, 128), 7.0, dtype=torch.bfloat16, device="cuda") for h in (8, 2))
        qkrope.qk_norm_rope(x[:, :8].cuda(), x[:, 8:].cuda(), p.cuda(), table.cuda(), w[0].cuda(), w[1].cuda(), axes=axes,
                            q_out=qo, k_out=ko, status=status)
        assert int(status) == _lib.MJ_DEV_BAD_POSITION
        assert (qo[t] == 7).all() and (ko[t] == 7).all()
        rest = [i for i in range(6) if i != t]
        want, slack = _plain(x[:, :8], w[0], table, pos, axes, False, 1e-6)
        _check(qo[rest], want[rest], slack[rest])


def test_replayed_from_a_graph():
    from mjolnir_b200 import qkrope

    x, table, w, pos, axes = _case(50, 10, 128, 128, torch.bfloat16, 3, seed=6)
    q, k, p, tab = x[:, :8].cuda(), x[:, 8:].cuda(), pos.cuda(), table.cuda()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    a = (tab, w[0].cuda(), w[1].cuda())
    qkrope.qk_norm_rope(q, k, p, *a, axes=axes, q_out=qo, k_out=ko)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qkrope.qk_norm_rope(q, k, p, *a, axes=axes, q_out=qo, k_out=ko)
    other = (pos + 11) % 64
    p.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    _check(qo, *_plain(x[:, :8], w[0], table, other, axes, False, 1e-6))
