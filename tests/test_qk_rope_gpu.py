"""Q/K norm with rotation against its formula in 64 bits."""

import pytest
import torch

from tests.block_helpers import UNIT

pytestmark = pytest.mark.gpu


def _plain(x, w, table, pos, interleaved, eps):
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    rot = table.shape[1]
    cos, sin = table.double()[pos, :rot // 2, ][:, None], table.double()[pos, rot // 2:][:, None]
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    out = y.clone()
    out[..., a] = y[..., a] * cos - y[..., b] * sin
    out[..., b] = y[..., b] * cos + y[..., a] * sin
    # 32-bit arithmetic: the row's sum of squares and each product round at most
    # a few dozen times 2^-24 of the largest normed element
    return out, 64 * 2.0**-24 * y.abs().amax(-1, keepdim=True)


def _check(got, want, slack):
    u = UNIT[got.dtype]
    err, tol = (got.double().cpu() - want).abs(), slack + u * (want.abs() + slack)
    if got.dtype == torch.float16:
        tol = tol + 2.0**-25
    assert (err <= tol).all(), (err / tol).max().item()


def _case(T, h_q, h_k, d, rot, dtype, seed=0, table_dtype=torch.float32, w_dtype=None, positions=64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, h_q + 2 * h_k, d, generator=g).to(dtype)
    table = torch.randn(positions, rot, generator=g).to(table_dtype)
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(w_dtype or dtype) for _ in (0, 1)]
    return x, table, w, torch.randint(0, positions, (T,), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (128, 32), (256, 256), (256, 64), (80, 48), (16, 16), (512, 512), (336, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_formula(dtype, d, rot, interleaved):
    from mjolnir_b200 import qkrope

    T, h_q, h_k = 21, 5, 2
    x, table, w, pos = _case(T, h_q, h_k, d, rot, dtype, seed=d + rot)
    fused = x.reshape(T, -1).cuda()
    q, k = fused.view(T, -1, d)[:, :h_q], fused.view(T, -1, d)[:, h_q:h_q + h_k]
    for wq, wk in ((w[0], w[1]), (None, w[1]), (w[0], None), (None, None)):
        qo, ko = qkrope.qk_norm_rope(q, k, pos.cuda(), table.cuda(), None if wq is None else wq.cuda(),
                                     None if wk is None else wk.cuda(), eps=1e-5, interleaved=interleaved)
        torch.cuda.synchronize()
        _check(qo, *_plain(x[:, :h_q], wq, table, pos, interleaved, 1e-5))
        _check(ko, *_plain(x[:, h_q:h_q + h_k], wk, table, pos, interleaved, 1e-5))
    assert torch.equal(fused.cpu(), x.reshape(T, -1))


@pytest.mark.parametrize("T,h_q,h_k", [(1, 1, 1), (1, 32, 8), (3, 0, 2), (3, 7, 0), (517, 32, 8), (0, 4, 4)])
def test_sizes(T, h_q, h_k):
    from mjolnir_b200 import qkrope

    x, table, w, pos = _case(T, h_q, h_k, 128, 128, torch.bfloat16, seed=T)
    qo, ko = qkrope.qk_norm_rope(x[:, :h_q].contiguous().cuda(), x[:, h_q:h_q + h_k].contiguous().cuda(), pos.cuda(), table.cuda(), w[0].cuda(), w[1].cuda())
    torch.cuda.synchronize()
    _check(qo, *_plain(x[:, :h_q], w[0], table, pos, False, 1e-6))
    _check(ko, *_plain(x[:, h_q:h_q + h_k], w[1], table, pos, False, 1e-6))


@pytest.mark.parametrize("table_dtype,w_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
def test_table_and_weight_types(table_dtype, w_dtype):
    from mjolnir_b200 import qkrope

    x, table, w, pos = _case(9, 4, 2, 128, 128, torch.float16, 3, table_dtype, w_dtype)
    qo, ko = qkrope.qk_norm_rope(x[:, :4].cuda(), x[:, 4:6].cuda(), pos.cuda(), table.cuda(), w[0].cuda(), w[1].cuda())
    torch.cuda.synchronize()
    _check(qo, *_plain(x[:, :4], w[0], table, pos, False, 1e-6))
    _check(ko, *_plain(x[:, 4:6], w[1], table, pos, False, 1e-6))


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_unaligned_rows_and_strided_table(interleaved):
    from mjolnir_b200 import qkrope

    T, h_q, h_k, d = 33, 3, 2, 128
    x, table, w, pos = _case(T, h_q, h_k, d, 64, torch.bfloat16, seed=4)
    wide = torch.zeros(T, (h_q + h_k) * (d + 1) + 3, dtype=torch.bfloat16, device="cuda")
    rows = wide[:, 3:].view(T, h_q + h_k, d + 1)[..., 1:]  # rows 2-byte aligned
    rows.copy_(x[:, :h_q + h_k])
    before = wide.clone()
    big = torch.zeros(64, 67, device="cuda")
    big[:, 1:65] = table.cuda()
    qkrope.qk_norm_rope(rows[:, :h_q], rows[:, h_q:], pos.cuda(), big[:, 1:65], w[0].cuda(), w[1].cuda(),
                        interleaved=interleaved, q_out=rows[:, :h_q], k_out=rows[:, h_q:])
    torch.cuda.synchronize()
    _check(rows[:, :h_q].contiguous(), *_plain(x[:, :h_q], w[0], table, pos, interleaved, 1e-6))
    _check(rows[:, h_q:].contiguous(), *_plain(x[:, h_q:h_q + h_k], w[1], table, pos, interleaved, 1e-6))
    rows.copy_(before[:, 3:].view(T, h_q + h_k, d + 1)[..., 1:])
    assert torch.equal(wide, before), "wrote between the rows"


def test_zero_rows_large_values_and_bad_positions():
    from mjolnir_b200 import qkrope

    x, table, w, pos = _case(6, 2, 1, 128, 128, torch.bfloat16, seed=5)
    x[0] = 0
    x[1] *= 1e15  # squares pass fp16 and bf16's precision, not 32 bits' range
    x[2, 0, 7] = float("nan")
    pos[3], pos[4] = -1, 64
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = [torch.full((6, n, 128), 5.0, dtype=torch.bfloat16, device="cuda") for n in (2, 1)]
    qkrope.qk_norm_rope(x[:, :2].cuda(), x[:, 2:3].cuda(), pos.cuda(), table.cuda(), w[0].cuda(), w[1].cuda(),
                        q_out=out[0], k_out=out[1], status=status)
    torch.cuda.synchronize()
    assert int(status) == 4  # MJ_DEV_BAD_POSITION
    assert (out[0][3:5] == 5).all() and (out[1][3:5] == 5).all()
    keep = [0, 1, 5]
    want, slack = _plain(x[keep, :2], w[0], table, pos[keep], False, 1e-6)
    _check(out[0][keep], want, slack)
    assert torch.isnan(out[0][2, 0]).all() and torch.isfinite(out[0][2, 1]).all()
