"""fp16 steps of single tokens and drafts are as exact behind a shared prefix as without one."""

import pytest
import torch

from tests.block_helpers import UNIT, Cache, attention_plain, values

pytestmark = pytest.mark.gpu


def step(monkeypatch, d, h_q, q_len, dtype, shared):
    """A step's (output, exact output, sum of p |v|) over a cache whose V is zero but for two tokens of the prefix: what their
    weights lost shows where their rows cancel."""
    from mjolnir_b200 import kvblock

    monkeypatch.setattr(kvblock.BlockAttention, "_worth", lambda self, *a: True)
    n, prefix = 6, 1024
    c = Cache([prefix + q_len + 3 * s for s in range(n)], h_k=2, d=d, seed=d + q_len, spread=0)
    c.table[1:, :prefix // c.page] = c.table[0, :prefix // c.page]
    codes = torch.zeros_like(c.codes[1])
    for token in (333, 777):
        page, row = int(c.table[0, token // c.page]), token % c.page
        codes[page, row] = c.codes[1][page, row]
    c.kv[1].copy_(codes.cuda())
    c.sc[1].fill_(131)  # outputs far above fp16's subnormals
    c.vals[1] = values(codes, torch.full_like(c.exps[1], 131))
    q_lens, scale = [q_len] * n, 0.5 * d**-0.5
    q = torch.randn(sum(q_lens), h_q, d, generator=c.g).to(dtype)
    r = kvblock.BlockAttention(num_heads=h_q, num_kv_heads=2, head_size=d, page_size=c.page, block_tokens=c.block, max_num_seqs=n,
                               max_num_tokens=sum(q_lens))
    plan = r.plan(q_lens, c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda(), shared=[(0, n, prefix)] if shared else [])
    assert plan.decode is not None and (plan.joins is not None) == shared
    got = r.run(plan, q.cuda(), torch.empty_like(q, device="cuda"), *c.args, scale)
    torch.cuda.synchronize()
    r.check_status()
    want, _, mag = attention_plain(c, q, q_lens, scale)
    return got.double().cpu(), want, mag


@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("d,h_q,q_len", [(128, 8, 1), (128, 24, 4), (128, 10, 3), (256, 8, 1), (256, 16, 2)])
def test_fp16_weights_of_decode_rows_keep_more_than_11_bits(monkeypatch, d, h_q, q_len, shared):
    """Scores below 8 (base 2) of at most 24 sums in 32 bits are off by 24 * 8 * 2^-23 = 2^-15.4 at most, polynomial
    exponentials by 2^-17.9, weights of two f16 terms by 2^-22: under 2^-14 of sum p |v| together. Weights of 11 bits are
    off by up to 2^-11. The decode kernel's three e4m3 terms are off by 2^-14 at most, together under 2^-13. Then one
    rounding of the output."""
    got, want, mag = step(monkeypatch, d, h_q, q_len, torch.float16, shared)
    tol = (2.0**-14 if shared else 2.0**-13) * mag
    worst = ((got - want).abs() / (tol + UNIT[torch.float16] * (want.abs() + tol))).max().item()
    assert worst <= 1.0, f"{worst:.3g} times the bound"


@pytest.mark.parametrize("d,h_q,q_len", [(128, 8, 1), (256, 8, 1)])
def test_bf16_weights_of_shared_prefixes_are_under_the_outputs_rounding(monkeypatch, d, h_q, q_len):
    """Two weights of 11 bits are off by 2^-11 of sum p |v| together, the rest as above: an eighth of bf16's half step of 2^-8."""
    got, want, mag = step(monkeypatch, d, h_q, q_len, torch.bfloat16, True)
    tol = (2.0**-11 + 2.0**-14) * mag
    worst = ((got - want).abs() / (tol + UNIT[torch.bfloat16] * (want.abs() + tol))).max().item()
    assert worst <= 1.0, f"{worst:.3g} times the bound"


@pytest.mark.parametrize("side", [0, 1])
def test_fp16_nan_in_the_prefix_reaches_every_row(monkeypatch, side):
    """A NaN code of K makes its KV head's rows NaN, one of V an element of them; the other KV head keeps its rows."""
    from mjolnir_b200 import kvblock

    monkeypatch.setattr(kvblock.BlockAttention, "_worth", lambda self, *a: True)
    c = Cache([600, 620, 640], h_k=2, seed=8)
    c.table[1:, :32] = c.table[0, :32]
    c.kv[side][int(c.table[0, 100 // 16]), 100 % 16, 0, 3] = 0x7F
    r = kvblock.BlockAttention(num_heads=4, num_kv_heads=2, head_size=128, page_size=16, max_num_seqs=3, max_num_tokens=3)
    plan = r.plan([1] * 3, c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda(), shared=[(0, 3, 512)])
    assert plan.joins is not None
    q = torch.randn(3, 4, 128, generator=c.g).half().cuda()
    out = r.run(plan, q, torch.zeros_like(q), *c.args, 128**-0.5).isnan().cpu()
    want = torch.zeros(3, 4, 128, dtype=torch.bool)
    want[:, :2] = True if side == 0 else torch.arange(128) == 3
    assert torch.equal(out, want)
