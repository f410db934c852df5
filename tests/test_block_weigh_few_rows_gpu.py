"""The weights of steps with a few rows a sequence, whose queries enter as three e4m3 terms, against 64 bits."""

import pytest
import torch

from tests.block_helpers import Cache, attention_plain, values
from tests.test_block_weigh_gpu import run, weigh_plain

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def check(c, q, q_lens, scale):
    """Beyond the sums' bound of the other tests: an element of a row that 2^x brings into [128, 256) is off by 2^-18 in
    that range at most, half a step of the third term, and not at all where its last bit stands at 2^-17 or above."""
    h_q, group = q.shape[1], q.shape[1] // c.h_k
    lse = attention_plain(c, q, q_lens, scale)[1].float()
    old = torch.rand(len(q_lens), c.h_k, max(c.lens), generator=c.g) / max(c.lens)
    got, status = run(c, q.cuda(), lse.cuda(), q_lens, old, scale)
    assert status == 0
    want, tol = weigh_plain(c, q, lse, q_lens, old, scale)
    up = torch.exp2((8 - torch.frexp(q.float().abs().amax(-1)).exponent).clamp(-126, 126).double())  # (tokens, h_q)
    lsb = 2.0 ** (torch.frexp(q.float()).exponent.double() - (8 if q.dtype == torch.bfloat16 else 11))
    lsb = torch.maximum(lsb, torch.full_like(lsb, 2.0**-133 if q.dtype == torch.bfloat16 else 2.0**-24))
    off = torch.where((lsb * up[..., None] >= 2.0**-17) | (q == 0), 0.0, 2.0**-18 / up[..., None])  # of each element
    at = 0
    for s, (m, L) in enumerate(zip(q_lens, c.lens)):
        k = c.rows(s, 0, L, 0)
        for h in range(h_q):
            sc = q[at:at + m, h].double() @ k[:, h // group].T * scale
            sees = torch.arange(L)[None] <= torch.arange(L - m, L)[:, None]
            p = torch.where(sees, (sc - lse[at:at + m, h].double()[:, None]).exp(), 0.0)
            lost = off[at:at + m, h] @ k[:, h // group].abs().T * scale
            tol[s, h // group, :L] += (p * torch.expm1(lost)).sum(0)
        at += m
        err = (got[s, :, :L].double() - want[s, :, :L]).abs()
        assert torch.isfinite(got[s, :, :L]).all() and (err <= tol[s, :, :L]).all(), (s, (err / tol[s, :, :L]).max().item())


def caches(d, **kw):
    return Cache([400, 33, 129], h_k=2, d=d, seed=d, **kw)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("q_len", [1, 2])
@pytest.mark.parametrize("dtype,q_scale,scale", [(torch.float16, 7.5e3, 1e-6), (torch.float16, 2.5e-6, 1e3), (torch.float16, 1.5e4, 1e-7),
                                                 (torch.bfloat16, 1e20, 1e-22), (torch.bfloat16, 1e30, 1e-32), (torch.bfloat16, 1e-30, 1e28)])
def test_large_and_small_queries(d, q_len, dtype, q_scale, scale):
    c = caches(d)
    check(c, (torch.randn(3 * q_len, 8, d, generator=c.g) * q_scale).to(dtype), [q_len] * 3, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [128, 256])
def test_wild_scales_and_growing_scores(d, dtype):
    for kw, q_scale in ((dict(k_ramp=8.0), 4.0), (dict(spread=10), 0.05)):
        c = caches(d, **kw)
        check(c, (torch.randn(6, 8, d, generator=c.g) * q_scale).to(dtype), [2] * 3, d**-0.5)


@pytest.mark.parametrize("dtype,size,scale", [(torch.bfloat16, 2.0**-133, 1e37), (torch.float16, 2.0**-24, 3e4)])
@pytest.mark.parametrize("d", [128, 256])
def test_rows_of_subnormals(d, dtype, size, scale):
    """Every element a few times the type's least one, one row with that alone."""
    c = caches(d)
    q = (torch.randint(-40, 41, (6, 8, d), generator=c.g).double() * size).to(dtype)
    q[1] = 0
    q[1, :, 5] = size
    check(c, q, [2] * 3, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [128, 256])
def test_rows_of_zeros(d, dtype):
    c = caches(d)
    q = torch.randn(6, 8, d, generator=c.g).to(dtype)
    q[0], q[3, 2:], q[5, :, d // 2:] = 0, 0, 0
    check(c, q, [2] * 3, d**-0.5)
    check(c, torch.zeros_like(q), [2] * 3, d**-0.5)


@pytest.mark.parametrize("used", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,above", [(128, 14), (128, 16), (128, 18), (256, 15), (256, 20)])
def test_one_element_far_above_the_others(d, above, dtype, used):
    """The other elements lose their last bits to it; where K has nothing there they alone make the scores."""
    c = caches(d)
    at = 37
    if not used:
        c.kv[0][..., at] = 0
        c.codes[0][..., at] = 0
        c.vals[0] = values(c.codes[0], c.exps[0])
    small = 2.0 ** (14 - above)  # the outlier stays inside fp16
    q = (torch.randn(6, 8, d, generator=c.g) * small).to(dtype)
    q[..., at] = torch.where(torch.rand(6, 8, generator=c.g) < 0.5, -1.0, 1.0) * 2.0**14
    check(c, q, [2] * 3, (2.0**-14 if used else 1 / small) * d**-0.5)
