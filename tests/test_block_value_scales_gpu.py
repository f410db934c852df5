"""Neighbouring blocks whose V scales are far apart.

What multiplies a V code is P' = 2^(score + log2(V scale) - m), m the running
maximum of those exponents, in fewer bits than 32: f16 in the chunk kernel, whose
half step below 2^-14 is 2^-25, with the largest P' at 1 or more; three e4m3 terms
in the decode kernel, whose last half step is 2^-18, with the largest P' at 112
or more. So beside its 2^-11 of sum p |v| an output element is off by at most that
floor times the largest P' times the sum of its codes: it matters to an element
that the large block holds zeros in."""

import math

import pytest
import torch

from tests.block_helpers import UNIT, Cache, values
from tests.test_block_attention_gpu import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [4, 12, 16, 20, 28, 40])
@pytest.mark.parametrize("large", [0, 21, 39])
@pytest.mark.parametrize("d,h_q,q_len,dtype", [(128, 4, 90, torch.bfloat16), (256, 2, 90, torch.float16), (128, 4, 1, torch.bfloat16),
                                               (256, 4, 2, torch.float16)])
def test_elements_that_the_large_block_holds_zeros_in(gap, large, d, h_q, q_len, dtype):
    L, block = 640, 16
    c = Cache([L], h_k=1, d=d, block=block, seed=gap + large, spread=0)
    c.exps[1][:] = 110
    page = int(c.table[0, large])
    c.exps[1][page] = 110 + gap
    c.codes[1][page, :, :, : d // 2] = 0
    c.vals[1] = values(c.codes[1], c.exps[1])
    c.kv[1].copy_(c.codes[1])
    c.sc[1].copy_(c.exps[1])
    q = (torch.randn(q_len, h_q, d, generator=c.g) * 0.05).to(dtype)
    got, _ = _run(c, q, [q_len])
    got = got.double().cpu()
    k, v = c.rows(0, 0, L, 0)[:, 0], c.rows(0, 0, L, 1)[:, 0]
    ev = torch.full((L,), -17.0, dtype=torch.float64)
    ev[large * block:(large + 1) * block] += gap
    # beyond 16 rows at head size 256 and 48 at 128 the chunk kernel serves
    floor = 2.0**-25 if q_len > 4 else 2.0**-18 / 112
    sees = torch.arange(L)[None] <= torch.arange(L - q_len, L)[:, None]
    for h in range(h_q):
        score = (q[:, h].double() @ k.T * d**-0.5).masked_fill(~sees, -math.inf)
        p = score.softmax(-1)
        want, mag = p @ v, p @ v.abs()
        top = (p * torch.exp2(ev)).amax(-1, keepdim=True)
        tol = 2.0**-10 * mag + floor * top * (sees.double() @ (v.abs() * torch.exp2(-ev)[:, None])) + 1e-12
        tol = tol + UNIT[dtype] * (want.abs() + tol) + (2.0**-25 if dtype == torch.float16 else 0)
        # an infinity where the value passes the output type, give or take the bound
        most, inf = torch.finfo(dtype).max, got[:, h].isinf()
        assert (want.abs() + tol)[inf].gt(most).all() and (got[:, h][inf].sign() == want[inf].sign()).all()
        assert (want.abs() - tol)[~inf].le(most).all()
        worst = ((got[:, h] - want).abs() / tol)[~inf].max().item()
        assert worst <= 1.0, f"head {h}: {worst:.3g} times the bound"
