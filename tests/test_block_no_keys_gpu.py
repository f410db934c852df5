"""Chunks whose whole row blocks see no key: empty sequences, and more queries
than tokens. Their outputs are zeros and their log-sum-exp -inf, whatever the
queries hold."""

import math

import pytest
import torch

from tests.block_helpers import Cache, assert_attention, attention_plain
from tests.test_block_attention_gpu import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,h_q,h_k", [(128, 1, 1), (128, 8, 2), (256, 1, 1), (256, 6, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,lens", [([300], [0]), ([300], [10]), ([700, 64, 90, 130], [3, 0, 200, 0])])
def test_rows_before_the_first_key(q_lens, lens, d, h_q, h_k, dtype, causal):
    c = Cache(lens, h_k=h_k, d=d, seed=d + h_q)
    q = torch.randn(sum(q_lens), h_q, d, generator=c.g).to(dtype)
    want, want_lse, mag = attention_plain(c, q, q_lens, d**-0.5, causal)
    none = torch.isinf(want_lse)
    assert none.any() or not causal
    for _ in range(5):
        got, lse = _run(c, q, q_lens, causal, lse=True)
        assert (got.cpu()[none] == 0).all() and (lse.cpu()[none] == -math.inf).all()
        assert_attention(got, want, mag)
