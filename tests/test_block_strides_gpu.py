"""Dims of extent 1 may carry any stride: single tokens, and single heads, as
views whose stride in that dim is no multiple of 16 bytes."""

import pytest
import torch

from tests.block_helpers import Cache

pytestmark = pytest.mark.gpu


def _odd(x, dim):
    """The same values as a 16-byte aligned view with a stride of 12345 in `dim` (extent 1)."""
    st = list(x.stride())
    st[dim] = 12345
    return x.as_strided(x.shape, st)


@pytest.mark.parametrize("tokens,h_k,dim", [(1, 2, 0), (1, 1, 0), (1, 1, 1), (40, 1, 1)])
def test_rows(tokens, h_k, dim):
    from mjolnir_b200 import kvblock

    c = Cache([tokens + 60], h_k=h_k, seed=tokens)
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(tokens, h_k, 128, generator=g, device="cuda").to(torch.bfloat16)
    caches = [kvblock.views(*kvblock.alloc(c.pages, 16, h_k, 128, 16)) for _ in (0, 1)]
    for cache, k in zip(caches, (x, _odd(x, dim))):
        kvblock.write(k, k, *cache, torch.arange(tokens, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(*caches))
    outs = []
    for pick in (lambda t: t, lambda t: _odd(t, dim)):
        k, v = (pick(torch.empty_like(x)) for _ in (0, 1))
        outs.append(kvblock.read(*c.args, c.table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"),
                                 torch.tensor([0, tokens], dtype=torch.int32, device="cuda"), k, v))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    r = kvblock.BlockAttention(num_heads=h_k, num_kv_heads=h_k, head_size=128, page_size=16, max_num_seqs=1, max_num_tokens=40)
    plan = r.plan([tokens], c.lens, c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda())
    want = r.run(plan, x, torch.empty_like(x), *c.args, 128**-0.5)
    got = r.run(plan, _odd(x, dim), _odd(torch.empty_like(x), dim), *c.args, 128**-0.5)
    assert torch.equal(got, want)
