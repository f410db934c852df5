"""The block-scaled write and read-back at pages of any multiple of the block,
powers of two or not: exact, and no other page is touched."""

import pytest
import torch

from tests.block_helpers import Cache
from tests.test_block_cache_gpu import Writer

pytestmark = pytest.mark.gpu

PAGES = [(48, 16), (80, 16), (96, 32), (144, 16), (192, 64), (384, 128), (1008, 16)]


@pytest.mark.parametrize("page,block", PAGES)
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (256, torch.float32)])
def test_write(page, block, d, dtype):
    """Whole pages, a run over a page's end, then single tokens of growing size."""
    g = torch.Generator().manual_seed(page)
    w = Writer(6, page, block, 2, d)
    slots = list(range(page - 5, page + 9)) + list(range(4 * page, 5 * page)) + [2 * page - 1, 6 * page - 1]
    k, v = (torch.randn(len(slots), 2, d, generator=g).to(dtype) for _ in (0, 1))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    w.write(k, v, slots, status=status)
    w.check()
    for step, slot in enumerate((page + 9, 5 * page, 2 * page - 2)):
        w.write(k[:1] * 3.0 ** (step + 1), v[:1], [slot], status=status)
        w.check()
    assert int(status) == 0
    w.write(k[:1], v[:1], [6 * page], status=status)
    w.check()
    assert int(status) == 1


@pytest.mark.parametrize("page,block", PAGES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_read(page, block, dtype):
    from mjolnir_b200 import kvblock

    lens, starts = [page + 7, 1, 2 * page], [page - 3, 0, 5]
    c = Cache(lens, h_k=3, page=page, block=block, seed=page)
    off = [0]
    for n, a in zip(lens, starts):
        off.append(off[-1] + n - a)
    out = [torch.empty(off[-1], 3, 128, dtype=dtype, device="cuda") for _ in (0, 1)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kvblock.read(*c.args, c.table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(off, dtype=torch.int32).cuda(),
                 *out, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for side in (0, 1):
        want = torch.cat([c.rows(s, a, n, side) for s, (a, n) in enumerate(zip(starts, lens))]).to(dtype)
        assert torch.equal(out[side].cpu(), want)


def test_many_pages():
    """Page numbers far beyond 16 bits."""
    from mjolnir_b200 import kvblock

    pages, page = 90_001, 48
    views = kvblock.views(*kvblock.alloc(pages, page, 1, 128, 16))
    x = torch.randn(100, 1, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16)
    table = torch.tensor([[pages - 1, 65_537, pages - 2]], dtype=torch.int32)
    pos = torch.arange(100)
    kvblock.write(x, -x, *views, (table[0, pos // page].long() * page + pos % page).cuda())
    k, v = torch.empty_like(x), torch.empty_like(x)
    kvblock.read(*views, table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"),
                 torch.tensor([0, 100], dtype=torch.int32, device="cuda"), k, v)
    torch.cuda.synchronize()
    assert torch.equal(k, -v)
    # the codes' page is where the table says, and no other row was written
    written = (views[0].view(pages, page, -1) != 0).any(-1).nonzero()
    assert written[:, 0].unique().tolist() == [65_537, pages - 2, pages - 1] and len(written) == 100
    # e4m3 keeps 4 significant bits; below 2^-6 of the scale its steps are 2^-9
    # of it, and the scale is under 2^-7 of the block's largest (< 8 here)
    err = (k.float() - x.float()).abs()
    assert (err <= x.float().abs() * 2.0**-4 + 2.0**-13).all()
