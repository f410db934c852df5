"""The block-scaled cache's write and read-back against their plain forms:
cache bytes and values are exact."""

import numpy as np
import pytest
import torch

from tests.block_helpers import Cache, write_plain

pytestmark = pytest.mark.gpu


class Writer:
    """A cache on the device beside its plain copy."""

    def __init__(self, pages, page, block, h_k, d, split=False):
        from mjolnir_b200 import kvblock

        self.page, self.block, self.h_k, self.d = page, block, h_k, d
        if split:  # token-major codes, head-last scales, K and V apart
            self.views = [torch.zeros(pages, page, h_k, d, dtype=torch.uint8, device="cuda") for _ in (0, 1)]
            self.views += [torch.zeros(pages, page // block, h_k, dtype=torch.uint8, device="cuda") for _ in (0, 1)]
        else:
            self.views = list(kvblock.views(*kvblock.alloc(pages, page, h_k, d, block)))
        for v in self.views:
            v.fill_(0xA5 if v.dim() == 4 else 0)
        self.plain = [v.cpu().numpy().copy() for v in self.views]

    def write(self, key, value, slots, **kw):
        from mjolnir_b200 import kvblock

        kvblock.write(key.cuda(), value.cuda(), *self.views, torch.as_tensor(slots).cuda(), **kw)
        torch.cuda.synchronize()
        good = [s if s < self.views[0].shape[0] * self.page else -1 for s in slots]
        for side, x in ((0, key), (1, value)):
            write_plain(x.double().numpy(), self.plain[side], self.plain[2 + side], good, self.page, self.block)

    def check(self):
        for name, got, want in zip(("K codes", "V codes", "K scales", "V scales"), self.views, self.plain):
            np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=name)


def _xy(g, T, h_k, d, dtype, ramp=None):
    x = torch.randn(T, h_k, d, generator=g)
    if ramp is not None:
        x = x * ramp[:, None, None]
    return x.to(dtype), (torch.randn(T, h_k, d, generator=g) * 0.1).to(dtype)


@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("d,dtype,split", [(128, torch.bfloat16, False), (256, torch.float16, True), (128, torch.float32, True)])
def test_whole_sequences_then_token_by_token(page, block, d, dtype, split):
    """Two ragged prompts, then single tokens whose size grows: scales grow and earlier rows follow."""
    g = torch.Generator().manual_seed(page + block)
    w = Writer(9, page, block, 3, d, split)
    perm = torch.randperm(9, generator=g).tolist()
    a, b = page + 5, 2 * page - 1
    slot = lambda first, i: perm[first + i // page] * page + i % page  # noqa: E731
    k, v = _xy(g, a + b, 3, d, dtype)
    w.write(k, v, [slot(0, i) for i in range(a)] + [slot(4, i) for i in range(b)])
    w.check()
    for step in range(6):
        k, v = _xy(g, 2, 3, d, dtype, torch.full((2,), 3.0 ** step))
        w.write(k, v, [slot(0, a + step), slot(4, b + step)])
        w.check()


def test_a_block_filled_token_by_token_equals_one_write():
    """Scales are powers of two, so the order of arrival leaves no trace (no code here becomes subnormal)."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(16, 2, 128, generator=g).sign() * (1 + torch.rand(16, 2, 128, generator=g)) * torch.linspace(0.2, 3, 16)[:, None, None]
    x = x.to(torch.bfloat16)
    one, many = Writer(2, 16, 16, 2, 128), Writer(2, 16, 16, 2, 128)
    one.write(x, x, list(range(16, 32)))
    for i in range(16):
        many.write(x[i:i + 1], x[i:i + 1], [16 + i])
    for p, q in zip(one.views, many.views):
        assert torch.equal(p, q)


def test_reused_page_forgets_its_old_scale():
    g = torch.Generator().manual_seed(6)
    w = Writer(1, 16, 16, 1, 128)
    big, _ = _xy(g, 16, 1, 128, torch.bfloat16)
    w.write(big * 1000, big, list(range(16)))
    w.write(big[:3] * 0.01, big[:3], [0, 1, 2])
    w.check()
    assert int(w.views[2].max()) < 120


def test_skips_order_and_single_rows():
    """Negative entries anywhere, rows out of order, rewritten rows, a block that starts mid-way."""
    g = torch.Generator().manual_seed(7)
    w = Writer(6, 32, 16, 2, 128)
    k, v = _xy(g, 12, 2, 128, torch.bfloat16)
    w.write(k, v, [-1, 35, -1, 33, 32, -1, -1, 100, -1, 0, 1, -1])
    w.check()
    w.write(k * 5, v, [-1, 33, -1, -1, 36, -1, -1, 101, 2, -1, -1, -1])
    w.check()
    w.write(k, v, [-1] * 12)
    w.check()


def test_long_gaps_of_skipped_tokens():
    g = torch.Generator().manual_seed(8)
    w = Writer(3, 128, 128, 1, 128)
    T = 700
    slots = [-1] * T
    for i, t in enumerate(range(3, T, 8)):  # every eighth token is this rank's
        slots[t] = 128 + i
    k, v = _xy(g, T, 1, 128, torch.bfloat16)
    w.write(k, v, slots)
    w.check()


def test_extreme_values():
    """Zeros, subnormals, infinities, NaN and magnitudes beyond the scale range."""
    w = Writer(4, 16, 16, 1, 128)
    x = torch.randn(64, 1, 128, generator=torch.Generator().manual_seed(9))
    x[:16] = 0
    x[16, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), -0.0])
    x[20:32] *= 1e-39
    x[32:48] = x[32:48] * 1e30
    x[48, 0, 0], x[49, 0, 1], x[50, 0, 2] = 448.0, 449.0, 1.75 * 2.0**20
    for dt in (torch.float32, torch.bfloat16):
        w.write(x.to(dt), x.to(dt), list(range(64)))
        w.check()


def test_every_bf16_value():
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).reshape(512, 1, 128)
    w = Writer(32, 16, 16, 1, 128)
    w.write(x, x.flip(0), list(range(512)))
    w.check()


def test_strided_rows_int32_slots_and_another_stream():
    from mjolnir_b200 import kvblock

    g = torch.Generator().manual_seed(10)
    w = Writer(4, 16, 16, 2, 128)
    fused = torch.randn(20, 8, 128, generator=g).to(torch.bfloat16).cuda()
    k, v = fused[:, 4:6], fused[:, 6:8]
    slots = torch.randperm(4, generator=g)[:2].repeat_interleave(10) * 16 + torch.arange(10).repeat(2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kvblock.write(k, v, *w.views, slots.int().cuda())
    torch.cuda.synchronize()
    for side, x in ((0, k), (1, v)):
        write_plain(x.double().cpu().numpy(), w.plain[side], w.plain[2 + side], slots.tolist(), 16, 16)
    w.check()


def test_empty_call_and_bad_slot():
    w = Writer(2, 16, 16, 1, 128)
    x = torch.randn(4, 1, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    w.write(x[:0], x[:0], [])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    w.write(x, x, [0, 1, 32, 17], status=status)
    w.check()
    assert int(status) == 1


@pytest.mark.parametrize("h_k,d,page,block,split", [(2, 128, 16, 16, False), (9, 128, 64, 32, True), (3, 256, 128, 128, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read(h_k, d, page, block, split, dtype):
    from mjolnir_b200 import kvblock

    lens = [1, 77, 0, 300, page]
    c = Cache(lens, h_k=h_k, d=d, page=page, block=block, split=split, seed=h_k)
    starts = [0, 5, 0, 123, 0]
    off = np.concatenate([[0], np.cumsum([n - a for n, a in zip(lens, starts)])]).astype(np.int32)
    total = int(off[-1])
    outs = [torch.full((total + 2, h_k + 1, d), -3.0, dtype=dtype, device="cuda") for _ in (0, 1)]
    got = kvblock.read(*c.args, c.table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), torch.from_numpy(off).cuda(),
                       *[o[:, :h_k] for o in outs])
    torch.cuda.synchronize()
    for side in (0, 1):
        want = torch.cat([c.rows(s, a, n, side) for s, (a, n) in enumerate(zip(starts, lens))]).to(dtype)
        assert torch.equal(got[side].cpu()[:total], want)
        assert (outs[side][total:] == -3).all() and (outs[side][:, h_k:] == -3).all(), "wrote a row it was not given"


def test_read_flags_bad_pages():
    from mjolnir_b200 import kvblock

    c = Cache([40, 40], h_k=1)
    table = c.table.clone()
    table[0, 1] = c.pages
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((80, 1, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    kvblock.read(*c.args, table.cuda(), torch.zeros(2, dtype=torch.int32).cuda(),
                 torch.tensor([0, 40, 80], dtype=torch.int32).cuda(), out, torch.empty_like(out), status=status)
    torch.cuda.synchronize()
    assert int(status) == 1
    assert (out[16:32] == 9).all()
    assert torch.equal(out[40:].cpu(), c.rows(1, 0, 40, 0).to(torch.bfloat16))


def test_pages_past_32_bit_offsets():
    """A cache of more than 2^32 bytes: its last pages write and read back."""
    from mjolnir_b200 import kvblock

    pages = (1 << 32) // (8 * 128 * 256) + 40
    views = kvblock.views(*kvblock.alloc(pages, 128, 8, 128, 16))
    x = torch.randn(300, 8, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    pos = torch.arange(300)
    slots = table[0, pos // 128].long() * 128 + pos % 128
    kvblock.write(x, -x, *views, slots.cuda())
    k, v = torch.empty_like(x), torch.empty_like(x)
    kvblock.read(*views, table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"),
                 torch.tensor([0, 300], dtype=torch.int32, device="cuda"), k, v)
    torch.cuda.synchronize()
    assert torch.equal(k, -v)
    # e4m3 keeps 4 significant bits; below 2^-6 of the scale its steps are 2^-9
    # of it, and the scale is under 2^-7 of the block's largest (< 8 here)
    err = (k.float() - x.float()).abs()
    assert (err <= x.float().abs() * 2.0**-4 + 2.0**-13).all()
