"""The operators of long-lived contexts as a layer would run them, one after
another, against the formulas in 64 bits: rotation by three axes, the cache
write, attention behind a shared prefix, the weights that the cached tokens
received, eviction by them, and single tokens over what is left."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H_Q, H_K, D, PAGE, BLOCK = 8, 2, 128, 16, 16
GROUP = H_Q // H_K


class Layer:
    """A cache and its runner; the tables and lengths of five sequences, the first three behind the same 384 tokens."""

    def __init__(self):
        from mjolnir_b200 import kvblock, qkrope

        g = torch.Generator("cuda").manual_seed(0)
        self.g, self.kv, self.rope = g, kvblock, qkrope
        self.cache, self.scales = kvblock.alloc(256, PAGE, H_K, D, BLOCK)
        self.views = kvblock.views(self.cache, self.scales)
        perm = torch.randperm(256, generator=g, device="cuda").int()
        self.table = perm[:5 * 48].view(5, 48).contiguous()
        self.table[1:3, :24] = self.table[0, :24]
        self.runner = kvblock.BlockAttention(num_heads=H_Q, num_kv_heads=H_K, head_size=D, page_size=PAGE, block_tokens=BLOCK,
                                             max_num_seqs=5, max_num_tokens=1216)
        self.norm = [(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(2)]
        inv = 1.0e4 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        angle = torch.arange(4096, device="cuda")[:, None] * inv
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
        self.axes = qkrope.angle_axes((24, 20, 20), alternate=True)
        self.weights = torch.zeros(5, H_K, 768, device="cuda")

    def project(self, n, position):
        """Q, K and V of n new tokens from a position on: images of 24 columns."""
        qkv = torch.randn(n, (H_Q + 2 * H_K) * D, generator=self.g, device="cuda").bfloat16()
        q, k, v = (x.view(n, -1, D) for x in qkv.split([H_Q * D, H_K * D, H_K * D], 1))
        i = torch.arange(n, device="cuda")
        pos = torch.stack([i * 0 + position, position + i // 24, position + i % 24])
        q, k = self.rope.qk_norm_rope(q, k, pos, self.cos_sin, *self.norm, axes=self.axes)
        return q, k, v

    def write(self, s, begin, k, v):
        pos = torch.arange(begin, begin + len(k), device="cuda")
        self.kv.write(k, v, *self.views, self.table[s, pos // PAGE].long() * PAGE + pos % PAGE)

    def rows(self, s, n):
        """What the cache holds of a sequence, (n, h_k, d) in 64 bits."""
        out = [torch.empty(n, H_K, D, device="cuda") for _ in range(2)]
        self.kv.read(*self.views, self.table[s:s + 1], torch.zeros(1, dtype=torch.int32, device="cuda"),
                     torch.tensor([0, n], dtype=torch.int32, device="cuda"), *out)
        return [x.double() for x in out]

    def attend(self, q, new, lens, shared=()):
        at = torch.tensor(lens, dtype=torch.int32, device="cuda")
        plan = self.runner.plan(new, lens, self.table, at, shared=shared)
        out, lse = torch.empty_like(q), torch.empty(len(q), H_Q, device="cuda")
        self.runner.run(plan, q, out, *self.views, D**-0.5, lse=lse)
        offsets = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        self.kv.weigh(q, lse, self.views[0], self.views[2], self.table, offsets, at, self.weights, D**-0.5)
        torch.cuda.synchronize()
        self.runner.check_status()
        return out, plan

    def check(self, q, out, new, lens, before):
        """Outputs and weights of a step, from what the cache holds."""
        at = 0
        for s, (n, L) in enumerate(zip(new, lens)):
            k, v = self.rows(s, L)
            sees = torch.arange(L, device="cuda") <= torch.arange(L - n, L, device="cuda")[:, None]
            received = torch.zeros(H_K, L, dtype=torch.float64, device="cuda")
            for h in range(H_Q):
                score = (q[at:at + n, h].double() @ k[:, h // GROUP].T * D**-0.5).masked_fill(~sees, -math.inf)
                p = score.softmax(-1)
                want, mag = p @ v[:, h // GROUP], p @ v[:, h // GROUP].abs()
                # P in 11 bits or more, scores as much again, one rounding of the output to bf16
                assert ((out[at:at + n, h].double() - want).abs() <= 2.0**-10 * mag + 2.0**-8 * want.abs() + 1e-6).all()
                received[h // GROUP] += p.sum(0)
            old = before[s, :, :L].double()
            old[:, L - n:] = 0
            # the lse that the step left is off by some 1e-5 at most, which is the weights' relative error
            assert ((self.weights[s, :, :L].double() - old - received).abs() <= 1e-4 * received + 1e-6 * old + 1e-7).all()
            at += n


@pytest.fixture
def share(monkeypatch):
    from mjolnir_b200 import kvblock

    monkeypatch.setattr(kvblock.BlockAttention, "_worth", lambda self, *a: True)  # (too small to pay)


def test_a_layer_over_a_long_life(share):
    m = Layer()
    prompts, shared = [500, 430, 390, 700, 333], [(0, 3, 384)]
    # prompts: the shared part once, then every sequence's own
    parts = [m.project(n - 384 if s in (1, 2) else n, 0 if s not in (1, 2) else 384) for s, n in enumerate(prompts)]
    for s, (_, k, v) in enumerate(parts):
        m.write(s, 384 if s in (1, 2) else 0, k, v)
    new = [116, 46, 6, 700, 333]
    q = torch.cat([parts[0][0][384:], parts[1][0], parts[2][0], parts[3][0], parts[4][0]])
    out, plan = m.attend(q, new, prompts, shared)
    assert plan.joins is not None
    m.check(q, out, new, prompts, torch.zeros_like(m.weights))
    # a few single tokens of each
    lens = list(prompts)
    for _ in range(3):
        now = [m.project(1, n) for n in lens]
        for s, (_, k, v) in enumerate(now):
            m.write(s, lens[s], k, v)
        lens = [n + 1 for n in lens]
        before, q = m.weights.clone(), torch.cat([x[0] for x in now])
        out, plan = m.attend(q, [1] * 5, lens, shared)
        assert plan.joins is not None
        m.check(q, out, [1] * 5, lens, before)
    # the last two, whose pages are their own, down to 256 tokens a head
    held = [m.rows(s, lens[s]) for s in (3, 4)]
    w = m.weights[3:].clone()
    kept, left = torch.empty(2, H_K, 256, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    m.kv.evict(m.weights[3:], *m.views, m.table[3:], torch.tensor(lens[3:], dtype=torch.int32, device="cuda"), left, kept, recent=32)
    assert left.tolist() == [256, 256]
    for i, s in enumerate((3, 4)):
        for h in range(H_K):
            at = kept[i, h].long()
            heavy = at[:224]
            assert (at[1:] > at[:-1]).all() and at[224:].tolist() == list(range(lens[s] - 32, lens[s]))
            rest = torch.ones(lens[s] - 32, dtype=torch.bool, device="cuda")
            rest[heavy] = False
            assert w[i, h, heavy].min() >= w[i, h, :lens[s] - 32][rest].max()
            assert torch.equal(m.weights[s, h, :256], w[i, h, at])
            for side, x in enumerate(m.rows(s, 256)):
                # e4m3 again: half a step of 2^-3, or of the block's subnormals, at its new scale
                old = held[i][side][at, h]
                top = old.view(16, 16, D).abs().amax((1, 2)).repeat_interleave(16)[:, None]
                assert ((x[:, h] - old).abs() <= torch.maximum(2.0**-4 * old.abs(), top * 2.0**-17)).all()
    # and on: single tokens over what is left, at the positions that they would have had
    positions, lens = list(lens), lens[:3] + [256, 256]
    for _ in range(2):
        now = [m.project(1, n) for n in positions]
        for s, (_, k, v) in enumerate(now):
            m.write(s, lens[s], k, v)
        positions, lens = [n + 1 for n in positions], [n + 1 for n in lens]
        before, q = m.weights.clone(), torch.cat([x[0] for x in now])
        out, _ = m.attend(q, [1] * 5, lens, shared)
        m.check(q, out, [1] * 5, lens, before)
