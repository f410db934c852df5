"""Plain 64-bit forms of the block-scaled cache operators, and builders for
their tests. Everything here runs on the CPU in numpy / torch."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import quant

E_MIN, E_MAX = 95, 159
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}  # relative half ulp


def exponent(amax: float) -> int:
    """Smallest e in range with amax <= 448 * 2^(e - 127)."""
    if not amax > 0:
        return E_MIN
    e = E_MIN
    while e < E_MAX and amax > 448.0 * 2.0 ** (e - 127):
        e += 1
    return e


def codes_of(x: np.ndarray, e: int) -> np.ndarray:
    """e4m3 bytes of float64 values at scale 2^(e - 127): nearest even, saturating, NaN -> 0x7F."""
    y = np.clip(np.asarray(x, np.float64) * 2.0 ** (127 - e), -448.0, 448.0)
    out = quant.quantize_rows_fp8(y.astype(np.float32).reshape(1, 1, -1), np.ones(1, np.float32)).reshape(y.shape)
    return np.where(np.isnan(x), 0x7F, out).astype(np.uint8)


def write_plain(x, codes, exps, slots, page, block) -> None:
    """The write of one side, in place: x (T, h, d) float64, codes (pages,
    page, h, d) and exps (pages, page / block, h) uint8 arrays."""
    T, h_k, d = x.shape
    runs: dict[int, list[int]] = {}
    for t, s in enumerate(slots):
        if s >= 0:
            runs.setdefault(s // block, []).append(t)
    for b, toks in runs.items():
        pg, sub = divmod(b, page // block)
        rows = [slots[t] % page for t in toks]
        opened = sub * block in rows
        for h in range(h_k):
            part = np.abs(x[toks, h])
            part = part[np.isfinite(part)]
            need = exponent(part.max() if part.size else 0.0)
            old = min(max(int(exps[pg, sub, h]), E_MIN), E_MAX)
            e = need if opened else max(old, need)
            if not opened and e > old:
                for r in range(sub * block, sub * block + block):
                    if r not in rows:
                        codes[pg, r, h] = codes_of(quant.decode_fp8(codes[pg, r, h]).astype(np.float64) * 2.0 ** (old - 127), e)
            exps[pg, sub, h] = e
            for t, r in zip(toks, rows):
                codes[pg, r, h] = codes_of(x[t, h], e)


def values(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """(pages, page, h, d) float64 values of code and exponent bytes."""
    page, blocks = codes.shape[1], exps.shape[1]
    v = torch.from_numpy(quant.decode_fp8(codes.numpy())).double()
    e = exps.long().clamp(E_MIN, E_MAX).repeat_interleave(page // blocks, 1)
    return v * torch.exp2(e.double() - 127)[..., None]


class Cache:
    """A filled paged cache on the device and its values on the host. Every
    byte no token owns is NaN code / a huge scale."""

    def __init__(self, lens, *, h_k=2, d=128, page=16, block=16, seed=0, split=False, spare=3, spread=2,
                 k_ramp=0.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.block, self.h_k, self.d = [int(x) for x in lens], page, block, h_k, d
        n = [-(-L // page) for L in self.lens]
        self.pages = sum(n) + spare
        perm = torch.randperm(self.pages, generator=g)
        self.table = torch.full((max(1, len(n)), max([1, *n]) + 1), -7, dtype=torch.int32)
        codes = torch.full((2, self.pages, page, h_k, d), 0x7F, dtype=torch.uint8)
        exps = torch.full((2, self.pages, page // block, h_k), 255, dtype=torch.uint8)
        at = 0
        for s, L in enumerate(self.lens):
            pg = perm[at:at + n[s]]
            at += n[s]
            self.table[s, :n[s]] = pg.int()
            for side in range(2):
                x = torch.randn(L, h_k, d, generator=g) * 70
                if side == 0 and k_ramp:
                    x = x * (1 + k_ramp * torch.arange(L)[:, None, None] / max(1, L)) / (1 + k_ramp)
                by = torch.from_numpy(quant.quantize_rows_fp8(x.numpy(), np.ones(1, np.float32)))
                pad = torch.full((n[s] * page, h_k, d), 0x7F, dtype=torch.uint8)
                pad[:L] = by
                codes[side, pg] = pad.view(n[s], page, h_k, d)
                e = torch.randint(121 - spread, 121 + spread + 1, (n[s] * page // block, h_k), generator=g)
                keep = -(-L // block)
                ee = torch.full((n[s] * page // block, h_k), 255, dtype=torch.uint8)
                ee[:keep] = e[:keep].to(torch.uint8)
                exps[side, pg] = ee.view(n[s], page // block, h_k)
        self.codes, self.exps, self.g = codes, exps, g
        self.vals = [values(codes[i], exps[i]) for i in (0, 1)]
        if split:  # separate (pages, page, h, d) tensors, scales head-last
            self.kv = [codes[i].cuda() for i in (0, 1)]
            self.sc = [exps[i].cuda() for i in (0, 1)]
        else:
            both = torch.cat([codes[0], codes[1]], -1).transpose(1, 2).contiguous().cuda()
            sc = torch.stack([exps[0], exps[1]], 1).permute(0, 3, 1, 2).contiguous().cuda()
            self.kv = [both[..., :d].transpose(1, 2), both[..., d:].transpose(1, 2)]
            self.sc = [sc[:, :, 0].transpose(1, 2), sc[:, :, 1].transpose(1, 2)]

    @property
    def args(self):
        return (*self.kv, *self.sc)

    def rows(self, s: int, begin: int, end: int, side: int) -> torch.Tensor:
        pos = torch.arange(begin, end)
        return self.vals[side][self.table[s, pos // self.page].long(), pos % self.page]


def attention_plain(cache: Cache, q: torch.Tensor, q_lens, scale: float, causal=True):
    """(O, LSE, sum of p |v|), all float64, of ragged queries (tokens, h_q, d)."""
    h_q, at = q.shape[1], 0
    group = h_q // cache.h_k
    out, mag = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for s, (m, L) in enumerate(zip(q_lens, cache.lens)):
        k, v = cache.rows(s, 0, L, 0), cache.rows(s, 0, L, 1)
        last = torch.arange(L - m, L) if causal else torch.full((m,), L - 1)
        sees = torch.arange(L)[None] <= last[:, None]
        for h in range(h_q if m and L else 0):
            sc = (q[at:at + m, h].double() @ k[:, h // group].T * scale).masked_fill(~sees, -math.inf)
            z = sc.logsumexp(-1)
            p = torch.where(sees, (sc - z[:, None]).exp(), 0.0)
            out[at:at + m, h], mag[at:at + m, h], lse[at:at + m, h] = p @ v[:, h // group], p @ v[:, h // group].abs(), z
        at += m
    return out, lse, mag


def check_attention(got, out, mag, what=""):
    """P is rounded to a type of 11 bits or finer, so its error is at most
    2^-11 of sum p |v|; scores (exact operands, 32-bit sums) are given as much
    again. Then one rounding of the output."""
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    return (got - out).abs(), 2.0**-10 * mag + 1e-12


def assert_attention(got: torch.Tensor, out, mag, what=""):
    err, tol = check_attention(got, out, mag, what)
    tol = tol + UNIT[got.dtype] * (out.abs() + tol)
    if got.dtype == torch.float16:
        tol = tol + 2.0**-25
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: error {worst:.3g} times the bound (max abs {err.max().item():.3g})"
