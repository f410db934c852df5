"""Cases and plain forms of the block-scaled KV-cache operators.

A layer's serving step over a KV cache held in e4m3 with one power-of-two scale
per (block of tokens, KV head):

* ``rope``  -- RMS norm of Q and K per head with the position rotation;
* ``write`` -- quantising new K / V rows into the paged cache;
* ``read``  -- gathering cached tokens back as contiguous rows;
* ``attn``  -- causal attention over the cache, for single tokens, drafts and
  chunks of ragged lengths.

A cache is (pages, h_k, page_size, K row | V row) bytes; its scales are
(pages, h_k, 2, page_size / block) exponent bytes e of the scale 2^(e - 127).
"""

import math
import random

import torch

own = False

E_MIN, E_MAX = 95, 159  # scale exponent bytes a writer produces: 2^-32 .. 2^32


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # Q/K norm and rotation of a decode step of 32 sequences (32 / 8 heads)
        dict(name="rope_step", op="rope", tokens=32, h_q=32, h_k=8, d=128, rot=128, interleaved=False, norm=True,
             dtype="bf16", shape_seed=1),
        # the same of a long prompt's prefill
        dict(name="rope_chunk", op="rope", tokens=8192, h_q=32, h_k=8, d=128, rot=128, interleaved=False, norm=True,
             dtype="bf16", shape_seed=2),
        # partial rotation of interleaved pairs at head size 256, an odd number of tokens
        dict(name="rope_partial", op="rope", tokens=1237, h_q=24, h_k=4, d=256, rot=64, interleaved=True, norm=True,
             dtype="fp16", shape_seed=3),
        # one new token for each of 128 running sequences, mostly into half-filled blocks
        dict(name="write_step", op="write", seqs=128, new=1, context=2000, h_k=8, d=128, page=16, block=16,
             dtype="bf16", shape_seed=4),
        # ragged prompt chunks of 8 sequences that continue half-filled blocks
        dict(name="write_chunk", op="write", seqs=8, new=1900, context=700, h_k=8, d=128, page=64, block=32,
             dtype="bf16", shape_seed=5),
        # a few short cached prefixes back as rows
        dict(name="read_prefix", op="read", seqs=3, tokens=2000, h_k=4, d=256, page=32, block=32, dtype="fp16",
             shape_seed=6),
        # a long cached context back as rows for a step that computes on them
        dict(name="read_long", op="read", seqs=6, tokens=16000, h_k=8, d=128, page=16, block=16, dtype="bf16",
             shape_seed=7),
        # a small decode step over short contexts
        dict(name="attn_step_short", op="attn", seqs=4, q_len=1, context=1000, h_q=32, h_k=8, d=128, page=16,
             block=16, dtype="bf16", shape_seed=8),
        # a large decode step over long ragged contexts
        dict(name="attn_step_long", op="attn", seqs=48, q_len=1, context=16384, h_q=32, h_k=8, d=128, page=16,
             block=16, dtype="bf16", shape_seed=9),
        # three draft positions at head size 256, large pages
        dict(name="attn_draft_256", op="attn", seqs=16, q_len=3, context=8000, h_q=24, h_k=4, d=256, page=128,
             block=64, dtype="fp16", shape_seed=10),
        # one long prompt from its first token
        dict(name="attn_prefill", op="attn", seqs=1, q_len=8192, context=0, h_q=32, h_k=8, d=128, page=16, block=16,
             dtype="bf16", shape_seed=11),
        # ragged prompt chunks of 5 sequences behind cached contexts
        dict(name="attn_chunks", op="attn", seqs=5, q_len=1500, context=6000, h_q=32, h_k=8, d=128, page=64,
             block=64, dtype="bf16", shape_seed=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attn", "attn"])
    d = rng.choice([128, 128, 256])
    h_k = rng.choice([1, 2, 4, 8])
    c = dict(op=op, d=d, h_k=h_k, dtype=rng.choice(["bf16", "bf16", "fp16"]), shape_seed=rng.randrange(1 << 30))
    if op == "rope":
        d = rng.choice([64, 128, 128, 256])
        return c | dict(d=d, tokens=_log(rng, 1, 8192 * 128 // max(128, d)), h_q=h_k * rng.choice([1, 3, 4]),
                        rot=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.8)
    c["page"] = rng.choice([16, 32, 64, 128])
    c["block"] = rng.choice([b for b in (16, 32, 64, 128) if b <= c["page"]])
    if op == "write":
        seqs = _log(rng, 1, 128)
        return c | dict(seqs=seqs, new=_log(rng, 1, max(1, 8192 // seqs)), context=_log(rng, 1, 2000))
    if op == "read":
        seqs = _log(rng, 1, 32)
        return c | dict(seqs=seqs, tokens=_log(rng, 1, max(1, 48000 // seqs)))
    c["h_q"] = h_k * rng.choice([1, 2, 4, 6])
    if rng.random() < 0.5:  # decode: a few positions of many sequences
        seqs = _log(rng, 1, 48)
        c |= dict(seqs=seqs, q_len=rng.choice([1, 1, 2, 4]), context=_log(rng, 16, max(16, min(30000, 300000 // seqs))))
    else:  # chunks: scores of seqs x q_len x (q_len + context) x h_q stay below the prefill case's
        seqs = _log(rng, 1, 8)
        q_len = _log(rng, 5, 2500 // seqs)
        c |= dict(seqs=seqs, q_len=q_len, context=_log(rng, 1, max(1, min(8000, 300_000_000 // (seqs * q_len * c["h_q"])))))
    return c


def _spread(case, most, least):
    """`seqs` ragged lengths of at most `most`, from the case alone."""
    rng = random.Random(case["shape_seed"])
    return [max(least, int(round(most * (1.0 if i == 0 else rng.uniform(0.4, 1.0))))) for i in range(case["seqs"])]


def _lens(case):
    """(new tokens, cached tokens before them) of each sequence."""
    ctx = _spread(case, case["context"], 0)
    new = case["new"] if case["op"] == "write" else case["q_len"]
    return (_spread(case, new, 1) if new > 4 else [new] * case["seqs"]), ctx


# ------------------------------------------------------------------- the work
def work(case):
    es, d, h_k = 2, case["d"], case["h_k"]
    if case["op"] == "rope":
        n = case["tokens"] * (case["h_q"] + h_k) * d
        return {"bytes": 2 * es * n + case["tokens"] * (case["rot"] * 4 + 8), "flops": 8 * n}
    g = case["block"]
    if case["op"] == "write":
        new, ctx = _lens(case)
        n = sum(new)
        blocks = sum((c + m - 1) // g - c // g + 1 for m, c in zip(new, ctx))
        return {"bytes": 2 * n * h_k * d * (es + 1) + 2 * blocks * h_k + 8 * n, "flops": 4 * n * h_k * d}
    if case["op"] == "read":
        n = sum(_spread(case, case["tokens"], 1))
        return {"bytes": 2 * n * h_k * d * (es + 1) + 2 * n * h_k // g, "flops": 2 * n * h_k * d}
    new, ctx = _lens(case)
    kv = sum(m + c for m, c in zip(new, ctx))
    seen = sum(m * c + m * (m + 1) // 2 for m, c in zip(new, ctx))
    return {"bytes": 2 * kv * h_k * d + 2 * kv * h_k // g + 2 * es * sum(new) * case["h_q"] * d,
            "flops": 4 * d * case["h_q"] * seen}


# ----------------------------------------------------------------- the inputs
def _dtype(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _table(lens, page, g, spare=4):
    """Shuffled pages for sequences of these lengths: (block table, number of pages)."""
    n = [max(1, -(-x // page)) for x in lens]
    pages = sum(n) + spare
    perm = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    cols = torch.arange(max(n), device="cuda")
    first = torch.tensor([sum(n[:i]) for i in range(len(n))], device="cuda")
    index = (first[:, None] + cols[None, :]).clamp(max=pages - 1)
    return torch.where(cols[None, :] < torch.tensor(n, device="cuda")[:, None], perm[index], 0).contiguous(), pages


def _cache(pages, case, g):
    """A filled cache: codes as quantised normal rows leave them, scales that vary by block."""
    h_k, page, d, block = case["h_k"], case["page"], case["d"], case["block"]
    cache = torch.empty(pages, h_k, page, 2 * d, dtype=torch.uint8, device="cuda")
    code = _rand(g, pages, h_k, page, 2 * d).mul_(75.0).clamp_(-448, 448)
    cache.view(torch.float8_e4m3fn).copy_(code)
    del code
    scales = torch.randint(119, 123, (pages, h_k, 2, page // block), generator=g, device="cuda", dtype=torch.int32)
    return cache, scales.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    s = {"case": case}
    dt = _dtype(case)
    if case["op"] == "rope":
        t, h_q, h_k, d, rot = case["tokens"], case["h_q"], case["h_k"], case["d"], case["rot"]
        # Q and K as views of the fused projection's rows, V between them and the next row
        qkv = _rand(g, t, (h_q + 2 * h_k) * d).mul_(1.5).to(dt)
        s["q"] = qkv[:, :h_q * d].view(t, h_q, d)
        s["k"] = qkv[:, h_q * d:(h_q + h_k) * d].view(t, h_k, d)
        s["q_weight"] = (1 + 0.2 * _rand(g, d)).to(dt) if case["norm"] else None
        s["k_weight"] = (1 + 0.2 * _rand(g, d)).to(dt) if case["norm"] else None
        most = max(4096, t)
        inv = 1.0e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        s["positions"] = torch.randint(0, most, (t,), generator=g, device="cuda")
        s["q_out"], s["k_out"] = torch.empty(t, h_q, d, dtype=dt, device="cuda"), torch.empty(t, h_k, d, dtype=dt, device="cuda")
        return s
    page, h_k, d = case["page"], case["h_k"], case["d"]
    if case["op"] == "read":
        lens = _spread(case, case["tokens"], 1)
        starts = [(i * 5) % (page + 3) for i in range(len(lens))]
        s["table"], pages = _table([a + n for a, n in zip(starts, lens)], page, g)
        s["cache"], s["scales"] = _cache(pages, case, g)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["offsets"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        s["k_out"] = torch.empty(sum(lens), h_k, d, dtype=dt, device="cuda")
        s["v_out"] = torch.empty(sum(lens), h_k, d, dtype=dt, device="cuda")
        return s
    new, ctx = _lens(case)
    s["table"], pages = _table([a + n for a, n in zip(ctx, new)], page, g)
    s["cache"], s["scales"] = _cache(pages, case, g)
    if case["op"] == "write":
        # the slot of every new token; K with a few large channels, V without
        seq = torch.tensor([i for i, n in enumerate(new) for _ in range(n)], device="cuda")
        pos = torch.tensor([c + j for n, c in zip(new, ctx) for j in range(n)], device="cuda")
        s["slots"] = s["table"][seq, pos // page].long() * page + pos % page
        spread = 1 + 6 * (torch.rand(h_k, d, generator=g, device="cuda") < 0.03)
        s["key"] = (_rand(g, len(pos), h_k, d) * spread).to(dt)
        s["value"] = _rand(g, len(pos), h_k, d).mul_(0.7).to(dt)
        return s
    s["q"] = _rand(g, sum(new), case["h_q"], d).to(dt)
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = d ** -0.5
    s["seq_lens"] = torch.tensor([a + n for a, n in zip(ctx, new)], dtype=torch.int32, device="cuda")
    s["q_lens"] = torch.tensor(new, device="cuda")
    s["q_most"], s["kv_most"] = max(new), max(a + n for a, n in zip(ctx, new))
    if own:
        from mjolnir_b200 import kvblock

        s["attention"] = kvblock.BlockAttention(
            num_heads=case["h_q"], num_kv_heads=h_k, head_size=d, page_size=page, block_tokens=case["block"],
            max_num_seqs=len(new), max_num_tokens=sum(new))
        s["plan"] = s["attention"].plan(new, [a + n for a, n in zip(ctx, new)], s["table"], s["seq_lens"])
    return s


# ------------------------------------------------------------ the plain forms
def _norm_rotate(x, w, cos_sin, rot, interleaved, eps=1e-6):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.float()
    cos, sin = cos_sin[:, None, :rot // 2], cos_sin[:, None, rot // 2:]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^(e - 127), within what a writer produces."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x + 118 + (m > 0.875).int(), E_MIN).clamp(E_MIN, E_MAX)


def _plain_write_side(x, codes, exps, slots, page, block):
    """codes (pages, h_k, page, d) e4m3 and exps (pages, h_k, page / block) uint8 views, written in place."""
    h_k, d = x.shape[1:]
    per = page // block
    x = x.float()
    size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)  # (tokens, h_k)
    at, which = torch.unique(slots // block, return_inverse=True)
    amax = torch.zeros(len(at), h_k, device=x.device).index_reduce(0, which, size, "amax")
    opened = torch.zeros(len(at), device=x.device).index_reduce(0, which, (slots % block == 0).float(), "amax") > 0
    pg, sub = at // per, at % per
    old = exps[pg, :, sub].int()  # (blocks, h_k)
    new = _exponent(amax)
    new = torch.where(opened[:, None], new, torch.maximum(old, new))
    # the rows of an open block that stay follow a scale that grew
    rows = sub[:, None] * block + torch.arange(block, device=x.device)
    here = codes[pg[:, None], :, rows]  # (blocks, block, h_k, d)
    shift = torch.where(opened[:, None], 0, old - new).float()
    moved = (here.float() * torch.exp2(shift)[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    codes[pg[:, None], :, rows] = moved
    exps[pg, :, sub] = new.to(torch.uint8)
    code = (x * torch.exp2(127.0 - new[which].float())[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    codes[slots // page, :, slots % page] = code


def _gather(codes, exps, table, pos, page, block):
    """Values in 32 bits of the tokens at `pos` (n, m) of the sequences of `table` (n, ...): (n, m, h_k, d)."""
    pg = table.long().gather(1, pos // page)
    row = pos % page
    return codes[pg, :, row].float() * torch.exp2(exps[pg, :, row // block].float() - 127.0)[..., None]


def _plain_attention(s, codes, exps, page, block):
    case = s["case"]
    h_k, h_q, d = case["h_k"], case["h_q"], case["d"]
    n, q_most, kv_most = len(s["q_lens"]), s["q_most"], s["kv_most"]
    kpos = torch.arange(kv_most, device="cuda")
    inside = torch.minimum(kpos[None, :], s["seq_lens"][:, None].long() - 1)
    first = torch.cumsum(s["q_lens"], 0) - s["q_lens"]
    qpos = torch.arange(q_most, device="cuda")
    qrow = first[:, None] + torch.minimum(qpos[None, :], s["q_lens"][:, None] - 1)
    q = s["q"][qrow].float().view(n, q_most, h_k, h_q // h_k, d)
    k = _gather(codes[..., :d], exps[:, :, 0], s["table"], inside, page, block)
    score = torch.einsum("nqhrd,nkhd->nhrqk", q, k).mul_(s["scale"])
    del k
    last = s["seq_lens"][:, None].long() - s["q_lens"][:, None] + qpos  # the last key each query sees
    score.masked_fill_(kpos > last[:, None, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    v = _gather(codes[..., d:], exps[:, :, 1], s["table"], inside, page, block)
    out = torch.einsum("nhrqk,nkhd->nqhrd", score, v).reshape(n * q_most, h_q, d)
    there = (qpos[None, :] < s["q_lens"][:, None]).flatten()
    return torch.zeros_like(s["q"]).index_copy(0, qrow.flatten()[there], out[there].to(s["q"].dtype))


def _views(s):
    """(k codes, v codes, k scales, v scales) as the framework's entry points take them: (pages, page_size, h_k, ...)."""
    d = s["case"]["d"]
    cache, scales = s["cache"], s["scales"]
    return (cache[..., :d].transpose(1, 2), cache[..., d:].transpose(1, 2),
            scales[:, :, 0].transpose(1, 2), scales[:, :, 1].transpose(1, 2))


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from mjolnir_b200 import kvblock, qkrope

        if op == "rope":
            return qkrope.qk_norm_rope(s["q"], s["k"], s["positions"], s["cos_sin"], s["q_weight"], s["k_weight"],
                                       eps=1e-6, interleaved=case["interleaved"], q_out=s["q_out"], k_out=s["k_out"])
        k, v, ks, vs = _views(s)
        if op == "write":
            kvblock.write(s["key"], s["value"], k, v, ks, vs, s["slots"])
            return s["cache"].view(torch.float8_e4m3fn), s["scales"]
        if op == "read":
            return kvblock.read(k, v, ks, vs, s["table"], s["starts"], s["offsets"], s["k_out"], s["v_out"])
        return s["attention"].run(s["plan"], s["q"], s["out"], k, v, ks, vs, s["scale"])
    if op == "rope":
        cs = s["cos_sin"][s["positions"]]
        return tuple(_norm_rotate(x, w, cs, case["rot"], case["interleaved"])
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    d, page, block = case["d"], case["page"], case["block"]
    codes, exps = s["cache"].view(torch.float8_e4m3fn), s["scales"]
    if op == "write":
        _plain_write_side(s["key"], codes[..., :d], exps[:, :, 0], s["slots"], page, block)
        _plain_write_side(s["value"], codes[..., d:], exps[:, :, 1], s["slots"], page, block)
        return codes, exps
    if op == "read":
        total = s["k_out"].shape[0]
        row = torch.arange(total, device="cuda")
        seq = torch.searchsorted(s["offsets"], row, right=True) - 1
        pos = (row - s["offsets"][seq] + s["starts"][seq])[:, None]
        table = s["table"][seq]
        return (_gather(codes[..., :d], exps[:, :, 0], table, pos, page, block)[:, 0].to(s["k_out"].dtype),
                _gather(codes[..., d:], exps[:, :, 1], table, pos, page, block)[:, 0].to(s["v_out"].dtype))
    return _plain_attention(s, codes, exps, page, block)


# ------------------------------------------- the same from the definition, in 64 bits
def _exact_rope(x, w, pos, table, rot, interleaved):
    y = x.double()
    if w is not None:
        y = y / ((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * w.double()
    out = y.clone()
    turn = torch.complex(table[pos, :rot // 2].double(), table[pos, rot // 2:].double())[:, None]
    first = torch.arange(0, rot, 2, device="cuda") if interleaved else torch.arange(rot // 2, device="cuda")
    second = first + (1 if interleaved else rot // 2)
    z = torch.complex(y[..., first], y[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _e4m3_values():
    """The 127 non-negative values of e4m3, from its definition."""
    low = [m * 2.0 ** -9 for m in range(8)]
    return torch.tensor(low + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:119],
                        dtype=torch.float64, device="cuda")


def _to_e4m3(x, values):
    """Nearest e4m3 value, ties to the even code, saturating."""
    a = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(values, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    down, up = a - values[lo], values[hi] - a
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return values[code] * torch.where(x < 0, -1.0, 1.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return tuple(_exact_rope(x, w, s["positions"], s["cos_sin"], case["rot"], case["interleaved"])
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    d, page, block = case["d"], case["page"], case["block"]
    if case["op"] == "write":
        if len(s["slots"]) // block + case["seqs"] > 2000:
            return None
        codes, exps = s["cache"].view(torch.float8_e4m3fn).double(), s["scales"].double() - 127
        values = _e4m3_values()

        def write_side(x, codes, exps, slots, page, block, values):
            """In place on 64-bit values of the codes and integer exponents; block by block of the call."""
            groups = {}
            for t, slot in enumerate(slots.tolist()):
                groups.setdefault(slot // block, []).append((t, slot))
            for at, members in groups.items():
                page_at, sub = at // (page // block), at % (page // block)
                rows = [slot % page for _, slot in members]
                part = x[[t for t, _ in members]].double()  # (m, h_k, d)
                big = part.abs().amax((0, 2))
                need = torch.ceil(torch.log2(big.clamp(min=1e-300) / 448)).clamp(-32, 32)
                need = torch.where(big > 448 * torch.exp2(need), need + 1, need)
                need = torch.where(big <= 448 * torch.exp2(need - 1), need - 1, need).clamp(-32, 32)
                before = exps[page_at, :, sub]
                after = need if sub * block in rows else torch.maximum(before, need)
                if sub * block not in rows:
                    span = slice(sub * block, sub * block + block)
                    codes[page_at, :, span] = _to_e4m3(codes[page_at, :, span] * torch.exp2(before - after)[:, None, None], values)
                exps[page_at, :, sub] = after
                codes[page_at][:, rows] = _to_e4m3(part * torch.exp2(-after)[None, :, None], values).transpose(0, 1)

        write_side(s["key"], codes[..., :d], exps[:, :, 0], s["slots"], page, block, values)
        write_side(s["value"], codes[..., d:], exps[:, :, 1], s["slots"], page, block, values)
        return codes, (exps + 127).to(torch.uint8)
    codes, scale = s["cache"].view(torch.float8_e4m3fn), torch.exp2(s["scales"].double() - 127)

    def rows(table, begin, end):
        pos = torch.arange(begin, end, device="cuda")
        pg, row = table[pos // page].long(), pos % page
        both = [codes[..., i * d:i * d + d][pg, :, row].double() * scale[:, :, i][pg, :, row // block][..., None] for i in (0, 1)]
        return both  # each (end - begin, h_k, d)

    if case["op"] == "read":
        off, begin = s["offsets"].tolist(), s["starts"].tolist()
        got = [rows(s["table"][i], begin[i], begin[i] + off[i + 1] - off[i]) for i in range(len(begin))]
        return tuple(torch.cat([x[i] for x in got]) for i in (0, 1))
    out, at, group = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, case["h_q"] // case["h_k"]
    for i, (m, length) in enumerate(zip(s["q_lens"].tolist(), s["seq_lens"].tolist())):
        k, v = rows(s["table"][i], 0, length)
        sees = torch.arange(length, device="cuda")[None, :] <= torch.arange(length - m, length, device="cuda")[:, None]
        for h in range(case["h_q"]):
            score = s["q"][at:at + m, h].double() @ k[:, h // group].T * s["scale"]
            weight = torch.where(sees, (score - score.where(sees, -math.inf).amax(-1, keepdim=True)).exp(), 0.0)
            out[at:at + m, h] = weight @ v[:, h // group] / weight.sum(-1, keepdim=True)
        at += m
    return out
