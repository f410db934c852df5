"""Cases and plain forms of operators around a long-lived block-scaled KV cache.

What a serving step over the e4m3 cache with one power-of-two scale per (block
of tokens, KV head) needs once contexts are long, shared or hold images:

* ``axes``   -- RMS norm of Q and K per head with the rotation by positions of
  several axes (time, height, width), each angle following one of them;
* ``shared`` -- attention of sequences that share a long cached prefix, whose
  keys are read once for all of them;
* ``weigh``  -- the attention weight that each cached token received in a step,
  added up per KV head;
* ``evict``  -- the tokens of least weight dropped per KV head, the others moved
  together in the sequence's own pages.

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
        # one token of each of 32 sequences, text and images mixed (32 / 8 heads)
        dict(name="axes_step", op="axes", tokens=32, h_q=32, h_k=8, d=128, rot=128, sections="16,24,24", alternate=False,
             interleaved=False, dtype="bf16", shape_seed=1),
        # the prefill of a long prompt with images
        dict(name="axes_image", op="axes", tokens=8192, h_q=32, h_k=8, d=128, rot=128, sections="24,20,20", alternate=True,
             interleaved=False, dtype="bf16", shape_seed=2),
        # partial rotation of interleaved pairs at head size 256, an odd number of tokens
        dict(name="axes_partial", op="axes", tokens=1237, h_q=24, h_k=4, d=256, rot=64, sections="10,11,11", alternate=False,
             interleaved=True, dtype="fp16", shape_seed=3),
        # four requests behind a short common instruction
        dict(name="shared_step_few", op="shared", groups="4", shared="1024", q_len=1, own_tokens=200, h_q=32, h_k=8, d=128,
             page=16, block=16, dtype="bf16", shape_seed=4),
        # a batch of requests about one long document
        dict(name="shared_step", op="shared", groups="64", shared="16384", q_len=1, own_tokens=500, h_q=32, h_k=8, d=128,
             page=16, block=16, dtype="bf16", shape_seed=5),
        # three draft positions at head size 256, large pages, a prefix that ends inside a tile
        dict(name="shared_draft_256", op="shared", groups="16", shared="8064", q_len=3, own_tokens=900, h_q=24, h_k=4, d=256,
             page=128, block=64, dtype="fp16", shape_seed=6),
        # short prompt ends behind two cached prefixes, and requests that share nothing
        dict(name="shared_chunks", op="shared", groups="16,8,3", shared="6000,2064,0", q_len=24, own_tokens=300, h_q=32, h_k=8,
             d=128, page=16, block=16, dtype="bf16", shape_seed=7),
        # the weights of a decode step of 32 sequences
        dict(name="weigh_step", op="weigh", seqs=32, q_len=1, context=8192, window=0, h_q=32, h_k=8, d=128, page=16, block=16,
             dtype="bf16", shape_seed=8),
        # a long prompt's, from its first token
        dict(name="weigh_prompt", op="weigh", seqs=1, q_len=8192, context=0, window=0, h_q=32, h_k=8, d=128, page=16, block=16,
             dtype="bf16", shape_seed=9),
        # those of the last 32 queries of ragged prompts, head size 256
        dict(name="weigh_window", op="weigh", seqs=6, q_len=1500, context=3000, window=32, h_q=24, h_k=4, d=256, page=64,
             block=32, dtype="fp16", shape_seed=10),
        # a few sequences that outgrew their budget by a page or two
        dict(name="evict_step", op="evict", seqs=4, tokens=1100, budget=1024, recent=128, h_k=8, d=128, page=16, block=16,
             shape_seed=11),
        # a batch of prompts cut down after their prefill
        dict(name="evict_prompts", op="evict", seqs=16, tokens=8000, budget=2048, recent=256, h_k=8, d=128, page=16, block=16,
             shape_seed=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["axes", "shared", "shared", "weigh", "weigh", "evict"])
    d = rng.choice([128, 128, 256])
    h_k = rng.choice([1, 2, 4, 8])
    c = dict(op=op, d=d, h_k=h_k, shape_seed=rng.randrange(1 << 30))
    if op != "evict":
        c |= dict(dtype=rng.choice(["bf16", "bf16", "fp16"]), h_q=h_k * rng.choice([1, 2, 3, 4, 6]))
    if op == "axes":
        d = rng.choice([64, 128, 128, 256])
        rot = rng.choice([d, d, d // 2])
        a = rng.choice([2, 3, 3, 4])
        rest = rot // 2 - a * (rot // 2 // a)
        sections = [rot // 2 // a + (rest if i == 0 else 0) for i in range(a)]
        move = rng.randrange(sections[1])  # from every other axis to the first
        sections = [x + (a - 1) * move if i == 0 else x - move for i, x in enumerate(sections)]
        return c | dict(d=d, tokens=_log(rng, 1, 8192 * 128 // max(128, d)), rot=rot, sections=",".join(map(str, sections)),
                        alternate=rng.random() < 0.5, interleaved=rng.random() < 0.3)
    c["page"] = rng.choice([16, 32, 64, 128])
    c["block"] = rng.choice([b for b in (16, 32, 64, 128) if b <= c["page"]])
    if op == "evict":
        seqs = _log(rng, 1, 24)
        tokens = _log(rng, 8, max(16, min(30000, 128000 // seqs)))
        budget = max(1, int(tokens * rng.choice([0.1, 0.25, 0.5, 0.9, 1.0])))
        return c | dict(seqs=seqs, tokens=tokens, budget=budget, recent=min(budget, rng.choice([0, 1, 16, budget // 4, budget])))
    if op == "shared":
        sizes = [_log(rng, 1, 40) for _ in range(rng.choice([1, 1, 2, 3]))]
        many = rng.random() < 0.4
        q_len = _log(rng, 5, max(6, 600 // sum(sizes))) if many else rng.choice([1, 1, 2, 4])
        most = min(20000, 900_000 // sum(sizes), 2_000_000_000 // (sum(sizes) * q_len * c["h_q"]))
        shared = [0 if i and rng.random() < 0.3 else _log(rng, 1, max(2, most // c["page"])) * c["page"] for i in range(len(sizes))]
        return c | dict(groups=",".join(map(str, sizes)), shared=",".join(map(str, shared)), q_len=q_len,
                        own_tokens=_log(rng, 1, 800))
    if rng.random() < 0.5:  # decode and draft steps
        seqs = _log(rng, 1, 48)
        return c | dict(seqs=seqs, q_len=rng.choice([1, 1, 2, 4]), context=_log(rng, 16, max(16, min(30000, 250000 // seqs))), window=0)
    seqs = _log(rng, 1, 8)
    q_len = _log(rng, 5, 2500 // seqs)
    return c | dict(seqs=seqs, q_len=q_len, context=_log(rng, 1, max(1, min(8000, 200_000_000 // (seqs * q_len * c["h_q"])))),
                    window=rng.choice([0, 0, 16, 32, 100]))


def _spread(case, count, most, least, salt=0):
    """`count` ragged lengths of at most `most`, from the case alone."""
    rng = random.Random(case["shape_seed"] + salt)
    return [max(least, int(round(most * (1.0 if i == 0 else rng.uniform(0.4, 1.0))))) for i in range(count)]


def _ints(text):
    return [int(x) for x in text.split(",")]


def _lens(case):
    """(new tokens, cached tokens before them, shared tokens) of each sequence."""
    if case["op"] == "shared":
        groups, shared = _ints(case["groups"]), _ints(case["shared"])
        prefix = [p for n, p in zip(groups, shared) for _ in range(n)]
        ctx = [p + c for p, c in zip(prefix, _spread(case, len(prefix), case["own_tokens"], 0))]
    else:
        prefix = [0] * case["seqs"]
        ctx = _spread(case, case["seqs"], case["context"], 0)
    n = len(ctx)
    new = _spread(case, n, case["q_len"], 1, 1) if case["q_len"] > 4 else [case["q_len"]] * n
    return new, ctx, prefix


# ------------------------------------------------------------------- the work
def work(case):
    es, d, h_k = 2, case["d"], case["h_k"]
    if case["op"] == "axes":
        n = case["tokens"] * (case["h_q"] + h_k) * d
        axes = len(_ints(case["sections"]))
        return {"bytes": 2 * es * n + case["tokens"] * (case["rot"] * 4 + 8 * axes), "flops": 8 * n}
    g = case["block"]
    if case["op"] == "evict":
        lens = _spread(case, case["seqs"], case["tokens"], 1)
        kept = sum(case["budget"] for n in lens if n > case["budget"])
        read = sum(n for n in lens if n > case["budget"])
        return {"bytes": h_k * (4 * read + kept * (4 * d + 4 + 4 + 4 / g) + 4 * sum(min(n, case["budget"]) for n in lens)),
                "flops": 4 * h_k * kept * d}
    new, ctx, prefix = _lens(case)
    if case["op"] == "weigh":
        seen_by = [min(m, case["window"]) if case["window"] else m for m in new]
        keys = sum(m + c for m, c in zip(new, ctx))
        pairs = sum(w * (c + m) - w * (w - 1) // 2 for w, m, c in zip(seen_by, new, ctx))
        return {"bytes": keys * h_k * d + keys * h_k // g + 4 * h_k * (keys + sum(ctx)) + sum(seen_by) * case["h_q"] * (es * d + 4),
                "flops": 2 * d * case["h_q"] * pairs}
    groups, shared = _ints(case["groups"]), _ints(case["shared"])
    kv = sum(m + c - p for m, c, p in zip(new, ctx, prefix)) + sum(shared)
    seen = sum(m * c + m * (m + 1) // 2 for m, c in zip(new, ctx))
    return {"bytes": 2 * kv * h_k * d + 2 * kv * h_k // g + 2 * es * sum(new) * case["h_q"] * d,
            "flops": 4 * d * case["h_q"] * seen}


# ----------------------------------------------------------------- the inputs
def _dtype(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _ints_on(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _table(lens, page, g, prefix=None, groups=None, spare=4):
    """Shuffled pages for sequences of these lengths, a group's first pages the same ones: (block table, number of pages)."""
    n = [max(1, -(-x // page)) for x in lens]
    common = [0] * len(n) if prefix is None else [p // page for p in prefix]
    leader = list(range(len(n))) if groups is None else [sum(groups[:i]) for i, m in enumerate(groups) for _ in range(m)]
    pages = sum(n) + spare
    perm = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    cols = torch.arange(max(n), device="cuda")[None, :]
    at = _ints_on([sum(n[:i]) for i in range(len(n))], torch.int64)[:, None]
    first = torch.where(cols < _ints_on(common)[:, None], at[_ints_on(leader, torch.int64)], at)
    table = perm[(first + cols).clamp(max=pages - 1)]
    return torch.where(cols < _ints_on(n)[:, None], table, 0).contiguous(), pages


def _cache(pages, case, g):
    """A filled cache: codes as quantised normal rows leave them, scales that vary by block."""
    h_k, page, d, block = case["h_k"], case["page"], case["d"], case["block"]
    cache = torch.empty(pages, h_k, page, 2 * d, dtype=torch.uint8, device="cuda")
    code = _rand(g, pages, h_k, page, 2 * d).mul_(75.0).clamp_(-448, 448)
    cache.view(torch.float8_e4m3fn).copy_(code)
    del code
    scales = torch.randint(119, 123, (pages, h_k, 2, page // block), generator=g, device="cuda", dtype=torch.int32)
    return cache, scales.to(torch.uint8)


def _axes_of(case):
    """The axis of each angle: sections one after the other, or taking turns while they last."""
    sections = _ints(case["sections"])
    n, a = sum(sections), len(sections)
    if case["alternate"]:
        return [i % a if i < a * sections[i % a] else 0 for i in range(n)]
    return [i for i, m in enumerate(sections) for _ in range(m)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    s = {"case": case}
    if case["op"] == "axes":
        dt = _dtype(case)
        t, h_q, h_k, d, rot = case["tokens"], case["h_q"], case["h_k"], case["d"], case["rot"]
        # Q and K as views of the fused projection's rows, V between them and the next row
        qkv = _rand(g, t, (h_q + 2 * h_k) * d).mul_(1.5).to(dt)
        s["q"] = qkv[:, :h_q * d].view(t, h_q, d)
        s["k"] = qkv[:, h_q * d:(h_q + h_k) * d].view(t, h_k, d)
        s["q_weight"], s["k_weight"] = (1 + 0.2 * _rand(g, d)).to(dt), (1 + 0.2 * _rand(g, d)).to(dt)
        most = max(4096, t)
        inv = 1.0e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        # images of 24 columns: a row and a column beside the time
        start = torch.randint(0, most - 200, (t,), generator=g, device="cuda").sort().values
        i, axes = torch.arange(t, device="cuda"), _axes_of(case)
        s["positions"] = torch.stack([start] + [start + (i // 24 ** k) % 24 for k in range(max(axes))]).contiguous()
        s["axes"] = tuple(axes)
        s["axis_of"] = _ints_on(axes, torch.int64)
        s["q_out"], s["k_out"] = torch.empty(t, h_q, d, dtype=dt, device="cuda"), torch.empty(t, h_k, d, dtype=dt, device="cuda")
        return s
    page, h_k, d = case["page"], case["h_k"], case["d"]
    if case["op"] == "evict":
        lens = _spread(case, case["seqs"], case["tokens"], 1)
        s["table"], pages = _table(lens, page, g)
        s["cache"], s["scales"] = _cache(pages, case, g)
        s["seq_lens"], s["most"] = _ints_on(lens), max(lens)
        # a few tokens hold most of the weight; many of the others have the same, none at all
        w = _rand(g, len(lens), h_k, max(lens)).mul_(2.0).exp_()
        s["weights"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.2, 0.0, w)
        s["new_lens"] = torch.empty(len(lens), dtype=torch.int32, device="cuda")
        s["kept"] = torch.empty(len(lens), h_k, case["budget"], dtype=torch.int32, device="cuda")
        return s
    dt = _dtype(case)
    new, ctx, prefix = _lens(case)
    lens = [a + n for a, n in zip(ctx, new)]
    groups = _ints(case["groups"]) if case["op"] == "shared" else None
    s["table"], pages = _table(lens, page, g, prefix, groups)
    s["cache"], s["scales"] = _cache(pages, case, g)
    s["q"] = _rand(g, sum(new), case["h_q"], d).to(dt)
    s["scale"] = d ** -0.5
    s["seq_lens"], s["q_lens"] = _ints_on(lens), _ints_on(new, torch.int64)
    s["offsets"] = _ints_on([sum(new[:i]) for i in range(len(new) + 1)])
    s["q_most"], s["kv_most"] = max(new), max(lens)
    if case["op"] == "weigh":
        if case["window"]:
            s["q_most"] = min(s["q_most"], case["window"])
        # the log-sum-exp as the step's attention left it, and what earlier steps added up
        s["lse"] = torch.zeros(sum(new), case["h_q"], device="cuda")
        s["lse"] = _plain_scores(s, True)
        s["weights"] = _rand(g, len(lens), h_k, max(lens) + 8).abs_().mul_(10 / max(lens))
        return s
    s["out"] = torch.empty_like(s["q"])
    if own:
        from mjolnir_b200 import kvblock

        s["attention"] = kvblock.BlockAttention(
            num_heads=case["h_q"], num_kv_heads=h_k, head_size=d, page_size=page, block_tokens=case["block"],
            max_num_seqs=len(new), max_num_tokens=sum(new))
        parts = [(sum(groups[:i]), n, p) for i, (n, p) in enumerate(zip(groups, _ints(case["shared"]))) if p]
        s["plan"] = s["attention"].plan(new, lens, s["table"], s["seq_lens"], shared=parts)
    return s


# ------------------------------------------------------------ the plain forms
def _norm_rotate(x, w, cos, sin, rot, interleaved, eps=1e-6):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _gather(codes, exps, table, pos, page, block):
    """Values in 32 bits of the tokens at `pos` (n, m) of the sequences of `table` (n, ...): (n, m, h_k, d)."""
    pg = table.long().gather(1, pos // page)
    row = pos % page
    return codes[pg, :, row].float() * torch.exp2(exps[pg, :, row // block].float() - 127.0)[..., None]


def _rows_of(s):
    """The query rows of every sequence that count, padded to the longest: rows (n, q), whether they are there, the last key each sees."""
    n = s["q_lens"]
    few = torch.minimum(n, torch.full_like(n, s["q_most"]))  # the last ones, where a window leaves the others out
    i = torch.arange(s["q_most"], device="cuda")[None, :]
    there = i < few[:, None]
    back = few[:, None] - torch.minimum(i, few[:, None] - 1)  # rows before the sequence's end
    return s["offsets"][1:].long()[:, None] - back, there, s["seq_lens"][:, None].long() - back


def _scores(s):
    """Scores of every query row that counts with every key, -inf where it sees none: (n, h_k, group, q, keys), and the rows."""
    case = s["case"]
    h_k, h_q, d, page, block = case["h_k"], case["h_q"], case["d"], case["page"], case["block"]
    rows, there, last = _rows_of(s)
    kpos = torch.arange(s["kv_most"], device="cuda")
    inside = torch.minimum(kpos[None, :], s["seq_lens"][:, None].long() - 1)
    q = s["q"][rows].float().view(*rows.shape, h_k, h_q // h_k, d)
    k = _gather(s["cache"].view(torch.float8_e4m3fn)[..., :d], s["scales"][:, :, 0], s["table"], inside, page, block)
    score = torch.einsum("nqhrd,nkhd->nhrqk", q, k).mul_(s["scale"])
    sees = (kpos <= last[..., None]) & there[..., None]
    return score.masked_fill_(~sees[:, None, None], -math.inf), rows, there, inside


def _plain_attention(s):
    case = s["case"]
    d, page, block = case["d"], case["page"], case["block"]
    score, rows, there, inside = _scores(s)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    v = _gather(s["cache"].view(torch.float8_e4m3fn)[..., d:], s["scales"][:, :, 1], s["table"], inside, page, block)
    out = torch.einsum("nhrqk,nkhd->nqhrd", score, v).flatten(2, 3)
    return torch.zeros_like(s["q"]).index_copy(0, rows[there], out[there].to(s["q"].dtype))


def _plain_scores(s, lse):
    """The log-sum-exp of every row that counts (with `lse`), or the weights of the step added to the earlier ones."""
    score, rows, there, _ = _scores(s)
    if lse:
        top = score.amax(-1, keepdim=True)
        got = score.sub_(top).exp_().sum(-1).log_().add_(top[..., 0]).permute(0, 3, 1, 2).flatten(2)  # (n, q, h_q)
        return s["lse"].index_copy(0, rows[there], got[there])
    h_k = s["case"]["h_k"]
    z = s["lse"][rows].view(*rows.shape, h_k, -1).permute(0, 2, 3, 1)
    step = score.sub_(z[..., None]).exp_().sum((2, 3))  # (n, h_k, keys)
    kpos = torch.arange(s["kv_most"], device="cuda")
    before = s["weights"][..., :s["kv_most"]]
    opened = kpos >= (s["seq_lens"] - s["q_lens"])[:, None, None]
    inside = kpos < s["seq_lens"][:, None, None]
    before.copy_(torch.where(inside, step + torch.where(opened, 0.0, before), before))
    return s["weights"]


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^(e - 127), within what a writer produces."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x + 118 + (m > 0.875).int(), E_MIN).clamp(E_MIN, E_MAX)


def _plain_evict(s):
    case = s["case"]
    h_k, d, page, block, budget, recent = (case[x] for x in ("h_k", "d", "page", "block", "budget", "recent"))
    codes, exps, lens = s["cache"].view(torch.float8_e4m3fn), s["scales"], s["seq_lens"].long()[:, None, None]
    most = max(s["most"], budget)
    pos = torch.arange(most, device="cuda")
    weights = torch.nn.functional.pad(s["weights"], (0, most - s["most"]))
    cut = lens > budget
    # the recent ones rank first, then the others by weight, the lowest index first among equals
    rank = torch.where(pos >= lens, -math.inf, torch.where((pos >= lens - recent) | ~cut, math.inf, weights))
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget].sort(dim=-1).values
    i = torch.arange(budget, device="cuda")
    there = i < torch.minimum(lens, torch.full_like(lens, budget))  # (n, 1, budget)
    kept = torch.where(there, kept, -1)
    # the rows, at the largest scale that a block of them needs
    table, src = s["table"].long()[:, None], kept.clamp(min=0)
    pg, row, h = table.expand(-1, h_k, -1).gather(2, src // page), src % page, torch.arange(h_k, device="cuda")[None, :, None]
    x = codes[pg, h, row].float().unflatten(-1, (2, d)) * torch.exp2(exps[pg, h, :, row // block].float() - 127.0)[..., None]
    pad = -budget % block
    size = torch.where(there[..., None], x.abs().amax(-1), 0.0)
    size = torch.nn.functional.pad(size, (0, 0, 0, pad)).unflatten(2, (-1, block)).amax(3)  # (n, h_k, blocks, 2)
    e = _exponent(size)
    x = x * torch.exp2(127.0 - e.repeat_interleave(block, 2)[:, :, :budget].float())[..., None]
    moves = there & cut
    to_page, to_row = table.expand(-1, h_k, -1).gather(2, (i // page).expand_as(kept)), (i % page).expand_as(kept)
    to_head, moves = h.expand_as(kept), moves.expand_as(kept)
    codes[to_page[moves], to_head[moves], to_row[moves]] = x.clamp(-448, 448).to(torch.float8_e4m3fn).flatten(-2)[moves]
    first = moves[..., ::block]
    exps[to_page[..., ::block][first], to_head[..., ::block][first], :, to_row[..., ::block][first] // block] = e[first].to(torch.uint8)
    span = min(budget, s["most"])
    moved = torch.where(moves, weights.gather(2, src), weights[..., :budget])
    s["weights"][..., :span] = moved[..., :span]
    new_lens = torch.minimum(s["seq_lens"], torch.full_like(s["seq_lens"], budget))
    return codes, exps, s["weights"], new_lens, kept.to(torch.int32)


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

        if op == "axes":
            return qkrope.qk_norm_rope(s["q"], s["k"], s["positions"], s["cos_sin"], s["q_weight"], s["k_weight"], eps=1e-6,
                                       interleaved=case["interleaved"], axes=s["axes"], q_out=s["q_out"], k_out=s["k_out"])
        k, v, ks, vs = _views(s)
        if op == "weigh":
            return kvblock.weigh(s["q"], s["lse"], k, ks, s["table"], s["offsets"], s["seq_lens"], s["weights"], s["scale"],
                                 window=case["window"])
        if op == "evict":
            kvblock.evict(s["weights"], k, v, ks, vs, s["table"], s["seq_lens"], s["new_lens"], s["kept"], recent=case["recent"])
            return s["cache"].view(torch.float8_e4m3fn), s["scales"], s["weights"], s["new_lens"], s["kept"]
        return s["attention"].run(s["plan"], s["q"], s["out"], k, v, ks, vs, s["scale"])
    if op == "axes":
        rot = case["rot"]
        at = s["positions"][s["axis_of"]].t()  # (tokens, rot / 2)
        cos, sin = s["cos_sin"][:, :rot // 2].gather(0, at)[:, None], s["cos_sin"][:, rot // 2:].gather(0, at)[:, None]
        return tuple(_norm_rotate(x, w, cos, sin, rot, case["interleaved"])
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    if op == "weigh":
        return _plain_scores(s, False)
    return _plain_evict(s) if op == "evict" else _plain_attention(s)


# ------------------------------------------- the same from the definition, in 64 bits
def _exact_axes(x, w, pos, table, axes, rot, interleaved):
    y = x.double()
    y = y / ((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * w.double()
    out = y.clone()
    for i, axis in enumerate(axes):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, t = table[pos[axis], i].double()[:, None], table[pos[axis], rot // 2 + i].double()[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * t
        out[..., b] = y[..., a] * t + y[..., b] * c
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


def _exact_evict(s):
    case = s["case"]
    h_k, d, page, block, budget, recent = (case[x] for x in ("h_k", "d", "page", "block", "budget", "recent"))
    values, lens = _e4m3_values(), s["seq_lens"].tolist()
    codes, exps, weights = s["cache"].view(torch.float8_e4m3fn).double(), s["scales"].clone(), s["weights"].double()
    kept = torch.full((len(lens), h_k, budget), -1, dtype=torch.int32, device="cuda")
    for i, n in enumerate(lens):
        if n <= budget:
            kept[i, :, :n] = torch.arange(n, dtype=torch.int32, device="cuda")
            continue
        pages = s["table"][i].long()
        for h in range(h_k):
            old = weights[i, h, :n - recent].cpu()
            order = sorted(range(n - recent), key=lambda t: -old[t].item())[:budget - recent]  # (a stable sort)
            order = sorted(order) + list(range(n - recent, n))
            at = torch.tensor(order, device="cuda")
            kept[i, h] = at.int()
            weights[i, h, :budget] = weights[i, h, at]
            e = exps[pages[at // page], h, :, at % page // block].double() - 127
            x = codes[pages[at // page], h, at % page].view(budget, 2, d) * torch.exp2(e)[..., None]
            for b in range(0, budget, block):
                part = x[b:b + block]
                big = part.abs().amax((0, 2))
                need = torch.ceil(torch.log2(big.clamp(min=1e-300) / 448)).clamp(-32, 32)
                need = torch.where(big > 448 * torch.exp2(need), need + 1, need)
                need = torch.where(big <= 448 * torch.exp2(need - 1), need - 1, need).clamp(-32, 32)
                rows = slice(b % page, b % page + len(part))
                codes[pages[b // page], h, rows] = _to_e4m3(part * torch.exp2(-need)[None, :, None], values).flatten(1)
                exps[pages[b // page], h, :, b % page // block] = (need + 127).to(torch.uint8)
    return codes, exps, weights, s["seq_lens"].clamp(max=budget), kept


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "axes":
        return tuple(_exact_axes(x, w, s["positions"], s["cos_sin"], _axes_of(case), case["rot"], case["interleaved"])
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    d, page, block = case["d"], case["page"], case["block"]
    if case["op"] == "evict":
        blocks = sum(case["budget"] // block + 1 for n in s["seq_lens"].tolist() if n > case["budget"]) * case["h_k"]
        return _exact_evict(s) if blocks <= 20000 else None
    codes, scale = s["cache"].view(torch.float8_e4m3fn), torch.exp2(s["scales"].double() - 127)

    def rows(i, length, side):
        pos = torch.arange(length, device="cuda")
        pg, row = s["table"][i][pos // page].long(), pos % page
        return codes[..., side * d:side * d + d][pg, :, row].double() * scale[:, :, side][pg, :, row // block][..., None]

    weigh, group = case["op"] == "weigh", case["h_q"] // case["h_k"]
    out = s["weights"].double() if weigh else torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begin = s["offsets"].tolist()
    for i, (m, length) in enumerate(zip(s["q_lens"].tolist(), s["seq_lens"].tolist())):
        k = rows(i, length, 0)
        count = min(m, case["window"]) if weigh and case["window"] else m
        at = begin[i + 1] - count
        sees = torch.arange(length, device="cuda")[None, :] <= torch.arange(length - count, length, device="cuda")[:, None]
        if weigh:
            out[i, :, length - m:length] = 0
        else:
            v = rows(i, length, 1)
        for h in range(case["h_q"]):
            score = s["q"][at:at + count, h].double() @ k[:, h // group].T * s["scale"]
            if weigh:
                score -= s["lse"][at:at + count, h].double()[:, None]
                out[i, h // group, :length] += torch.where(sees, score.exp(), 0.0).sum(0)
                continue
            weight = torch.where(sees, (score - score.where(sees, -math.inf).amax(-1, keepdim=True)).exp(), 0.0)
            out[at:at + count, h] = weight @ v[:, h // group] / weight.sum(-1, keepdim=True)
    return out
