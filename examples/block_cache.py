"""One attention layer over the block-scaled KV cache: two prompts in ragged
chunks, then single tokens, through Q/K norm and rotation, the quantising
write, and attention; at the end the cache is read back.

    python examples/block_cache.py

Prints how far the outputs are from attention over the unquantised K and V
(e4m3 keeps four significant bits).
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mjolnir_b200 import kvblock, qkrope  # noqa: E402

H_Q, H_K, D, PAGE, BLOCK = 32, 8, 128, 16, 16


def main() -> None:
    g = torch.Generator("cuda").manual_seed(0)
    prompts, decodes = [700, 1234], 4
    most = max(prompts) + decodes
    blocks = -(-most // PAGE)
    cache, scales = kvblock.alloc(2 * blocks, PAGE, H_K, D, BLOCK)
    views = kvblock.views(cache, scales)
    table = torch.randperm(2 * blocks, generator=g, device="cuda").int().view(2, blocks)
    attention = kvblock.BlockAttention(num_heads=H_Q, num_kv_heads=H_K, head_size=D, page_size=PAGE, block_tokens=BLOCK,
                                       max_num_seqs=2, max_num_tokens=1024)
    weights = [1 + 0.1 * torch.randn(D, generator=g, device="cuda").bfloat16() for _ in range(2)]
    inv = 1.0e6 ** (-torch.arange(0, D, 2, device="cuda") / D)
    angle = torch.arange(most, device="cuda")[:, None] * inv
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
    full = [[torch.empty(0, H_K, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)] for _ in range(2)]  # unquantised K, V
    done, worst = [0, 0], 0.0

    def step(new: list[int]) -> float:
        """A step of `new` tokens of each sequence; returns its error."""
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(new)).cuda()
        pos = torch.cat([torch.arange(d, d + n) for d, n in zip(done, new)]).cuda()
        slots = table[seq, pos // PAGE].long() * PAGE + pos % PAGE
        qkv = torch.randn(len(pos), (H_Q + 2 * H_K) * D, generator=g, device="cuda").bfloat16()
        q, k, v = (x.view(len(pos), -1, D) for x in qkv.split([H_Q * D, H_K * D, H_K * D], 1))
        q, k = qkrope.qk_norm_rope(q, k, pos, cos_sin, *weights)
        kvblock.write(k, v, *views, slots)
        lens = [d + n for d, n in zip(done, new)]
        plan = attention.plan(new, lens, table, torch.tensor(lens, dtype=torch.int32).cuda())
        out = attention.run(plan, q, torch.empty_like(q), *views, D**-0.5)
        err, at = 0.0, 0
        for s, n in enumerate(new):
            full[s] = [torch.cat([full[s][i], x[at:at + n]]) for i, x in enumerate((k, v))]
            kf, vf = (x.float().repeat_interleave(H_Q // H_K, 1).transpose(0, 1) for x in full[s])
            score = q[at:at + n].float().transpose(0, 1) @ kf.transpose(1, 2) * D**-0.5
            score.masked_fill_(torch.arange(lens[s], device="cuda") > torch.arange(done[s], lens[s], device="cuda")[:, None], -1e30)
            want = (score.softmax(-1) @ vf).transpose(0, 1)
            err = max(err, ((out[at:at + n].float() - want).norm() / want.norm()).item())
            at += n
            done[s] = lens[s]
        return err

    while any(d < p for d, p in zip(done, prompts)):
        worst = max(worst, step([min(512, p - d) for d, p in zip(done, prompts)]))
    for _ in range(decodes):
        worst = max(worst, step([1, 1]))
    attention.check_status()
    offsets = torch.tensor([0, done[0], sum(done)], dtype=torch.int32, device="cuda")
    k, v = (torch.empty(sum(done), H_K, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kvblock.read(*views, table, torch.zeros(2, dtype=torch.int32, device="cuda"), offsets, k, v)
    back = [((x.float() - torch.cat([full[0][i], full[1][i]]).float()).norm() / x.float().norm()).item() for i, x in enumerate((k, v))]
    print(f"{sum(done)} tokens of 2 sequences: attention off by at most {worst:.4f} (relative), K {back[0]:.4f}, V {back[1]:.4f} read back")
    # e4m3 rounds each value by at most 2^-4 of it, by 2^-4 / sqrt(3) at random
    if worst > 0.0625 or max(back) > 0.0625:
        raise SystemExit("further off than e4m3's rounding")


if __name__ == "__main__":
    main()
