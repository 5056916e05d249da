"""Several samples of one prompt over shared pages: prompt -> fork -> decode
steps -> some samples end -> compaction -> more steps.

A toy transformer with random weights (no checkpoint): per layer one q / k / v
projection, then ``TorchBlockAllocator.layer_step_shared`` -- the new tokens' q
and k normalised and rotated, k and v appended to the pages, the attention with
the prompt's pages read once for all samples -- and an output projection.  With
``check`` every attention output is compared with the plain decode
(``ops.paged_attention_v3``), which reads every sample's whole context.

    python examples/parallel_sampling.py [--samples 8] [--prompt 1000] [--steps 32]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "gb10-attn_b200"))
from pa_b200 import ops  # noqa: E402
from pa_b200.kv import KVConfig, ModelConfig, TorchBlockAllocator  # noqa: E402


class Toy:
    def __init__(self, cfg: ModelConfig, vocab: int, max_len: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        h, hk, d = cfg.n_head, cfg.kv_heads, cfg.head_dim
        width = h * d

        def w(*shape):
            x = torch.randn(shape, device="cuda", generator=g) * shape[0] ** -0.5
            return x.bfloat16()

        self.cfg, self.embed = cfg, w(vocab, width) * vocab ** 0.5
        self.qkv = [w(width, (h + 2 * hk) * d) for _ in range(cfg.n_layer)]
        self.out = [w(width, width) for _ in range(cfg.n_layer)]
        self.q_norm = [(1 + 0.1 * torch.randn(d, device="cuda", generator=g)).bfloat16()
                       for _ in range(cfg.n_layer)]
        self.k_norm = [(1 + 0.1 * torch.randn(d, device="cuda", generator=g)).bfloat16()
                       for _ in range(cfg.n_layer)]
        self.cos_sin = ops.rope_table(max_len, d)

    def project(self, layer, x):
        c = self.cfg
        y = (x @ self.qkv[layer]).view(x.shape[0], c.n_head + 2 * c.kv_heads, c.head_dim)
        return y.split((c.n_head, c.kv_heads, c.kv_heads), 1)


def prefill(toy, alloc, prompt, tokens):
    """The prompt's keys and values into its pages; the last hidden state."""
    n = len(tokens)
    none = torch.empty(0, device="cuda")
    table = alloc.block_table([prompt])
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    ctx = torch.tensor([n], dtype=torch.int32, device="cuda")
    x = toy.embed[tokens]
    for layer in range(toy.cfg.n_layer):
        kc, vc = alloc.layer_kv(layer)
        q = ops.qk_norm_rope_append(*toy.project(layer, x), toy.q_norm[layer], toy.k_norm[layer], 1e-6,
                                    toy.cos_sin, False, pos, torch.zeros_like(pos), kc, vc, table, none, none)
        o = ops.paged_attention_prefill(q.float()[None], kc, vc, table, ctx, toy.cfg.head_dim ** -0.5)
        x = x + o[0].bfloat16().flatten(1) @ toy.out[layer]
    return x[-1:]


def run(samples=8, prompt_len=1000, steps=32, layers=2, heads=32, kv_heads=8, head_dim=128, vocab=512,
        check=False, seed=0):
    torch.manual_seed(seed)
    cfg = ModelConfig("toy", layers, heads, head_dim, kv_heads)
    block = 16
    blocks = -(-prompt_len // block) + samples * (2 + -(-steps // block))
    alloc = TorchBlockAllocator(KVConfig(block, blocks, "bfloat16"), cfg, "cuda")
    toy = Toy(cfg, vocab, prompt_len + steps + 1, seed)
    tokens = torch.randint(0, vocab, (prompt_len,), device="cuda")
    prompt = alloc.allocate(range(prompt_len))
    x = prefill(toy, alloc, prompt, tokens)

    batch = alloc.fork(prompt, samples)
    alloc.free(prompt.block_ids)
    x = x.expand(samples, -1)
    worst, text = 0.0, [[] for _ in batch]
    for step in range(steps):
        if step == steps // 2 and len(batch) > 1:
            # every other sample has ended: its pages go back, the rest move down
            for a in batch[1::2]:
                alloc.free(a.block_ids)
            batch, x, text = batch[::2], x[::2], text[::2]
            alloc.compact(batch)
        logits = x.float() @ toy.embed.float().T
        new = torch.multinomial(torch.softmax(logits / logits.std(), -1), 1)[:, 0]
        for a, t, out in zip(batch, new.tolist(), text):
            alloc.extend(a, [t])
            out.append(t)
        # a scheduler keeps these between steps and changes what a new page changes
        table, (starts, lens) = alloc.block_table(batch), alloc.prefix_groups(batch)
        ctx = torch.tensor([a.num_tokens for a in batch], dtype=torch.int32, device="cuda")
        x = toy.embed[new]
        for layer in range(layers):
            q, k, v = toy.project(layer, x)
            o = alloc.layer_step_shared(layer, q, k, v, toy.q_norm[layer], toy.k_norm[layer], toy.cos_sin, ctx - 1,
                                        table, ctx, starts, lens)
            if check:
                none = torch.empty(0, device="cuda")
                kc, vc = alloc.layer_kv(layer)
                q2 = ops.qk_norm_rope_append(q, k, v, toy.q_norm[layer], toy.k_norm[layer], 1e-6, toy.cos_sin, False,
                                             ctx - 1, none, kc, vc, table, none, none)
                ref = ops.paged_attention_v3(q2.float(), kc, vc, table, ctx, head_dim ** -0.5, 0)
                worst = max(worst, float((o.float() - ref).abs().max() / ref.abs().max()))
            x = x + o.flatten(1) @ toy.out[layer]
    used = alloc.kv_cfg.num_blocks - alloc.num_free_blocks
    apart = samples * -(-(prompt_len + steps) // block)
    return {"text": text, "blocks_used": used, "blocks_apart": apart, "worst": worst, "alloc": alloc, "batch": batch}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    r = run(a.samples, a.prompt, a.steps, check=True)
    print(f"{len(r['text'])} samples left of {a.samples}; {r['blocks_used']} blocks in use at the end, "
          f"{r['blocks_apart']} if every sample had kept its own; attention within {r['worst']:.1e} of the plain decode")
