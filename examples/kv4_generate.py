"""Greedy generation through a stack of attention layers on one MI355X, as a server would run it: MXFP4
projections, the head norm and rotation into a 4-bit paged cache, attention over it, forked sequences,
drafted tokens that are rejected, and a compaction between steps.

  python examples/kv4_generate.py [--layers 4] [--prompt 700] [--steps 24]

Weights are random (synthetic.weights); each layer is x + o_proj(attention(qkv(norm(x)))), with no MLP.
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vllm_sly_radiance_amd import radiance_kv4 as kv4  # noqa: E402
from vllm_sly_radiance_amd import radiance_mxfp4 as mxfp4  # noqa: E402
from vllm_sly_radiance_amd import synthetic  # noqa: E402
from vllm_sly_radiance_amd.kv4_pool import PagePool  # noqa: E402


class Linear:
    """An MXFP4 linear through the quant method that a model would use."""

    def __init__(self, n, k, seed, device):
        w, ws = synthetic.weights(n, k, seed)
        self.layer = torch.nn.Module()
        for name, x in (("weight", w), ("weight_scale", ws)):
            setattr(self.layer, name, torch.nn.Parameter(torch.from_numpy(x).to(device),
                                                         requires_grad=False))
        self.kernel = mxfp4.kernel_class()()
        self.kernel.process_weights_after_loading(self.layer)

    def __call__(self, x):
        return self.kernel.apply_weights(self.layer, x)


class AttentionLayer:
    """x -> o_proj(attention(qkv(x))), its keys and values in `cache` (one layer of kv4.new_cache)."""

    def __init__(self, hidden, heads, kv_heads, d, table, seed, device):
        self.heads, self.kv_heads, self.d, self.table = heads, kv_heads, d, table
        self.qkv = Linear((heads + 2 * kv_heads) * d, hidden, seed, device)
        self.o_proj = Linear(hidden, heads * d, seed + 1, device)
        g = np.random.default_rng(seed + 2)
        self.q_weight, self.k_weight = (torch.from_numpy(1 + 0.1 * g.standard_normal(d, np.float32))
                                        .to(device, torch.bfloat16) for _ in range(2))

    def __call__(self, x, cache, step):
        T = x.shape[0]
        q, k, v = self.qkv(x).view(T, -1, self.d).split([self.heads, self.kv_heads, self.kv_heads], 1)
        q = kv4.qk_norm_rope_append(q, k, v, self.q_weight, self.k_weight, self.table, step.positions,
                                    cache, step.slots)
        return self.o_proj(kv4.attention(q, cache, *step.attention).view(T, -1))


class Stack:
    def __init__(self, layers=4, hidden=2048, heads=16, kv_heads=4, d=128, vocabulary=512, positions=8192,
                 pages=512, page=16, device="cuda"):
        at = torch.arange(positions, device=device, dtype=torch.float32)[:, None]
        at = at * 1e4 ** (-torch.arange(0, d, 2, device=device, dtype=torch.float32) / d)
        table = torch.cat([at.cos(), at.sin()], 1)
        self.layers = [AttentionLayer(hidden, heads, kv_heads, d, table, 10 * i, device)
                       for i in range(layers)]
        self.pool = PagePool(kv4.new_cache(pages, kv_heads, page, d, device, layers=layers))
        g = np.random.default_rng(99)
        self.embedding, self.unembedding = (
            torch.from_numpy(g.standard_normal((vocabulary, hidden), np.float32))
            .to(device, torch.bfloat16) for _ in range(2))

    def forward(self, sequences, tokens):
        """Logits fp32 [total, vocabulary] of the new tokens (a list a sequence), which join the cache."""
        step = self.pool.extend(sequences, [len(t) for t in tokens])
        flat = torch.tensor([t for ts in tokens for t in ts], dtype=torch.int64)
        x = self.embedding[flat.to(self.embedding.device)]
        for i, layer in enumerate(self.layers):
            y = layer(torch.nn.functional.rms_norm(x, x.shape[-1:]), self.pool.cache[i], step)
            x = x + torch.nn.functional.rms_norm(y, y.shape[-1:])
        return x.float() @ self.unembedding.float().T


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--prompt", type=int, default=700)
    p.add_argument("--steps", type=int, default=24)
    a = p.parse_args(argv)
    with torch.no_grad():
        s = Stack(layers=a.layers)
        rng = np.random.default_rng(1)
        prompt = rng.integers(0, 512, a.prompt).tolist()
        done_soon, first = s.pool.add(), s.pool.add()
        s.forward([done_soon], [prompt[:100]])
        nexts = [int(s.forward([first], [prompt])[-1].argmax())]
        # a second continuation from the same prompt, whose pages both share
        ids = [first, s.pool.fork(first)]
        nexts.append((nexts[0] + 1) % 512)
        out = [[], []]
        torch.cuda.synchronize()
        start = time.perf_counter()
        for i in range(a.steps):
            draft = rng.integers(0, 512, (2, 3)).tolist() if i % 4 == 3 else [[], []]
            logits = s.forward(ids, [[n] + t for n, t in zip(nexts, draft)])
            rows = 1 + len(draft[0])
            for b, sequence in enumerate(ids):
                out[b].append(nexts[b])
                # drafted tokens count while they are what the model would have said
                good = 0
                said = logits[b * rows:(b + 1) * rows].argmax(1).tolist()
                while good < len(draft[b]) and draft[b][good] == said[good]:
                    good += 1
                out[b] += draft[b][:good]
                nexts[b] = said[good]
                s.pool.truncate(sequence, s.pool.length(sequence) - (len(draft[b]) - good))
            if i == a.steps // 2:
                s.pool.free(done_soon)
                moved = s.pool.compact()
        torch.cuda.synchronize()
        took = time.perf_counter() - start
    print(f"{a.steps} steps of 2 sequences over {a.layers} layers: {1e3 * took / a.steps:.2f} ms a step, "
          f"{s.pool.pages - s.pool.free_pages} pages in use, {moved} moved")
    for o in out:
        print("  ", *o)
    return s, ids, prompt, out


if __name__ == "__main__":
    main()
