"""Sampled generation through a hybrid stack on one MI355X, as a server would run it: three linear-attention
layers (MXFP4 projections, the short convolution, the gated delta rule, the gated norm that quantizes for the
output projection) for one of attention over the 4-bit paged cache, tokens by temperature, top-k, top-p and
min-p, a forked sequence, and drafted tokens of which the states after each are kept until it is known how many
count.

  python examples/gdn_generate.py [--layers 4] [--prompt 700] [--steps 24]

Weights are random (synthetic.weights); layers have no MLP.
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from examples.kv4_generate import AttentionLayer, Linear  # noqa: E402
from vllm_sly_radiance_amd import radiance_fused_norm as fused  # noqa: E402
from vllm_sly_radiance_amd import radiance_gdn as gdn  # noqa: E402
from vllm_sly_radiance_amd import radiance_kv4 as kv4  # noqa: E402
from vllm_sly_radiance_amd.kv4_pool import PagePool  # noqa: E402
from vllm_sly_radiance_amd.radiance_sample import sample  # noqa: E402

DRAFT = 3       # drafted tokens of a step at most


class GdnLayer:
    """x -> o_proj(norm(delta rule(conv(in_proj(x))), z)), its states in one layer of the pools."""

    def __init__(self, hidden, k_heads, v_heads, d, width, seed, device):
        self.k_heads, self.v_heads, self.d = k_heads, v_heads, d
        self.channels = (2 * k_heads + v_heads) * d
        self.in_proj = Linear(self.channels + v_heads * d, hidden, seed, device)
        self.o_proj = Linear(hidden, v_heads * d, seed + 1, device)
        g = np.random.default_rng(seed + 2)
        bf16 = lambda x: torch.from_numpy(x.astype(np.float32)).to(device, torch.bfloat16)  # noqa: E731
        self.conv_weight = bf16(g.standard_normal((self.channels, width)) / width ** 0.5)
        self.gates = bf16(g.standard_normal((hidden, 2 * v_heads)) / hidden ** 0.5)
        self.norm_weight = bf16(1 + 0.1 * g.standard_normal(d))
        self.a_log = torch.from_numpy(np.log(g.uniform(1, 16, v_heads)).astype(np.float32)).to(device)
        self.dt_bias = torch.from_numpy(g.uniform(-6, -2, v_heads).astype(np.float32)).to(device)

    def __call__(self, x, conv_state, state, *batch):
        T = x.shape[0]
        mixed, z = self.in_proj(x).split([self.channels, self.v_heads * self.d], 1)
        a, b = (x @ self.gates).split(self.v_heads, 1)
        mixed = gdn.causal_conv(mixed, self.conv_weight, None, conv_state, *batch)
        q, k, v = mixed.view(T, -1, self.d).split([self.k_heads, self.k_heads, self.v_heads], 1)
        o = gdn.gated_delta_rule(q, k, v, a, b, self.a_log, self.dt_bias, state, *batch)
        return self.o_proj(fused.call_gdn_norm_quant(o.view(T, -1), z, self.norm_weight, 1e-6))


class Hybrid:
    def __init__(self, layers=4, hidden=2048, k_heads=8, v_heads=16, heads=16, kv_heads=4, d=128, width=4,
                 vocabulary=512, positions=8192, pages=512, page=16, sequences=8, device="cuda"):
        at = torch.arange(positions, device=device, dtype=torch.float32)[:, None]
        at = at * 1e4 ** (-torch.arange(0, d, 2, device=device, dtype=torch.float32) / d)
        table = torch.cat([at.cos(), at.sin()], 1)
        self.layers = [AttentionLayer(hidden, heads, kv_heads, d, table, 10 * i, device) if i % 4 == 3 else
                       GdnLayer(hidden, k_heads, v_heads, d, width, 10 * i, device) for i in range(layers)]
        attention = sum(isinstance(x, AttentionLayer) for x in self.layers)
        self.pool = PagePool(kv4.new_cache(pages, kv_heads, page, d, device, layers=max(attention, 1)))
        # a sequence's slots: its state, or those after a token and each of the drafted ones behind it
        slots = sequences * (1 + DRAFT)
        self.conv_state = gdn.new_conv_state(slots, (2 * k_heads + v_heads) * d, width, device, layers - attention)
        self.state = gdn.new_state(slots, v_heads, d, d, device, layers - attention)
        self.free, self.base, self.now = list(range(0, slots, 1 + DRAFT)), {}, {}
        g = np.random.default_rng(99)
        self.embedding, self.unembedding = (
            torch.from_numpy(g.standard_normal((vocabulary, hidden), np.float32))
            .to(device, torch.bfloat16) for _ in range(2))

    def _room(self):
        if not self.free:
            raise RuntimeError(f"there are {len(self.base)} sequences, as many as there is room for")

    def add(self):
        self._room()
        sequence = self.pool.add()
        self.base[sequence], self.now[sequence] = self.free.pop(), -1
        return sequence

    def fork(self, sequence):
        self._room()
        other = self.pool.fork(sequence)
        self.base[other], self.now[other] = self.free.pop(), -1
        if self.now[sequence] >= 0:         # (else there is nothing to go on from)
            self.now[other] = self.base[other]
            for pool in (self.conv_state, self.state):
                pool[:, self.base[other]] = pool[:, self.now[sequence]]
        return other

    def drop(self, sequence):
        self.pool.free(sequence)
        self.free.append(self.base.pop(sequence))
        del self.now[sequence]

    def keep(self, sequence, drafted, good):
        """Of the last `drafted` tokens of forward(..., drafts=True), the first `good` count."""
        self.pool.truncate(sequence, self.pool.length(sequence) - (drafted - good))
        self.now[sequence] = self.base[sequence] + good

    def forward(self, sequences, tokens, drafts=False):
        """Logits fp32 [total, vocabulary] of the new tokens (a list a sequence). drafts: the states after
        each are kept, for `keep` to choose from; one and DRAFT behind it at most."""
        if drafts and max(map(len, tokens), default=0) > 1 + DRAFT:
            raise ValueError(f"more than {DRAFT} drafted tokens behind one of a sequence")
        step = self.pool.extend(sequences, [len(t) for t in tokens])
        _, _, starts, max_q, _ = step.attention
        device = self.embedding.device
        flat = torch.tensor([t for ts in tokens for t in ts], dtype=torch.int64).to(device)
        read = torch.tensor([self.now[s] for s in sequences], dtype=torch.int32).to(device)
        write = torch.tensor([self.base[s] for s in sequences], dtype=torch.int32).to(device)
        if drafts:
            write = write[:, None] + torch.arange(max_q, dtype=torch.int32, device=device)
        x, linear, attention = self.embedding[flat], 0, 0
        for layer in self.layers:
            y = torch.nn.functional.rms_norm(x, x.shape[-1:])
            if isinstance(layer, AttentionLayer):
                y = layer(y, self.pool.cache[attention], step)
                attention += 1
            else:
                y = layer(y, self.conv_state[linear], self.state[linear], starts, read, write, max_q)
                linear += 1
            x = x + torch.nn.functional.rms_norm(y, y.shape[-1:])
        for s, t in zip(sequences, tokens):
            if t or not drafts:             # (the state after each of no tokens is written nowhere)
                self.now[s] = self.base[s] + (len(t) - 1 if drafts else 0)
        return x.float() @ self.unembedding.float().T / x.shape[1] ** 0.5


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--prompt", type=int, default=700)
    p.add_argument("--steps", type=int, default=24)
    a = p.parse_args(argv)
    how = dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.02)
    with torch.no_grad():
        s = Hybrid(layers=a.layers)
        rng = np.random.default_rng(1)
        chance = torch.Generator("cuda").manual_seed(7)
        said = lambda logits: sample(  # noqa: E731
            logits, torch.rand(len(logits), device="cuda", generator=chance), **how).tolist()
        prompt = rng.integers(0, 512, a.prompt).tolist()
        first = s.add()
        after = s.forward([first], [prompt])[-1:]
        ids = [first, s.fork(first)]
        nexts = said(after.expand(2, -1))
        out, taken = [[], []], 0
        torch.cuda.synchronize()
        start = time.perf_counter()
        for i in range(a.steps):
            # every other step verifies drafted tokens
            draft = [[], []]
            if i % 2:
                draft = rng.integers(0, 512, (2, DRAFT)).tolist()
            logits = s.forward(ids, [[n] + t for n, t in zip(nexts, draft)], drafts=True)
            rows = 1 + len(draft[0])
            tokens = said(logits)
            for b, sequence in enumerate(ids):
                out[b].append(nexts[b])
                row, good = tokens[b * rows:(b + 1) * rows], 0
                while good < len(draft[b]) and draft[b][good] == row[good]:
                    good += 1
                out[b] += draft[b][:good]
                taken += good
                nexts[b] = row[good]
                s.keep(sequence, len(draft[b]), good)
        torch.cuda.synchronize()
        took = time.perf_counter() - start
    print(f"{a.steps} steps of 2 sequences over {a.layers} layers: {1e3 * took / a.steps:.2f} ms a step, "
          f"{taken} drafted tokens taken")
    for o in out:
        print("  ", *o)
    return s, ids, prompt, out


if __name__ == "__main__":
    main()
