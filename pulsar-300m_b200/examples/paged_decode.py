"""Serving attention layers of Pulsar from a paged 4-bit KV cache: a few sequences of unequal length are
prefilled in chunks, decode together, verify a block of drafts and take part of it back.

    python pulsar-300m_b200/examples/paged_decode.py [--sequences 6] [--prompt 700] [--steps 8]

Layers 0 (local: window 1024) and 3 (global: theta 1e6, long-context query gain) of a random-init model
(``make_state_dict``) run on random hidden states. Every row's attention is compared with the same
attention over unquantised keys and values in 32 bits; the differences printed are what 4 bits cost.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pulsar_b200 import paged  # noqa: E402
from pulsar_b200.config import PulsarConfig  # noqa: E402
from pulsar_b200.weights import make_state_dict  # noqa: E402

PAGE = 64


class Layer:
    """One attention layer up to the output projection, on a paged cache and beside it in 32 bits."""

    def __init__(self, cfg, state, index, num_pages, max_pos, device):
        b = f"core.{index}.attn."
        self.cfg, self.window = cfg, 0 if index in (3, 7) else 1024
        self.wqkv = state[b + "wqkv.weight"].to(device, torch.bfloat16)
        # random-init heads have equal norm weights; spread them as training does
        g = torch.Generator().manual_seed(index)
        self.q_norm = (state[b + "q_norm_weight"][0] + 0.1 * torch.randn(cfg.n_heads, 64, generator=g)).to(device)
        self.k_norm = (state[b + "k_norm_weight"][0] + 0.1 * torch.randn(cfg.n_kv_heads, 64, generator=g)).to(device)
        theta = cfg.rope_theta_local if self.window else cfg.rope_theta_global
        self.cos, self.sin = paged.rope_tables(max_pos, 64, theta, device=device)
        at = torch.arange(1, max_pos + 1, device=device).clamp(min=cfg.base_seq_len)
        self.q_gain = None if self.window else 1 + 0.1 * torch.log(at / cfg.base_seq_len)
        self.pages = paged.kv4_pages(num_pages, cfg.n_kv_heads, 64, PAGE, device)
        self.kept = {}                  # sequence -> unquantised (k, v) so far

    def __call__(self, x, batch):
        """x [rows, d_model]: append every row's key and value, then attend."""
        cfg, qd, kd = self.cfg, self.cfg.n_heads * 64, self.cfg.n_kv_heads * 64
        q, k, v = (t.unflatten(-1, (-1, 64)) for t in F.linear(x, self.wqkv).split([qd, kd, kd], -1))
        queries = paged.kv4_append(q, k, v, self.pages, batch.slots, batch.positions, self.cos, self.sin,
                                   q_norm=self.q_norm, k_norm=self.k_norm, eps=cfg.rms_eps, q_gain=self.q_gain)
        out = paged.kv4_attention(queries, self.pages, batch.table, batch.lens, batch.cu, max_q=batch.max_q,
                                  max_kv=batch.max_kv, window=self.window)
        return out, self._plain(queries, k, v, batch)

    def _plain(self, queries, k, v, batch):
        k = k.float()
        k = self.k_norm * (k * torch.rsqrt(k.pow(2).mean(-1, keepdim=True) + self.cfg.rms_eps))
        c, s = (t[batch.positions.long()][:, None] for t in (self.cos, self.sin))
        a, b = k.chunk(2, -1)
        k = torch.cat([a * c - b * s, b * c + a * s], -1)
        out = torch.empty_like(queries, dtype=torch.float32)
        for i, (seq, n0, n1) in enumerate(batch.parts):
            lo, hi = batch.rows[i], batch.rows[i + 1]
            old = self.kept.get(seq, (k[:0], v[:0].float()))
            kk, vv = (torch.cat([o[:n0], t[lo:hi].float()]) for o, t in zip(old, (k, v)))
            self.kept[seq] = kk, vv
            at, pos = torch.arange(n1, device=k.device), torch.arange(n0, n1, device=k.device)[:, None]
            hide = (at > pos) | (at <= pos - self.window if self.window else at < 0)
            g = queries.shape[1] // kk.shape[1]
            score = torch.einsum("qhd,khd->hqk", queries[lo:hi].float(), kk.repeat_interleave(g, 1)) / 8
            out[lo:hi] = torch.einsum("hqk,khd->qhd", score.masked_fill(hide, -torch.inf).softmax(-1),
                                      vv.repeat_interleave(g, 1))
        return out


class Batch:
    """The rows of one step: ``parts`` lists (sequence, its length before, its length with its rows)."""

    def __init__(self, tables, parts, device):
        self.parts = parts
        counts = [n1 - n0 for _, n0, n1 in parts]
        self.rows = [sum(counts[:i]) for i in range(len(parts) + 1)]
        self.max_q, self.max_kv = max(counts), max(n1 for _, _, n1 in parts)
        width = max(len(tables[s]) for s, _, _ in parts)
        self.table = torch.tensor([tables[s] + [-1] * (width - len(tables[s])) for s, _, _ in parts],
                                  dtype=torch.int32, device=device)
        self.lens = torch.tensor([n1 for _, _, n1 in parts], dtype=torch.int32, device=device)
        self.cu = None if self.max_q == 1 else torch.tensor(self.rows, dtype=torch.int32, device=device)
        at = [(s, i) for s, n0, n1 in parts for i in range(n0, n1)]
        self.positions = torch.tensor([i for _, i in at], dtype=torch.int32, device=device)
        self.slots = torch.tensor([tables[s][i // PAGE] * PAGE + i % PAGE for s, i in at], device=device)


def run(sequences=6, prompt=700, steps=8, drafts=4, seed=0, device="cuda"):
    """Largest relative difference (2-norm) of each kind of step from the unquantised attention."""
    cfg = PulsarConfig()
    state = make_state_dict(cfg, seed=seed)
    gen = torch.Generator().manual_seed(seed)
    lens = [1 + int(i) for i in torch.randint(prompt, (sequences,), generator=gen)]
    lens[0] = prompt
    max_pos = prompt + steps + drafts + 2
    num_pages = sum(-(-(n + steps + drafts + 2) // PAGE) for n in lens)
    free = torch.randperm(num_pages, generator=gen).tolist()
    layers = [Layer(cfg, state, i, num_pages, max_pos, device) for i in (0, 3)]
    tables, have, worst = [[] for _ in lens], [0] * sequences, {}

    def step(kind, counts):
        parts = [(s, have[s], have[s] + c) for s, c in enumerate(counts) if c]
        for s, _, n1 in parts:
            while len(tables[s]) * PAGE < n1:
                tables[s].append(free.pop())
            have[s] = n1
        batch = Batch(tables, parts, device)
        x = torch.randn(batch.rows[-1], cfg.d_model, generator=gen).to(device, torch.bfloat16)
        for layer in layers:
            out, ref = layer(x, batch)
            worst[kind] = max(worst.get(kind, 0.0), ((out.float() - ref).norm() / ref.norm()).item())

    chunk = max(1, prompt // 2)
    step("first chunk", [min(n, chunk) for n in lens])
    if any(n > chunk for n in lens):
        step("second chunk", [max(0, n - chunk) for n in lens])
    for _ in range(steps):
        step("decode", [1] * sequences)
    step("verify", [drafts + 1] * sequences)
    for s in range(sequences):     # keep the first s % (drafts + 1) drafts: the length is the rollback
        have[s] -= drafts - s % (drafts + 1)
    step("decode after rollback", [1] * sequences)
    return worst, layers[0].pages.numel(), sum(len(t) for t in tables) * PAGE


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--sequences", type=int, default=6)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    worst, nbytes, tokens = run(a.sequences, a.prompt, a.steps)
    for kind, off in worst.items():
        print(f"{kind:22s} off by {100 * off:.2f} % of the unquantised attention")
    print(f"cache: {nbytes / 2**20:.2f} MiB a layer for {tokens} token places, bf16: {tokens * 4 * 64 * 4 / 2**20:.2f} MiB")


if __name__ == "__main__":
    main()
