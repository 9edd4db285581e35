"""A decoder's attention layer served from GLINT planes and a 4-bit cache.

    python examples/attention_layer.py [--budget 512] [--steps 64]

What runs, all of it on this library's kernels: the q|k|v linear (device.htile) on packed
prompts, attention over them (attn_prompt), their keys and values into a paged 4-bit
cache (kv4_append); the cache's weights seeded by the last tokens of each prompt
(kv4_attn with several rows) and the cache cut to a budget (kv4_evict); then tokens one
at a time: q|k|v, append, attention with running weights, eviction every few steps,
and the o linear.  Random weights; sizes of one Llama-3-8B layer.  Rotary embedding and
the rest of a model are the caller's: `rope(q, k, positions)` is applied to the views.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import Callable, List, Optional

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from glint_b200 import attn, device  # noqa: E402


class AttentionLayer:
    """One layer's linears, cache and book-keeping for a fixed set of sequences.

    wqkv, wo: (hole, plug, absmax) planes of the [(heads + 2 kv_heads) * head_dim, hidden] and
    [hidden, heads * head_dim] weights.  Each sequence may hold `capacity` slots; beyond
    `budget` (plus `slack`, so that eviction runs once in `slack` steps) the slots of
    least weight go, the `recent` newest tokens excepted.  A call that would take a sequence
    past its slots raises ValueError."""

    def __init__(self, wqkv, wo, hidden: int, heads: int, kv_heads: int, head_dim: int, seqs: int, capacity: int,
                 budget: int, recent: int, slack: int = 16, window: int = 8, page_size: int = 64,
                 rope: Optional[Callable] = None):
        self.wqkv, self.wo, self.hidden, self.heads, self.rope = wqkv, wo, hidden, heads, rope
        self.kv_heads, self.head_dim, self.budget, self.recent = kv_heads, head_dim, budget, recent
        self.slack, self.window = slack, window
        per = -(-capacity // page_size)
        self.cache = attn.KV4Cache.empty(seqs * per, kv_heads, head_dim, page_size)
        # every sequence owns its pages from the start; a server would hand them out as lengths grow
        self.table = torch.arange(seqs * per, dtype=torch.int32, device="cuda").view(seqs, per)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.seen = torch.zeros_like(self.lens)
        # two pairs that take turns: eviction reads one and writes the other
        self.weight = [torch.zeros(seqs, kv_heads, per * page_size, device="cuda") for _ in range(2)]
        self.pos = [torch.zeros(seqs, kv_heads, per * page_size, dtype=torch.int32, device="cuda") for _ in range(2)]
        self.longest = 0  # an upper bound of lens, kept on the host

    def _qkv(self, x: torch.Tensor, positions: torch.Tensor):
        n = (self.heads + 2 * self.kv_heads) * self.head_dim
        y = device.htile(x, *self.wqkv, n, mode="fast", out_dtype=torch.bfloat16)
        y = y.view(x.shape[0], self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], 1)  # views: no copy
        return (*self.rope(q, k, positions), v) if self.rope else (q, k, v)

    def _o(self, o: torch.Tensor) -> torch.Tensor:
        o = o.reshape(-1, self.heads * self.head_dim)
        return device.htile(o, *self.wo, self.hidden, mode="fast", out_dtype=torch.bfloat16)

    def _room(self, longest: int) -> None:
        have = self.table.shape[1] * self.cache.page_size
        if longest > have:  # an index past the table would end the process's use of the GPU
            raise ValueError(f"{longest} slots wanted of a sequence's {have}: a larger capacity or a smaller budget")

    def _slots(self, seq: torch.Tensor, at: torch.Tensor) -> torch.Tensor:
        page = self.cache.page_size
        return self.table[seq, at // page] * page + (at % page).to(torch.int32)

    def prompt(self, x: torch.Tensor, lens: List[int]) -> torch.Tensor:
        """x [sum(lens), hidden]: the prompts, packed; each fills its sequence from the start."""
        if len(lens) != self.table.shape[0] or min(lens) < 1 or sum(lens) != x.shape[0]:
            raise ValueError(f"a prompt of a token or more for each of {self.table.shape[0]} sequences, packed")
        self._room(max(lens))
        n = torch.tensor(lens, device="cuda")
        ends = torch.zeros(len(lens) + 1, dtype=torch.int32, device="cuda")
        ends[1:] = n.cumsum(0)
        seq = torch.arange(len(lens), device="cuda").repeat_interleave(n)
        at = torch.arange(x.shape[0], device="cuda") - ends[seq]
        q, k, v = self._qkv(x, at)
        o, _ = attn.attn_prompt(q, k, v, ends)
        attn.kv4_append(self.cache, k, v, self._slots(seq, at))
        self.lens.copy_(n)
        self.seen.copy_(n)
        self.longest = max(lens)
        wide = self.pos[0].shape[2]
        self.pos[0].copy_(torch.arange(wide, dtype=torch.int32, device="cuda").expand_as(self.pos[0]))
        # which slots matter: what the prompts' last tokens look at
        w = min(self.window, min(lens))
        last = (ends[1:, None] - w + torch.arange(w, device="cuda")).view(-1)
        attn.kv4_attn(q[last].view(len(lens), w, self.heads, self.head_dim), self.cache, self.table, self.lens,
                      weight_out=self.weight[0])
        self._evict(0)
        return self._o(o)

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """x [seqs, hidden]: one token of every sequence."""
        seqs = x.shape[0]
        if seqs != self.table.shape[0]:
            raise ValueError(f"a token of each of {self.table.shape[0]} sequences, not {seqs}")
        self._room(self.longest + 1)
        q, k, v = self._qkv(x, self.seen)
        seq = torch.arange(seqs, device="cuda")
        attn.kv4_append(self.cache, k, v, self._slots(seq, self.lens))
        self.pos[0][seq, :, self.lens.long()] = self.seen[:, None]
        self.lens += 1
        self.seen += 1
        self.longest += 1
        self.attended, _ = attn.kv4_attn(q[:, None], self.cache, self.table, self.lens, weight=self.weight[0],
                                         weight_out=self.weight[0])
        self._evict(self.slack)
        return self._o(self.attended)

    def _evict(self, slack: int) -> None:
        if self.longest <= self.budget + slack:
            return
        _, self.lens = attn.kv4_evict(self.cache, self.table, self.lens, self.weight[0], self.pos[0], self.seen,
                                      self.budget, self.recent, weight_out=self.weight[1], pos_out=self.pos[1])
        self.weight.reverse()
        self.pos.reverse()
        self.longest = self.budget


def random_planes(n: int, k: int, g: torch.Generator):
    w = (torch.randn(n, k, device="cuda", generator=g) * k ** -0.5).bfloat16()
    return device.encode(w)


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--budget", type=int, default=512)
    p.add_argument("--steps", type=int, default=64)
    args = p.parse_args()
    hidden, heads, kv, dim = 4096, 32, 8, 128
    lens = [700, 1, 33, 1500, 260]
    g = torch.Generator(device="cuda").manual_seed(0)
    layer = AttentionLayer(random_planes((heads + 2 * kv) * dim, hidden, g), random_planes(hidden, heads * dim, g),
                           hidden, heads, kv, dim, len(lens), max(lens) + args.steps, args.budget, args.budget // 8)
    y = layer.prompt(torch.randn(sum(lens), hidden, device="cuda", generator=g).bfloat16(), lens)
    print(f"prompts of {lens} tokens -> {tuple(y.shape)}; slots held {layer.lens.tolist()}")
    x = torch.randn(len(lens), hidden, device="cuda", generator=g).bfloat16()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(args.steps):
        x = layer.step(x)
    end.record()
    end.synchronize()
    bits = 4 + 32 / attn.BLOCK
    print(f"{args.steps} steps, {begin.elapsed_time(end) / args.steps * 1e3:.0f} us each; slots held "
          f"{layer.lens.tolist()} of {layer.seen.tolist()} tokens seen, {bits} bits a value; "
          f"output finite: {bool(x.isfinite().all())}")


if __name__ == "__main__":
    main()
