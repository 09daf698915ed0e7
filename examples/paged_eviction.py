"""Samples of one prompt under a budget of cached tokens: the prompt's pages are shared, every step's attention reads
them once, its softmax weights are summed per key, and a sequence that grows past the budget gives up the tokens that
got the least.

One attention layer with random projections stands for the model.  Every step is checked against dense attention (fp32)
over the tokens that each head still has, which the loop keeps beside the pool, and so are the sums and the choice.

    python examples/paged_eviction.py            # needs a B200
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from attention_kernel_triton_b200.paged_kv_append import append_paged_kv_cache  # noqa: E402
from attention_kernel_triton_b200.paged_kv_eviction import (accumulate_attention_weights_paged,  # noqa: E402
                                                            evict_paged_kv_cache, select_kept_tokens)
from attention_kernel_triton_b200.paged_kv_pages import fork_paged_kv_cache, free_kv_pages  # noqa: E402
from attention_kernel_triton_b200.paged_prefix_attention import (  # noqa: E402
    flash_attention_shared_prefix_paged_with_lse, shared_prefix_pages)
from attention_kernel_triton_b200.rotary_embedding import apply_rotary_qk, rotary_cos_sin  # noqa: E402


class EvictingServer:
    def __init__(self, budget=96, sinks=4, recent=32, samples=3, Hq=8, Hkv=2, D=64, page_size=16, num_pages=96,
                 width=512, dtype=torch.float16, device="cuda", seed=0):
        self.Hq, self.Hkv, self.D, self.P, self.dev = Hq, Hkv, D, page_size, torch.device(device)
        self.budget, self.sinks, self.recent, self.samples, self.width = budget, sinks, recent, samples, width
        self.pool = torch.zeros((num_pages, 2, Hkv, page_size, D), dtype=dtype, device=device)
        self.cos_sin = rotary_cos_sin(4096, D, device=device)
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.pages, self.lens, self.seen = [[]], [0], [0]  # page table on the host; tokens in the pool, tokens so far
        self.sums = torch.zeros((1, Hkv, width), device=device)
        self.dense = [torch.zeros((0, 2, Hkv, D), device=device)]  # what the pool should hold, slot by slot
        self.worst = dict(attention=0.0, sums=0.0)

    def i32(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.dev)

    def table(self):
        starts = [0]
        for p in self.pages:
            starts.append(starts[-1] + len(p))
        last = [n - self.P * (len(p) - 1) if p else 0 for n, p in zip(self.lens, self.pages)]
        return self.i32(starts), self.i32([x for p in self.pages for x in p]), self.i32(last)

    def keep_table(self, starts, indices, last):
        starts, indices, last = starts.tolist(), indices.tolist(), last.tolist()
        self.pages = [indices[starts[b]:starts[b + 1]] for b in range(len(last))]
        self.lens = [self.P * (len(p) - 1) + n if p else 0 for p, n in zip(self.pages, last)]

    def step(self, new):
        """`new` tokens to every sequence: positions, append, attention, sums."""
        B = len(self.lens)
        free, count = free_kv_pages(self.pool.shape[0], self.table()[1])
        free = free[:int(count)].tolist()
        for b in range(B):
            self.lens[b] += new
            while len(self.pages[b]) * self.P < self.lens[b]:
                self.pages[b].append(free.pop(0))
        qkv = torch.randn((B * new, self.Hq + 2 * self.Hkv, self.D), generator=self.gen, device=self.dev).to(self.pool.dtype)
        q, k, v = qkv.split((self.Hq, self.Hkv, self.Hkv), 1)
        # the positions are those in the text, which the cache's slots no longer show once tokens are gone
        at = torch.cat([torch.arange(n, n + new, dtype=torch.int32, device=self.dev) for n in self.seen])
        q, k = apply_rotary_qk(q, k, self.cos_sin, at)
        self.seen = [n + new for n in self.seen]
        rows, table = self.i32(list(range(0, B * new + 1, new))), self.table()
        append_paged_kv_cache(self.pool, k, v, rows, *table)
        # one group: all samples of the prompt
        groups = self.i32([0, B])
        out, lse = flash_attention_shared_prefix_paged_with_lse(q, rows, self.pool, *table, groups)
        before = self.sums.clone()
        accumulate_attention_weights_paged(self.sums, q, rows, self.pool, *table, lse)
        for b in range(B):
            part = slice(b * new, (b + 1) * new)
            self.dense[b] = torch.cat((self.dense[b], torch.stack((k[part], v[part]), 1).float()))
            self.check(b, q[part].float(), out[part].float(), before[b])
        return out

    def check(self, b, q, out, before):
        L, n, G = self.lens[b], q.shape[0], self.Hq // self.Hkv
        keys, values = self.dense[b].unbind(1)
        x = torch.einsum("nhgd,lhd->nhgl", q.unflatten(1, (self.Hkv, G)), keys) / math.sqrt(self.D)
        pos = torch.arange(L - n, L, device=self.dev)
        w = x.masked_fill(torch.arange(L, device=self.dev) > pos[:, None, None, None], -math.inf).softmax(-1)
        want = torch.einsum("nhgl,lhd->nhgd", w, values).flatten(1, 2)
        self.worst["attention"] = max(self.worst["attention"], (out - want).abs().max().item())
        sums = before[:, :L] + w.sum((0, 2))
        self.worst["sums"] = max(self.worst["sums"], ((self.sums[b, :, :L] - sums).abs() / (1 + sums)).max().item())

    def fork(self):
        """The prompt becomes `samples` sequences that share its full pages."""
        parents = [0] * self.samples
        self.keep_table(*fork_paged_kv_cache(self.pool, *self.table(), self.i32(parents),
                                             max_entries=len(self.pages[0]) * self.samples))
        self.sums = self.sums[parents]
        self.dense = [self.dense[0].clone() for _ in parents]
        self.seen = [self.seen[0]] * self.samples

    def evict(self):
        """Every sequence back to the budget; returns the tokens that each head of each kept."""
        lens = self.i32(self.lens)
        keep, kept = select_kept_tokens(self.sums, lens, self.budget, sinks=self.sinks, recent=self.recent)
        table = evict_paged_kv_cache(self.pool, *self.table(), keep, kept, weights=self.sums)
        starts, indices, last = table
        self.keep_table(starts, indices, last)
        for b, n in enumerate(kept.tolist()):
            rows = keep[b, :, :n].long()  # [Hkv, n]
            self.dense[b] = torch.stack([self.dense[b][rows[h], :, h] for h in range(self.Hkv)], 2)
        return keep, kept

    def shared(self):
        starts, indices, last = self.table()
        return shared_prefix_pages(self.i32([0, len(self.lens)]), starts, indices, last, self.P).item()


def main(verbose=True):
    server = EvictingServer()

    def say(what):
        if verbose:
            print(f"{what:62s} attention {server.worst['attention']:.1e}  sums {server.worst['sums']:.1e}")

    server.step(100)
    say("a prompt of 100 tokens")
    server.fork()
    shared = server.shared()
    for _ in range(4):
        server.step(5)
    say(f"three samples, {shared} pages shared, five tokens a step")
    server.evict()
    say(f"back to {server.lens[0]} tokens, {server.shared()} pages shared")
    for _ in range(20):
        server.step(1)
        if max(server.lens) > server.budget + 12:
            server.evict()
    say("20 single tokens under the budget")
    return server


if __name__ == "__main__":
    s = main()
    # fp16 rounding of the rows, weights and outputs, on values below 4; sums in fp32 of scores of fp16 rows
    sys.exit(0 if s.worst["attention"] <= 8e-3 and s.worst["sums"] <= 1e-4 else 1)
