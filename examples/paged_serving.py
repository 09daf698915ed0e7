"""A serving loop over a paged cache: prompts in chunks, samples forked from one prompt, drafted tokens verified,
sequences dropped and the pool compacted -- with the package's operators only.

One attention layer with random projections stands for the model; every step's output is checked against the same
attention over dense tensors that the loop keeps beside the pool (fp32), so the script also shows that the table,
the rotary positions and the forks fit together.

    python examples/paged_serving.py            # needs a B200
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from attention_kernel_triton_b200.paged_chunk_attention import flash_attention_chunk_paged  # noqa: E402
from attention_kernel_triton_b200.paged_kv_pages import (compact_paged_kv_cache, fork_paged_kv_cache,  # noqa: E402
                                                         free_kv_pages)
from attention_kernel_triton_b200.rotary_embedding import append_rotary_paged_kv_cache, rotary_cos_sin  # noqa: E402


class PagedServer:
    """Sequences in a pool of pages; ``step`` appends new tokens to each and attends from them."""

    def __init__(self, num_pages=64, Hq=8, Hkv=2, D=128, page_size=16, max_positions=1024, dtype=torch.float16,
                 device="cuda", seed=0):
        self.Hq, self.Hkv, self.D, self.P, self.dev = Hq, Hkv, D, page_size, torch.device(device)
        self.pool = torch.zeros((num_pages, 2, Hkv, page_size, D), dtype=dtype, device=device)
        self.table = rotary_cos_sin(max_positions, D, device=device)
        self.pages, self.lens = [], []  # the page table as the host keeps it
        self.dense = []                 # per sequence: rotated keys and values [len, 2, Hkv, D], for the check
        self.gen = torch.Generator(device=device).manual_seed(seed)

    def i32(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.dev)

    def device_table(self):
        starts = [0]
        for p in self.pages:
            starts.append(starts[-1] + len(p))
        last = [n - self.P * (len(p) - 1) if p else 0 for n, p in zip(self.lens, self.pages)]
        return self.i32(starts), self.i32([x for p in self.pages for x in p]), self.i32(last)

    def add_sequence(self):
        self.pages.append([])
        self.lens.append(0)
        self.dense.append(torch.zeros((0, 2, self.Hkv, self.D), device=self.dev))

    def grow(self, news):
        """Pages for the new tokens, the lowest dead ones."""
        named = self.device_table()[1]
        free, count = free_kv_pages(self.pool.shape[0], named)
        free = free[:int(count)].tolist()
        for b, n in enumerate(news):
            while len(self.pages[b]) * self.P < self.lens[b] + n:
                self.pages[b].append(free.pop(0))
            self.lens[b] += n

    def step(self, news):
        """Appends ``news[b]`` tokens to sequence ``b``; returns their attention and its largest difference from the
        dense computation."""
        total = sum(news)
        qkv = torch.randn((total, self.Hq + 2 * self.Hkv, self.D), generator=self.gen, device=self.dev).to(self.pool.dtype)
        q, k, v = qkv.split((self.Hq, self.Hkv, self.Hkv), 1)
        self.grow(news)
        at = self.i32([0, *torch.tensor(news).cumsum(0).tolist()])
        table = self.device_table()
        q_rot = append_rotary_paged_kv_cache(self.pool, q, k, v, at, *table, self.table)
        out = flash_attention_chunk_paged(q_rot, at, self.pool, *table)
        return out, self.check(news, q, k, v, out)

    def check(self, news, q, k, v, out):
        half, worst, row = self.D // 2, 0.0, 0
        for b, n in enumerate(news):
            if not n:
                continue
            pos = torch.arange(self.lens[b] - n, self.lens[b], device=self.dev)
            c, s = self.table[pos][:, None, :half], self.table[pos][:, None, half:]
            turn = lambda x: torch.cat((x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s), -1)  # noqa: E731
            part = slice(row, row + n)
            new = torch.stack((turn(k[part].float()), v[part].float()), 1)
            self.dense[b] = torch.cat((self.dense[b], new))
            keys, values = self.dense[b].unbind(1)
            group = self.Hq // self.Hkv
            x = torch.einsum("nhgd,lhd->nhgl", turn(q[part].float()).unflatten(1, (self.Hkv, group)), keys) / math.sqrt(self.D)
            x = x.masked_fill(torch.arange(self.lens[b], device=self.dev) > pos[:, None, None, None], -math.inf)
            want = torch.einsum("nhgl,lhd->nhgd", x.softmax(-1), values).flatten(1, 2)
            worst = max(worst, (out[part].float() - want).abs().max().item())
            row += n
        return worst

    def fork(self, parents):
        """The batch becomes one continuation of each parent; sequences that none names are dropped."""
        entries = sum(len(self.pages[p]) for p in parents)
        starts, indices, _ = (t.tolist() for t in fork_paged_kv_cache(self.pool, *self.device_table(), self.i32(parents),
                                                                      max_entries=entries))
        self.pages = [indices[starts[i]:starts[i + 1]] for i in range(len(parents))]
        self.lens = [self.lens[p] for p in parents]
        self.dense = [self.dense[p].clone() for p in parents]

    def compact(self):
        starts, named, _ = self.device_table()
        indices, used = compact_paged_kv_cache(self.pool, named)
        starts, indices = starts.tolist(), indices.tolist()
        self.pages = [indices[starts[i]:starts[i + 1]] for i in range(len(self.pages))]
        return int(used)


def main(verbose=True):
    server, worst = PagedServer(), 0.0

    def say(what, error):
        nonlocal worst
        worst = max(worst, error)
        if verbose:
            print(f"{what:58s} largest difference {error:.1e}")

    for _ in range(3):
        server.add_sequence()
    say("prompts of 100, 37 and 5 tokens", server.step([100, 37, 5])[1])
    say("a second chunk of the first prompt beside decoding", server.step([70, 1, 1])[1])
    server.fork([0, 0, 1, 0])  # three samples of the first prompt, the second goes on, the third is dropped
    say("three samples and one sequence decode a token", server.step([1, 1, 1, 1])[1])
    say("five drafted tokens verified in each", server.step([5, 5, 5, 5])[1])
    server.fork([3, 2])
    used = server.compact()
    say(f"two sequences stay, the pool compacted to {used} pages", server.step([1, 4])[1])
    return worst, used


if __name__ == "__main__":
    error, _ = main()
    # fp16 rounding of the rotated rows, the weights and the outputs, on values below 4
    sys.exit(0 if error <= 8e-3 else 1)
