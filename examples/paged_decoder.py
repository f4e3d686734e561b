"""The attention block of a decoder layer that serves several users from a paged key/value cache.

    python examples/paged_decoder.py                     # 8 users, prompts of up to 700 tokens, 64 tokens each, Mistral-7B's widths

A step takes any number of new tokens of every user: whole prompts, chunks of them, single tokens, all in one call of each
operator.  The weights are random block floats (there is no checkpoint here), the hidden states random numbers.  With rotary_dim, queries and
keys turn by their positions on the way from the projection to attention and cache; with a window, a conversation's last tokens and its
first few (sinks) are what attention looks at, and release() gives the pages between them back; fork() lets requests go on from others."""
from __future__ import annotations

import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-metal_amd"))

import ttnn  # noqa: E402


class PagedAttention:
    """x -> attention(x w_qkv) w_o, with the keys and values of `users` requests in `pages` pages of `page_size` tokens."""

    def __init__(self, device, *, hidden, heads, kv_heads, head_dim, users, pages, page_size, longest, cache_dtype, window=None, sinks=0,
                 rotary_dim=None, interleaved=False, norms=(None, None)):
        """rotary_dim: elements of a head that turn (None: no positions); norms: weights of the norms of query and key heads, float32 [head_dim], or None."""
        self.device, self.heads, self.kv_heads, self.head_dim, self.page_size, self.window, self.sinks = device, heads, kv_heads, head_dim, page_size, window, sinks
        self.pages, self.interleaved = pages, interleaved
        self.frequencies = None if rotary_dim is None else ttnn.experimental.rotary_frequencies(rotary_dim, device=device)
        self.query_norm, self.key_norm = (None if w is None else ttnn.from_torch(w.float(), device=device) for w in norms)
        self.w_qkv = self._weights(hidden, (heads + 2 * kv_heads) * head_dim)
        self.w_o = self._weights(heads * head_dim, hidden)
        self.keys, self.values = (ttnn.experimental.allocate_paged_cache(pages, kv_heads, page_size, head_dim, dtype=cache_dtype, device=device) for _ in range(2))
        self.page_table = self._integers([[-1] * -(-longest // page_size)] * users)
        self.free_pages = list(range(pages))
        self.lengths = [0] * users

    def _weights(self, rows, columns):
        return ttnn.from_torch(torch.randn(1, 1, rows, columns) * rows ** -0.5, dtype=ttnn.bfloat8_b, layout=ttnn.TILE_LAYOUT, device=self.device)

    def _integers(self, values):
        return ttnn.from_torch(torch.tensor(values, dtype=torch.int32), device=self.device)

    def step(self, x, new):
        """x: bfloat16 [1, 1, sum(new), hidden], the new tokens of all users one after the other, new[u] of user u."""
        E, width = ttnn.experimental, self.head_dim * self.kv_heads
        cached = self._integers(self.lengths)
        # once per step, for all layers of a model
        self.page_table, slots, row_starts, counts = E.paged_tables(cached, self._integers(new), self.page_table, self._integers(self.free_pages), page_size=self.page_size, num_tokens=sum(new))
        # per layer
        qkv = ttnn.linear(x, self.w_qkv)
        columns = {"key_column": self.heads * self.head_dim, "value_column": self.heads * self.head_dim + width}
        if self.frequencies is None:
            queries = qkv
            E.write_paged_cache(qkv, self.keys, self.values, slots, **columns)
        else:
            queries = E.rotate_write_paged_cache(qkv, self.keys, self.values, slots, cached, row_starts, self.frequencies, num_heads=self.heads, **columns, interleaved=self.interleaved,
                                                 query_norm=self.query_norm, key_norm=self.key_norm)
        context = E.attend_paged_cache(queries, self.keys, self.values, self.page_table, cached, row_starts, num_heads=self.heads, window=self.window, sinks=self.sinks)
        y = ttnn.linear(context, self.w_o)
        taken, missing = ttnn.to_torch(ttnn.from_device(counts)).flatten().tolist()
        if missing:
            raise RuntimeError(f"{missing} pages short")
        self.free_pages = self.free_pages[taken:]
        self.lengths = [length + n for length, n in zip(self.lengths, new)]
        return y

    def fork(self, parents):
        """User u goes on from where user parents[u] is (-1: from scratch).  The caches of all layers of a model would be copied by the one call."""
        E = ttnn.experimental
        self.page_table, lengths, sources, targets, counts = E.fork_paged_tables(self.page_table, self._integers(self.lengths), self._integers(parents), self._integers(self.free_pages), page_size=self.page_size)
        E.copy_paged_pages([self.keys, self.values], sources, targets)
        missing = ttnn.to_torch(ttnn.from_device(counts)).flatten().tolist()[1]
        if missing:
            raise RuntimeError(f"{missing} pages short")
        self.lengths = ttnn.to_torch(ttnn.from_device(lengths)).flatten().tolist()
        self.release()

    def release(self):
        """The pages that no user needs any longer come back."""
        self.page_table, free, counts = ttnn.experimental.release_paged_pages(self.page_table, self._integers(self.lengths), page_size=self.page_size, num_pages=self.pages, window=self.window, sinks=self.sinks)
        there = ttnn.to_torch(ttnn.from_device(counts)).flatten().tolist()[0]
        self.free_pages = ttnn.to_torch(ttnn.from_device(free)).flatten().tolist()[:there]


def main():
    torch.manual_seed(0)
    device = ttnn.open_device(0)
    hidden, prompts, tokens = 4096, [700, 33, 512, 1, 260, 90, 411, 128], 64
    block = PagedAttention(device, hidden=hidden, heads=32, kv_heads=8, head_dim=128, users=len(prompts), pages=200, page_size=64, longest=1024, cache_dtype=ttnn.bfloat8_b,
                           window=256, sinks=4, rotary_dim=128)
    states = lambda n: ttnn.from_torch(torch.randn(1, 1, n, hidden).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device)
    y = block.step(states(sum(prompts)), prompts)
    print("prompts of", prompts, "tokens:", tuple(y.shape))
    x = states(len(prompts))
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for _ in range(tokens):
        y = block.step(x, [1] * len(prompts))
    torch.cuda.synchronize()
    print(f"{tokens} tokens for each of {len(prompts)} users: {(time.perf_counter() - begin) / tokens * 1e6:.0f} us per step, lengths now {block.lengths}, {len(block.free_pages)} pages free")
    block.release()
    print(f"behind the window of {block.window}: {len(block.free_pages)} pages free")
    block.fork([0, 0, 0, 0, 4, 4, 4, 4])
    block.step(x, [1] * len(prompts))
    print(f"eight answers to two prompts: lengths {block.lengths}, {len(block.free_pages)} pages free")
    ttnn.close_device(device)


if __name__ == "__main__":
    main()
