"""The attention block of a decoder layer that serves several users from a paged key/value cache.

    python examples/paged_decoder.py                     # 8 users, prompts of up to 700 tokens, 64 tokens each, Mistral-7B's widths

A step takes any number of new tokens of every user: whole prompts, chunks of them, single tokens, all in one call of each
operator.  The weights are random block floats (there is no checkpoint here), the hidden states random numbers.  Queries and keys go into
attention and cache as they are projected: a model with rotary positions rotates them in the qkv rows first, which is not done here."""
from __future__ import annotations

import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-metal_amd"))

import ttnn  # noqa: E402


class PagedAttention:
    """x -> attention(x w_qkv) w_o, with the keys and values of `users` requests in `pages` pages of `page_size` tokens."""

    def __init__(self, device, *, hidden, heads, kv_heads, head_dim, users, pages, page_size, longest, cache_dtype, window=None):
        self.device, self.heads, self.kv_heads, self.head_dim, self.page_size, self.window = device, heads, kv_heads, head_dim, page_size, window
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
        E.write_paged_cache(qkv, self.keys, self.values, slots, key_column=self.heads * self.head_dim, value_column=self.heads * self.head_dim + width)
        context = E.attend_paged_cache(qkv, self.keys, self.values, self.page_table, cached, row_starts, num_heads=self.heads, window=self.window)
        y = ttnn.linear(context, self.w_o)
        taken, missing = ttnn.to_torch(ttnn.from_device(counts)).flatten().tolist()
        if missing:
            raise RuntimeError(f"{missing} pages short")
        self.free_pages = self.free_pages[taken:]
        self.lengths = [length + n for length, n in zip(self.lengths, new)]
        return y


def main():
    torch.manual_seed(0)
    device = ttnn.open_device(0)
    hidden, prompts, tokens = 4096, [700, 33, 512, 1, 260, 90, 411, 128], 64
    block = PagedAttention(device, hidden=hidden, heads=32, kv_heads=8, head_dim=128, users=len(prompts), pages=200, page_size=64, longest=1024, cache_dtype=ttnn.bfloat8_b)
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
    ttnn.close_device(device)


if __name__ == "__main__":
    main()
