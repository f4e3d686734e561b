"""The attention block of examples/paged_decoder.py, as a server runs it, against the same block computed in one go in 64 bits.

Tolerance, in the norm of a token's row: four roundings to bf16 lie between the two (the projection, the weights of the softmax, the
context, the result), each at most 2^-8 of what it rounds, and 2^-6 is their sum; with the block floats of the cache one more on
either side of the softmax, 2^-7 each of a value's 16 neighbours, hence 2^-5."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decoder.py")
    spec = importlib.util.spec_from_file_location("paged_decoder", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("cache,tolerance", [("bfloat16", 2.0 ** -6), ("bfloat8_b", 2.0 ** -5)])
@pytest.mark.parametrize("window", [None, 40])
def test_the_block_of_a_decoder_layer(example, cache, tolerance, window):
    import ttnn

    torch.manual_seed(4)
    device = ttnn.open_device(0)
    hidden, heads, kv_heads, dim = 256, 4, 2, 64
    block = example.PagedAttention(device, hidden=hidden, heads=heads, kv_heads=kv_heads, head_dim=dim, users=3, pages=20, page_size=32, longest=200, cache_dtype=getattr(ttnn, cache), window=window)
    # prompts (one in two chunks), single tokens, one that comes later, tokens that are checked several at once
    steps = [[70, 33, 0], [25, 1, 0], [1, 1, 0], [1, 1, 100], [3, 1, 1], [1, 4, 1]]
    total = [sum(s[u] for s in steps) for u in range(3)]
    x = [torch.randn(n, hidden).bfloat16() for n in total]
    got, at = [[] for _ in total], [0, 0, 0]
    for new in steps:
        rows = torch.cat([x[u][at[u]:at[u] + n] for u, n in enumerate(new)])
        y = ttnn.to_torch(block.step(ttnn.from_torch(rows[None, None], layout=ttnn.TILE_LAYOUT, device=device), new).cpu())[0, 0].double()
        for u, n in enumerate(new):
            got[u].append(y[:n])
            y, at[u] = y[n:], at[u] + n
    assert block.lengths == total and len(block.free_pages) == 20 - sum(-(-n // 32) for n in total)
    w_qkv, w_o = (ttnn.to_torch(w.cpu())[0, 0].double() for w in (block.w_qkv, block.w_o))
    for u, n in enumerate(total):
        qkv = (x[u].double() @ w_qkv).view(n, heads + 2 * kv_heads, dim).transpose(0, 1)
        q, k, v = qkv[:heads], qkv[heads:heads + kv_heads].repeat_interleave(heads // kv_heads, 0), qkv[heads + kv_heads:].repeat_interleave(heads // kv_heads, 0)
        i, j = torch.arange(n)[:, None], torch.arange(n)
        hidden_from = (j > i) | (j <= i - (window or n))
        want = (torch.softmax((q @ k.transpose(1, 2) * dim ** -0.5).masked_fill(hidden_from, float("-inf")), -1) @ v).transpose(0, 1).reshape(n, heads * dim) @ w_o
        off = (torch.cat(got[u]) - want).norm(dim=1) / want.norm(dim=1)
        assert (off <= tolerance).all(), f"user {u}: {off.max():.4f} at token {off.argmax().item()}"
    ttnn.close_device(device)


def test_too_few_pages_are_noticed(example):
    import ttnn

    device = ttnn.open_device(0)
    block = example.PagedAttention(device, hidden=256, heads=4, kv_heads=2, head_dim=64, users=2, pages=3, page_size=32, longest=200, cache_dtype=ttnn.bfloat16)
    x = ttnn.from_torch(torch.randn(1, 1, 130, 256).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device)
    with pytest.raises(RuntimeError, match="3 pages short"):
        block.step(x, [65, 65])                                    # three pages each, three in all
    ttnn.close_device(device)
