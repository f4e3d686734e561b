"""The attention block of examples/paged_decoder.py with positions, norms, a window with sinks, forks and pages that come back, as a server runs it, against the same
block computed in one go in 64 bits.

Tolerance, in the norm of a token's row: six roundings to bf16 lie between the two (the projection, the rotated queries and keys, the weights of the
softmax, the context, the result), each at most 2^-8 of what it rounds: 2^-5.4, hence 2^-5.  With the block floats of the cache one more on either side
of the softmax, 2^-7 each of a value's 16 neighbours: 2^-4.6, hence 2^-4."""
import importlib.util
import os

import pytest
import torch

import paged_more_model as model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decoder.py")
    spec = importlib.util.spec_from_file_location("paged_decoder", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("cache,tolerance", [("bfloat16", 2.0 ** -5), ("bfloat8_b", 2.0 ** -4)])
@pytest.mark.parametrize("window,sinks,norms,interleaved,rotary_dim", [(None, 0, False, False, 64), (40, 5, True, False, 64), (33, 0, False, True, 32), (64, 40, True, True, 48)])
def test_the_block_of_a_decoder_layer(example, cache, tolerance, window, sinks, norms, interleaved, rotary_dim):
    import ttnn

    torch.manual_seed(4)
    device = ttnn.open_device(0)
    hidden, heads, kv_heads, dim, users, pages = 256, 4, 2, 64, 4, 24
    weights = [1 + 0.2 * torch.randn(dim) if norms else None for _ in range(2)]
    block = example.PagedAttention(device, hidden=hidden, heads=heads, kv_heads=kv_heads, head_dim=dim, users=users, pages=pages, page_size=32, longest=220, cache_dtype=getattr(ttnn, cache), window=window,
                                   sinks=sinks, rotary_dim=rotary_dim, interleaved=interleaved, norms=weights)
    x, got = [torch.zeros(0, hidden).bfloat16()] * users, [torch.zeros(0, hidden, dtype=torch.float64)] * users
    # prompts, single tokens, forks of two of them and one from scratch, drafts, forks again; pages come back every now and then
    for step in [[70, 33, 0, 5], [25, 1, 0, 0], "release", [1, 1, 1, 1], ("fork", [0, 1, 0, 0]), [1, 1, 1, 1], [3, 1, 2, 4], "release", [1, 40, 1, 1], ("fork", [1, 1, -1, 3]), "release",
                 [1, 1, 1, 1], [20, 2, 3, 1], "release", [1, 1, 1, 1]]:
        if step == "release":
            block.release()
            needed = {page for row in block.page_table._buf.tolist() for page in row if page >= 0}
            assert sorted(block.free_pages) == [page for page in range(pages) if page not in needed]
            if window and not sinks:                               # a request holds what its window reaches and no more
                assert all(sum(page >= 0 for page in row) <= window // 32 + 2 for row in block.page_table._buf.tolist())
            continue
        if step[0] == "fork":
            block.fork(step[1])
            x, got = ([side[u] if u >= 0 else side[0][:0] for u in step[1]] for side in (x, got))
            assert block.lengths == [len(rows) for rows in x]
            continue
        rows = [torch.randn(n, hidden).bfloat16() for n in step]
        y = ttnn.to_torch(block.step(ttnn.from_torch(torch.cat(rows)[None, None], layout=ttnn.TILE_LAYOUT, device=device), step).cpu())[0, 0].double()
        for u, n in enumerate(step):
            x[u], got[u], y = torch.cat([x[u], rows[u]]), torch.cat([got[u], y[:n]]), y[n:]
    w_qkv, w_o = (ttnn.to_torch(w.cpu())[0, 0].double() for w in (block.w_qkv, block.w_o))
    frequencies = (10000.0 ** (-torch.arange(rotary_dim // 2, dtype=torch.float64) / (rotary_dim // 2))).float()
    for u in range(users):
        n = len(x[u])
        qkv = x[u].double() @ w_qkv
        turned = [model.rotate(part, [(0, p) for p in range(n)], h, dim, frequencies, interleaved, w, 1e-6)[0].transpose(0, 1)
                  for part, h, w in ((qkv[:, :heads * dim], heads, weights[0]), (qkv[:, heads * dim:(heads + kv_heads) * dim], kv_heads, weights[1]))]
        v = qkv[:, (heads + kv_heads) * dim:].view(n, kv_heads, dim).transpose(0, 1).repeat_interleave(heads // kv_heads, 0)
        q, k = turned[0], turned[1].repeat_interleave(heads // kv_heads, 0)
        i, j = torch.arange(n)[:, None], torch.arange(n)
        unseen = (j > i) | ((j <= i - (window or n)) & (j >= sinks))
        want = (torch.softmax((q @ k.transpose(1, 2) * dim ** -0.5).masked_fill(unseen, float("-inf")), -1) @ v).transpose(0, 1).reshape(n, heads * dim) @ w_o
        off = (got[u] - want).norm(dim=1) / want.norm(dim=1)
        assert (off <= tolerance).all(), f"user {u}: {off.max():.4f} at token {off.argmax().item()} of {n}"
    ttnn.close_device(device)


def test_forks_without_pages_are_noticed(example):
    import ttnn

    device = ttnn.open_device(0)
    block = example.PagedAttention(device, hidden=256, heads=4, kv_heads=2, head_dim=64, users=2, pages=3, page_size=32, longest=200, cache_dtype=ttnn.bfloat16, rotary_dim=64)
    block.step(ttnn.from_torch(torch.randn(1, 1, 70, 256).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device), [70, 0])
    with pytest.raises(RuntimeError, match="1 pages short"):
        block.fork([0, 0])
    ttnn.close_device(device)


def test_the_example_runs(example, capsys):
    example.main()
    assert "eight answers" in capsys.readouterr().out
