"""Attention over a paged cache with a window and sinks on the GPU, against a plain statement of it in 64 bits (tests/paged_more_model.py, where the
tolerance is derived)."""
import pytest
import torch

import paged_model
import paged_more_model as model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def device():
    import ttnn

    dev = ttnn.open_device(0)
    yield dev
    ttnn.close_device(dev)


def integers(device, values):
    import ttnn

    return ttnn.from_torch(torch.as_tensor(values, dtype=torch.int32), device=device)


def needed(cached, new, window, sinks):
    """Tokens that some row of a request sees."""
    reach = range(cached + new)
    return [j for j in reach if j < sinks or j > cached - window] if new else []


def sinks_case(oracle, device, *, cached, new, heads, kv_heads, head_dim, page_size, window, sinks, dtype="bfloat16", layout="TILE_LAYOUT", spare=0, scale=None, seed=3, spread=2.0, calls=1, odd=None):
    """Pages that hold nothing that is seen are not in the table; everything that is not seen is rubbish: NaN and infinities where the cache can hold them."""
    import ttnn
    from ttmi import capi

    g = torch.Generator().manual_seed(seed)
    E, requests = ttnn.experimental, len(cached)
    width = max([-(-(c + n) // page_size) for c, n in zip(cached, new)] + [1]) + 1
    seen_pages = [sorted({j // page_size for j in needed(c, n, window, sinks)}) for c, n in zip(cached, new)]
    pages = sum(map(len, seen_pages)) + 2
    order = torch.randperm(pages, generator=g).tolist()
    table, seen = [[-1] * width for _ in cached], torch.zeros(pages, page_size, dtype=torch.bool)
    for r, (c, n) in enumerate(zip(cached, new)):
        for j in seen_pages[r]:
            table[r][j] = order.pop()
        for j in needed(c, n, window, sinks):
            seen[table[r][j // page_size], j % page_size] = True
    tokens, starts = sum(new) + spare, [sum(new[:r]) for r in range(requests + 1)]
    rows = (torch.randn(tokens, heads * head_dim, generator=g) * spread).bfloat16()
    caches, values = [], []
    for which in range(2):
        x = torch.randn(pages, kv_heads, page_size, head_dim, generator=g).bfloat16()
        if odd is not None and which == 1:
            odd(x, table)
        cache = E.allocate_paged_cache(pages, kv_heads, page_size, head_dim, dtype=getattr(ttnn, dtype), device=device)
        bad = ~seen[:, None, :, None].expand_as(x)
        if dtype == "bfloat16":
            values.append(x.double())
            rubbish = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38]).bfloat16()[torch.randint(0, 4, x.shape, generator=g)]
            cache._buf.copy_(capi.tilize(torch.where(bad, rubbish, x).cuda()))
        else:
            values.append(paged_model.bfloat8_b(oracle, x).double())
            cache._buf.copy_(capi.pack_tensor(capi.BFLOAT8_B, torch.where(bad, torch.tensor(-3.3e38).bfloat16(), x).float().cuda()))
        caches.append(cache)
    given = ttnn.from_torch(rows[None, None], dtype=ttnn.bfloat16, layout=getattr(ttnn, layout), device=device)
    arguments = [given, *caches, integers(device, table), integers(device, cached), integers(device, starts)]
    for _ in range(calls):
        out = E.attend_paged_cache(*arguments, num_heads=heads, scale=scale, window=window, sinks=sinks)
    got = ttnn.to_torch(ttnn.from_device(out))[0, 0].double()
    want, bound = model.attention(rows, values[0], values[1], table, cached, starts, heads, head_dim, page_size, 0, scale, window, sinks)
    if odd is not None:
        return got, want, bound
    assert not torch.isnan(got).any(), "NaN: " + str(torch.isnan(got).nonzero()[:4].tolist())
    off = (got - want).abs()
    assert (off <= bound).all(), f"{(off > bound).sum()} of {off.numel()} outside, worst {(off / bound).max():.2f} of the bound at {(off / bound).argmax().item()}"


SHAPES = [(1, 1, 64), (8, 2, 128), (71, 1, 64), (16, 16, 64), (12, 4, 96), (16, 2, 256), (34, 2, 128), (80, 1, 64)]
LENGTHS = {"decode": ([0, 1, 31, 32, 63, 64, 200, 517], [1] * 8), "drafts": ([0, 90, 400, 33], [5, 3, 4, 0]), "chunks": ([0, 65, 3, 390, 0], [40, 0, 1, 55, 97]), "a prompt": ([0], [330])}


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", SHAPES)
@pytest.mark.parametrize("step", LENGTHS)
def test_steps(oracle, device, dtype, heads, kv_heads, head_dim, step):
    """Every kernel: few and many rows, one and several row tiles, all head sizes; a gap that is none, small and large."""
    cached, new = LENGTHS[step]
    for window, sinks in [(40, 4), (100, 33)]:
        sinks_case(oracle, device, cached=cached, new=new, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_size=32, window=window, sinks=sinks, dtype=dtype, spare=2)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [70, 1, 33, 1], [300, 257, 0, 280]])
@pytest.mark.parametrize("sinks", [0, 1, 31, 32, 33, 64, 65, 96, 200, 2 ** 31 - 1])
def test_sinks_at_the_ends_of_blocks(oracle, device, dtype, new, sinks):
    """Sinks that end in, at and behind a block and a step, that reach into the window and past the tokens; windows of one and more tokens."""
    for window in [1, 31, 32, 33, 150]:
        sinks_case(oracle, device, cached=[0, 7, 130, 500], new=new, heads=4, kv_heads=2, head_dim=64, page_size=64, dtype=dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("page_size", [32, 96, 160, 256])
def test_layouts_and_page_sizes(oracle, device, layout, page_size):
    sinks_case(oracle, device, cached=[10, 700, 159], new=[60, 1, 2], heads=8, kv_heads=4, head_dim=64, page_size=page_size, layout=layout, spare=5, scale=-0.3, window=64, sinks=37)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_long_contexts_are_cut_and_joined(oracle, device, dtype):
    """The tokens of one request go to many workgroups, pieces with sinks, with window and with both among them; twice, the second call finds the buffers of the first."""
    sinks_case(oracle, device, cached=[9000, 3], new=[1, 1], heads=4, kv_heads=1, head_dim=64, page_size=64, dtype=dtype, calls=2, window=2500, sinks=700)
    sinks_case(oracle, device, cached=[6100], new=[40], heads=4, kv_heads=1, head_dim=128, page_size=128, dtype=dtype, calls=2, window=1500, sinks=500)
    sinks_case(oracle, device, cached=[6100], new=[290], heads=2, kv_heads=1, head_dim=64, page_size=128, dtype=dtype, calls=2, window=1500, sinks=50)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("head_dim,page_size", [(64, 64), (256, 32)])
def test_more_pieces_than_workgroups(oracle, device, dtype, head_dim, page_size):
    """Whole prompts: workgroups ask for further pieces, the second call finds the counter as the first one found it."""
    kv_heads = 8 if head_dim == 64 else 4
    sinks_case(oracle, device, cached=[0, 500], new=[1290, 1270], heads=4 * kv_heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, dtype=dtype, calls=2, window=60, sinks=20)


@pytest.mark.parametrize("new", [1, 200])
def test_sinks_without_a_window_or_within_it(device, new):
    """All tokens are seen: bit for bit the attention without a window; and without sinks, that with the window alone."""
    import ttnn
    from ttmi import capi

    torch.manual_seed(5)
    E, pages = ttnn.experimental, 12
    caches = [E.allocate_paged_cache(pages, 2, 64, 128, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    for cache in caches:
        cache._buf.copy_(capi.tilize(torch.randn(pages, 2, 64, 128).cuda().bfloat16()))
    rows = ttnn.from_torch(torch.randn(1, 1, new, 8 * 128).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device)
    step = lambda **kw: E.attend_paged_cache(rows, *caches, integers(device, [list(range(pages))]), integers(device, [500]), integers(device, [0, new]), num_heads=8, **kw)._buf
    assert torch.equal(step(sinks=50), step()) and torch.equal(step(window=100, sinks=0), step(window=100))


@pytest.mark.parametrize("new", [3, 120])
def test_sinks_without_a_page(oracle, device, new):
    """The page of the sinks is gone: what is left is the window; a request of which nothing is left is zeros."""
    import ttnn
    from ttmi import capi

    torch.manual_seed(6)
    E, pages, dim = ttnn.experimental, 16, 64
    keys, values = torch.randn(pages, 1, 32, dim).bfloat16(), torch.randn(pages, 1, 32, dim).bfloat16()
    caches = [E.allocate_paged_cache(pages, 1, 32, dim, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    for cache, x in zip(caches, (keys, values)):
        cache._buf.copy_(capi.tilize(x.cuda()))
    table = [[-1] + list(range(1, 16)), [99] * 16]
    rows = torch.randn(2 * new, 4 * dim).bfloat16()
    given = ttnn.from_torch(rows[None, None], layout=ttnn.ROW_MAJOR_LAYOUT, device=device)
    out = E.attend_paged_cache(given, *caches, integers(device, table), integers(device, [300, 300]), integers(device, [0, new, 2 * new]), num_heads=4, window=50, sinks=8)
    got = ttnn.to_torch(out.cpu())[0, 0].double()
    want, bound = model.attention(rows, keys.double(), values.double(), table, [300, 300], [0, new, 2 * new], 4, dim, 32, window=50, sinks=8)
    assert ((got - want).abs() <= bound).all() and not got[new:].any()


@pytest.mark.parametrize("new", [[1, 1], [150, 1]])
def test_infinite_and_nan_values_that_count_come_out(oracle, device, new):
    """A NaN and infinities among the sinks, and one in the window: the answers of the rows that see them in those columns, and no others."""
    def odd(x, table):
        x[table[0][0], 0, 2, 5] = float("nan")
        x[table[0][0], 0, 3, 6] = float("inf")
        x[table[0][0], 0, 3, 7] = -float("inf")

    got, want, bound = sinks_case(oracle, device, cached=[300, 10], new=new, heads=2, kv_heads=1, head_dim=64, page_size=32, window=40, sinks=5, odd=odd)
    rows = slice(0, new[0])
    for head in (0, 64):
        assert torch.isnan(got[rows, head + 5]).all() and (got[rows, head + 6] == float("inf")).all() and (got[rows, head + 7] == -float("inf")).all()
    rest = torch.ones_like(got, dtype=torch.bool)
    for head in (0, 64):
        rest[rows, head + 5:head + 8] = False
    assert ((got - want).abs() <= bound)[rest].all()


def test_far_positions(device):
    """More tokens from before than the table names, positions at 2^31: the sinks are seen, the window lies behind the table."""
    from ttmi import capi

    torch.manual_seed(7)
    keys, values = (torch.randn(3, 2, 32, 64).bfloat16() for _ in range(2))
    for tokens in (4, 150):
        rows = torch.randn(tokens, 256).bfloat16()
        out = torch.empty(tokens, 256, dtype=torch.bfloat16, device="cuda")
        put = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        held = [capi.tilize(keys.cuda()), capi.tilize(values.cuda()), rows.cuda(), put([[2, 0, 1]]), put([2 ** 31 - 3]), put([0, tokens])]
        k, v, r, table, cached, starts = (x.data_ptr() for x in held)
        capi.check(capi.lib().ttmi_paged_attention_sinks(r, 0, tokens, 256, 0, k, v, capi.BFLOAT16, 3, 2, 32, 64, table, 1, 3, cached, starts, 4, 0.125, 1000, 40, out.data_ptr(), None, 0, capi._stream()))
        want, bound = model.attention(rows, keys.double(), values.double(), [[2, 0, 1]], [2 ** 31 - 3], [0, tokens], 4, 64, 32, window=1000, sinks=40)
        assert ((out.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_graphs_side_by_side(device, dtype):
    """A step of single tokens and a chunk, captured on one stream, replayed at once on two others on other lengths: the bits of the eager calls."""
    import ttnn
    from ttmi import capi

    torch.manual_seed(8)
    E, heads, kv_heads, dim, pages = ttnn.experimental, 8, 2, 128, 64
    caches = [E.allocate_paged_cache(pages, kv_heads, 64, dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)]
    for cache in caches:
        x = torch.randn(pages, kv_heads, 64, dim, device="cuda")
        cache._buf.copy_(capi.tilize(x.bfloat16()) if dtype == "bfloat16" else capi.pack_tensor(capi.BFLOAT8_B, x))
    table = integers(device, [list(range(pages))])
    rows = [ttnn.from_torch(torch.randn(1, 1, n, heads * dim).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device) for n in (1, 200)]
    cached, starts = [integers(device, [3000]), integers(device, [3500])], [integers(device, [0, 1]), integers(device, [0, 200])]
    step = lambda i: E.attend_paged_cache(rows[i], *caches, table, cached[i], starts[i], num_heads=heads, window=900, sinks=70)
    stream, streams, graphs, outs = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    torch.cuda.synchronize()
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=stream):
            outs.append(step(i))
    for lengths in [(3000, 3500), (700, 1800), (3999, 40)]:
        for c, n in zip(cached, lengths):
            c._buf.fill_(n)
        want = [step(i)._buf.clone() for i in range(2)]
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i]._buf, want[i])


def test_the_host_layer_refuses(device):
    import ttnn

    E = ttnn.experimental
    caches = [E.allocate_paged_cache(2, 2, 32, 64, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    rows = ttnn.from_torch(torch.randn(1, 1, 4, 256).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device)
    for bad in [-1, 1.5, 2 ** 31]:
        with pytest.raises(RuntimeError, match="sinks"):
            E.attend_paged_cache(rows, *caches, integers(device, [[0, 1]]), integers(device, [0]), integers(device, [0, 4]), num_heads=4, window=8, sinks=bad)
