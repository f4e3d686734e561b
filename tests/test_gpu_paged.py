"""The paged key/value cache on the GPU: page tables, writes and attention over it, against plain statements of them in 64 bits
(tests/paged_model.py, where the tolerance of attention is derived; tables and writes are exact)."""
import pytest
import torch

import paged_model

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


def as_list(tensor):
    return tensor._buf.cpu().tolist()


def activations(device, rows, layout):
    import ttnn

    return ttnn.from_torch(rows[None, None], dtype=ttnn.bfloat16, layout=getattr(ttnn, layout), device=device)


def fill_cache(cache, values):
    """values: [pages, kv_heads, page_size, head_dim] bf16 -> into the cache's buffer, as the codec packs them."""
    import ttnn
    from ttmi import capi

    values = values.cuda()
    if cache.dtype == ttnn.bfloat16:
        cache._buf.copy_(capi.tilize(values.bfloat16()))
    else:
        cache._buf.copy_(capi.pack_tensor(capi.BFLOAT8_B, values.float()))


def read_cache(cache):
    """[pages, kv_heads, page_size, head_dim] float32 on the CPU."""
    import ttnn

    return ttnn.to_torch(ttnn.from_device(cache)).float()


# ---- tables ---------------------------------------------------------------------------------------------------------------------------
TABLES = {
    "one request, one token": ([0], [1], 32, 2, 3),
    "decode": ([31, 32, 33, 64], [1, 1, 1, 1], 32, 4, 9),
    "some requests without tokens": ([0, 5, 0, 70, 0], [0, 0, 40, 0, 7], 32, 5, 9),
    "page size no power of two": ([95, 96, 97, 200], [1, 1, 300, 0], 96, 7, 20),
    "too few pages": ([10, 20, 30], [100, 100, 100], 32, 8, 5),
    "rows too short": ([10, 200, 0], [100, 5, 33], 32, 3, 50),
    "no requests": ([], [], 64, 4, 4),
    "no tokens": ([7, 0], [0, 0], 64, 4, 0),
    "negative lengths": ([-3, 40], [5, -2], 32, 4, 6),
    "many requests": ([(i * 37) % 150 for i in range(1000)], [(i * 13) % 5 for i in range(1000)], 32, 6, 700),
}


@pytest.mark.parametrize("name", TABLES)
@pytest.mark.parametrize("spare_tokens", [0, 13])
def test_tables(device, name, spare_tokens):
    import ttnn

    cached, new, page_size, width, free = TABLES[name]
    generator = torch.Generator().manual_seed(5)
    table = torch.randint(0, 10000, (len(cached), width), generator=generator)
    free = torch.randperm(free, generator=generator) + 20000
    tokens = sum(max(n, 0) for n in new) + spare_tokens
    out = ttnn.experimental.paged_tables(integers(device, cached), integers(device, new), integers(device, table.reshape(len(cached), width)), integers(device, free),
                                         page_size=page_size, num_tokens=tokens)
    want = paged_model.tables(cached, new, table.tolist(), free.tolist(), page_size, tokens)
    for got, expected in zip(out, want):
        assert as_list(got) == expected


def test_tables_with_fewer_rows_than_tokens(device):
    import ttnn

    cached, new = [3, 0, 9], [4, 6, 5]
    out = ttnn.experimental.paged_tables(integers(device, cached), integers(device, new), integers(device, [[1, 2]] * 3), integers(device, range(8)), page_size=32, num_tokens=7)
    want = paged_model.tables(cached, new, [[1, 2]] * 3, range(8), 32, 7)
    assert [as_list(t) for t in out] == list(want) and as_list(out[2]) == [0, 4, 7, 7]


def test_tables_may_overwrite_the_old_ones(device):
    from ttmi import capi

    cached, new = [40, 64, 0], [60, 1, 32]
    table, free = [[3, 4, 9, 9], [5, 6, 9, 9], [9, 9, 9, 9]], [10, 11, 12, 13, 14]
    at = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    c, n, t, f = at(cached), at(new), at(table), at(free)
    slots, starts, counts = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (93, 4, 2))
    p = lambda x: x.data_ptr()
    capi.check(capi.lib().ttmi_paged_tables(p(c), p(n), 3, 32, p(t), 4, p(f), 5, 93, p(t), p(slots), p(starts), p(counts), capi._stream()))
    assert [x.tolist() for x in (t, slots, starts, counts)] == list(paged_model.tables(cached, new, table, free, 32, 93))


# ---- writes ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("tokens,kv_heads,page_size,head_dim,extra", [(1, 1, 32, 32, 0), (5, 8, 64, 128, 64), (33, 2, 96, 96, 32), (70, 3, 32, 256, 0), (32, 1, 128, 64, 8)])
def test_write(oracle, device, layout, dtype, tokens, kv_heads, page_size, head_dim, extra):
    """Slots in any order, some tokens without one; what else lies in the pages stays, bit for bit."""
    import ttnn

    if extra % 32 and layout == "TILE_LAYOUT":
        pytest.skip("rows in TILE layout are whole tiles wide")
    torch.manual_seed(6)
    pages, wide = 5, kv_heads * head_dim
    caches = [ttnn.experimental.allocate_paged_cache(pages, kv_heads, page_size, head_dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)]
    before = [torch.randn(pages, kv_heads, page_size, head_dim).bfloat16() for _ in range(2)]
    for cache, values in zip(caches, before):
        fill_cache(cache, values)
    rows = torch.randn(tokens, 64 + 2 * wide + extra).bfloat16() * torch.exp2(torch.randint(-12, 12, (tokens, 64 + 2 * wide + extra)).float()).bfloat16()
    rows[tokens // 2, 64:64 + 16] = 0.0
    slots = torch.randperm(pages * page_size)[:tokens]
    if tokens > 4:
        slots[3], slots[4] = -1, pages * page_size                 # neither is a slot
    ttnn.experimental.write_paged_cache(activations(device, rows, layout), *caches, integers(device, slots), key_column=64 + wide, value_column=64)
    for cache, values, column in zip(caches, before, (64 + wide, 64)):
        want = values.float() if dtype == "bfloat16" else paged_model.bfloat8_b(oracle, values)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page_size:
                new = rows[t, column:column + wide].float().view(kv_heads, head_dim)
                if dtype == "bfloat8_b":
                    new = paged_model.bfloat8_b(oracle, new[:, None].expand(-1, 32, -1).contiguous())[:, 0]
                want[slot // page_size, :, slot % page_size] = new
        assert torch.equal(read_cache(cache), want)


# ---- attention ------------------------------------------------------------------------------------------------------------------------
def attention_case(oracle, device, *, cached, new, heads, kv_heads, head_dim, page_size, dtype="bfloat16", layout="TILE_LAYOUT", window=0, scale=None, query_column=0,
                   spare_rows=0, drop_pages=0, seed=7, spread=1.0, calls=1):
    """Random tables, values and rows; NaN and infinities (in BFLOAT8_B: the largest exponent) in every slot that no token of a request
    lies in; compares with the definition."""
    import ttnn

    generator = torch.Generator().manual_seed(seed)
    requests, width = len(cached), max([-(-(c + n) // page_size) for c, n in zip(cached, new)] + [1]) + 1
    pages = sum(-(-(c + n) // page_size) for c, n in zip(cached, new)) + 2
    order = torch.randperm(pages, generator=generator).tolist()
    table, owned = [], torch.zeros(pages, page_size, dtype=torch.bool)
    for c, n in zip(cached, new):
        row = [order.pop() for _ in range(-(-(c + n) // page_size))]
        for p in range(c + n):
            owned[row[p // page_size], p % page_size] = True
        table.append(row + [-1] * (width - len(row)))
    for i in range(drop_pages):                                    # requests with a hole, or a number that is no page
        r = i % requests
        held = -(-(cached[r] + new[r]) // page_size)
        if held:
            table[r][(i * 7) % held] = -1 if i % 2 else pages + i
    tokens = sum(new) + spare_rows
    starts = [sum(new[:r]) for r in range(requests + 1)]
    rows = (torch.randn(tokens, query_column + heads * head_dim, generator=generator) * spread).bfloat16()
    caches, values = [], []
    for _ in range(2):
        x = torch.randn(pages, kv_heads, page_size, head_dim, generator=generator).bfloat16()
        cache = ttnn.experimental.allocate_paged_cache(pages, kv_heads, page_size, head_dim, dtype=getattr(ttnn, dtype), device=device)
        bad = ~owned[:, None, :, None].expand_as(x)
        if dtype == "bfloat16":
            values.append(x.double())
            rubbish = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38]).bfloat16()[torch.randint(0, 4, x.shape, generator=generator)]
            fill_cache(cache, torch.where(bad, rubbish, x))
        else:
            values.append(paged_model.bfloat8_b(oracle, x).double())
            fill_cache(cache, torch.where(bad, torch.tensor(-3.3e38).bfloat16(), x))
        caches.append(cache)
    put = lambda v: integers(device, v)
    arguments = [activations(device, rows, layout), *caches, put(table), put(cached), put(starts)]
    for _ in range(calls):
        out = ttnn.experimental.attend_paged_cache(*arguments, num_heads=heads, query_column=query_column, scale=scale, window=window or None)
    assert tuple(out.shape) == (1, 1, tokens, heads * head_dim) and out.dtype == ttnn.bfloat16 and out.layout == getattr(ttnn, layout)
    if layout == "TILE_LAYOUT":                                    # the rows that fill up the last tiles are zeros
        whole = out._buf.cpu().view(-1, heads * head_dim // 32, 2, 2, 16, 16).permute(0, 2, 4, 1, 3, 5).reshape(-1, heads * head_dim)
        assert not whole[tokens:].any()
    got = ttnn.to_torch(ttnn.from_device(out))[0, 0].double()
    want, bound = paged_model.attention(rows, values[0], values[1], table, cached, starts, heads, head_dim, page_size, query_column, scale, window)
    off = (got - want).abs()
    assert not torch.isnan(got).any(), "NaN: " + str(torch.isnan(got).nonzero()[:4].tolist())
    assert (off <= bound).all(), f"{(off > bound).sum()} of {off.numel()} outside, worst {(off / bound).max():.2f} of the bound at {(off / bound).argmax().item()}"
    return out


SHAPES = [(1, 1, 64), (32, 8, 128), (71, 1, 64), (16, 16, 64), (12, 4, 96), (16, 2, 256), (6, 2, 128)]


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", SHAPES)
def test_decode(oracle, device, dtype, heads, kv_heads, head_dim):
    """One new token each; contexts that end at, before and behind the ends of tiles and pages."""
    attention_case(oracle, device, cached=[0, 1, 30, 31, 32, 63, 64, 127, 200], new=[1] * 9, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_size=64, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", SHAPES)
def test_chunks(oracle, device, dtype, heads, kv_heads, head_dim):
    """Requests with none, one, a few and many new tokens, from scratch and behind others."""
    attention_case(oracle, device, cached=[0, 65, 3, 90, 0], new=[40, 0, 1, 5, 97], heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_size=96, dtype=dtype, spare_rows=3)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("window", [1, 2, 31, 33, 64, 100])
def test_window(oracle, device, dtype, layout, window):
    attention_case(oracle, device, cached=[0, 7, 130, 500], new=[70, 1, 33, 1], heads=8, kv_heads=2, head_dim=64, page_size=32, dtype=dtype, layout=layout, window=window)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 1, 3, 65]])
def test_missing_pages_are_left_out(oracle, device, dtype, new):
    """Holes in a table, numbers that are no page, and a request of which nothing is left."""
    attention_case(oracle, device, cached=[100, 20, 300, 10], new=new, heads=8, kv_heads=2, head_dim=128, page_size=32, dtype=dtype, drop_pages=7)


@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("page_size", [32, 64, 96, 160, 256])
def test_layouts_and_page_sizes(oracle, device, layout, page_size):
    attention_case(oracle, device, cached=[10, 300, 159], new=[60, 1, 2], heads=8, kv_heads=4, head_dim=64, page_size=page_size, layout=layout, query_column=96, spare_rows=11, scale=0.3)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_long_contexts_are_cut_and_joined(oracle, device, dtype):
    """One user and few heads: the tokens go to many workgroups; twice, the second call finds the buffers that the first one left."""
    attention_case(oracle, device, cached=[6000, 3], new=[1, 1], heads=4, kv_heads=1, head_dim=64, page_size=64, dtype=dtype, calls=2)
    attention_case(oracle, device, cached=[3100], new=[34], heads=4, kv_heads=1, head_dim=128, page_size=128, dtype=dtype, calls=2)


def test_large_scores(oracle, device):
    """Scores of some hundreds: the running maximum moves, most weights vanish."""
    attention_case(oracle, device, cached=[400, 0], new=[1, 150], heads=4, kv_heads=2, head_dim=64, page_size=32, spread=30.0, seed=11)


def test_no_rows_and_no_requests(device):
    import ttnn

    cache = [ttnn.experimental.allocate_paged_cache(2, 2, 32, 64, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    out = ttnn.experimental.attend_paged_cache(activations(device, torch.randn(3, 256).bfloat16(), "ROW_MAJOR_LAYOUT"), *cache, integers(device, torch.zeros(0, 4)), integers(device, []),
                                               integers(device, [0]), num_heads=4)
    assert torch.equal(ttnn.to_torch(out.cpu()), torch.zeros(1, 1, 3, 256).bfloat16())
    out = ttnn.experimental.attend_paged_cache(activations(device, torch.randn(3, 256).bfloat16(), "TILE_LAYOUT"), *cache, integers(device, [[-1, -1], [-1, -1]]), integers(device, [5, 0]),
                                               integers(device, [0, 1, 2]), num_heads=4)
    assert torch.equal(out._buf.cpu(), torch.zeros(32 * 256).bfloat16())


def test_infinite_and_nan_values_that_count_come_out(device):
    """A NaN in a value that a row sees is the row's answer in that column, and no other's; a row before it does not see it."""
    import ttnn

    torch.manual_seed(3)
    keys, values = (torch.randn(2, 1, 32, 64).bfloat16() for _ in range(2))
    values[0, 0, 20, 5] = float("nan")
    caches = [ttnn.experimental.allocate_paged_cache(2, 1, 32, 64, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    for cache, x in zip(caches, (keys, values)):
        fill_cache(cache, x)
    rows = torch.randn(24, 64).bfloat16()
    out = ttnn.experimental.attend_paged_cache(activations(device, rows, "ROW_MAJOR_LAYOUT"), *caches, integers(device, [[0, 1]]), integers(device, [0]), integers(device, [0, 24]), num_heads=1)
    nan = torch.isnan(ttnn.to_torch(out.cpu())[0, 0])
    want = torch.zeros(24, 64, dtype=torch.bool)
    want[20:, 5] = True
    assert torch.equal(nan, want)


# ---- a step as it is used ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_steps_of_a_graph(device, dtype):
    """Tables, write and attention captured once and replayed on other lengths and rows, against the same calls made eagerly; work of
    other kinds and synchronisations in between."""
    import ttnn

    torch.manual_seed(9)
    heads, kv_heads, dim, page_size, requests, pages = 8, 2, 64, 32, 3, 24
    wide, tokens = (heads + 2 * kv_heads) * dim, 64
    caches = [[ttnn.experimental.allocate_paged_cache(pages, kv_heads, page_size, dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)] for _ in range(2)]
    for pair in caches:
        for cache in pair:
            fill_cache(cache, torch.zeros(pages, kv_heads, page_size, dim))
    rows = activations(device, torch.zeros(tokens, wide).bfloat16(), "TILE_LAYOUT")
    cached, new, table, free = integers(device, [0] * requests), integers(device, [0] * requests), integers(device, [[-1] * 8] * requests), integers(device, range(pages))

    def step(pair):
        t, slots, starts, counts = ttnn.experimental.paged_tables(cached, new, table, free, page_size=page_size, num_tokens=tokens)
        ttnn.experimental.write_paged_cache(rows, *pair, slots, key_column=heads * dim, value_column=(heads + kv_heads) * dim)
        return t, slots, ttnn.experimental.attend_paged_cache(rows, *pair, t, cached, starts, num_heads=heads)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(caches[1])                                            # buffers of the library for this stream
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = step(caches[1])
    for c, n in [([0, 0, 0], [20, 1, 33]), ([20, 1, 33], [1, 1, 1]), ([21, 2, 34], [30, 0, 34]), ([51, 2, 68], [1, 1, 0])]:
        cached._buf.copy_(torch.tensor(c, dtype=torch.int32))
        new._buf.copy_(torch.tensor(n, dtype=torch.int32))
        rows._buf.copy_(torch.randn(tokens * wide).bfloat16())
        eager = step(caches[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, captured):
            assert torch.equal(a._buf, b._buf)
        for a, b in zip(caches[0], caches[1]):
            assert torch.equal(a._buf, b._buf)
        assert not torch.isnan(eager[2]._buf.float()).any()
        held = torch.stack([(torch.tensor(c) + torch.tensor(n) + page_size - 1) // page_size]).max().item()
        assert held <= 8
        used = set(eager[0]._buf[eager[0]._buf >= 0].tolist())
        table._buf.copy_(eager[0]._buf)
        left = [p for p in range(pages) if p not in used]
        free._buf.copy_(torch.tensor(left + [-1] * (pages - len(left)), dtype=torch.int32))


def test_on_another_stream(oracle, device):
    """The calls run on torch's current stream, with buffers of that stream."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attention_case(oracle, device, cached=[700, 20], new=[1, 40], heads=8, kv_heads=2, head_dim=64, page_size=32)
    stream.synchronize()


def test_a_workspace_of_the_callers(device):
    """ttmi_paged_attention with a workspace of its own, which needs no initialisation, gives the bits of a call without one; one that
    is too small, or not aligned, is refused."""
    from ttmi import capi

    torch.manual_seed(10)
    L, heads, kv_heads, dim, page_size, pages, length = capi.lib(), 8, 2, 64, 64, 40, 2500
    rows = torch.randn(1, heads * dim, device="cuda").bfloat16()
    keys, values = (capi.tilize(torch.randn(pages, kv_heads, page_size, dim, device="cuda").bfloat16()) for _ in range(2))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, cached, starts = ints([list(range(pages))]), ints([length - 1]), ints([0, 1])
    out = [torch.empty(heads * dim, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    size = L.ttmi_paged_attention_workspace_bytes(1, 1, heads, capi.BFLOAT16, kv_heads, dim)
    memory = torch.full((max(size, 256) + 256,), 255, dtype=torch.uint8, device="cuda")
    base = (memory.data_ptr() + 255) // 256 * 256
    p = lambda t: t.data_ptr()

    def call(o, workspace, nbytes):
        return L.ttmi_paged_attention(p(rows), capi.ROW_MAJOR, 1, heads * dim, 0, p(keys), p(values), capi.BFLOAT16, pages, kv_heads, page_size, dim, p(table), 1, pages, p(cached), p(starts),
                                      heads, dim ** -0.5, 0, p(o), workspace, nbytes, capi._stream())

    capi.check(call(out[0], None, 0))
    capi.check(call(out[1], base, size))
    capi.check(call(out[2], base, size))
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
    if size:
        assert call(out[1], base, size - 1) == 1 and call(out[1], base + 16, size) == 1


# ---- refusals --------------------------------------------------------------------------------------------------------------------------
def test_refusals(device):
    import ttnn

    E = ttnn.experimental
    ints = lambda v: integers(device, v)
    cache = lambda *shape, dtype=ttnn.bfloat16: E.allocate_paged_cache(*shape, dtype=dtype, device=device)
    k, v = cache(3, 2, 32, 64), cache(3, 2, 32, 64)
    rows = activations(device, torch.zeros(4, 512).bfloat16(), "ROW_MAJOR_LAYOUT")
    slots, table, cached, starts = ints([0, 1, 2, 3]), ints([[0, 1]]), ints([0]), ints([0, 4])
    with pytest.raises(RuntimeError, match="multiples of 32"):
        cache(3, 2, 40, 64)
    with pytest.raises(RuntimeError, match="BFLOAT16 or BFLOAT8_B"):
        cache(3, 2, 32, 64, dtype=ttnn.bfloat4_b)
    with pytest.raises(RuntimeError, match="at least 1"):
        cache(0, 2, 32, 64)
    with pytest.raises(RuntimeError, match="same requests"):
        E.paged_tables(ints([1, 2]), ints([1]), ints([[0], [0]]), ints([1]), page_size=32, num_tokens=1)
    with pytest.raises(RuntimeError, match="page size"):
        E.paged_tables(ints([1]), ints([1]), ints([[0]]), ints([1]), page_size=48, num_tokens=1)
    with pytest.raises(RuntimeError, match=r"\[requests, pages\]"):
        E.paged_tables(ints([1]), ints([1]), ints([[0], [0]]), ints([1]), page_size=32, num_tokens=1)
    with pytest.raises(RuntimeError, match="UINT32"):
        E.paged_tables(activations(device, torch.zeros(1, 32).bfloat16(), "ROW_MAJOR_LAYOUT"), ints([1]), ints([[0]]), ints([1]), page_size=32, num_tokens=1)
    with pytest.raises(RuntimeError, match="at most 4096"):
        E.paged_tables(ints([0] * 4097), ints([0] * 4097), ints([[0]] * 4097), ints([1]), page_size=32, num_tokens=1)
    with pytest.raises(RuntimeError, match="3 slots for 4 tokens"):
        E.write_paged_cache(rows, k, v, ints([0, 1, 2]), key_column=0, value_column=128)
    with pytest.raises(RuntimeError, match="same memory"):
        E.write_paged_cache(rows, k, k, slots, key_column=0, value_column=128)
    with pytest.raises(RuntimeError, match="outside rows"):
        E.write_paged_cache(rows, k, v, slots, key_column=0, value_column=416)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        E.write_paged_cache(rows, k, v, slots, key_column=16, value_column=128)
    with pytest.raises(RuntimeError, match="same shape, dtype and layout"):
        E.write_paged_cache(rows, k, cache(4, 2, 32, 64), slots, key_column=0, value_column=128)
    with pytest.raises(RuntimeError, match="must be BFLOAT16"):
        E.write_paged_cache(ttnn.from_torch(torch.zeros(1, 1, 4, 512), device=device), k, v, slots, key_column=0, value_column=128)
    attend = lambda **kw: E.attend_paged_cache(rows, k, v, table, cached, starts, **{"num_heads": 4, **kw})
    with pytest.raises(RuntimeError, match="no multiple of 2 key heads"):
        attend(num_heads=3)
    with pytest.raises(RuntimeError, match="do not fit"):
        attend(num_heads=16)
    with pytest.raises(RuntimeError, match="outside rows"):
        attend(num_heads=8, query_column=32)
    with pytest.raises(RuntimeError, match="scale must be finite"):
        attend(scale=float("inf"))
    with pytest.raises(RuntimeError, match="window must be"):
        attend(window=0)
    with pytest.raises(RuntimeError, match="one element more"):
        E.attend_paged_cache(rows, k, v, table, cached, ints([0, 4, 4]), num_heads=4)
    with pytest.raises(RuntimeError, match="head dimension 32"):
        E.attend_paged_cache(rows, cache(3, 2, 32, 32), cache(3, 2, 32, 32), table, cached, starts, num_heads=4)
    with pytest.raises(RuntimeError, match="without padding"):
        flat = ttnn.from_torch(torch.zeros(3, 2, 20, 64).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device)
        E.attend_paged_cache(rows, flat, flat, table, cached, starts, num_heads=4)
    with pytest.raises(RuntimeError, match="needs to be on device"):
        E.attend_paged_cache(ttnn.from_device(rows), k, v, table, cached, starts, num_heads=4)
    with pytest.raises(RuntimeError, match="must be a ttnn.Tensor"):
        E.attend_paged_cache(rows, k, v, [[0, 1]], cached, starts, num_heads=4)
