"""Pages of a cache that are shared, copied and given back, on the GPU: integers and bytes, exactly those of the plain statements in tests/paged_more_model.py."""
import ctypes

import pytest
import torch

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


def as_list(tensor):
    return tensor._buf.cpu().tolist()


# ---- forks ------------------------------------------------------------------------------------------------------------------------------
FORKS = {
    "one to four": ([700], [0, 0, 0, 0], 64, 12, 9),
    "whole pages have nothing to copy": ([64, 128], [0, 0, 1, 1, 1], 64, 3, 5),
    "a beam step": ([33, 70, 1, 95], [2, 2, 0, 2], 32, 4, 10),
    "empty, negative, unknown": ([0, -5, 40], [0, 1, 2, 2, -1, 3, 2 ** 30, 0], 32, 3, 4),
    "too few pages": ([10, 20, 30], [0, 0, 0, 1, 1, 2, 2, 2], 32, 2, 3),
    "no free pages": ([10], [0, 0], 32, 1, 0),
    "lengths past the row": ([1000, 95], [0, 0, 1, 1], 32, 3, 5),
    "no continuations": ([10, 20], [], 32, 2, 3),
    "no requests": ([], [0, -1], 32, 2, 3),
    "many": ([(i * 37) % 200 for i in range(1000)], [(i * i * 7) % 1000 for i in range(4096)], 32, 8, 3000),
    "as many as there may be": ([i % 100 + 1 for i in range(4096)], [4095 - i // 2 for i in range(4096)], 32, 4, 5000),
}


@pytest.mark.parametrize("name", FORKS)
def test_forks(device, name):
    import ttnn

    lengths, parents, page_size, width, free = FORKS[name]
    g = torch.Generator().manual_seed(4)
    table = torch.randint(0, 100000, (len(lengths), width), generator=g)
    free = torch.randperm(max(free, 1), generator=g)[:free] + 200000
    out = ttnn.experimental.fork_paged_tables(integers(device, table.view(len(lengths), width)), integers(device, lengths), integers(device, parents), integers(device, free), page_size=page_size)
    rows, *rest = model.fork(table.tolist(), lengths, parents, free.tolist(), page_size)
    if not lengths:
        rows = [[-1] * width for _ in parents]
    assert as_list(out[0]) == rows and [as_list(t) for t in out[1:]] == rest
    assert tuple(out[0].shape) == (len(parents), width)


def test_forks_of_rows_with_holes(device):
    """A begun page that is not there is nothing to copy; a number in the list that is no page is handed on, and not copied into."""
    import ttnn

    table, lengths, parents, free = [[5, -1, 7], [8, 9, -1]], [40, 45], [0, 0, 1, 1, 1], [-1, 3]
    out = ttnn.experimental.fork_paged_tables(integers(device, table), integers(device, lengths), integers(device, parents), integers(device, free), page_size=32)
    rows, *rest = model.fork(table, lengths, parents, free, 32)
    assert as_list(out[0]) == rows and [as_list(t) for t in out[1:]] == rest


# ---- copies -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("count,pages,kv_heads,page_size,head_dim,pairs", [(1, 2, 1, 32, 32, 1), (2, 9, 2, 64, 64, 4), (3, 20, 8, 96, 128, 9), (2, 7, 3, 32, 96, 3), (130, 6, 1, 32, 64, 3), (2, 5, 16, 256, 128, 2)])
def test_copies(device, dtype, count, pages, kv_heads, page_size, head_dim, pairs):
    """Every byte of the targets, in every cache; pairs with a number that is no page are left out, all other pages stay."""
    import ttnn

    torch.manual_seed(5)
    E = ttnn.experimental
    caches = [E.allocate_paged_cache(pages, kv_heads, page_size, head_dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(count)]
    for c in caches:
        c._buf.view(torch.uint8).copy_(torch.randint(0, 256, (c._buf.view(torch.uint8).numel(),), dtype=torch.uint8))
    before = [c._buf.cpu().view(torch.uint8).view(pages, -1) for c in caches]
    order = torch.randperm(pages).tolist()
    targets, sources = order[:pairs], [order[pairs + i % (pages - pairs)] for i in range(pairs)]
    none = [(-1, order[-1]), (order[-1], -1), (pages, order[-1]), (order[-1], pages), (-2 ** 31, 2 ** 31 - 1), (order[-1], order[-1])]
    given = list(zip(sources, targets))
    given = none[:3] + given[:1] + none[3:] + given[1:]
    E.copy_paged_pages(caches, integers(device, [s for s, _ in given]), integers(device, [t for _, t in given]))
    for c, b in zip(caches, before):
        want = b.clone()
        for s, t in zip(sources, targets):
            want[t] = b[s]
        assert torch.equal(c._buf.cpu().view(torch.uint8).view(pages, -1), want)


def test_copies_past_4_gib(device):
    """Pages whose bytes lie beyond what 32 bits count."""
    import ttnn

    E, pages = ttnn.experimental, 4400
    cache = E.allocate_paged_cache(pages, 8, 128, 512, dtype=ttnn.bfloat16, device=device)     # 1 MiB a page
    whole = cache._buf.view(pages, -1)
    whole.zero_()
    whole[4399], whole[7] = 3.0, 5.0
    E.copy_paged_pages([cache], integers(device, [4399, 7]), integers(device, [303, 4398]))
    assert (whole[303] == 3).all() and (whole[4398] == 5).all() and not whole[302].any() and not whole[304].any() and not whole[4397].any()


# ---- releases -----------------------------------------------------------------------------------------------------------------------------
def release_case(device, table, lengths, page_size, pages, window=0, sinks=0):
    import ttnn

    width = len(table[0]) if table else 3
    out = ttnn.experimental.release_paged_pages(integers(device, torch.tensor(table, dtype=torch.int32).view(len(table), width)), integers(device, lengths), page_size=page_size, num_pages=pages,
                                                window=window or None, sinks=sinks)
    rows, free, counts = model.release(table, lengths, page_size, pages, window, sinks)
    assert as_list(out[2]) == counts and as_list(out[1]) == free and as_list(out[0]) == rows


@pytest.mark.parametrize("pages", [1, 31, 32, 33, 64, 1000, 2047, 2048, 2049, 100000])
def test_releases(device, pages):
    """Pools that end in and at a word and a workgroup's share; pages in several rows, numbers that are none, rows that are over."""
    g = torch.Generator().manual_seed(pages)
    table = torch.randint(-2, pages + 2, (7, 9), generator=g).tolist()
    release_case(device, table, [0, 1, 32, 33, 288, 1000, -4], 32, pages)


@pytest.mark.parametrize("window", [1, 31, 32, 33, 64, 100, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 1, 32, 33, 100])
def test_windows(device, window, sinks):
    lengths = [0, 1, 31, 32, 33, 63, 64, 65, 95, 96, 97, 130, 500]
    table = torch.arange(13 * 6).view(13, 6).tolist()
    release_case(device, table, lengths, 32, 90, window, sinks)
    release_case(device, table, [3 * n for n in lengths], 96, 90, window, sinks)


@pytest.mark.parametrize("requests,width,pages", [(1, 5000, 9000), (900, 70, 70000), (4096, 20, 300000), (5000, 3, 20000), (256, 64, 65536), (255, 64, 65535), (256, 64, 65537), (257, 64, 60000), (1024, 16, 3000), (4096, 4, 65536)])
def test_large_tables(device, requests, width, pages):
    g = torch.Generator().manual_seed(3)
    table = torch.randint(0, pages, (requests, width), generator=g)
    lengths = torch.randint(0, width * 32, (requests,), generator=g)
    release_case(device, table.tolist(), lengths.tolist(), 32, pages, 300, 40)


def test_no_requests_and_a_pool_without_tables(device):
    release_case(device, [], [], 32, 70)


def test_releases_may_overwrite_the_table(device):
    from ttmi import capi

    table, lengths = [[3, 1, 2], [0, 4, 9]], [70, 33]
    at = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    t, n, free, counts = at(table), at(lengths), at([7] * 6), at([7] * 3)
    size = capi.lib().ttmi_paged_release_workspace_bytes(2, 3, 5)
    space = torch.empty(max(size, 4), dtype=torch.uint8, device="cuda")
    p = lambda x: x.data_ptr()
    capi.check(capi.lib().ttmi_paged_release(p(t), p(n), 2, 3, 32, 0, 0, 5, p(t), p(free), p(counts), p(space), size, capi._stream()))
    rows, want, c = model.release(table, lengths, 32, 5)
    assert t.tolist() == rows and free.tolist() == want + [7] and counts.tolist() == c + [7]


# ---- as they are used -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_a_graph_of_forks_copies_and_releases(device, dtype):
    """Captured once and replayed on other lengths and parents, against the same calls made eagerly."""
    import ttnn

    torch.manual_seed(6)
    E, pages, requests, width = ttnn.experimental, 40, 4, 6
    caches = [[E.allocate_paged_cache(pages, 2, 32, 64, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)] for _ in range(2)]
    table, lengths, parents = integers(device, torch.randperm(pages)[:requests * width].view(requests, width)), integers(device, [0] * requests), integers(device, [0] * requests)

    def step(pair):
        kept, free, counts = E.release_paged_pages(table, lengths, page_size=32, num_pages=pages, window=100, sinks=4)
        made = E.fork_paged_tables(kept, lengths, parents, free, page_size=32)
        E.copy_paged_pages(pair, made[2], made[3])
        return [kept, free, counts, *made]

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        captured = step(caches[1])
    for n, p in [([5, 70, 150, 33], [0, 0, 1, 1]), ([0, 190, 190, 64], [1, 2, 2, 3]), ([33, 33, 33, 33], [3, 3, 3, 3])]:
        lengths._buf.copy_(torch.tensor(n, dtype=torch.int32))
        parents._buf.copy_(torch.tensor(p, dtype=torch.int32))
        fresh = torch.randint(0, 256, (2, caches[0][0]._buf.view(torch.uint8).numel()), dtype=torch.uint8)
        for pair in caches:
            for cache, x in zip(pair, fresh):
                cache._buf.view(torch.uint8).copy_(x)
        eager = step(caches[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, captured):
            assert torch.equal(a._buf, b._buf)
        for a, b in zip(*caches):
            assert torch.equal(a._buf.view(torch.uint8), b._buf.view(torch.uint8))
        kept, free, _ = model.release(table._buf.view(requests, width).tolist(), n, 32, pages, 100, 4)
        rows = model.fork(kept, n, p, free, 32)[0]
        assert as_list(eager[3]) == rows


def test_the_host_layer_refuses(device):
    import ttnn

    E = ttnn.experimental
    table, lengths, free = integers(device, [[0, 1], [2, 3]]), integers(device, [3, 40]), integers(device, [4, 5])
    for bad in [dict(page_size=40), dict(lengths=integers(device, [1])), dict(parents=None), dict(page_table=lengths), dict(free_pages=table.cpu())]:
        with pytest.raises(RuntimeError):
            E.fork_paged_tables(**{**dict(page_table=table, lengths=lengths, parents=lengths, free_pages=free, page_size=32), **bad})
    for bad in [dict(page_size=40), dict(num_pages=0), dict(window=0), dict(sinks=-1), dict(lengths=free.cpu()), dict(page_table=free)]:
        with pytest.raises(RuntimeError):
            E.release_paged_pages(**{**dict(page_table=table, lengths=lengths, page_size=32, num_pages=6), **bad})
    caches = [E.allocate_paged_cache(4, 1, 32, 64, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    other = E.allocate_paged_cache(4, 1, 64, 64, dtype=ttnn.bfloat16, device=device)
    E.copy_paged_pages([], free, free)
    for c, s, t in [([caches[0], other], free, free), ([caches[0], caches[0]], free, free), (caches, free, integers(device, [1])), ([lengths], free, free), (caches, free, table.cpu())]:
        with pytest.raises(RuntimeError):
            E.copy_paged_pages(c, s, t)
