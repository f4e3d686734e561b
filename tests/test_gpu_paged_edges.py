"""Attention over the paged cache where it can go wrong: values and keys that are not finite, scales of either sign and none,
caches and rows past 4 GiB, thousands of requests, steps of random shapes, streams side by side, a capture without scratch.

Tolerances are those of tests/paged_model.py plus 2^-9 of the result: bf16 has 8 significant bits, so that the result's own
rounding takes up to 2^-8 of it, of which the bound there holds half.  Where a call has to give the same bits, bits are compared."""
import random

import pytest
import torch

import paged_model
from test_gpu_paged import activations, attention_case, device, fill_cache, integers, read_cache  # noqa: F401 (device is a fixture)

pytestmark = pytest.mark.gpu


def caches_of(device, keys, values, dtype="bfloat16"):
    import ttnn

    caches = []
    for x in (keys, values):
        caches.append(ttnn.experimental.allocate_paged_cache(*x.shape, dtype=getattr(ttnn, dtype), device=device))
        fill_cache(caches[-1], x)
    return caches


def inside(got, want, bound):
    off = (got.double() - want).abs()
    assert (off <= bound + 2.0 ** -9 * want.abs()).all(), f"worst {(off / bound).max():.2f} of the bound at {(off / bound).argmax().item()}"


# ---- values and keys that are not finite ------------------------------------------------------------------------------------------------
# requests' lengths, heads, key heads, elements of a head, window: single tokens, rows of several lengths in both kernels
BAD = {
    "decode": ([70, 33, 5], [1, 1, 1], 4, 2, 64, 0),
    "drafts": ([70, 33, 0], [3, 5, 4], 8, 2, 128, 0),
    "a prompt": ([0], [400], 4, 2, 128, 0),
    "a prompt, wide heads": ([40], [300], 2, 1, 256, 0),
    "a prompt, 96 elements": ([100], [200], 6, 2, 96, 0),
    "a prompt, window": ([100], [300], 4, 1, 64, 50),
    "a prompt cut into pieces": ([3000], [260], 2, 2, 128, 0),
    "prompts and single tokens": ([10, 130, 64, 1], [150, 1, 0, 70], 4, 1, 128, 0),
}


@pytest.mark.parametrize("name", BAD)
def test_values_that_are_not_finite(device, name):
    """Infinities and NaN among the values: a row's column has what adding them up would give if a token that it sees has one there (NaN for a
    NaN, or for infinities of both signs), and no trace of those that it does not see."""
    import ttnn

    cached, new, heads, kv_heads, dim, window = BAD[name]
    generator = torch.Generator().manual_seed(len(name))
    page_size, requests, tokens = 32, len(cached), sum(new)
    width = max(-(-(c + n) // page_size) for c, n in zip(cached, new))
    table = torch.randperm(requests * width, generator=generator).view(requests, width).tolist()
    starts = [sum(new[:r]) for r in range(requests + 1)]
    keys, values = (torch.randn(requests * width, kv_heads, page_size, dim, generator=generator).bfloat16() for _ in range(2))
    share = 2.0 / max(cached + new)                                # about one value in each column that a row looks at
    kind = torch.randint(0, 3, values.shape, generator=generator)
    special = torch.tensor([float("nan"), float("inf"), -float("inf")]).bfloat16()[kind]
    bad = torch.rand(values.shape, generator=generator) < share
    rows = torch.randn(tokens, heads * dim, generator=generator).bfloat16()
    out = ttnn.experimental.attend_paged_cache(activations(device, rows, "TILE_LAYOUT"), *caches_of(device, keys, torch.where(bad, special, values)), integers(device, table),
                                               integers(device, cached), integers(device, starts), num_heads=heads, window=window or None)
    got = ttnn.to_torch(out.cpu())[0, 0].view(tokens, heads, dim)
    finite, bound = paged_model.attention(rows, keys.double(), torch.where(bad, torch.zeros_like(values), values).double(), table, cached, starts, heads, dim, page_size, window=window)
    finite, bound = finite.view(tokens, heads, dim), bound.view(tokens, heads, dim)
    where = lambda k: torch.where(bad & (kind == k), 1.0, 0.0).double()
    ones = torch.zeros_like(keys).double()                         # equal scores: a mean of the marks, positive where one is seen
    marks = [paged_model.attention(rows, ones, where(k), table, cached, starts, heads, dim, page_size, window=window)[0].view(tokens, heads, dim) > 0 for k in range(3)]
    nan, up, down = marks[0] | (marks[1] & marks[2]), marks[1], marks[2]
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got == float("inf"), up & ~nan) and torch.equal(got == -float("inf"), down & ~nan)
    fine = ~(nan | up | down)
    assert fine.any() and not fine.all()
    inside(got[fine], finite[fine], bound[fine])


@pytest.mark.parametrize("name", BAD)
def test_a_key_that_is_not_a_number(device, name):
    """It makes all of a row's weights NaN, for the heads that share it and the rows that see it; the others do not notice."""
    import ttnn

    cached, new, heads, kv_heads, dim, window = BAD[name]
    generator = torch.Generator().manual_seed(len(name) + 100)
    page_size, requests, tokens = 32, len(cached), sum(new)
    width = max(-(-(c + n) // page_size) for c, n in zip(cached, new))
    table = torch.randperm(requests * width, generator=generator).view(requests, width).tolist()
    starts = [sum(new[:r]) for r in range(requests + 1)]
    keys, values = (torch.randn(requests * width, kv_heads, page_size, dim, generator=generator).bfloat16() for _ in range(2))
    rows = torch.randn(tokens, heads * dim, generator=generator).bfloat16()
    want, bound = (x.view(tokens, heads, dim) for x in paged_model.attention(rows, keys.double(), values.double(), table, cached, starts, heads, dim, page_size, window=window))
    nan = torch.zeros(tokens, heads, dim, dtype=torch.bool)
    for r in range(0, requests, 2):                                # in every other request, one key of the last key head
        at = cached[r] + new[r] // 2 if new[r] > 1 else cached[r] // 2
        keys[table[r][at // page_size], kv_heads - 1, at % page_size, dim // 2] = float("nan")
        for i in range(new[r]):
            p = cached[r] + i
            if at <= p and (not window or at > p - window):
                nan[starts[r] + i, heads - heads // kv_heads:] = True
    out = ttnn.experimental.attend_paged_cache(activations(device, rows, "ROW_MAJOR_LAYOUT"), *caches_of(device, keys, values), integers(device, table), integers(device, cached), integers(device, starts),
                                               num_heads=heads, window=window or None)
    got = ttnn.to_torch(out.cpu())[0, 0].view(tokens, heads, dim)
    assert torch.equal(torch.isnan(got), nan) and nan.any()
    inside(got[~nan], want[~nan], bound[~nan])


@pytest.mark.parametrize("new", [[1, 1], [90, 1], [300]])
def test_block_floats_that_were_not_finite(oracle, device, new):
    """Rows of 16 block floats with the exponent 255, as infinities and NaN leave them, behind a request's last token and in pages of
    nobody: nothing of them is seen."""
    import ttnn

    generator = torch.Generator().manual_seed(5)
    cached, heads, kv_heads, dim, page_size = [45] * len(new), 4, 2, 64, 64
    width = max(-(-(c + n) // page_size) for c, n in zip(cached, new))
    table = torch.randperm(len(new) * width, generator=generator).view(len(new), width).tolist()
    pages, tokens = len(new) * width + 1, sum(new)
    starts = [sum(new[:r]) for r in range(len(new) + 1)]
    keys, values = (torch.randn(pages, kv_heads, page_size, dim, generator=generator).bfloat16() for _ in range(2))
    owned = torch.zeros(pages, page_size, dtype=torch.bool)
    for r, n in enumerate(new):
        for p in range(cached[r] + n):
            owned[table[r][p // page_size], p % page_size] = True
    rubbish = torch.tensor([float("inf"), float("nan"), -float("inf"), 1.0]).bfloat16()[torch.randint(0, 4, keys.shape, generator=generator)]
    keep = owned[:, None, :, None]
    caches = caches_of(device, torch.where(keep, keys, rubbish), torch.where(keep, values, rubbish), "bfloat8_b")
    rows = torch.randn(tokens, heads * dim, generator=generator).bfloat16()
    out = ttnn.experimental.attend_paged_cache(activations(device, rows, "TILE_LAYOUT"), *caches, integers(device, table), integers(device, cached), integers(device, starts), num_heads=heads)
    want, bound = paged_model.attention(rows, paged_model.bfloat8_b(oracle, keys).double(), paged_model.bfloat8_b(oracle, values).double(), table, cached, starts, heads, dim, page_size)
    inside(ttnn.to_torch(out.cpu())[0, 0], want, bound)


# ---- scales -------------------------------------------------------------------------------------------------------------------------------
def same_as_model(oracle, device, cached, new, heads, kv_heads, dim, page_size, dtype="bfloat16", layout="TILE_LAYOUT", window=0, scale=None, query_column=0, seed=0, spread=1.0, hole=False):
    import ttnn

    generator = torch.Generator().manual_seed(seed)
    requests, tokens = len(cached), sum(new)
    width = max(-(-(c + n) // page_size) for c, n in zip(cached, new)) + seed % 2
    table = torch.randperm(requests * width + 1, generator=generator)[:requests * width].view(requests, width).tolist()
    if hole:
        for r in range(requests):
            table[r][(r * 5) % width] = -1
    starts = [sum(new[:r]) for r in range(requests + 1)]
    keys, values = (torch.randn(requests * width + 1, kv_heads, page_size, dim, generator=generator).bfloat16() for _ in range(2))
    caches = caches_of(device, keys, values, dtype)
    if dtype == "bfloat8_b":
        keys, values = (paged_model.bfloat8_b(oracle, x) for x in (keys, values))
    rows = (torch.randn(tokens, query_column + heads * dim, generator=generator) * spread).bfloat16()
    out = ttnn.experimental.attend_paged_cache(activations(device, rows, layout), *caches, integers(device, table), integers(device, cached), integers(device, starts), num_heads=heads,
                                               query_column=query_column, scale=scale, window=window or None)
    want, bound = paged_model.attention(rows, keys.double(), values.double(), table, cached, starts, heads, dim, page_size, query_column, scale, window)
    inside(ttnn.to_torch(out.cpu())[0, 0], want, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("new", [[1, 1, 1], [300], [5, 90, 1]])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-12, 0.7])
def test_scales(oracle, device, dtype, new, scale):
    same_as_model(oracle, device, [130, 0, 65][:len(new)], new, 8, 2, 64, 32, dtype=dtype, scale=scale, seed=3)


# ---- steps of random shapes -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(40))
def test_random_steps(oracle, device, seed):
    r = random.Random(seed)
    requests = r.choice([1, 1, 2, 3, 7, 20])
    kv_heads, group, dim = r.choice([1, 2, 4]), r.choice([1, 2, 3, 4, 5, 8, 17]), r.choice([64, 96, 128, 256])
    longest = r.choice([1, 2, 8, 40, 300]) if requests < 7 else r.choice([1, 6, 30])
    new = [r.choice([1, r.randint(0, longest), r.randint(1, longest)]) for _ in range(requests)]
    new[0] = max(new[0], 1)
    cached = [r.choice([0, r.randint(0, 70), r.randint(0, 900)]) for _ in range(requests)]
    same_as_model(oracle, device, cached, new, kv_heads * group, kv_heads, dim, r.choice([32, 64, 96, 128]), dtype=r.choice(["bfloat16", "bfloat8_b"]),
                  layout=r.choice(["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"]), window=r.choice([0, 0, r.randint(1, 200)]), query_column=r.choice([0, 32, 256]), seed=seed, spread=r.choice([1.0, 4.0]), hole=r.random() < 0.25)


# ---- many requests, long caches, many rows ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("requests,longest", [(1500, 1), (700, 3), (4096, 1)])
def test_many_requests(oracle, device, requests, longest):
    """More requests than a wavefront has lanes: every lane has several, some of them without new tokens."""
    r = random.Random(requests)
    new = [r.randint(0, longest) if i % 3 else 1 for i in range(requests)]
    same_as_model(oracle, device, [r.choice([0, 3, 40, 100]) for _ in range(requests)], new, 2, 1, 64, 32, seed=2)


@pytest.mark.parametrize("dtype,pages", [("bfloat16", 40000), ("bfloat8_b", 70000)])
def test_a_cache_of_more_than_four_gibibytes(device, dtype, pages):
    """Tokens written to the far end of such a cache and attended to there: the bits that a small cache gives."""
    import ttnn

    torch.manual_seed(6)
    heads, kv_heads, dim, page_size, cached, new = 16, 8, 128, 64, [100, 300], [1, 40]
    width, tokens = 6, sum(c + n for c, n in zip(cached, new))
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * dim).bfloat16()
    near = torch.arange(2 * width).view(2, width)
    steps = activations(device, qkv[:sum(new)], "ROW_MAJOR_LAYOUT")
    results = []
    for count, table in ((2 * width, near), (pages, pages - 1 - near)):
        caches = [ttnn.experimental.allocate_paged_cache(count, kv_heads, page_size, dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)]
        assert count == 2 * width or caches[0]._buf.numel() * caches[0]._buf.element_size() > 1 << 32
        slots = torch.cat([table[r, torch.arange(cached[r] + new[r]) // page_size] * page_size + torch.arange(cached[r] + new[r]) % page_size for r in range(2)])
        ttnn.experimental.write_paged_cache(activations(device, qkv, "TILE_LAYOUT"), *caches, integers(device, slots), key_column=heads * dim, value_column=(heads + kv_heads) * dim)
        for rows in (steps, activations(device, qkv[:2], "ROW_MAJOR_LAYOUT")):
            lengths = new if rows is steps else [1, 1]
            out = ttnn.experimental.attend_paged_cache(rows, *caches, integers(device, table.contiguous()), integers(device, cached), integers(device, [0, lengths[0], sum(lengths)]), num_heads=heads)
            results.append(ttnn.to_torch(out.cpu()))
        del caches
    assert torch.equal(results[0], results[2]) and torch.equal(results[1], results[3])
    assert all(r.float().abs().sum() > 0 for r in results)


@pytest.mark.parametrize("layout", [0, 1])
def test_rows_of_more_than_four_gibibytes(layout):
    """One prompt of 270,000 tokens, 64 heads on one key head, window 40: keys and values come from the far end of the rows, the last
    rows are compared with the definition."""
    from ttmi import capi

    torch.manual_seed(7)
    L, tokens, heads, dim, page_size, window, looked_at = capi.lib(), 270016, 64, 128, 128, 40, 32
    width, pages = (heads + 2) * dim, -(-tokens // page_size)
    rows = torch.randn(looked_at + window, width, device="cuda").bfloat16()
    whole = torch.zeros(tokens, width, dtype=torch.bfloat16, device="cuda")
    assert whole.numel() * 2 > 1 << 32
    whole[-rows.shape[0]:] = rows
    if layout:
        whole = whole.view(tokens // 32, 2, 16, width // 32, 2, 16).permute(0, 3, 1, 4, 2, 5).reshape(tokens, width)
    caches = [torch.zeros(pages * page_size * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ints = lambda v: torch.as_tensor(v, dtype=torch.int32, device="cuda")
    p = lambda t: t.data_ptr()
    table, slots, cached, starts = ints(list(range(pages))), torch.arange(tokens, dtype=torch.int32, device="cuda"), ints([0]), ints([0, tokens])
    out = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device="cuda")
    capi.check(L.ttmi_paged_write(p(whole), layout, tokens, width, heads * dim, (heads + 1) * dim, p(slots), p(caches[0]), p(caches[1]), 0, pages, 1, page_size, dim, capi._stream()))
    capi.check(L.ttmi_paged_attention(p(whole), layout, tokens, width, 0, p(caches[0]), p(caches[1]), 0, pages, 1, page_size, dim, p(table), 1, pages, p(cached), p(starts), heads, dim ** -0.5, window,
                                      p(out), None, 0, capi._stream()))
    got = out[-32:].cpu()
    if layout:
        got = got.reshape(heads * dim // 32, 2, 2, 16, 16).permute(1, 3, 0, 2, 4).reshape(32, heads * dim)
    rows = rows.cpu()
    k, v = rows[:, heads * dim:(heads + 1) * dim].double(), rows[:, (heads + 1) * dim:].double()
    last = torch.zeros(96, dim, dtype=torch.float64)
    pad = lambda x: torch.cat([x, last])[:96].view(1, 1, 96, dim)
    want, bound = paged_model.attention(rows[-32:, :heads * dim], pad(k), pad(v), [[0]], [window], [0, looked_at], heads, dim, 96, window=window)
    inside(got, want, bound)
    assert not out[:tokens - rows.shape[0] - 64].any()


# ---- streams ------------------------------------------------------------------------------------------------------------------------------------
def test_streams_side_by_side(device):
    """Two streams at once, each with scratch of its own: the bits of calls one after the other, every time."""
    import ttnn

    torch.manual_seed(8)
    heads, kv_heads, dim, page_size, pages = 8, 2, 128, 64, 64
    caches = caches_of(device, *(torch.randn(pages, kv_heads, page_size, dim).bfloat16() for _ in range(2)))
    table = integers(device, torch.arange(pages)[None])
    rows = [activations(device, torch.randn(n, heads * dim).bfloat16(), "TILE_LAYOUT") for n in (1, 200)]
    lengths = [(integers(device, [3000]), integers(device, [0, 1])), (integers(device, [3500]), integers(device, [0, 200]))]
    step = lambda i: ttnn.experimental.attend_paged_cache(rows[i], *caches, table, *lengths[i], num_heads=heads)
    want = [ttnn.to_torch(step(i).cpu()) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs.append((i, step(i)))
    torch.cuda.synchronize()
    for i, out in outs:
        assert torch.equal(ttnn.to_torch(out.cpu()), want[i])


def test_a_capture_without_scratch_is_refused():
    """A stream that has none yet cannot allocate it while it is captured; with a workspace of the caller's the call is captured, and its
    replays follow the lengths."""
    from ttmi import capi

    torch.manual_seed(9)
    L, heads, kv_heads, dim, page_size, pages = capi.lib(), 4, 1, 64, 64, 48
    rows = torch.randn(1, heads * dim, device="cuda").bfloat16()
    keys, values = (capi.tilize(torch.randn(pages, kv_heads, page_size, dim, device="cuda").bfloat16()) for _ in range(2))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, cached, starts = ints([list(range(pages))]), ints([2000]), ints([0, 1])
    out, want = (torch.empty(heads * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    size = L.ttmi_paged_attention_workspace_bytes(1, 1, heads, capi.BFLOAT16, kv_heads, dim)
    memory = torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda")
    base = (memory.data_ptr() + 255) // 256 * 256

    def call(o, workspace, nbytes):
        return L.ttmi_paged_attention(rows.data_ptr(), capi.ROW_MAJOR, 1, heads * dim, 0, keys.data_ptr(), values.data_ptr(), capi.BFLOAT16, pages, kv_heads, page_size, dim, table.data_ptr(), 1, pages,
                                      cached.data_ptr(), starts.data_ptr(), heads, dim ** -0.5, 0, o.data_ptr(), workspace, nbytes, capi._stream())

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    capi.release_scratch()                                         # torch hands out streams again, which may have some
    with torch.cuda.graph(graph, stream=stream):
        refused = call(out, None, 0)
        message = L.ttmi_last_error().decode()
        captured = call(out, base, size)
    assert refused == 3 and "captured call" in message and captured == 0
    for length in (2000, 5, 3071, 640):
        cached.fill_(length)
        graph.replay()
        torch.cuda.synchronize()
        capi.check(call(want, None, 0))
        assert torch.equal(out, want)
