"""Calls of the paged cache's attention that a server makes besides its ordinary steps: a step without requests, calls captured into
graphs, row starts that are not those of a plain step, lengths near the end of an int32.

Where a value is computed, the tolerance is that of tests/paged_model.py plus 2^-9 of the result (bf16 has 8 significant bits: the result's own
rounding takes up to 2^-8, of which the bound there holds half)."""
import pytest
import torch

import paged_model
from ttmi import capi

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE = 4, 2, 64, 32


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def attend(rows, caches, table, cached, starts, out, layout=capi.ROW_MAJOR, heads=HEADS, dim=DIM, page_size=PAGE, window=0, scale=None, workspace=None, workspace_bytes=0, tokens=None):
    """The C entry on bf16 caches [pages, kv_heads, page_size, dim] given as (keys, values, pages, kv_heads); its status."""
    keys, values, pages, kv_heads = caches
    requests, width = table.shape
    return capi.lib().ttmi_paged_attention(rows.data_ptr(), layout, rows.shape[0] if tokens is None else tokens, rows.shape[1], 0, keys.data_ptr(), values.data_ptr(), capi.BFLOAT16, pages, kv_heads, page_size,
                                           dim, table.data_ptr(), requests, width, cached.data_ptr(), starts.data_ptr(), heads, dim ** -0.5 if scale is None else scale, window, out.data_ptr(),
                                           workspace, workspace_bytes, capi._stream())


def caches_of(pages, kv_heads=KV_HEADS, page_size=PAGE, dim=DIM):
    keys, values = (torch.randn(pages, kv_heads, page_size, dim, device="cuda").bfloat16() for _ in range(2))
    return (capi.tilize(keys), capi.tilize(values), pages, kv_heads), (keys.cpu().double(), values.cpu().double())


# ---- no requests ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [3, 200])
def test_no_requests_and_a_workspace(tokens):
    """A step without requests needs no workspace: one of the size that is asked for, no bytes, stays untouched, and the rows are zeros."""
    torch.manual_seed(1)
    caches, _ = caches_of(2)
    assert capi.lib().ttmi_paged_attention_workspace_bytes(tokens, 0, HEADS, capi.BFLOAT16, KV_HEADS, DIM) == 0
    neighbour = torch.full((1 << 15,), 0x5a, dtype=torch.uint8, device="cuda")
    rows, out = torch.randn(tokens, HEADS * DIM, device="cuda").bfloat16(), torch.ones(tokens, HEADS * DIM, dtype=torch.bfloat16, device="cuda")
    base = (neighbour.data_ptr() + 255) // 256 * 256
    capi.check(attend(rows, caches, ints([]).view(0, 2), ints([]), ints([0]), out, workspace=base, workspace_bytes=0))
    assert (neighbour == 0x5a).all() and not out.any()


# ---- graphs -----------------------------------------------------------------------------------------------------------------------------
def test_a_captured_call_takes_no_buffer_of_a_stream():
    """Also where the stream has one: the graph may be replayed on another stream, while the next call of this one has the buffer."""
    torch.manual_seed(2)
    caches, _ = caches_of(60)
    table, cached, starts = ints([list(range(60))]), ints([1900]), ints([0, 1])
    rows, out = torch.randn(1, HEADS * DIM, device="cuda").bfloat16(), torch.empty(1, HEADS * DIM, dtype=torch.bfloat16, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        capi.check(attend(rows, caches, table, cached, starts, out))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        status = attend(rows, caches, table, cached, starts, out)
        message = capi.lib().ttmi_last_error().decode()
        empty = attend(rows, caches, table[:0], cached, starts, out)          # no requests: nothing that needs memory
    assert status == 3 and "captured call" in message and empty == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_graphs_of_one_stream_side_by_side(dtype):
    """A step of single tokens and a chunk, captured one after the other on one stream and replayed at once on two others, beside eager calls on
    the stream of the capture: every replay has the bits of the eager call, also after the library has given its buffers back."""
    import ttnn

    torch.manual_seed(3)
    device = ttnn.open_device(0)
    heads, kv_heads, dim, page_size, pages = 8, 2, 128, 64, 64
    E = ttnn.experimental
    caches = [E.allocate_paged_cache(pages, kv_heads, page_size, dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)]
    for cache in caches:
        x = torch.randn(pages, kv_heads, page_size, dim, device="cuda")
        cache._buf.copy_(capi.tilize(x.bfloat16()) if dtype == "bfloat16" else capi.pack_tensor(capi.BFLOAT8_B, x))
    put = lambda v: ttnn.from_torch(torch.tensor(v, dtype=torch.int32), device=device)
    table = put([list(range(pages))])
    rows = [ttnn.from_torch(torch.randn(1, 1, n, heads * dim).bfloat16(), layout=ttnn.TILE_LAYOUT, device=device) for n in (1, 200)]
    cached, starts = [put([3000]), put([3500])], [put([0, 1]), put([0, 200])]
    step = lambda i: E.attend_paged_cache(rows[i], *caches, table, cached[i], starts[i], num_heads=heads)
    captured_on = torch.cuda.Stream()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=captured_on):
            outs.append(step(i))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for replay, lengths in enumerate([(3000, 3500), (700, 1800), (3999, 40), (2, 3333)]):
        for c, n in zip(cached, lengths):
            c._buf.fill_(n)
        want = [step(i)._buf.clone() for i in range(2)]
        for out in outs:
            out._buf.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(captured_on):
            beside = [step(i)._buf for i in (0, 1, 0)]
        torch.cuda.synchronize()
        for i, got in [(0, outs[0]._buf), (1, outs[1]._buf), (0, beside[0]), (1, beside[1]), (0, beside[2])]:
            assert torch.equal(got, want[i]), (replay, i)
        if replay == 1:
            capi.release_scratch()
    ttnn.close_device(device)


# ---- row starts -----------------------------------------------------------------------------------------------------------------------
def check_rows(layout, tokens, starts, owners, cached, window=0, width=20, scale=None):
    """One call with these row starts into memory full of ones: owners = (first row, rows) of every request as they should be taken; every other row,
    those that fill up the last tiles among them, is zeros, and what lies behind the output stays."""
    torch.manual_seed(4)
    requests = len(cached)
    caches, (keys, values) = caches_of(requests * width + 1)
    table = torch.arange(requests * width).view(requests, width)
    rows = torch.randn(tokens, HEADS * DIM).bfloat16()
    wide, whole = HEADS * DIM, (tokens + 31) // 32 * 32 if layout == capi.TILE else tokens
    padded = torch.cat([rows, torch.zeros(whole - tokens, wide).bfloat16()])
    given = capi.tilize(padded.cuda()[None]) if layout == capi.TILE else rows.cuda()
    out = torch.ones(whole * wide + 4096, dtype=torch.bfloat16, device="cuda")
    capi.check(attend(given.view(-1, wide), caches, ints(table.tolist()).view(requests, width), ints(cached), ints(starts), out, layout=layout, window=window, scale=scale, tokens=tokens))
    assert (out[whole * wide:] == 1).all()
    got = out[:whole * wide].cpu()
    if layout == capi.TILE:
        got = got.view(-1, wide // 32, 2, 2, 16, 16).permute(0, 2, 4, 1, 3, 5)
    got = got.reshape(whole, wide).double()
    taken = torch.zeros(whole, dtype=torch.bool)
    for r, (first, n) in enumerate(owners):
        taken[first:first + n] = True
        if n:
            want, bound = paged_model.attention(rows[first:first + n], keys, values, [table[r].tolist()], [cached[r]], [0, n], HEADS, DIM, PAGE, window=window, scale=scale)
            off = (got[first:first + n] - want).abs()
            assert (off <= bound + 2.0 ** -9 * want.abs()).all(), f"request {r}: worst {(off / bound).max():.2f} of the bound"
    assert not got[~taken].any()


@pytest.mark.parametrize("layout", [capi.ROW_MAJOR, capi.TILE])
@pytest.mark.parametrize("tokens,starts,owners,cached", [
    (9, [3, 4, 6], [(3, 1), (4, 2)], [50, 33]),                    # a slice of a step's starts: rows before the first one
    (33, [3, 5, 40], [(3, 2), (5, 28)], [0, 64]),                  # more rows said than there are
    (333, [70, 71, 400], [(70, 1), (71, 262)], [100, 3]),          # the same in the kernel for many rows
    (40, [35], [], []),                                            # no requests at all
    (40, [-7, 2, 5], [(0, 2), (2, 3)], [9, 40]),                   # below zero is zero
    (5, [9, 12, 40], [(5, 0), (5, 0)], [9, 40]),                   # all of it past the last row
])
def test_rows_of_no_request_are_zeros(layout, tokens, starts, owners, cached):
    check_rows(layout, tokens, starts, owners, cached)


def owners_of(starts, tokens):
    """Every request's rows where a start below an earlier one is read as that one."""
    at, owners = min(max(starts[0], 0), tokens), []
    for s in starts[1:]:
        to = max(at, min(max(s, 0), tokens))
        owners.append((at, to - at))
        at = to
    return owners


@pytest.mark.parametrize("layout", [capi.ROW_MAJOR, capi.TILE])
@pytest.mark.parametrize("tokens,starts,cached", [
    (10, [0, 5, 3, 8], [40, 3, 70]),
    (10, [0, 8, 4], [33, 5]),                                      # the last start lies inside the first request's rows
    (10, [6, 2, 9], [64, 31]),
    (260, [0, 200, 100, 1, 250], [10, 0, 7, 90]),                  # the kernel for many rows
    (70, [0, 40, 1, 41, 0, 42], [5, 0, 9, 300, 20]),               # both kernels, or one for a mixture
    (300, [(37 * i) % 290 for i in range(200)], [(11 * i) % 90 for i in range(199)]),         # several requests to a lane
])
def test_row_starts_that_do_not_ascend(layout, tokens, starts, cached):
    """No row belongs to two requests; the rows that are some request's hold its answer, the same every time."""
    check_rows(layout, tokens, starts, owners_of(starts, tokens), cached)


def test_a_step_after_row_starts_that_do_not_ascend():
    """Long contexts, cut into pieces: nothing is left of them in the counters that the next call on the stream finds."""
    for _ in range(2):
        check_rows(capi.ROW_MAJOR, 6, [0, 3, 1, 2, 5, 0], owners_of([0, 3, 1, 2, 5, 0], 6), [3000, 2500, 100, 3100, 900], width=100)
        check_rows(capi.ROW_MAJOR, 5, [0, 1, 2, 3, 4, 5], [(i, 1) for i in range(5)], [3000, 2500, 100, 3100, 900], width=100)


# ---- a scale of zero ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 150])
def test_a_scale_of_zero_weighs_all_alike(tokens):
    """Scores of 2^120 and more times 0: the mean of the values that a row sees."""
    torch.manual_seed(5)
    pages, cached = 12, 200
    keys, values = torch.randn(pages, KV_HEADS, PAGE, DIM).bfloat16() * 2.0 ** 60, torch.randn(pages, KV_HEADS, PAGE, DIM).bfloat16()
    rows = (torch.randn(tokens, HEADS * DIM) * 2.0 ** 60).bfloat16()
    out = torch.empty(tokens, HEADS * DIM, dtype=torch.bfloat16, device="cuda")
    caches = (capi.tilize(keys.cuda()), capi.tilize(values.cuda()), pages, KV_HEADS)
    capi.check(attend(rows.cuda(), caches, ints([list(range(pages))]), ints([cached]), ints([0, tokens]), out, scale=0.0))
    want, bound = paged_model.attention(rows, keys.double(), values.double(), [list(range(pages))], [cached], [0, tokens], HEADS, DIM, PAGE, scale=0.0)
    assert ((out.cpu().double() - want).abs() <= bound + 2.0 ** -9 * want.abs()).all()


# ---- lengths ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [0, 2 ** 31 - 40])
@pytest.mark.parametrize("tokens", [4, 150])
def test_positions_of_two_to_the_31_and_more(tokens, window):
    """A request that has more tokens from before than its row of the page table holds, with new ones at 2^31: every one of them sees the tokens that have
    a page, or, of those, what its window reaches (here: a window that ends before the first token from the 40th new one on)."""
    torch.manual_seed(6)
    caches, (keys, values) = caches_of(3)
    rows = torch.randn(tokens, HEADS * DIM).bfloat16()
    cached, out = 2 ** 31 - 3, torch.empty(tokens, HEADS * DIM, dtype=torch.bfloat16, device="cuda")
    capi.check(attend(rows.cuda(), caches, ints([[2, 0, 1]]), ints([cached]), ints([0, tokens]), out, window=window))
    k, v = (x[[2, 0, 1]].transpose(0, 1).reshape(KV_HEADS, 96, DIM) for x in (keys, values))
    got = out.cpu().double().view(tokens, HEADS, DIM)
    for t in range(tokens):
        first = max(0, cached + t - window + 1) if window else 0
        if first >= 96:
            assert not got[t].any(), t
            continue
        want, bound = paged_model.attention(rows[t:t + 1], k[None, :, first:], v[None, :, first:], [[0]], [95 - first], [0, 1], HEADS, DIM, 96 - first)
        assert ((got[t].flatten() - want[0]).abs() <= bound[0] + 2.0 ** -9 * want[0].abs()).all(), t


@pytest.mark.parametrize("tokens", [3, 200])
def test_lengths_and_page_numbers_that_are_none(tokens):
    """Negative lengths are 0, lengths past the table's row see what it holds, numbers outside the cache are no pages: answers by the definition."""
    torch.manual_seed(7)
    pages, requests = 6, 3
    caches, (keys, values) = caches_of(pages)
    table = torch.tensor([[-2 ** 31, 5, 2 ** 31 - 1, 0], [6, -1, 7, 1 << 30], [3, 1, 4, 2]])
    cached = [-2 ** 31, 50, 10 ** 6]
    starts = [0, tokens - 2, tokens - 1, tokens]
    rows, out = torch.randn(tokens, HEADS * DIM).bfloat16(), torch.ones(tokens + 8, HEADS * DIM, dtype=torch.bfloat16, device="cuda")
    capi.check(attend(rows.cuda(), caches, table.to(torch.int32).cuda(), ints(cached), ints(starts), out))
    assert (out[tokens:] == 1).all()
    lengths = [0, 50, 4 * PAGE - 1]                                # the last one: its row sees all four pages
    want, bound = paged_model.attention(rows, keys, values, table.tolist(), lengths, starts, HEADS, DIM, PAGE)
    off = (out[:tokens].cpu().double() - want).abs()
    assert (off <= bound + 2.0 ** -9 * want.abs()).all() and not out[tokens - 2].any() and out[tokens - 1].any()
