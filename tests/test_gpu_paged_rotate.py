"""Rotated heads, with their norms, and rotated keys and values into a paged cache, on the GPU, against plain statements of them in 64 bits
(tests/paged_more_model.py, where the tolerances are derived)."""
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


def floats(device, values):
    import ttnn

    return None if values is None else ttnn.from_torch(values.float(), device=device)


def activations(device, rows, layout):
    import ttnn

    return ttnn.from_torch(rows[None, None], dtype=ttnn.bfloat16, layout=getattr(ttnn, layout), device=device)


def whole_rows(tensor, width):
    """Every row that is in memory, those that fill up the last tiles among them."""
    flat = tensor._buf.cpu()
    if "TILE" in str(tensor.layout):
        flat = flat.view(-1, width // 32, 2, 2, 16, 16).permute(0, 2, 4, 1, 3, 5)
    return flat.reshape(-1, width)


def frequencies_of(rotary_dim, theta=10000.0):
    return (theta ** (-torch.arange(rotary_dim // 2, dtype=torch.float64) / max(rotary_dim // 2, 1))).float()


def check(got, out, bound):
    off = (got.double() - out).abs()
    assert (off <= bound).all(), f"{(off > bound).sum()} of {off.numel()} outside, worst {(off / bound).max():.2f} of the bound at {(off / bound).argmax().item()}"


def rotate_case(device, *, cached, new, heads, head_dim, rotary_dim=None, layout="TILE_LAYOUT", interleaved=False, norm=False, magnitude=1.0, epsilon=1e-5, column=0, spare=0, starts=None, seed=1,
                spread=1.0):
    import ttnn

    torch.manual_seed(seed)
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    starts = starts or [sum(new[:r]) for r in range(len(new) + 1)]
    tokens, wide = sum(new) + spare, heads * head_dim
    extra = 32 if layout == "TILE_LAYOUT" else 8
    rows = (torch.randn(tokens, column + wide + extra) * spread).bfloat16()
    weights = 1 + 0.3 * torch.randn(head_dim) if norm else None
    f = frequencies_of(rotary_dim)
    out = ttnn.experimental.rotate_heads(activations(device, rows, layout), integers(device, cached), integers(device, starts), floats(device, f), num_heads=heads, head_dim=head_dim,
                                         column=column, interleaved=interleaved, norm=floats(device, weights), epsilon=epsilon, magnitude=magnitude)
    assert tuple(out.shape) == (1, 1, tokens, wide) and out.dtype == ttnn.bfloat16 and out.layout == getattr(ttnn, layout)
    got = whole_rows(out, wide)
    assert not got[tokens:].any()
    owners = model.owners(cached, starts, tokens)
    want, bound = model.rotate(rows[:, column:column + wide], owners, heads, head_dim, f, interleaved, weights, epsilon, magnitude)
    check(got[:tokens].view(want.shape), want, model.as_bfloat16(want, bound))
    nobody = torch.tensor([o is None for o in owners])
    assert not got[:tokens][nobody].any()


@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,head_dim,rotary_dim", [(1, 64, 64), (5, 64, 16), (71, 64, 48), (3, 96, 96), (4, 96, 32), (2, 96, 80), (32, 128, 128), (3, 128, 112), (2, 256, 256), (3, 256, 64), (2, 256, 240), (2, 128, 16)])
def test_heads(device, layout, interleaved, norm, heads, head_dim, rotary_dim):
    """Every head size, whole and in part, behind other columns; requests with none, one and many tokens."""
    rotate_case(device, cached=[0, 1000, 5, 31], new=[3, 1, 0, 14], heads=heads, head_dim=head_dim, rotary_dim=rotary_dim, layout=layout, interleaved=interleaved, norm=norm, column=64, magnitude=1.2)


@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 32, 33, 100, 257])
def test_row_counts(device, layout, tokens):
    rotate_case(device, cached=[7], new=[tokens], heads=3, head_dim=64, layout=layout, spare=tokens % 3)


@pytest.mark.parametrize("requests", [63, 64, 65, 127, 128, 129, 300, 4096])
def test_many_requests(device, requests):
    """Single tokens, some requests without any: row starts over several chunks of the search."""
    new = [0 if r % 7 == 3 else 1 for r in range(requests)]
    rotate_case(device, cached=[(r * 37) % 500 for r in range(requests)], new=new, heads=1, head_dim=64, layout="ROW_MAJOR_LAYOUT", spare=5)


def test_many_heads_of_many_tokens(device):
    """Items of several heads, the last one of fewer."""
    rotate_case(device, cached=[0, 90], new=[3000, 1100], heads=71, head_dim=64, rotary_dim=32, layout="ROW_MAJOR_LAYOUT", norm=True)
    rotate_case(device, cached=[0], new=[2100], heads=33, head_dim=128, layout="TILE_LAYOUT")


@pytest.mark.parametrize("cached", [131071, 2 ** 24 + 1, 2 ** 31 - 2])
def test_far_positions(device, cached):
    """Angles of millions of turns."""
    rotate_case(device, cached=[cached, 3], new=[4, 1], heads=2, head_dim=128)


def test_no_rotation_is_the_norm_alone(device):
    rotate_case(device, cached=[4], new=[9], heads=4, head_dim=128, rotary_dim=0, norm=True)
    rotate_case(device, cached=[4], new=[9], heads=4, head_dim=128, rotary_dim=0, layout="ROW_MAJOR_LAYOUT")


@pytest.mark.parametrize("starts,tokens", [([3, 4, 6], 9), ([3, 5, 40], 33), ([-7, 2, 5], 40), ([9, 12, 40], 5), ([0, 5, 3, 8], 10), ([6, 2, 9], 64), ([35], 40), ([0, 40, 1, 41, 0, 42], 70)])
@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
def test_row_starts_of_any_content(device, starts, tokens, layout):
    """Rows of no request are zeros; a start below an earlier one is read as that one."""
    requests = len(starts) - 1
    rotate_case(device, cached=[(r * 50 - 20) for r in range(requests)], new=[tokens], heads=2, head_dim=64, starts=starts, layout=layout)


def test_no_tokens(device):
    import ttnn
    from ttmi import capi

    f = floats(device, frequencies_of(64))
    capi.check(capi.lib().ttmi_rotate_heads(None, 0, 0, 128, 0, 2, 64, None, integers(device, [0])._buf.data_ptr(), 0, f._buf.data_ptr(), 64, 0, None, 0.0, 1.0, None, capi._stream()))
    out = ttnn.experimental.rotate_heads(activations(device, torch.randn(3, 128).bfloat16(), "TILE_LAYOUT"), integers(device, []), integers(device, [0]), f, num_heads=2, head_dim=64)
    assert not out._buf.any()


def test_infinities_stay_in_their_pairs(device):
    """An infinite or NaN element comes out in its pair alone; elements that do not turn are copied, whatever they are."""
    import ttnn

    rows = torch.randn(1, 64).bfloat16()
    rows[0, 3], rows[0, 40], rows[0, 41] = float("nan"), float("inf"), float("nan")
    out = ttnn.experimental.rotate_heads(activations(device, rows, "ROW_MAJOR_LAYOUT"), integers(device, [9]), integers(device, [0, 1]), floats(device, frequencies_of(32)), num_heads=1, head_dim=64)
    got = ttnn.to_torch(out.cpu())[0, 0, 0]
    assert torch.isnan(got).nonzero().flatten().tolist() == [3, 19, 41] and got[40] == float("inf") and torch.equal(got[42:], rows[0, 42:])


# ---- straight into the cache ----------------------------------------------------------------------------------------------------------
def write_case(oracle, device, *, cached, new, heads, kv_heads, head_dim, page_size, dtype, layout="TILE_LAYOUT", rotary_dim=None, interleaved=False, norms=(False, False), magnitude=1.0, seed=2,
               spare=0, lost=()):
    """Slots in any order, tokens of `lost` without one; what else lies in the pages stays, bit for bit."""
    import ttnn
    from ttmi import capi

    torch.manual_seed(seed)
    E = ttnn.experimental
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    tokens, f = sum(new) + spare, frequencies_of(rotary_dim)
    pages = -(-tokens // page_size) + 2
    slots = torch.randperm(pages * page_size)[:tokens].tolist()
    for i, t in enumerate(lost):
        slots[t] = [-1, pages * page_size, -2 ** 31][i % 3]
    starts = [sum(new[:r]) for r in range(len(new) + 1)]
    q, wide = heads * head_dim, kv_heads * head_dim
    columns = 32, 32 + q, 32 + q + wide + 32                       # queries, keys, values
    rows = torch.randn(tokens, columns[2] + wide).bfloat16()
    weights = [1 + 0.3 * torch.randn(head_dim) if n else None for n in norms]
    before = [torch.randn(pages, kv_heads, page_size, head_dim) for _ in range(2)]
    caches = []
    for x in before:
        cache = E.allocate_paged_cache(pages, kv_heads, page_size, head_dim, dtype=getattr(ttnn, dtype), device=device)
        cache._buf.copy_(capi.tilize(x.cuda().bfloat16()) if dtype == "bfloat16" else capi.pack_tensor(capi.BFLOAT8_B, x.cuda()))
        caches.append(cache)
    old = [ttnn.to_torch(ttnn.from_device(c)).float() for c in caches]
    given = activations(device, rows, layout)
    common = dict(interleaved=interleaved, epsilon=1e-5, magnitude=magnitude)
    lengths = integers(device, cached), integers(device, starts), floats(device, f)
    out = E.rotate_write_paged_cache(given, *caches, integers(device, slots), *lengths, num_heads=heads, query_column=columns[0], key_column=columns[1], value_column=columns[2],
                                     query_norm=floats(device, weights[0]), key_norm=floats(device, weights[1]), **common)
    alone = E.rotate_heads(given, *lengths, num_heads=heads, head_dim=head_dim, column=columns[0], norm=floats(device, weights[0]), **common)
    assert torch.equal(out._buf, alone._buf)                       # the queries, whose values test_heads checks
    owners = model.owners(cached, starts, tokens)
    keys, bound = model.rotate(rows[:, columns[1]:columns[1] + wide], owners, kv_heads, head_dim, f, interleaved, weights[1], 1e-5, magnitude)
    values = rows[:, columns[2]:].double().view(tokens, kv_heads, head_dim)
    if dtype == "bfloat8_b":
        values = torch.from_numpy(oracle.to_torch_bfp_tiles(3, oracle.from_torch_bfp_tiles(3, torch.nn.functional.pad(rows[:, columns[2]:].float(), (0, 0, 0, -tokens % 32)).numpy()),
                                                            (-(-tokens // 32) * 32, wide)))[:tokens].double().view(values.shape)
    bound = model.as_bfloat16(keys, bound) if dtype == "bfloat16" else model.as_bfloat8_b(keys, bound)
    written = torch.zeros(pages, page_size, dtype=torch.bool)
    for which, (cache, want) in enumerate(zip(caches, (keys, values))):
        now = ttnn.to_torch(ttnn.from_device(cache)).float()
        for t, (slot, owner) in enumerate(zip(slots, owners)):
            if owner is None or not 0 <= slot < pages * page_size:
                continue
            page, at = divmod(slot, page_size)
            written[page, at] = True
            got = now[page, :, at].double()
            if which:
                assert torch.equal(got, want[t]), t
            else:
                check(got, want[t], bound[t])
        same = ~written[:, None, :, None].expand_as(now)
        assert torch.equal(now[same], old[which][same])


@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("heads,kv_heads,head_dim,rotary_dim", [(4, 4, 64, 64), (7, 1, 64, 16), (8, 2, 96, 96), (4, 2, 96, 48), (32, 8, 128, 128), (6, 3, 128, 48), (4, 2, 256, 64), (2, 1, 256, 256)])
def test_writes(oracle, device, layout, dtype, heads, kv_heads, head_dim, rotary_dim):
    """Pairs whose partners share an exponent with others in the same lane and in other lanes; tokens without a slot, rows of no request."""
    write_case(oracle, device, cached=[0, 70, 3], new=[5, 1, 34], heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary_dim=rotary_dim, page_size=64, dtype=dtype, layout=layout, spare=2,
               lost=[0, 7, 20, 39])


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, True)])
def test_writes_with_norms(oracle, device, dtype, interleaved, norms):
    for head_dim, rotary_dim in [(64, 32), (96, 80), (128, 128), (256, 240)]:
        write_case(oracle, device, cached=[900, 0], new=[1, 20], heads=4, kv_heads=2, head_dim=head_dim, rotary_dim=rotary_dim, page_size=32, dtype=dtype, interleaved=interleaved, norms=norms,
                   magnitude=0.7)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_prompts_are_written(oracle, device, dtype):
    """Items of several heads."""
    write_case(oracle, device, cached=[0, 17], new=[1800, 333], heads=32, kv_heads=8, head_dim=128, page_size=96, dtype=dtype, norms=(True, True), spare=1)


@pytest.mark.parametrize("rotary_dim", [128, 48])
def test_keys_are_those_of_rotate_heads(device, rotary_dim):
    """A bf16 cache holds the bits that rotate_heads gives for the key columns; values are copied whatever they hold."""
    import ttnn
    from ttmi import capi

    torch.manual_seed(8)
    E, tokens, kv_heads, dim = ttnn.experimental, 70, 2, 128
    rows = torch.randn(tokens, 3 * kv_heads * dim).bfloat16()
    odd = torch.randint(-32768, 32767, (tokens, kv_heads * dim), dtype=torch.int16).view(torch.bfloat16)
    rows[:, 2 * kv_heads * dim:] = odd
    caches = [E.allocate_paged_cache(3, kv_heads, 32, dim, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    given, lengths = activations(device, rows, "ROW_MAJOR_LAYOUT"), (integers(device, [5]), integers(device, [0, tokens]), floats(device, frequencies_of(rotary_dim)))
    norm = floats(device, 1 + 0.2 * torch.randn(dim))
    E.rotate_write_paged_cache(given, *caches, integers(device, range(tokens)), *lengths, num_heads=kv_heads, key_column=kv_heads * dim, value_column=2 * kv_heads * dim, key_norm=norm)
    alone = ttnn.to_torch(E.rotate_heads(given, *lengths, num_heads=kv_heads, head_dim=dim, column=kv_heads * dim, norm=norm).cpu())[0, 0]
    keys, values = (c._buf.cpu().view(3, kv_heads, 1, dim // 32, 2, 2, 16, 16).permute(0, 2, 4, 6, 1, 3, 5, 7).reshape(96, kv_heads * dim)[:tokens] for c in caches)
    assert torch.equal(keys, alone) and torch.equal(values.contiguous().view(torch.int16), odd.view(torch.int16))


@pytest.mark.parametrize("layout", ["TILE_LAYOUT", "ROW_MAJOR_LAYOUT"])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -90, 2.0 ** -100, 2.0 ** -122, 2.0 ** -133, 2.0 ** 127])
def test_numbers_at_the_ends_of_the_range_are_packed_as_elsewhere(device, layout, scale):
    """Without frequencies and norms a BFLOAT8_B cache holds the bits that write_paged_cache gives: tiny and huge numbers, infinities and NaN, rows of zeros, among ordinary ones."""
    import ttnn

    torch.manual_seed(10)
    E, tokens, kv_heads, dim = ttnn.experimental, 45, 2, 96
    wide = kv_heads * dim
    rows = (torch.randn(tokens, 3 * wide) * scale).bfloat16()
    rows[3], rows[4, ::2], rows[5:9] = 0.0, -0.0, torch.randn(4, 3 * wide).bfloat16()
    rows[10, ::37], rows[11, ::41], rows[12, 5::16] = float("inf"), float("nan"), -float("inf")
    given, slots = activations(device, rows, layout), integers(device, torch.randperm(96)[:tokens])
    caches = [[E.allocate_paged_cache(3, kv_heads, 32, dim, dtype=ttnn.bfloat8_b, device=device) for _ in range(2)] for _ in range(2)]
    for pair in caches:
        for cache in pair:
            cache._buf.zero_()
    E.write_paged_cache(given, *caches[0], slots, key_column=wide, value_column=2 * wide)
    E.rotate_write_paged_cache(given, *caches[1], slots, integers(device, [7]), integers(device, [0, tokens]), floats(device, frequencies_of(0)), num_heads=kv_heads, key_column=wide, value_column=2 * wide)
    for a, b in zip(*caches):
        assert torch.equal(a._buf, b._buf)


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_a_graph_replayed_on_other_lengths_and_streams(device, dtype):
    import ttnn

    torch.manual_seed(9)
    E, heads, kv_heads, dim, tokens = ttnn.experimental, 8, 2, 128, 33
    wide = (heads + 2 * kv_heads) * dim
    rows = activations(device, torch.randn(tokens, wide).bfloat16(), "TILE_LAYOUT")
    cached, starts, slots, f = integers(device, [0, 0]), integers(device, [0, 1, tokens]), integers(device, range(tokens)), floats(device, frequencies_of(dim))
    caches = [[E.allocate_paged_cache(4, kv_heads, 32, dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)] for _ in range(2)]
    for pair in caches:
        for cache in pair:
            cache._buf.zero_()
    step = lambda pair: E.rotate_write_paged_cache(rows, *pair, slots, cached, starts, f, num_heads=heads, key_column=heads * dim, value_column=(heads + kv_heads) * dim)
    graph, stream, other = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        captured = step(caches[1])
    for lengths in [(0, 0), (700, 3), (5, 100000)]:
        cached._buf.copy_(torch.tensor(lengths, dtype=torch.int32))
        rows._buf.copy_(torch.randn(rows._buf.numel()).bfloat16())
        slots._buf.copy_(torch.randperm(128)[:tokens].int())
        eager = step(caches[0])
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager._buf, captured._buf)
        for a, b in zip(*caches):
            assert torch.equal(a._buf.view(torch.uint8), b._buf.view(torch.uint8))


def test_rows_past_4_gib(device):
    """Activations whose bytes are more than 32 bits count, in both layouts; the last rows are turned as the first ones."""
    from ttmi import capi

    torch.manual_seed(11)
    tokens, width, dim = 270016, 8192, 128
    rows = torch.zeros(tokens, width, dtype=torch.bfloat16, device="cuda")
    few = torch.randn(64, dim).bfloat16()
    f = frequencies_of(dim)
    put = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    cached, starts, freq = put([5, 900]), put([0, tokens - 40, tokens]), f.cuda()
    want, bound = model.rotate(few, [(0, 5 + tokens - 64 + i) if i < 24 else (1, 900 + i - 24) for i in range(64)], 1, dim, f)
    bound = model.as_bfloat16(want, bound)
    for layout in (capi.ROW_MAJOR, capi.TILE):
        rows.zero_()
        if layout == capi.ROW_MAJOR:
            rows[-64:, 8064:] = few.cuda()
        else:
            rows.view(-1, width // 32, 2, 2, 16, 16)[-2:, 252:].copy_(few.view(2, 2, 16, 4, 2, 16).permute(0, 3, 1, 4, 2, 5))
        out = torch.empty(tokens, dim, dtype=torch.bfloat16, device="cuda")
        capi.check(capi.lib().ttmi_rotate_heads(rows.data_ptr(), layout, tokens, width, 8064, 1, dim, cached.data_ptr(), starts.data_ptr(), 2, freq.data_ptr(), dim, 0, None, 0.0, 1.0, out.data_ptr(),
                                                capi._stream()))
        got = out[-64:].cpu() if layout == capi.ROW_MAJOR else out.view(-1, 4, 2, 2, 16, 16)[-2:].cpu().permute(0, 2, 4, 1, 3, 5).reshape(64, dim)
        check(got.view(want.shape), want, bound)
        assert not out[:1000].any()


@pytest.mark.parametrize("dtype", ["bfloat16", "bfloat8_b"])
def test_pages_past_4_gib(device, dtype):
    """Keys and values into the last pages of large caches, and attention over a window there behind sinks in the first ones: the bits of the same pages in small caches."""
    import ttnn

    torch.manual_seed(12)
    E, kv_heads, dim, page_size, heads, tokens = ttnn.experimental, 8, 128, 128, 16, 40
    many = 20000 if dtype == "bfloat16" else 36000
    wide = (heads + 2 * kv_heads) * dim
    rows = activations(device, torch.randn(300, wide).bfloat16(), "TILE_LAYOUT")
    chunk = activations(device, torch.randn(tokens, wide).bfloat16(), "TILE_LAYOUT")
    f = floats(device, frequencies_of(dim))
    answers = []
    for pages, table in [(3, [0, 1, 2]), (many, [1, many - 2, many - 1])]:
        caches = [E.allocate_paged_cache(pages, kv_heads, page_size, dim, dtype=getattr(ttnn, dtype), device=device) for _ in range(2)]
        made = []
        for given, n, cached in ((rows, 300, 0), (chunk, tokens, 300)):
            slots = integers(device, [table[p // page_size] * page_size + p % page_size for p in range(cached, cached + n)])
            lengths = integers(device, [cached]), integers(device, [0, n])
            queries = E.rotate_write_paged_cache(given, *caches, slots, *lengths, f, num_heads=heads, key_column=heads * dim, value_column=(heads + kv_heads) * dim)
            made.append(E.attend_paged_cache(queries, *caches, integers(device, [table]), *lengths, num_heads=heads, window=64, sinks=4)._buf.cpu())
        answers.append(made)
        del caches
    for a, b in zip(*answers):
        assert torch.equal(a, b) and not torch.isnan(a.float()).any()


# ---- frequencies, refusals of the host layer --------------------------------------------------------------------------------------------
def test_frequencies(device):
    import math

    import ttnn

    make = lambda *a, **kw: ttnn.to_torch(ttnn.experimental.rotary_frequencies(*a, device=device, **kw).cpu()).flatten().double()
    plain = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    assert torch.allclose(make(128), plain, rtol=2.0 ** -23)
    assert torch.allclose(make(128, theta=500000.0, factor=4.0), 500000.0 ** (-torch.arange(64, dtype=torch.float64) / 64) / 4, rtol=2.0 ** -23)
    got, turns = make(128, factor=8.0, original_length=8192), plain * 8192 / (2 * math.pi)
    assert torch.allclose(got[turns <= 1], plain[turns <= 1] / 8, rtol=2.0 ** -23) and torch.allclose(got[turns >= 4], plain[turns >= 4], rtol=2.0 ** -23)
    between = (turns > 1) & (turns < 4)
    share = (turns - 1) / 3
    assert between.any() and torch.allclose(got[between], (plain * (share + (1 - share) / 8))[between], rtol=2.0 ** -22)
    for bad in [dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=64, theta=0.0), dict(rotary_dim=64, factor=-1.0), dict(rotary_dim=64, original_length=0),
                dict(rotary_dim=64, original_length=8192, low_turns=4.0, high_turns=1.0)]:
        with pytest.raises(RuntimeError, match="rotary_frequencies"):
            ttnn.experimental.rotary_frequencies(**bad, device=device)


def test_the_host_layer_refuses(device):
    import ttnn

    E = ttnn.experimental
    rows, f = activations(device, torch.randn(4, 512).bfloat16(), "TILE_LAYOUT"), floats(device, frequencies_of(64))
    cached, starts, slots = integers(device, [0]), integers(device, [0, 4]), integers(device, range(4))
    rotate = lambda **kw: E.rotate_heads(**{**dict(input_tensor=rows, cached_lengths=cached, row_starts=starts, frequencies=f, num_heads=4, head_dim=64), **kw})
    rotate()
    for bad in [dict(num_heads=9), dict(num_heads=0), dict(head_dim=48), dict(column=288), dict(column=8), dict(frequencies=floats(device, torch.ones(40))), dict(frequencies=floats(device, torch.ones(4))),
                dict(frequencies=cached), dict(frequencies=None), dict(norm=floats(device, torch.ones(32))), dict(norm=cached), dict(row_starts=cached), dict(cached_lengths=f), dict(epsilon=-1.0),
                dict(magnitude=float("nan")), dict(input_tensor=f), dict(input_tensor=rows.cpu())]:
        with pytest.raises(RuntimeError):
            rotate(**bad)
    caches = [E.allocate_paged_cache(2, 2, 32, 64, dtype=ttnn.bfloat16, device=device) for _ in range(2)]
    write = lambda **kw: E.rotate_write_paged_cache(**{**dict(input_tensor=rows, key_cache=caches[0], value_cache=caches[1], slots=slots, cached_lengths=cached, row_starts=starts, frequencies=f,
                                                              num_heads=4, key_column=256, value_column=384), **kw})
    write()
    for bad in [dict(num_heads=9), dict(key_column=416), dict(value_column=8), dict(slots=cached), dict(value_cache=caches[0]), dict(key_norm=floats(device, torch.ones(128))), dict(row_starts=cached),
                dict(frequencies=floats(device, torch.ones(64))), dict(key_cache=rows)]:
        with pytest.raises(RuntimeError):
            write(**bad)
