"""The paged key/value cache of a decoder layer: the calls whose speed counts, from one token of one user to long prompts.

Three operators of ``ttnn.experimental`` work on it, in the order in which a serving step calls them:

  tables   paged_tables: the page tables, the slots of the new tokens and the row starts of a step, from the requests' lengths
  write    write_paged_cache: the new keys and values of a fused qkv projection go into their slots, bf16 or BFLOAT8_B
  attend   attend_paged_cache: the new tokens' queries against everything that their requests have in the cache

A case is a dict of plain values; its requests' lengths follow from these alone (``_lengths``), its values and the places of
its pages from the seed.  ``run`` computes the plain form in elementary torch operations in 32 bits, or, where ``own`` is
true, makes the calls of a user.  Both work on the same memory: caches, rows and outputs lie in TILE layout (32 x 32 tiles of
four 16 x 16 faces), or row-major where the case says so.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_GOLDEN = (5 ** 0.5 - 1) / 2


def listed():
    return [
        # one decode step of 32 users: the smallest call, launch latency counts
        {"name": "tables_decode", "kind": "tables", "requests": 32, "page_size": 64, "max_pages": 64, "cached_low": 1, "cached_high": 4000, "new_low": 1, "new_high": 1},
        # a step that takes in 257 prompts of many lengths, some of them empty, some with a common prefix already there
        {"name": "tables_prompts", "kind": "tables", "requests": 257, "page_size": 32, "max_pages": 300, "cached_low": 0, "cached_high": 4000, "new_low": 0, "new_high": 250},
        # one decode step of 32 users into a bf16 cache: 32 rows scattered over the pages
        {"name": "write_decode", "kind": "write", "requests": 32, "page_size": 64, "cached_low": 1, "cached_high": 500, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bf16", "layout": "tile"},
        # prompts of 4000 tokens in all into a BFLOAT8_B cache, which is then read back as the values it holds
        {"name": "write_prompts", "kind": "write", "requests": 5, "page_size": 64, "cached_low": 0, "cached_high": 90, "new_low": 500, "new_high": 1100, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bfp8_b", "layout": "tile"},
        # one user, one token, a short conversation: latency
        {"name": "decode_one", "kind": "attend", "requests": 1, "page_size": 64, "cached_low": 1500, "cached_high": 1500, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bf16", "window": 0, "layout": "tile"},
        # a decode step of 32 users, conversations of any length up to 4096, four query heads to a key head: the ordinary step
        {"name": "decode_32", "kind": "attend", "requests": 32, "page_size": 64, "cached_low": 1, "cached_high": 4095, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bf16", "window": 0, "layout": "tile"},
        # eight users with documents of up to 32768 tokens in a BFLOAT8_B cache: the largest reads
        {"name": "decode_long", "kind": "attend", "requests": 8, "page_size": 128, "cached_low": 20000, "cached_high": 32767, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bfp8_b", "window": 0, "layout": "tile"},
        # Falcon-7B's 71 query heads on one key head, 64 users, BFLOAT8_B cache
        {"name": "decode_one_key_head", "kind": "attend", "requests": 64, "page_size": 32, "cached_low": 500, "cached_high": 8000, "new_low": 1, "new_high": 1, "heads": 71, "kv_heads": 1, "head_dim": 64, "cache": "bfp8_b", "window": 0, "layout": "tile"},
        # five tokens each of 16 users, drafted by a small model and checked at once; row-major rows
        {"name": "check_drafts", "kind": "attend", "requests": 16, "page_size": 32, "cached_low": 900, "cached_high": 8000, "new_low": 5, "new_high": 5, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bf16", "window": 0, "layout": "rows"},
        # a chunk of 512 tokens of one long prompt behind the 7680 before it
        {"name": "chunk_512", "kind": "attend", "requests": 1, "page_size": 64, "cached_low": 7680, "cached_high": 7680, "new_low": 512, "new_high": 512, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bf16", "window": 0, "layout": "tile"},
        # a chunk of 300 tokens among 31 users who decode
        {"name": "mixed_step", "kind": "attend", "requests": 32, "page_size": 64, "cached_low": 1, "cached_high": 2000, "new_low": 1, "new_high": 1, "prompts": 1, "prompt": 300, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bf16", "window": 0, "layout": "tile"},
        # two whole prompts of 5000 and some tokens, every token looks at the 4096 before it, BFLOAT8_B cache: bound by the matrix cores
        {"name": "prompts_windowed", "kind": "attend", "requests": 2, "page_size": 64, "cached_low": 0, "cached_high": 0, "new_low": 5000, "new_high": 5500, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "bfp8_b", "window": 4096, "layout": "tile"},
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    def between(name, low, high):
        return {name + "_low": low, name + "_high": high}

    kind = rng.choice(["tables", "write", "attend", "attend", "attend", "attend"])
    page_size = rng.choice([32, 64, 64, 96, 128, 256])
    if kind == "tables":
        longest = _spread(rng, 64, 9000)
        new = _spread(rng, 1, 250)
        return {"kind": kind, "requests": _spread(rng, 1, 300), "page_size": page_size, "max_pages": -(-(longest + new) // page_size) + rng.randint(0, 5),
                **between("cached", rng.randint(0, longest), longest), **between("new", rng.randint(0, new), new)}
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (71, 1, 64), (16, 16, 64), (12, 4, 96), (16, 2, 256)])
    shared = {"page_size": page_size, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "cache": rng.choice(["bf16", "bfp8_b"]),
              "layout": rng.choice(["tile", "tile", "rows"])}
    if kind == "write":
        total = _spread(rng, 1, 3800)
        requests = rng.randint(1, min(total, 40))
        new = total // requests
        return {"kind": kind, "requests": requests, **between("cached", 0, _spread(rng, 1, 500)), **between("new", new, new), **shared}
    while True:
        style = rng.choice(["decode", "decode", "drafts", "chunks", "prompts"])
        requests = _spread(rng, 1, {"decode": 96, "drafts": 32, "chunks": 4, "prompts": 8}[style])
        new = {"decode": 1, "drafts": rng.randint(2, 16), "chunks": _spread(rng, 17, 1024), "prompts": _spread(rng, 32, 4096)}[style]
        longest = 1 if style == "prompts" else _spread(rng, 64, 32000)
        case = {"kind": kind, "requests": requests, **between("cached", *((0, 0) if style == "prompts" else (rng.randint(1, longest), longest))),
                **between("new", rng.randint(1, new) if style == "prompts" else new, new), "window": rng.choice([0, 0, 0, _spread(rng, 16, 4096)]), **shared}
        largest = {w: max(work(c)[w] for c in listed()) for w in ("bytes", "flops")}
        padded = requests * heads * new * (longest + new)          # scores of the plain form, every request as long as the longest
        if all(work(case)[w] <= largest[w] for w in largest) and padded <= 2 * 32 * 5500 ** 2 and requests * kv_heads * head_dim * (longest + new) <= 8 * 8 * 128 * 32768:
            return case


# ---- what follows from a case alone ----------------------------------------------------------------------------------------------
def _lengths(case):
    """(cached, new) of every request: spread evenly over the case's ranges, in no order."""
    def spaced(name, turn):
        low, high = case[name + "_low"], case[name + "_high"]
        return [low + int((high - low + 1) * ((i * _GOLDEN + turn) % 1.0)) for i in range(case["requests"])]
    cached, new = spaced("cached", 0.37), spaced("new", 0.71)
    for i in range(case.get("prompts", 0)):
        new[i * case["requests"] // case["prompts"]] = case["prompt"]
    return cached, new


def _pages(length, page_size):
    return -(-length // page_size)


def _columns(case):
    """Columns of a row of the fused qkv projection: first key column, first value column, all."""
    queries, keys = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    return queries, queries + keys, queries + 2 * keys


def _element_bytes(case):
    return 2.0 if case["cache"] == "bf16" else 1088 / 1024


def work(case):
    cached, new = _lengths(case)
    tokens, requests = sum(new), case["requests"]
    if case["kind"] == "tables":
        return {"bytes": 4 * (2 * requests + 2 * requests * case["max_pages"] + tokens + requests + 3), "flops": 0}
    per_token = 2 * case["kv_heads"] * case["head_dim"]
    if case["kind"] == "write":
        return {"bytes": tokens * (per_token * (2.0 + _element_bytes(case)) + 4), "flops": 0}
    window = case["window"] or 1 << 30
    pairs = sum(_sum_of_reach(c, n, window) for c, n in zip(cached, new))
    seen = sum(min(c + n, n + window - 1) for c, n in zip(cached, new) if n)
    return {"bytes": seen * per_token * _element_bytes(case) + tokens * case["heads"] * case["head_dim"] * 4 + 4 * (seen / case["page_size"] + 2 * requests),
            "flops": 4 * case["head_dim"] * case["heads"] * pairs}


def _sum_of_reach(cached, new, window):
    """sum over the new tokens of how many tokens each looks at: min(its position + 1, window)."""
    growing = max(0, min(new, window - cached))                    # tokens that the window does not cut off
    return growing * cached + growing * (growing + 1) // 2 + (new - growing) * window


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _tiles(x):
    """[..., h, w] -> the same elements in the order of whole 32 x 32 tiles of four 16 x 16 faces: [..., h/32, w/32, 2, 2, 16, 16]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32, 0, -x.shape[-2] % 32))
    h, w = x.shape[-2:]
    x = x.reshape(*x.shape[:-2], h // 32, 2, 16, w // 32, 2, 16)
    n = x.dim()
    return x.permute(*range(n - 6), n - 6, n - 3, n - 5, n - 2, n - 4, n - 1)


def _cache_shape(case, pages):
    """A cache as both sides see it: [pages, heads, tile rows, tile columns] and a tile, 2 x 2 faces of 16 x 16 or its packed bytes."""
    grid = (pages, case["kv_heads"], case["page_size"] // 32, case["head_dim"] // 32)
    return grid + ((2, 2, 16, 16) if case["cache"] == "bf16" else (1088,))


def _inputs(case, seed):
    """The values of a case as plain tensors: rows bf16, caches in TILE layout, tables and lengths int32."""
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    cached, new = _lengths(case)
    requests, page_size, tokens = case["requests"], case["page_size"], sum(new)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    held = [_pages(c, page_size) for c in cached]
    want = [_pages(c + n, page_size) for c, n in zip(cached, new)]
    width = case.get("max_pages", max(want) + 1)
    spare = 4
    order = torch.randperm(sum(want) + spare, generator=generator, device="cuda").int()
    there = held if case["kind"] == "tables" else want             # a step that has its tables has its pages
    ends = torch.tensor(there, device="cuda").cumsum(0)
    column = torch.arange(width, device="cuda")
    index = (ends - torch.tensor(there, device="cuda"))[:, None] + column
    table = torch.where(column < torch.tensor(there, device="cuda")[:, None], order[index.clamp(max=order.numel() - 1)], -1).int()
    state = {"kind": case["kind"], "page_size": page_size, "page_table": table, "cached": ints(cached), "new": ints(new)}
    if case["kind"] == "tables":
        state["free_pages"] = order[sum(held):].contiguous()
        state["tokens"] = (tokens + 31) // 32 * 32                 # rows of the step's activations: whole tiles
        return state
    starts = [sum(new[:r]) for r in range(requests + 1)]
    state["row_starts"], state["tokens"], state["columns"] = ints(starts), tokens, _columns(case)
    state["rows"] = torch.randn(tokens, _columns(case)[2], generator=generator, device="cuda").bfloat16()
    if case["kind"] == "attend":
        state["rows"] *= 2                                         # scores with a spread of 2: some tokens count, most do not
    shape = _cache_shape(case, sum(want) + spare)
    for name in ("keys", "values"):
        values = torch.randn(shape[:4] + (2, 2, 16, 16), generator=generator, device="cuda")
        state[name] = values.bfloat16() if case["cache"] == "bf16" else _packed(values)
        del values
    if case["kind"] == "write":
        position = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).cuda()
        request = torch.repeat_interleave(torch.arange(requests), torch.tensor(new)).cuda()
        state["slots"] = (table[request, position // page_size] * page_size + position % page_size).int()
    state["layout"], state["cache"], state["heads"], state["head_dim"], state["window"] = (case.get(k) for k in ("layout", "cache", "heads", "head_dim", "window"))
    state["longest"], state["most_new"] = max(c + n for c, n in zip(cached, new)), max(new)
    return state


def _step(exponent):
    """2^(exponent - 133), what a mantissa of 1 stands for, put together from its bits; numbers under 2^-126 are not among the values here."""
    return ((exponent - 6).clamp(min=1) << 23).view(torch.float32)


def _exponent_and_codes(x):
    """Block floats of 16 neighbours each (the last dimension): the exponent byte that they share and sign | 7-bit mantissa bytes, rounded half up."""
    exponent = (x.view(torch.int32) >> 23 & 0xff).amax(dim=-1, keepdim=True)
    mantissa = torch.where(exponent == 0, 0.0, torch.floor(x.abs() / _step(exponent) + 0.5).clamp(max=127.0)).to(torch.uint8)
    return exponent[..., 0].to(torch.uint8), mantissa | (x.view(torch.int32) >> 31 & 1).to(torch.uint8) << 7


def _packed(x):
    """[..., 2, 2, 16, 16] -> [..., 1088]: 64 exponent bytes, then 1024 codes, face by face."""
    exponents, codes = _exponent_and_codes(x)
    return torch.cat([exponents.flatten(-3), codes.flatten(-4)], dim=-1)


def _unpacked(tiles):
    """[..., 1088] packed bytes -> the values in 32 bits, [..., 2, 2, 16, 16]."""
    code = tiles[..., 64:].unflatten(-1, (2, 2, 16, 16)).int()
    return (code & 127).float() * _step(tiles[..., :64].unflatten(-1, (2, 2, 16, 1)).int()) * (1 - (code >> 7) * 2)


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        state["handles"] = _handles(case, state)
    return state


def _package():
    package = os.path.join(os.getcwd(), "tt-metal_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import ttnn

    return ttnn


def _handles(case, state):
    """The ttnn tensors that a serving program holds: lengths and tables, the activations of the layer, the caches."""
    ttnn = _package()
    device = ttnn.open_device(torch.cuda.current_device())
    handles = {"ttnn": ttnn}
    handles |= {name: ttnn.from_torch(state[name], device=device) for name in ("cached", "new", "page_table", "free_pages", "row_starts", "slots") if name in state}
    if case["kind"] == "tables":
        return handles
    layout = ttnn.TILE_LAYOUT if case["layout"] == "tile" else ttnn.ROW_MAJOR_LAYOUT
    handles["rows"] = ttnn.from_torch(state["rows"][None, None], dtype=ttnn.bfloat16, layout=layout, device=device)
    dtype = ttnn.bfloat16 if case["cache"] == "bf16" else ttnn.bfloat8_b
    for name in ("keys", "values"):
        cache = ttnn.experimental.allocate_paged_cache(state[name].shape[0], case["kv_heads"], case["page_size"], case["head_dim"], dtype=dtype, device=device)
        cache._buf.view(torch.uint8).copy_(state[name].flatten().view(torch.uint8))
        handles[name] = cache
    return handles


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state, state["handles"])
    return {"tables": _plain_tables, "write": _plain_write, "attend": _plain_attend}[state["kind"]](state)


def _own(state, handles):
    ttnn = handles["ttnn"]
    if state["kind"] == "tables":
        made = ttnn.experimental.paged_tables(handles["cached"], handles["new"], handles["page_table"], handles["free_pages"],
                                              page_size=state["page_size"], num_tokens=state["tokens"])
        return [t._buf for t in made]
    if state["kind"] == "write":
        ttnn.experimental.write_paged_cache(handles["rows"], handles["keys"], handles["values"], handles["slots"],
                                            key_column=state["columns"][0], value_column=state["columns"][1])
        if state["cache"] == "bf16":
            return [handles["keys"]._buf, handles["values"]._buf]
        return [ttnn.clone(handles[name], dtype=ttnn.bfloat16)._buf for name in ("keys", "values")]
    out = ttnn.experimental.attend_paged_cache(handles["rows"], handles["keys"], handles["values"], handles["page_table"], handles["cached"], handles["row_starts"],
                                               num_heads=state["heads"], window=state["window"] or None)
    return out._buf


def _plain_tables(state):
    page_size, table, free = state["page_size"], state["page_table"], state["free_pages"]
    cached, new = state["cached"], state["new"]
    requests, width = table.shape
    held = ((cached + page_size - 1) // page_size).clamp(max=width)
    want = ((cached + new + page_size - 1) // page_size).clamp(max=width)
    taken = (want - held).cumsum(0).int()
    column = torch.arange(width, dtype=torch.int32, device="cuda")
    index = (taken - want)[:, None] + column                       # base + j - held
    fresh = torch.where((column < want[:, None]) & (index < free.numel()), free[index.clamp(0, free.numel() - 1)], -1)
    out = torch.where(column < held[:, None], table, fresh)
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0).int()])
    token = torch.arange(state["tokens"], dtype=torch.int32, device="cuda")
    request = (token[:, None] >= starts[1:]).sum(dim=1).clamp(max=requests - 1)
    position = cached[request] + token - starts[request]
    page = out[request, (position // page_size).clamp(max=width - 1)]
    there = (token < starts[-1]) & (position // page_size < width) & (page >= 0)
    slots = torch.where(there, page * page_size + position % page_size, -1)
    got = taken[-1:].clamp(max=free.numel())
    return [out, slots, starts, torch.cat([got, taken[-1:] - got])]


def _plain_write(state):
    slots = state["slots"].long()
    page, within = slots // state["page_size"], slots % state["page_size"]
    out = []
    for name, column in (("keys", state["columns"][0]), ("values", state["columns"][1])):
        cache = state[name]
        heads, across = cache.shape[1], cache.shape[3]
        rows = state["rows"][:, column:column + heads * across * 32].view(-1, heads, across, 2, 16)
        tile, down, row = within // 32, within // 16 % 2, within % 16
        if state["cache"] == "bf16":
            cache[page, :, tile, :, down, :, row] = rows           # tokens, heads, tile columns, face columns, 16 elements
            out.append(cache.view(-1))
            continue
        exponents, codes = _exponent_and_codes(rows.float())
        cache[..., :64].unflatten(-1, (2, 2, 16))[page, :, tile, :, down, :, row] = exponents
        cache[..., 64:].unflatten(-1, (2, 2, 16, 16))[page, :, tile, :, down, :, row] = codes
        out.append(_unpacked(cache).bfloat16().view(-1))
    return out


def _gathered(state, name):
    """[requests, heads, tokens, head dim] in 32 bits: the pages of every request in order, as far as the longest request goes."""
    pages = -(-state["longest"] // state["page_size"])
    tiles = state[name][state["page_table"][:, :pages].clamp(min=0).long()]
    tiles = tiles.float() if state["cache"] == "bf16" else _unpacked(tiles)
    requests, pages, heads, down, across = tiles.shape[:5]
    return tiles.permute(0, 2, 1, 3, 5, 7, 4, 6, 8).reshape(requests, heads, pages * down * 32, across * 32)


def _plain_attend(state):
    tokens, heads, dim = state["tokens"], state["heads"], state["head_dim"]
    keys, values = _gathered(state, "keys"), _gathered(state, "values")
    requests, kv_heads, length = keys.shape[:3]
    group, most = heads // kv_heads, state["most_new"]
    starts, new = state["row_starts"][:-1, None].long(), state["new"][:, None]
    step = torch.arange(most, device="cuda")
    at = (starts + step).clamp(max=tokens - 1)                     # row of each request's new tokens, the shorter ones padded
    query = state["rows"][:, :heads * dim].float()[at].view(requests, most, kv_heads, group, dim)
    query = query.permute(0, 2, 3, 1, 4).reshape(requests, kv_heads, group * most, dim)
    scores = torch.matmul(query, keys.transpose(2, 3).contiguous()) * dim ** -0.5
    position, place = state["cached"][:, None] + step, torch.arange(length, device="cuda")
    seen = place <= position[..., None]
    if state["window"]:
        seen = seen & (place > position[..., None] - state["window"])
    scores = scores.view(requests, kv_heads, group, most, length).masked_fill_(~seen[:, None, None], -math.inf)
    scores = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.view(requests, kv_heads, group * most, length), values).view(requests, kv_heads, group, most, dim) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(requests * most, heads * dim)
    token = torch.arange(tokens, device="cuda")
    request = (token[:, None] >= state["row_starts"][1:]).sum(dim=1)
    out = out[request * most + token - state["row_starts"][request]].bfloat16()
    return _tiles(out).reshape(-1) if state["layout"] == "tile" else out[None, None]


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------
def _held(tiles, cache):
    """What a cache holds, in 64 bits."""
    if cache == "bf16":
        return tiles.double()
    signs, sizes = 1.0 - 2.0 * (tiles[..., 64:] >= 128), (tiles[..., 64:] % 128).double()
    scale = torch.exp2(tiles[..., :64].double() - 133.0).repeat_interleave(16, dim=-1)
    return (signs * sizes * scale).unflatten(-1, (2, 2, 16, 16))


def exact(case, seed):
    state = _inputs(case, seed)
    cached, new = _lengths(case)
    page_size = case["page_size"]
    if case["kind"] == "tables":
        table, free = state["page_table"].tolist(), iter(state["free_pages"].tolist())
        width, slots, starts, taken = case["max_pages"], [], [0], 0
        for row, c, n in zip(table, cached, new):
            for j in range(_pages(c, page_size), min(width, _pages(c + n, page_size))):
                row[j] = next(free)
                taken += 1
            slots += [row[p // page_size] * page_size + p % page_size for p in range(c, c + n)]
            starts.append(starts[-1] + n)
        slots += [-1] * (state["tokens"] - len(slots))
        return [torch.tensor(v, dtype=torch.int32) for v in (table, slots, starts, [taken, 0])]
    if case["kind"] == "write":
        out = []
        for name, column in zip(("keys", "values"), _columns(case)):
            cache = _held(state[name], case["cache"])
            pages, heads, down, across = cache.shape[:4]
            cache = cache.permute(0, 1, 2, 4, 6, 3, 5, 7).reshape(pages, heads, down * 32, across * 32).contiguous()
            rows = state["rows"][:, column:column + heads * across * 32].double().view(-1, heads, across * 2, 16)
            if case["cache"] != "bf16":
                step = torch.exp2(torch.frexp(rows.abs().amax(dim=-1, keepdim=True))[1].double() - 7)
                rows = torch.sign(rows) * torch.clamp(torch.floor(rows.abs() / step + 0.5), max=127) * step
            slots = state["slots"].long()
            cache[slots // page_size, :, slots % page_size] = rows.flatten(2)
            out.append(_tiles(cache).reshape(-1))
        return out
    heads, dim, group = case["heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(state["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    first = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        table = state["page_table"][r, :_pages(c + n, page_size)].long()
        both = []
        for name in ("keys", "values"):
            tiles = _held(state[name][table], case["cache"])
            both.append(tiles.permute(1, 0, 2, 4, 6, 3, 5, 7).reshape(case["kv_heads"], -1, dim)[:, :c + n])
        query = state["rows"][first:first + n, :heads * dim].double().view(n, heads, dim)
        position, place = torch.arange(c, c + n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
        seen = (place <= position) & (place > position - (case["window"] or 1 << 30))
        for h in range(heads):
            scores = query[:, h] @ both[0][h // group].T / math.sqrt(dim)
            out[first:first + n, h] = torch.softmax(scores.masked_fill(~seen, -math.inf), dim=-1) @ both[1][h // group]
        first += n
    out = out.flatten(1)
    return _tiles(out).reshape(-1) if case["layout"] == "tile" else out[None, None]
