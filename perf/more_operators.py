"""What a decoder layer does around its paged key/value cache: positions, long conversations, several continuations of one.

Five operators of ``ttnn.experimental``, which stand beside those that make the tables of a step, write and attend:

  rotate    rotate_heads: the norm of every head and the rotation by its token's position, from the rows of a fused qkv projection
  write     rotate_write_paged_cache: the same for queries and keys, the keys and the values going straight into their pages
  attend    attend_paged_cache with a window and sinks: the last tokens of a conversation and its first few
  fork      fork_paged_tables and copy_paged_pages: several continuations share what they have in common, and copy the page they go on in
  release   release_paged_pages: pages that nobody needs any longer, from lengths and tables

A case is a dict of plain values; its requests' lengths follow from these alone (``_lengths``), its values and the places of
its pages from the seed.  ``run`` computes the plain form in elementary torch operations in 32 bits (angles in 64), or, where
``own`` is true, makes the calls of a user.  Both work on the same memory: caches, rows and outputs lie in TILE layout (32 x 32
tiles of four 16 x 16 faces), or row-major where the case says so.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_GOLDEN = (5 ** 0.5 - 1) / 2
_EPSILON = 1e-5


def listed():
    return [
        # queries of one decode step of 32 users, conversations of up to 4000 tokens: the smallest call, launch latency counts
        {"name": "rotate_decode", "kind": "rotate", "requests": 32, "cached_low": 1, "cached_high": 4000, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "rotary_dim": 128, "interleaved": False, "norm": False, "factor": 1.0, "magnitude": 1.0, "layout": "tile"},
        # prompts of 8000 tokens in all, Falcon-7B's 71 heads of 64 elements, neighbours rotated together, a quarter of them at rest; row-major rows
        {"name": "rotate_prompts", "kind": "rotate", "requests": 3, "cached_low": 0, "cached_high": 30000, "new_low": 2100, "new_high": 3060, "heads": 71, "kv_heads": 1, "head_dim": 64,
         "rotary_dim": 48, "interleaved": True, "norm": False, "factor": 8.0, "magnitude": 1.2, "layout": "rows"},
        # one decode step of 32 users: queries and keys with their norms, into a bf16 cache
        {"name": "write_decode", "kind": "write", "requests": 32, "cached_low": 1, "cached_high": 500, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "rotary_dim": 128, "interleaved": False, "norm": True, "factor": 1.0, "magnitude": 1.0, "layout": "tile", "page_size": 64, "cache": "bf16"},
        # five drafted tokens of each of 23 users, heads of 256 elements of which a quarter turns, no norms; row-major rows
        {"name": "write_drafts", "kind": "write", "requests": 23, "cached_low": 100, "cached_high": 900, "new_low": 5, "new_high": 5, "heads": 16, "kv_heads": 2, "head_dim": 256,
         "rotary_dim": 64, "interleaved": False, "norm": False, "factor": 1.0, "magnitude": 1.0, "layout": "rows", "page_size": 32, "cache": "bf16"},
        # prompts of 8000 tokens in all with norms into a BFLOAT8_B cache, which is then read back as the values it holds
        {"name": "write_prompts", "kind": "write", "requests": 5, "cached_low": 0, "cached_high": 90, "new_low": 1200, "new_high": 2000, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "rotary_dim": 128, "interleaved": False, "norm": True, "factor": 8.0, "magnitude": 1.2, "layout": "tile", "page_size": 64, "cache": "bfp8_b"},
        # one user, one token, a conversation of 60000 tokens of which the last 1024 and the first four count: latency
        {"name": "sinks_one", "kind": "attend", "requests": 1, "cached_low": 60000, "cached_high": 60000, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "layout": "tile", "page_size": 64, "cache": "bf16", "window": 1024, "sinks": 4},
        # a decode step of 32 users, conversations of up to 12000 tokens, the last 4096 and the first four of each: the ordinary step
        {"name": "sinks_decode", "kind": "attend", "requests": 32, "cached_low": 1, "cached_high": 12000, "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "layout": "tile", "page_size": 64, "cache": "bf16", "window": 4096, "sinks": 4},
        # two whole prompts of 5000 and some tokens, BFLOAT8_B cache, a window of 1024 behind a common preamble of 100: bound by the matrix cores
        {"name": "sinks_prompts", "kind": "attend", "requests": 2, "cached_low": 0, "cached_high": 0, "new_low": 5000, "new_high": 5500, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "layout": "tile", "page_size": 64, "cache": "bfp8_b", "window": 1024, "sinks": 100},
        # one prompt goes on in four ways, one layer: the smallest fork
        {"name": "fork_prompt", "kind": "fork", "requests": 1, "cached_low": 700, "cached_high": 700, "beams": 1, "children": 4, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "cache": "bf16", "layers": 1},
        # a step of beam search, four beams for each of 24 users, the caches of eight layers
        {"name": "fork_beams", "kind": "fork", "requests": 96, "cached_low": 100, "cached_high": 400, "beams": 4, "children": 96, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "cache": "bf16", "layers": 8},
        # a pool of 4096 pages, 32 users, behind the window of 1024
        {"name": "release_decode", "kind": "release", "requests": 32, "cached_low": 1, "cached_high": 4000, "page_size": 64, "max_pages": 64, "num_pages": 4096, "window": 1024, "sinks": 4,
         "shared": 2},
        # a large server's pool of 300000 pages, 1000 conversations of up to 16000 tokens with a common preamble
        {"name": "release_server", "kind": "release", "requests": 1000, "cached_low": 300, "cached_high": 16000, "page_size": 32, "max_pages": 512, "num_pages": 300000, "window": 0, "sinks": 0,
         "shared": 8},
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    def between(name, low, high):
        return {name + "_low": low, name + "_high": high}

    kind = rng.choice(["rotate", "write", "attend", "attend", "attend", "fork", "release"])
    page_size = rng.choice([32, 64, 64, 96, 128, 256])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (71, 1, 64), (16, 16, 64), (12, 4, 96), (16, 2, 256)])
    shape = {"heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}
    cache = {"page_size": page_size, "cache": rng.choice(["bf16", "bfp8_b"])}
    if kind == "release":
        longest = _spread(rng, 64, 16000)
        requests = _spread(rng, 1, 900)
        width = -(-longest // page_size) + rng.randint(0, 5)
        shared = rng.randint(0, 8)
        return {"kind": kind, "requests": requests, **between("cached", rng.randint(0, longest), longest), "page_size": page_size, "max_pages": width,
                "num_pages": shared + min(requests * width + _spread(rng, 1, 1000), 299000), "window": rng.choice([0, _spread(rng, 16, 8000)]), "sinks": rng.choice([0, 1, 4, 100]), "shared": shared}
    if kind == "fork":
        beams = rng.randint(1, 6)
        users = _spread(rng, 1, 16)
        longest = _spread(rng, 32, 400)
        layers = 1 if cache["cache"] == "bfp8_b" else rng.choice([1, 2, 4])
        return {"kind": kind, "requests": users * beams, **between("cached", rng.randint(1, longest), longest), "beams": beams, "children": users * beams * rng.choice([1, 1, 2]),
                **shape, **cache, "page_size": min(page_size, 128), "layers": layers}
    layout = {"layout": rng.choice(["tile", "tile", "rows"])}
    turn = {"rotary_dim": rng.choice([head_dim, head_dim, head_dim // 2, head_dim - 16, 16]), "interleaved": rng.choice([False, False, True]), "norm": rng.choice([False, True]),
            "factor": rng.choice([1.0, 4.0, 8.0]), "magnitude": rng.choice([1.0, 1.2])}
    if kind in ("rotate", "write"):
        total = _spread(rng, 1, 7000)
        requests = rng.randint(1, min(total, 40))
        new = total // requests
        case = {"kind": kind, "requests": requests, **between("cached", 0, _spread(rng, 1, 100000 if kind == "rotate" else 400)), **between("new", new, new), **shape, **turn, **layout}
        return {**case, **cache} if kind == "write" else case
    while True:
        style = rng.choice(["decode", "decode", "drafts", "chunks", "prompts"])
        requests = _spread(rng, 1, {"decode": 96, "drafts": 32, "chunks": 4, "prompts": 8}[style])
        new = {"decode": 1, "drafts": rng.randint(2, 16), "chunks": _spread(rng, 17, 1024), "prompts": _spread(rng, 32, 4096)}[style]
        longest = 1 if style == "prompts" else _spread(rng, 64, 32000)
        case = {"kind": kind, "requests": requests, **between("cached", *((0, 0) if style == "prompts" else (rng.randint(1, longest), longest))),
                **between("new", rng.randint(1, new) if style == "prompts" else new, new), "window": _spread(rng, 16, 4096), "sinks": rng.choice([1, 4, 4, 32, rng.randint(1, 300)]),
                **shape, **cache, **layout}
        largest = {w: max(work(c)[w] for c in listed()) for w in ("bytes", "flops")}
        padded = requests * heads * new * min(longest + new, case["window"] + case["sinks"] + new)
        if all(work(case)[w] <= largest[w] for w in largest) and padded <= 2 * 32 * 5500 ** 2 and requests * kv_heads * head_dim * (longest + new) <= 8 * 8 * 128 * 32768:
            return case


# ---- what follows from a case alone ----------------------------------------------------------------------------------------------
def _lengths(case):
    """(cached, new) of every request: spread evenly over the case's ranges, in no order."""
    def spaced(name, turn):
        low, high = case.get(name + "_low", 0), case.get(name + "_high", 0)
        return [low + int((high - low + 1) * ((i * _GOLDEN + turn) % 1.0)) for i in range(case["requests"])]
    return spaced("cached", 0.37), spaced("new", 0.71)


def _parents(case):
    """Which request every continuation goes on from: one of the beams of its user, some of them more than once."""
    each = case["children"] * case["beams"] // case["requests"]    # continuations of a user
    return [i // each * case["beams"] + int(case["beams"] * ((i * _GOLDEN + 0.19) % 1.0)) for i in range(case["children"])]


def _copies(case):
    """(child, its parent) for every continuation that needs a copy of a page begun: all of a parent's but the first."""
    cached, seen, copies = _lengths(case)[0], set(), []
    for child, parent in enumerate(_parents(case)):
        if parent in seen and cached[parent] % case["page_size"]:
            copies.append((child, parent))
        seen.add(parent)
    return copies


def _pages(length, page_size):
    return -(-length // page_size)


def _columns(case):
    """Columns of a row of the fused qkv projection: first key column, first value column, all."""
    queries, keys = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    return queries, queries + keys, queries + 2 * keys


def _element_bytes(case):
    return 2.0 if case["cache"] == "bf16" else 1088 / 1024


def _page_bytes(case):
    return case["kv_heads"] * case["page_size"] * case["head_dim"] * _element_bytes(case)


def work(case):
    cached, new = _lengths(case)
    tokens, requests = sum(new), case["requests"]
    if case["kind"] == "release":
        return {"bytes": 4 * (2 * requests * case["max_pages"] + requests + case["num_pages"] + 2), "flops": 0}
    if case["kind"] == "fork":
        children, copies = case["children"], len(_copies(case))
        width = _pages(max(cached), case["page_size"]) + 1
        return {"bytes": 4 * (2 * children * width + requests + 4 * children + copies) + 4 * case["layers"] * copies * _page_bytes(case), "flops": 0}
    queries, keys = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    if case["kind"] in ("rotate", "write"):
        turned = tokens * (queries + (keys if case["kind"] == "write" else 0))
        written = tokens * 2 * keys * (2.0 + _element_bytes(case)) + 4 * tokens if case["kind"] == "write" else 0
        return {"bytes": tokens * queries * 4 + written + 8 * requests + 2 * case["rotary_dim"], "flops": turned * (3 + (4 if case["norm"] else 0))}
    window, sinks = case["window"], case["sinks"]
    pairs = seen = 0
    for c, n in zip(cached, new):
        pairs += sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(c, c + n))
        seen += min(c + n, n + window - 1 + min(sinks, max(0, c + 1 - window)))
    return {"bytes": seen * 2 * keys * _element_bytes(case) + tokens * queries * 4 + 4 * (seen / case["page_size"] + 2 * requests), "flops": 4 * case["head_dim"] * case["heads"] * pairs}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _tiles(x):
    """[..., h, w] -> the same elements in the order of whole 32 x 32 tiles of four 16 x 16 faces: [..., h/32, w/32, 2, 2, 16, 16]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32, 0, -x.shape[-2] % 32))
    h, w = x.shape[-2:]
    x = x.reshape(*x.shape[:-2], h // 32, 2, 16, w // 32, 2, 16)
    n = x.dim()
    return x.permute(*range(n - 6), n - 6, n - 3, n - 5, n - 2, n - 4, n - 1)


def _frequencies(case):
    """Angles per token, [rotary_dim / 2] in 64 bits: powers of 10000; for a context longer than the 8192 tokens of training, those that turn less
    than once in it are divided by the factor, those that turn more than four times stay, the ones between go from the one to the other."""
    pairs = case["rotary_dim"] // 2
    plain = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    stays = ((plain * 8192 / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
    return plain * (stays + (1.0 - stays) / case["factor"])


def _inputs(case, seed):
    """The values of a case as plain tensors: rows bf16, caches in TILE layout, tables and lengths int32."""
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    cached, new = _lengths(case)
    requests, tokens = case["requests"], sum(new)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device="cuda")

    state = {"kind": case["kind"], "cached": ints(cached), "tokens": tokens, **{k: v for k, v in case.items() if k not in ("name", "requests")}}
    if case["kind"] != "rotate":
        page_size = case["page_size"]
        want = [_pages(c + n, page_size) for c, n in zip(cached, new)]
        width = case.get("max_pages", max(want) + 1)
        pool = case.get("num_pages", sum(want) + (case["children"] if case["kind"] == "fork" else 4))
        order = torch.randperm(pool, generator=generator, device="cuda").int()
        shared = case.get("shared", 0)                             # pages of a preamble that all have in common
        lengths = torch.tensor(want, device="cuda")
        column = torch.arange(width, device="cuda")
        index = shared + (lengths.cumsum(0) - lengths)[:, None] + column
        table = torch.where(column < shared, order[column.clamp(max=pool - 1)], order[index % pool])
        state["page_table"] = torch.where(column < lengths[:, None], table, -1).int()
        state["pages"] = pool
        if case["kind"] == "release":
            return state
    if case["kind"] == "fork":
        state["parents"], state["free_pages"] = ints(_parents(case)), order[sum(want):].contiguous()
    else:
        state["row_starts"], state["columns"] = ints([sum(new[:r]) for r in range(requests + 1)]), _columns(case)
        state["rows"] = normal(tokens, _columns(case)[2]).bfloat16()
    if case["kind"] in ("rotate", "write"):
        state["frequencies"] = _frequencies(case).float().cuda()
        for name in ("query_norm", "key_norm"):
            state[name] = 1.0 + 0.2 * normal(case["head_dim"]) if case["norm"] else None
    if case["kind"] == "rotate":
        return state
    if case["kind"] == "attend":
        state["rows"] *= 2                                         # scores with a spread of 2: some tokens count, most do not
        state["longest"], state["most_new"] = max(c + n for c, n in zip(cached, new)), max(new)
        state["reach"] = max(c + n - max(0, c + 1 - case["window"] - case["sinks"]) for c, n in zip(cached, new))
    if case["kind"] == "write":
        position = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).cuda()
        request = torch.repeat_interleave(torch.arange(requests), torch.tensor(new)).cuda()
        state["slots"] = (state["page_table"][request, position // page_size] * page_size + position % page_size).int()
    shape = (pool, case["kv_heads"], page_size // 32, case["head_dim"] // 32, 2, 2, 16, 16)
    state["caches"] = []                                           # keys, values, layer by layer
    for _ in range(2 * case.get("layers", 1)):
        values = normal(*shape)
        state["caches"].append(values.bfloat16() if case["cache"] == "bf16" else _packed(values))
        del values
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


def _values_of(codes, exponents):
    """Codes [..., 16] and the exponent bytes [...] that they share -> the values in 32 bits."""
    code = codes.int()
    return (code & 127).float() * _step(exponents.int()[..., None]) * (1 - (code >> 7) * 2)


def _unpacked(tiles):
    """[..., 1088] packed bytes -> the values in 32 bits, [..., 2, 2, 16, 16]."""
    return _values_of(tiles[..., 64:].unflatten(-1, (2, 2, 16, 16)), tiles[..., :64].unflatten(-1, (2, 2, 16)))


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
    """The ttnn tensors that a serving program holds: lengths and tables, frequencies and norms, the activations of the layer, the caches."""
    ttnn = _package()
    device = ttnn.open_device(torch.cuda.current_device())
    handles = {"ttnn": ttnn, "query_norm": None, "key_norm": None}
    names = ("cached", "page_table", "free_pages", "row_starts", "slots", "parents", "frequencies", "query_norm", "key_norm")
    handles |= {name: ttnn.from_torch(state[name], device=device) for name in names if state.get(name) is not None}
    if "rows" in state:
        layout = ttnn.TILE_LAYOUT if case["layout"] == "tile" else ttnn.ROW_MAJOR_LAYOUT
        handles["rows"] = ttnn.from_torch(state["rows"][None, None], dtype=ttnn.bfloat16, layout=layout, device=device)
    handles["caches"] = []
    for values in state.get("caches", ()):
        dtype = ttnn.bfloat16 if case["cache"] == "bf16" else ttnn.bfloat8_b
        cache = ttnn.experimental.allocate_paged_cache(values.shape[0], case["kv_heads"], case["page_size"], case["head_dim"], dtype=dtype, device=device)
        cache._buf.view(torch.uint8).copy_(values.flatten().view(torch.uint8))
        handles["caches"].append(cache)
    return handles


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state, state["handles"])
    return {"rotate": _plain_rotate, "write": _plain_write, "attend": _plain_attend, "fork": _plain_fork, "release": _plain_release}[state["kind"]](state)


def _own(state, handles):
    ttnn, kind = handles["ttnn"], state["kind"]
    if kind == "rotate":
        return ttnn.experimental.rotate_heads(handles["rows"], handles["cached"], handles["row_starts"], handles["frequencies"], num_heads=state["heads"], head_dim=state["head_dim"],
                                              interleaved=state["interleaved"], norm=handles["query_norm"], epsilon=_EPSILON, magnitude=state["magnitude"])._buf
    if kind == "attend":
        keys, values = handles["caches"]
        return ttnn.experimental.attend_paged_cache(handles["rows"], keys, values, handles["page_table"], handles["cached"], handles["row_starts"], num_heads=state["heads"],
                                                    window=state["window"], sinks=state["sinks"])._buf
    if kind == "release":
        made = ttnn.experimental.release_paged_pages(handles["page_table"], handles["cached"], page_size=state["page_size"], num_pages=state["pages"],
                                                     window=state["window"] or None, sinks=state["sinks"])
        return [t._buf for t in made]
    if kind == "write":
        keys, values = handles["caches"]
        queries = ttnn.experimental.rotate_write_paged_cache(handles["rows"], keys, values, handles["slots"], handles["cached"], handles["row_starts"], handles["frequencies"],
                                                             num_heads=state["heads"], key_column=state["columns"][0], value_column=state["columns"][1], interleaved=state["interleaved"],
                                                             query_norm=handles["query_norm"], key_norm=handles["key_norm"], epsilon=_EPSILON, magnitude=state["magnitude"])
        out = [queries._buf]
    else:
        made = ttnn.experimental.fork_paged_tables(handles["page_table"], handles["cached"], handles["parents"], handles["free_pages"], page_size=state["page_size"])
        ttnn.experimental.copy_paged_pages(handles["caches"], made[2], made[3])
        out = [t._buf for t in made]
    return out + [(c if state["cache"] == "bf16" else ttnn.clone(c, dtype=ttnn.bfloat16))._buf for c in handles["caches"]]


def _positions(state):
    """Request and position of every row."""
    token = torch.arange(state["tokens"], device="cuda")
    request = (token[:, None] >= state["row_starts"][1:]).sum(dim=1)
    return request, state["cached"][request] + token - state["row_starts"][request]


def _rotated(state, x, norm, position):
    """x [tokens, heads, head_dim] bf16 -> its norm and rotation in 32 bits."""
    x, turning = x.float(), state["rotary_dim"]
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPSILON) * norm
    angle = position.double()[:, None] * state["frequencies"].double()
    cos, sin = (f(angle).float()[:, None] * state["magnitude"] for f in (torch.cos, torch.sin))
    turned = x[..., :turning]
    if state["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :turning // 2], turned[..., turning // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., turning:]], dim=-1)


def _laid_out(state, x):
    """[tokens, width] -> as the activations lie."""
    return _tiles(x).reshape(-1) if state["layout"] == "tile" else x[None, None]


def _plain_rotate(state):
    heads, dim = state["heads"], state["head_dim"]
    queries = _rotated(state, state["rows"][:, :heads * dim].view(-1, heads, dim), state["query_norm"], _positions(state)[1])
    return _laid_out(state, queries.bfloat16().flatten(1))


def _plain_write(state):
    dim, kv_heads, (first_key, first_value, _) = state["head_dim"], state["kv_heads"], state["columns"]
    position = _positions(state)[1]
    keys = _rotated(state, state["rows"][:, first_key:first_value].view(-1, kv_heads, dim), state["key_norm"], position)
    values = state["rows"][:, first_value:].view(-1, kv_heads, dim).float()
    slots = state["slots"].long()
    page, within = slots // state["page_size"], slots % state["page_size"]
    tile, down, row = within // 32, within // 16 % 2, within % 16
    out = [_plain_rotate(state)]
    for cache, x in zip(state["caches"], (keys, values)):
        x = x.reshape(-1, kv_heads, dim // 32, 2, 16)
        if state["cache"] == "bf16":
            cache[page, :, tile, :, down, :, row] = x.bfloat16()   # tokens, heads, tile columns, face columns, 16 elements
            out.append(cache.view(-1))
            continue
        exponents, codes = _exponent_and_codes(x.contiguous())
        cache[..., :64].unflatten(-1, (2, 2, 16))[page, :, tile, :, down, :, row] = exponents
        cache[..., 64:].unflatten(-1, (2, 2, 16, 16))[page, :, tile, :, down, :, row] = codes
        out.append(_unpacked(cache).bfloat16().view(-1))
    return out


def _plain_attend(state):
    tokens, heads, dim, window, sinks, page_size = (state[k] for k in ("tokens", "heads", "head_dim", "window", "sinks", "page_size"))
    cached, starts, most = state["cached"].long(), state["row_starts"][:-1].long(), state["most_new"]
    requests = cached.numel()
    # what some row of a request sees: its first tokens, then those from the first row's window on
    place = torch.arange(state["reach"], device="cuda")
    place = place + torch.where(place < sinks, 0, (cached + 1 - window - sinks).clamp(min=0)[:, None])
    page = state["page_table"].gather(1, (place // page_size).clamp(max=state["page_table"].shape[1] - 1)).clamp(min=0).long()
    within = place % page_size
    where = (page, slice(None), within // 32, slice(None), within // 16 % 2, slice(None), within % 16)
    keys, values = (c[where].float() if state["cache"] == "bf16" else
                    _values_of(c[..., 64:].unflatten(-1, (2, 2, 16, 16))[where], c[..., :64].unflatten(-1, (2, 2, 16))[where]) for c in state["caches"])
    keys, values = (x.flatten(3).transpose(1, 2) for x in (keys, values))                          # requests, heads, tokens, head dim
    kv_heads, length = keys.shape[1:3]
    group = heads // kv_heads
    step = torch.arange(most, device="cuda")
    at = (starts[:, None] + step).clamp(max=tokens - 1)            # row of each request's new tokens, the shorter ones padded
    query = state["rows"][:, :heads * dim].float()[at].view(requests, most, kv_heads, group, dim)
    query = query.permute(0, 2, 3, 1, 4).reshape(requests, kv_heads, group * most, dim)
    scores = torch.matmul(query, keys.transpose(2, 3).contiguous()) * dim ** -0.5
    position = (cached[:, None] + step)[..., None]
    seen = (place[:, None] <= position) & ((place[:, None] > position - window) | (place[:, None] < sinks))
    scores = scores.view(requests, kv_heads, group, most, length).masked_fill_(~seen[:, None, None], -math.inf)
    scores = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.view(requests, kv_heads, group * most, length), values.contiguous()).view(requests, kv_heads, group, most, dim) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(requests * most, heads * dim)
    request, position = _positions(state)
    return _laid_out(state, out[request * most + position - state["cached"][request]].bfloat16())


def _plain_fork(state):
    page_size, table, free = state["page_size"], state["page_table"], state["free_pages"]
    parents = state["parents"].long()
    lengths, rows = state["cached"][parents], table[parents]
    child = torch.arange(parents.numel(), device="cuda")
    again = ((parents[:, None] == parents) & (child < child[:, None])).any(dim=1)                 # not the first one of its parent
    begun = lengths // page_size
    page = rows.gather(1, begun[:, None].long())[:, 0]
    copied = again & (lengths % page_size != 0) & (page >= 0)
    index = copied.cumsum(0) - 1
    fresh = torch.where(index < free.numel(), free[index.clamp(0, free.numel() - 1)], -1)
    column = torch.arange(table.shape[1], device="cuda")
    rows = torch.where(column < ((lengths + page_size - 1) // page_size)[:, None], rows, -1)
    rows = torch.where(copied[:, None] & (column == begun[:, None]), fresh[:, None], rows)
    sources, targets = (torch.where(copied & (fresh >= 0), x, -1) for x in (page, fresh))
    wanted = copied.sum()
    taken = wanted.clamp(max=free.numel())
    there = targets >= 0
    out = [rows, lengths, sources, targets, torch.stack([taken, wanted - taken]).int()]
    for cache in state["caches"]:
        cache[targets[there].long()] = cache[sources[there].long()]
        out.append((cache if state["cache"] == "bf16" else _unpacked(cache).bfloat16()).view(-1))
    return out


def _plain_release(state):
    page_size, table, pages, lengths = state["page_size"], state["page_table"], state["pages"], state["cached"][:, None]
    first = torch.arange(table.shape[1], device="cuda") * page_size
    kept = first < lengths
    if state["window"]:
        kept = kept & ((first + page_size > lengths + 1 - state["window"]) | (first < state["sinks"]))
    table = torch.where(kept, table, -1)
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(table >= 0, table, pages).long()] = True
    free = torch.where(used[:pages], pages, torch.arange(pages, device="cuda")).sort()[0]
    taken = used[:pages].sum()
    return [table.int(), torch.where(free < pages, free, -1).int(), torch.stack([pages - taken, taken]).int()]


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------
def _held(tiles, cache):
    """What a cache holds, in 64 bits."""
    if cache == "bf16":
        return tiles.double()
    signs, sizes = 1.0 - 2.0 * (tiles[..., 64:] >= 128), (tiles[..., 64:] % 128).double()
    scale = torch.exp2(tiles[..., :64].double() - 133.0).repeat_interleave(16, dim=-1)
    return (signs * sizes * scale).unflatten(-1, (2, 2, 16, 16))


def _turned(case, x, norm, frequencies, position):
    """x [tokens, heads, head_dim] times the complex number of its token and pair, in 64 bits."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + _EPSILON) * norm.double()
    turning, pairs = case["rotary_dim"], case["rotary_dim"] // 2
    by = torch.polar(torch.full((x.shape[0], pairs), case["magnitude"], dtype=torch.float64, device="cuda"), position.double()[:, None] * frequencies.double())[:, None]
    order = torch.arange(turning, device="cuda").view(pairs, 2) if case["interleaved"] else torch.arange(turning, device="cuda").view(2, pairs).T
    out = x.clone()
    out[..., order.flatten()] = torch.view_as_real(torch.view_as_complex(x[..., order].contiguous()) * by).flatten(-2)
    return out


def exact(case, seed):
    state = _inputs(case, seed)
    cached, new = _lengths(case)
    page_size = case.get("page_size")
    if case["kind"] == "release":
        table, used = state["page_table"].tolist(), set()
        for row, c in zip(table, cached):
            seen_from = max(0, c + 1 - case["window"]) if case["window"] else 0
            for j in range(len(row)):
                tokens = range(j * page_size, min(c, (j + 1) * page_size))
                if not tokens or (tokens.start + page_size <= seen_from and tokens.start >= case["sinks"]):
                    row[j] = -1
                else:
                    used.add(row[j])
        free = [page for page in range(state["pages"]) if page not in used]
        return [torch.tensor(v, dtype=torch.int32) for v in (table, free + [-1] * len(used), [len(free), len(used)])]
    if case["kind"] == "fork":
        parents, old, free = _parents(case), state["page_table"].tolist(), state["free_pages"].tolist()
        table = [[old[p][j] if j * page_size < cached[p] else -1 for j in range(len(old[p]))] for p in parents]
        sources, targets = [-1] * len(parents), [-1] * len(parents)
        for (child, parent), page in zip(_copies(case), free):
            begun = cached[parent] // page_size
            sources[child], targets[child], table[child][begun] = old[parent][begun], page, page
        out = [torch.tensor(v, dtype=torch.int32) for v in (table, [cached[p] for p in parents], sources, targets, [len(_copies(case)), 0])]
        for cache in state["caches"]:
            for source, target in zip(sources, targets):
                if target >= 0:
                    cache[target] = cache[source]
            out.append(_held(cache, case["cache"]).reshape(-1))
        return out
    heads, dim, kv_heads, (first_key, first_value, _) = case["heads"], case["head_dim"], case["kv_heads"], _columns(case)
    lay = (lambda x: _tiles(x).reshape(-1)) if case["layout"] == "tile" else (lambda x: x[None, None])
    if case["kind"] in ("rotate", "write"):
        position = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).cuda()
        queries = _turned(case, state["rows"][:, :first_key].view(-1, heads, dim), state["query_norm"], state["frequencies"], position)
        if case["kind"] == "rotate":
            return lay(queries.flatten(1))
        keys = _turned(case, state["rows"][:, first_key:first_value].view(-1, kv_heads, dim), state["key_norm"], state["frequencies"], position)
        out, slots = [lay(queries.flatten(1))], state["slots"].long()
        for cache, x in zip(state["caches"], (keys, state["rows"][:, first_value:].double())):
            cache = _held(cache, case["cache"])
            pages, _, down, across = cache.shape[:4]
            cache = cache.permute(0, 1, 2, 4, 6, 3, 5, 7).reshape(pages, kv_heads, down * 32, across * 32).contiguous()
            x = x.reshape(-1, kv_heads, across * 2, 16)
            if case["cache"] != "bf16":
                step = torch.exp2(torch.frexp(x.abs().amax(dim=-1, keepdim=True))[1].double() - 7)
                x = torch.sign(x) * torch.clamp(torch.floor(x.abs() / step + 0.5), max=127) * step
            cache[slots // page_size, :, slots % page_size] = x.flatten(2)
            out.append(_tiles(cache).reshape(-1))
        return out
    group = heads // kv_heads
    out = torch.zeros(state["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    first = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        table = state["page_table"][r, :_pages(c + n, page_size)].long()
        both = []
        for cache in state["caches"]:
            tiles = _held(cache[table], case["cache"])
            both.append(tiles.permute(1, 0, 2, 4, 6, 3, 5, 7).reshape(kv_heads, -1, dim)[:, :c + n])
        query = state["rows"][first:first + n, :heads * dim].double().view(n, heads, dim)
        position, place = torch.arange(c, c + n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
        seen = (place <= position) & ((place > position - case["window"]) | (place < case["sinks"]))
        for h in range(heads):
            scores = query[:, h] @ both[0][h // group].T / math.sqrt(dim)
            out[first:first + n, h] = torch.softmax(scores.masked_fill(~seen, -math.inf), dim=-1) @ both[1][h // group]
        first += n
    return lay(out.flatten(1))
