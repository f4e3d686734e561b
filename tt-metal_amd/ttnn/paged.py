"""``ttnn.experimental``: a key/value cache in pages, and attention over it.

No counterpart under these names in tt-metal.  A step of a decoder layer, the tables once for all layers:

    page_table, slots, row_starts, counts = ttnn.experimental.paged_tables(cached, new, page_table, free_pages, page_size=64, num_tokens=tokens)
    qkv = ttnn.linear(x, w_qkv)                                       # queries | keys | values of all heads
    queries = ttnn.experimental.rotate_write_paged_cache(qkv, keys, values, slots, cached, row_starts, frequencies, num_heads=32, key_column=..., value_column=...)
    context = ttnn.experimental.attend_paged_cache(queries, keys, values, page_table, cached, row_starts, num_heads=32)
    y = ttnn.linear(context, w_o)

A model without rotary positions has write_paged_cache(qkv, ...) there, and its queries in qkv.  Between steps, requests fork (fork_paged_tables, copy_paged_pages), and
pages come back (release_paged_pages).

Lengths, tables and slots are uint32 tensors on the device (0xffffffff: no page, no slot) and stay there; they may not change while a call that reads
them runs (calls on one stream run one after the other).  The shapes and the rules are checked by the C++ host layer; the kernels run on torch's current stream, behind ttmi_paged_* of include/ttmi.h."""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from tt_lib.tensor import DataType, Device, Tensor, _m, _wrap

from .core import to_device


def _handle(operation_name, name, t):
    if not isinstance(t, Tensor):
        raise RuntimeError(f"{operation_name}: {name} must be a ttnn.Tensor")
    if t._t is None:
        raise RuntimeError(f"{operation_name}: {name} has been deallocated")
    return t._t


def _handles(operation_name, **tensors):
    return [_handle(operation_name, name, t) for name, t in tensors.items()]


def _count(operation_name, name, value, least=0):
    if type(value) is int and least <= value <= 0x7FFFFFFF:
        return value
    if int(value) != value or not least <= value <= 0x7FFFFFFF:
        raise RuntimeError(f"{operation_name}: {name} must be a whole number of at least {least}, got {value}")
    return int(value)


def allocate_paged_cache(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, *, dtype: DataType, device: Device) -> Tensor:
    """A cache for the keys, or the values, of one layer: [num_pages, num_kv_heads, page_size, head_dim], TILE layout, dtype
    bfloat16 or bfloat8_b, page_size and head_dim multiples of 32.  What it holds is undefined, and no attention looks at a slot
    that has not been written."""
    name = "ttnn.experimental.allocate_paged_cache"
    extents = [_count(name, n, v, 1) for n, v in (("num_pages", num_pages), ("num_kv_heads", num_kv_heads), ("page_size", page_size), ("head_dim", head_dim))]
    return _wrap(_m().allocate_paged_cache(*extents, int(DataType(dtype)), device.device_id))


def paged_tables(cached_lengths: Tensor, new_lengths: Tensor, page_table: Tensor, free_pages: Tensor, *, page_size: int,
                 num_tokens: int) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """What a step needs, from its requests' lengths: (page_table, slots, row_starts, counts).

    Request r has cached_lengths[r] tokens from before and adds new_lengths[r].  The new page table keeps the pages that it holds
    and goes on with pages from free_pages, in order, request by request; entries without a page are 0xffffffff.  slots[t] is
    where token t of the step goes (num_tokens of them, 0xffffffff behind the last token and without a page), row_starts the
    first token of every request and the number of all, counts = (pages taken, pages wanted and not there).  The arguments do not
    change.  At most 4096 requests.  The four share an allocation, which lives as long as any of them."""
    name = "ttnn.experimental.paged_tables"
    handles = _handles(name, cached_lengths=cached_lengths, new_lengths=new_lengths, page_table=page_table, free_pages=free_pages)
    return tuple(_wrap(t) for t in _m().paged_tables(*handles, _count(name, "page_size", page_size), _count(name, "num_tokens", num_tokens), name))


def write_paged_cache(input_tensor: Tensor, key_cache: Tensor, value_cache: Tensor, slots: Tensor, *, key_column: int, value_column: int) -> None:
    """Writes the new keys and values into their slots of both caches, in place.  input_tensor: bfloat16 [1, 1, tokens, width] in
    either layout, as a fused qkv projection leaves it; key_column and value_column say where in a row the keys and the values of
    all key heads start (multiples of 32).  Tokens without a slot are left out; a slot may be named once."""
    name = "ttnn.experimental.write_paged_cache"
    handles = _handles(name, input_tensor=input_tensor, key_cache=key_cache, value_cache=value_cache, slots=slots)
    _m().paged_write(*handles, _count(name, "key_column", key_column), _count(name, "value_column", value_column), name)


def attend_paged_cache(input_tensor: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, cached_lengths: Tensor, row_starts: Tensor, *,
                       num_heads: int, query_column: int = 0, scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0) -> Tensor:
    """Attention of the step's tokens over everything their requests have in the cache, themselves included: causal, and no
    further back than the last `window` tokens where one is given, but for the first `sinks` tokens of a request, which stay
    visible.  What lies between them needs no pages.  input_tensor: bfloat16 [1, 1, tokens, width] in either layout,
    num_heads queries of head_dim elements in every row from query_column on; head h looks at key head
    h // (num_heads // num_kv_heads).  scale: 1 / sqrt(head_dim) if not given.  Returns bfloat16 [1, 1, tokens, num_heads * head_dim]
    in input_tensor's layout.  A request may have any number of new tokens; rows of no request (before row_starts[0], behind the last
    one's), and rows with nothing to look at (no page), are zeros.  Row starts ascend; one below an earlier one is read as that one.

    Scores, maxima and sums are held in 32 bits; the weights of the softmax are rounded to bfloat16 for the product with the values.

    While the stream is captured into a graph, the call takes memory of its own from torch's allocator, so replays may run on any stream."""
    name = "ttnn.experimental.attend_paged_cache"
    handles = _handles(name, input_tensor=input_tensor, key_cache=key_cache, value_cache=value_cache, page_table=page_table, cached_lengths=cached_lengths,
                       row_starts=row_starts)
    return _wrap(_m().paged_attention(*handles, _count(name, "num_heads", num_heads, 1), _count(name, "query_column", query_column),
                                      None if scale is None else float(scale), 0 if window is None else _count(name, "window", window, 1), _count(name, "sinks", sinks), name))


def rotary_frequencies(rotary_dim: int, *, theta: float = 10000.0, factor: float = 1.0, original_length: Optional[int] = None, low_turns: float = 1.0,
                       high_turns: float = 4.0, device: Device) -> Tensor:
    """Angles per token of the rotary_dim / 2 pairs, theta ** (-2 i / rotary_dim), as float32 on the device.

    For contexts longer than the model was trained for, all are divided by `factor`; or, where original_length (the tokens of training) is given, those
    that turn at most low_turns times in it, while those that turn high_turns times or more stay and the ones between are
    a mixture, linear in the number of turns.  A model with other frequencies has them as a tensor of its own."""
    name = "ttnn.experimental.rotary_frequencies"
    pairs = _count(name, "rotary_dim", rotary_dim, 16) // 2
    if rotary_dim % 16:
        raise RuntimeError(f"{name}: rotary_dim must be a multiple of 16, got {rotary_dim}")
    if not (theta > 0 and factor > 0 and math.isfinite(theta) and math.isfinite(factor)):
        raise RuntimeError(f"{name}: theta and factor must be positive, got {theta} and {factor}")
    frequencies = float(theta) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    stays = torch.zeros(pairs, dtype=torch.float64)
    if original_length is not None:
        if not 0 <= low_turns < high_turns:
            raise RuntimeError(f"{name}: low_turns must be below high_turns, got {low_turns} and {high_turns}")
        turns = frequencies * _count(name, "original_length", original_length, 1) / (2 * math.pi)
        stays = ((turns - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
    return to_device(Tensor((frequencies * (stays + (1.0 - stays) / factor)).float(), None), device)


def rotate_heads(input_tensor: Tensor, cached_lengths: Tensor, row_starts: Tensor, frequencies: Tensor, *, num_heads: int, head_dim: int, column: int = 0,
                 interleaved: bool = False, norm: Optional[Tensor] = None, epsilon: float = 1e-6, magnitude: float = 1.0) -> Tensor:
    """The heads of the step's tokens, turned by their positions: token i of a request's new ones is at cached_lengths + i.

    input_tensor: bfloat16 [1, 1, tokens, width] in either layout, num_heads heads of head_dim (64, 96, 128 or 256) elements in every row from
    `column` on (a multiple of 32).  The first 2 * len(frequencies) elements of a head turn, element i with element i + len(frequencies), or 2 i with
    2 i + 1 where `interleaved`; the angle is position * frequency, the result is multiplied with `magnitude`.  The rest of the head stays.  norm
    (float32, head_dim elements): before that, the head is divided by its root mean square, sqrt(mean(x^2) + epsilon), and multiplied with these
    weights.  Returns bfloat16 [1, 1, tokens, num_heads * head_dim] in input_tensor's layout; rows of no request are zeros.
    In 32 bits, angles reduced in 64, rounded once."""
    name = "ttnn.experimental.rotate_heads"
    handles = _handles(name, input_tensor=input_tensor, cached_lengths=cached_lengths, row_starts=row_starts, frequencies=frequencies)
    return _wrap(_m().rotate_heads(*handles, _count(name, "num_heads", num_heads, 1), _count(name, "head_dim", head_dim, 1), _count(name, "column", column), bool(interleaved),
                                   None if norm is None else _handle(name, "norm", norm), float(epsilon), float(magnitude), name))


def rotate_write_paged_cache(input_tensor: Tensor, key_cache: Tensor, value_cache: Tensor, slots: Tensor, cached_lengths: Tensor, row_starts: Tensor, frequencies: Tensor, *,
                             num_heads: int, key_column: int, value_column: int, query_column: int = 0, interleaved: bool = False, query_norm: Optional[Tensor] = None,
                             key_norm: Optional[Tensor] = None, epsilon: float = 1e-6, magnitude: float = 1.0) -> Tensor:
    """What a fused qkv projection leaves, in one pass: rotate_heads of the queries, which are returned for attend_paged_cache, and of the keys, which go
    into their slots with the values beside them (write_paged_cache).  Keys of a bfloat8_b cache are packed from 32 bits.  Tokens of no request, and
    tokens without a slot, are left out of the caches; a slot may be named once."""
    name = "ttnn.experimental.rotate_write_paged_cache"
    handles = _handles(name, input_tensor=input_tensor, key_cache=key_cache, value_cache=value_cache, slots=slots, cached_lengths=cached_lengths, row_starts=row_starts,
                       frequencies=frequencies)
    return _wrap(_m().paged_rotate_write(*handles, _count(name, "num_heads", num_heads, 1), _count(name, "key_column", key_column), _count(name, "value_column", value_column),
                                         _count(name, "query_column", query_column), bool(interleaved), None if query_norm is None else _handle(name, "query_norm", query_norm),
                                         None if key_norm is None else _handle(name, "key_norm", key_norm), float(epsilon), float(magnitude), name))


def fork_paged_tables(page_table: Tensor, lengths: Tensor, parents: Tensor, free_pages: Tensor, *, page_size: int) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Requests that go on from others (several answers to one prompt, beams): (page_table, lengths, sources, targets, counts).

    Row i of the new table continues request parents[i] (0xffffffff: an empty row) with its length.  They share its full pages, which nobody writes into as
    long as no length goes back behind the fork.  The
    page that it is about to go on in stays with the first of them; each other one takes a page from free_pages, in order, and
    copy_paged_pages(caches, sources, targets) has to copy it before the next write.  counts = (entries taken, pages wanted at the end of the list); a row that
    got none has no page there.  The arguments do not change.  At most 4096 requests and as many continuations.  The five share an allocation."""
    name = "ttnn.experimental.fork_paged_tables"
    handles = _handles(name, page_table=page_table, lengths=lengths, parents=parents, free_pages=free_pages)
    return tuple(_wrap(t) for t in _m().paged_fork(*handles, _count(name, "page_size", page_size), name))


def copy_paged_pages(caches: Sequence[Tensor], sources: Tensor, targets: Tensor) -> None:
    """Page sources[i] to page targets[i] in every one of the caches, in place: the keys and the values of all layers, of one shape and dtype.
    Pairs in which either is no page are left out.  All are moved at once: a target may be named once, and is not a source."""
    name = "ttnn.experimental.copy_paged_pages"
    _m().paged_copy([_handle(name, "a cache", t) for t in caches], *_handles(name, sources=sources, targets=targets), name)


def release_paged_pages(page_table: Tensor, lengths: Tensor, *, page_size: int, num_pages: int, window: Optional[int] = None, sinks: int = 0) -> Tuple[Tensor, Tensor, Tensor]:
    """What is left of the tables, and the pages that nobody needs: (page_table, free_pages, counts).

    Entries behind a request's length become 0xffffffff (a request that is over has length 0), and, with a window, those that no later token will see: before
    the window of the token at `length`, without one of the first `sinks` tokens.  Pages may be shared.  free_pages: those of the num_pages that no entry names, ascending, then
    0xffffffff; counts = (free, in use): a later step that takes more than `free` entries of the list has run out of pages.  The arguments do not change.  The three share an allocation."""
    name = "ttnn.experimental.release_paged_pages"
    handles = _handles(name, page_table=page_table, lengths=lengths)
    return tuple(_wrap(t) for t in _m().paged_release(*handles, _count(name, "page_size", page_size), _count(name, "num_pages", num_pages, 1),
                                                      0 if window is None else _count(name, "window", window, 1), _count(name, "sinks", sinks), name))
