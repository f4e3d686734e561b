"""``ttnn.experimental``: a key/value cache in pages, and attention over it.

No counterpart under these names in tt-metal.  A step of a decoder layer, the tables once for all layers:

    page_table, slots, row_starts, counts = ttnn.experimental.paged_tables(cached, new, page_table, free_pages, page_size=64, num_tokens=tokens)
    qkv = ttnn.linear(x, w_qkv)                                       # queries | keys | values of all heads
    ttnn.experimental.write_paged_cache(qkv, keys, values, slots, key_column=..., value_column=...)
    context = ttnn.experimental.attend_paged_cache(qkv, keys, values, page_table, cached, row_starts, num_heads=32)
    y = ttnn.linear(context, w_o)

Lengths, tables and slots are uint32 tensors on the device (0xffffffff: no page, no slot) and stay there.  The shapes and the
rules are checked by the C++ host layer; the kernels run on torch's current stream, behind ttmi_paged_* of include/ttmi.h."""
from __future__ import annotations

from typing import Optional, Tuple

from tt_lib.tensor import DataType, Device, Tensor, _m, _wrap


def _handles(operation_name, **tensors):
    for name, t in tensors.items():
        if not isinstance(t, Tensor):
            raise RuntimeError(f"{operation_name}: {name} must be a ttnn.Tensor")
        if not t.is_allocated():
            raise RuntimeError(f"{operation_name}: {name} has been deallocated")
    return [t._t for t in tensors.values()]


def _count(operation_name, name, value, least=0):
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
                       num_heads: int, query_column: int = 0, scale: Optional[float] = None, window: Optional[int] = None) -> Tensor:
    """Attention of the step's tokens over everything their requests have in the cache, themselves included: causal, and no
    further back than the last `window` tokens where one is given.  input_tensor: bfloat16 [1, 1, tokens, width] in either layout,
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
                                      None if scale is None else float(scale), 0 if window is None else _count(name, "window", window, 1), name))
