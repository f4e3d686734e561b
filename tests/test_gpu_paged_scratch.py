"""What a call of the paged cache's attention may find in the library's own buffer: anything, if the lengths of an earlier call changed while it ran."""
import ctypes

import pytest
import torch

from ttmi import capi

pytestmark = pytest.mark.gpu

SCRATCH_PAGED, COUNTERS = 2, 4096              # csrc/ttmi_internal.h, csrc/paged_attention.hip


def counters_of_the_last_call(L, stream):
    """What the last call on the stream counted with, as a tensor of the library's memory."""
    L.ttmi_test_scratch.restype = None
    L.ttmi_test_scratch.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_size_t), ctypes.POINTER(ctypes.c_uint32)]
    ptr, size, uses = ctypes.c_void_p(), ctypes.c_size_t(), ctypes.c_uint32()
    L.ttmi_test_scratch(SCRATCH_PAGED, stream, ctypes.byref(ptr), ctypes.byref(size), ctypes.byref(uses))
    assert ptr.value and uses.value and size.value >= 2 * COUNTERS * 4

    class Memory:
        __cuda_array_interface__ = dict(shape=(COUNTERS,), typestr="<i4", data=(ptr.value + (uses.value - 1) % 2 * COUNTERS * 4, False), version=2)

    return torch.as_tensor(Memory(), device="cuda")


# A step whose lengths another stream writes over while it runs comes to any result, its workgroups having cut different steps into pieces, and leaves counters that
# are not back at zero: pieces asked for, or parts of a row arrived.  The sizes are of more pieces than workgroups (units of 256 rows), and of rows in parts, in
# both kernels and in one call of both.
@pytest.mark.parametrize("heads,kv_heads,dim,cached,new,window", [
    (16, 16, 64, [0, 7], [1100, 1205], 0),             # 16 * (5 + 5) units in two parts each: more pieces than workgroups
    (32, 8, 128, [0] * 3, [990, 700, 810], 300),       # 40 tiles of 8 units
    (8, 2, 64, [2100], [300], 0),                      # few units in many parts
    (8, 2, 64, [900, 1800, 33], [1, 1, 1], 0),         # single tokens
    (8, 2, 128, [1500] * 6 + [40], [1] * 6 + [350], 0),                # single tokens and a prompt: both kernels
])
@pytest.mark.parametrize("left", [1, 7, 0x7FFFFFFF])
def test_counters_that_an_earlier_call_left(test_library, heads, kv_heads, dim, cached, new, window, left):
    page_size = 64
    g = torch.Generator(device="cuda").manual_seed(heads + sum(new))
    width = max(-(-(c + n) // page_size) for c, n in zip(cached, new))
    pages, tokens = len(new) * width, sum(new)
    keys, values = (capi.tilize(torch.randn(pages, kv_heads, page_size, dim, device="cuda", generator=g).bfloat16()) for _ in range(2))
    rows = torch.randn(tokens, heads * dim, device="cuda", generator=g).bfloat16()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    table, lengths, starts = ints(list(range(pages))).view(len(new), width), ints(cached), ints([sum(new[:r]) for r in range(len(new) + 1)])

    def attend(workspace=None):
        out = torch.full((tokens, heads * dim), 7.0, device="cuda", dtype=torch.bfloat16)
        capi.check(test_library.ttmi_paged_attention(rows.data_ptr(), capi.ROW_MAJOR, tokens, heads * dim, 0, keys.data_ptr(), values.data_ptr(), capi.BFLOAT16, pages, kv_heads, page_size, dim,
                                                     table.data_ptr(), len(new), width, lengths.data_ptr(), starts.data_ptr(), heads, dim ** -0.5, window, out.data_ptr(),
                                                     None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.numel(), capi._stream()))
        return out

    size = test_library.ttmi_paged_attention_workspace_bytes(tokens, len(new), heads, capi.BFLOAT16, kv_heads, dim)
    expected = attend(torch.empty(size, dtype=torch.uint8, device="cuda"))         # its counters are cleared by the call itself
    capi.release_scratch()                                         # other tests' streams may have had this handle
    attend()
    for _ in range(3):                                             # whichever of the buffer's parts a call has
        counters_of_the_last_call(test_library, capi._stream()).fill_(left)
        for _ in range(3):
            assert torch.equal(attend(), expected)
    capi.release_scratch()                                         # with what the last of them left


def test_two_threads_on_one_stream():
    """Steps of more pieces than workgroups and of rows in parts, called by two threads on a stream that they share: one buffer, whose counters go from call to call.  It grows meanwhile."""
    import threading

    page_size, dim = 64, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    stream = torch.cuda.Stream()

    def step(heads, kv_heads, cached, new):
        width = max(-(-(c + n) // page_size) for c, n in zip(cached, new))
        pages, tokens = len(new) * width, sum(new)
        keys, values = (capi.tilize(torch.randn(pages, kv_heads, page_size, dim, device="cuda", generator=g).bfloat16()) for _ in range(2))
        rows = torch.randn(tokens, heads * dim, device="cuda", generator=g).bfloat16()
        return (tokens, heads, kv_heads, pages, width, rows, keys, values, ints(list(range(pages))), ints(cached), ints([sum(new[:r]) for r in range(len(new) + 1)]))

    def attend(what, on):
        tokens, heads, kv_heads, pages, width, rows, keys, values, table, cached, starts = what
        out = torch.full((tokens, heads * dim), 7.0, device="cuda", dtype=torch.bfloat16)
        on.wait_stream(torch.cuda.current_stream())
        capi.check(capi.lib().ttmi_paged_attention(rows.data_ptr(), capi.ROW_MAJOR, tokens, heads * dim, 0, keys.data_ptr(), values.data_ptr(), capi.BFLOAT16, pages, kv_heads, page_size, dim,
                                                   table.data_ptr(), cached.numel(), width, cached.data_ptr(), starts.data_ptr(), heads, dim ** -0.5, 0, out.data_ptr(), None, 0, on.cuda_stream))
        return out

    steps = [step(8, 2, [900], [1]), step(8, 2, [2100], [300]), step(16, 16, [0, 7], [1100, 1205]), step(8, 2, [900, 1800, 33], [1, 1, 1])]
    expected = [attend(what, torch.cuda.current_stream()) for what in steps]
    torch.cuda.synchronize()
    results = [[], []]

    def calls(mine):
        for i in range(24):
            n = (i + 2 * mine) % len(steps)
            results[mine].append((n, attend(steps[n], stream)))

    threads = [threading.Thread(target=calls, args=(mine,)) for mine in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert [len(r) for r in results] == [24, 24]
    for got in results:
        for n, out in got:
            assert torch.equal(out, expected[n])
