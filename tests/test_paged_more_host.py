"""What the C entries for positions, sinks and pages that change hands refuse: the checks come before anything is launched, so these calls reach no
GPU.  The pointers are numbers that nothing looks behind.  And the plain forms that the kernels are compared with, by hand."""
import ctypes
import math

import pytest
import torch

import paged_model
import paged_more_model

INVALID, UNSUPPORTED = 1, 3
SOMEWHERE = 1 << 20                                                # aligned, and not null


@pytest.fixture(scope="module")
def capi():
    import os

    from ttmi import capi

    if not os.path.exists(capi.LIB_PATH):
        pytest.skip("libttmi.so not built in this checkout (python tt-metal_amd/build.py)")
    return capi


def refused(capi, name, defaults, changes):
    status = getattr(capi.lib(), name)(*{**defaults, **changes}.values())
    message = capi.lib().ttmi_last_error().decode()
    assert status in (INVALID, UNSUPPORTED) and "paged" in message, (status, message)


ROWS = dict(rows=SOMEWHERE, layout=0, tokens=5, width=512)
CACHE = dict(key_cache=SOMEWHERE, value_cache=2 * SOMEWHERE, cache_dtype=0, pages=3, kv_heads=2, page_size=32, head_dim=64)
TURN = dict(frequencies=SOMEWHERE, rotary_dim=64, interleaved=0)
LENGTHS = dict(cached=SOMEWHERE, row_starts=SOMEWHERE, requests=2)
ROTATE = dict(**ROWS, column=0, heads=4, head_dim=64, **LENGTHS, **TURN, norm=None, epsilon=1e-6, magnitude=1.0, out=2 * SOMEWHERE, stream=None)
WRITE = dict(**ROWS, query_column=0, heads=4, key_column=256, value_column=384, slots=SOMEWHERE, **CACHE, **LENGTHS, **TURN, query_norm=None, key_norm=None, epsilon=1e-6, magnitude=1.0,
             out=2 * SOMEWHERE, stream=None)
TURNS = [dict(head_dim=32), dict(head_dim=160), dict(heads=0), dict(heads=0xfffffffe), dict(rotary_dim=24), dict(rotary_dim=80), dict(rotary_dim=0xfffffff0), dict(requests=4097), dict(row_starts=None),
         dict(cached=None), dict(frequencies=None), dict(frequencies=SOMEWHERE + 4), dict(cached=SOMEWHERE + 2), dict(row_starts=SOMEWHERE + 1), dict(epsilon=-1.0), dict(epsilon=float("nan")),
         dict(epsilon=float("inf")), dict(magnitude=float("inf")), dict(magnitude=float("nan")), dict(layout=7), dict(width=516), dict(layout=1, width=504), dict(tokens=0x7fffffff), dict(rows=None),
         dict(out=None), dict(rows=SOMEWHERE + 8), dict(out=SOMEWHERE + 8), dict(out=SOMEWHERE + 1024)]


@pytest.mark.parametrize("change", TURNS + [dict(column=16), dict(column=288), dict(norm=SOMEWHERE + 4)])
def test_rotations_refuse(capi, change):
    refused(capi, "ttmi_rotate_heads", ROTATE, change)


CACHES = [dict(cache_dtype=4), dict(cache_dtype=1), dict(pages=0), dict(kv_heads=0), dict(page_size=40), dict(page_size=0), dict(head_dim=48), dict(pages=1 << 27), dict(key_cache=None),
          dict(value_cache=None), dict(key_cache=SOMEWHERE + 8)]


@pytest.mark.parametrize("change", TURNS + CACHES + [dict(query_column=16), dict(query_column=288), dict(key_column=400), dict(value_column=416), dict(key_column=0xffffffe0), dict(slots=None),
                                                     dict(slots=SOMEWHERE + 2), dict(query_norm=SOMEWHERE + 8), dict(key_norm=SOMEWHERE + 4)])
def test_rotated_writes_refuse(capi, change):
    refused(capi, "ttmi_paged_rotate_write", WRITE, change)


ATTEND = dict(**ROWS, query_column=0, **CACHE, page_table=SOMEWHERE, requests=2, max_pages=2, cached=SOMEWHERE, row_starts=SOMEWHERE, heads=4, scale=0.125, window=16, sinks=4, out=SOMEWHERE,
              workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize("change", CACHES + [dict(sinks=0x80000000), dict(sinks=0xffffffff), dict(head_dim=32), dict(heads=3), dict(query_column=288), dict(requests=4097), dict(scale=float("nan")),
                                             dict(page_table=None), dict(out=SOMEWHERE + 8), dict(workspace=SOMEWHERE, workspace_bytes=16)])
def test_attention_with_sinks_refuses(capi, change):
    refused(capi, "ttmi_paged_attention_sinks", ATTEND, change)


FORK = dict(page_table=SOMEWHERE, lengths=SOMEWHERE, requests=3, max_pages=4, page_size=64, parents=SOMEWHERE, children=5, free_pages=SOMEWHERE, free_count=6, page_table_out=2 * SOMEWHERE,
            lengths_out=3 * SOMEWHERE, sources=SOMEWHERE, targets=SOMEWHERE, counts=SOMEWHERE, stream=None)


@pytest.mark.parametrize("change", [dict(page_size=0), dict(page_size=48), dict(requests=4097), dict(children=4097), dict(free_count=1 << 31)] +
                         [{name: None} for name in ("page_table", "lengths", "parents", "free_pages", "page_table_out", "lengths_out", "sources", "targets", "counts")] +
                         [dict(parents=SOMEWHERE + 2), dict(targets=SOMEWHERE + 1), dict(page_table_out=SOMEWHERE), dict(lengths_out=SOMEWHERE + 8)])
def test_forks_refuse(capi, change):
    refused(capi, "ttmi_paged_fork", FORK, change)


def test_copies_refuse(capi):
    at = lambda *p: (ctypes.c_void_p * len(p))(*p)
    copy = dict(caches=at(SOMEWHERE, 2 * SOMEWHERE), count=2, cache_dtype=0, pages=3, kv_heads=2, page_size=32, head_dim=64, sources=SOMEWHERE, targets=SOMEWHERE, pairs=4, stream=None)
    for change in [dict(cache_dtype=4), dict(pages=0), dict(kv_heads=0), dict(page_size=40), dict(head_dim=48), dict(caches=None), dict(caches=at(SOMEWHERE, None)), dict(caches=at(SOMEWHERE, SOMEWHERE + 8)),
                   dict(sources=None), dict(targets=None), dict(sources=SOMEWHERE + 2), dict(pairs=1 << 31)]:
        refused(capi, "ttmi_paged_copy", copy, change)


RELEASE = dict(page_table=SOMEWHERE, lengths=SOMEWHERE, requests=3, max_pages=4, page_size=64, window=16, sinks=4, pages=100, page_table_out=SOMEWHERE, free_pages=SOMEWHERE, counts=SOMEWHERE,
               workspace=SOMEWHERE, workspace_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change", [dict(page_size=0), dict(page_size=48), dict(pages=0), dict(pages=1 << 31), dict(page_table=None), dict(lengths=None), dict(page_table_out=None),
                                    dict(free_pages=None), dict(counts=None), dict(lengths=SOMEWHERE + 2), dict(page_table_out=SOMEWHERE + 4)])
def test_releases_refuse(capi, change):
    refused(capi, "ttmi_paged_release", RELEASE, change)


def test_releases_of_a_large_pool_need_a_workspace(capi):
    large = dict(RELEASE, requests=1000, max_pages=500, pages=3000000)
    size = capi.lib().ttmi_paged_release_workspace_bytes(1000, 500, 3000000)
    assert size > 0
    for change in [dict(workspace=None), dict(workspace_bytes=size - 1), dict(workspace=SOMEWHERE + 16)]:
        refused(capi, "ttmi_paged_release", large, change)


def test_a_copy_into_nothing_needs_no_gpu(capi):
    at = (ctypes.c_void_p * 1)(SOMEWHERE)
    assert capi.lib().ttmi_paged_copy(at, 1, 0, 3, 2, 32, 64, None, None, 0, None) == 0
    assert capi.lib().ttmi_paged_copy(None, 0, 0, 3, 2, 32, 64, SOMEWHERE, SOMEWHERE, 4, None) == 0


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------
def test_the_plain_rotation_by_hand():
    """A quarter turn takes (a, b) to (-b, a); elements behind the turning ones stay; without a request, zeros."""
    x = torch.arange(1.0, 9.0)[None].repeat(3, 1)
    f = torch.tensor([math.pi / 2, 0.0], dtype=torch.float64)
    out, _ = paged_more_model.rotate(x, [(0, 0), (0, 1), None], 1, 8, f)
    assert torch.allclose(out[0, 0], x[0].double()) and not out[2].any()
    assert torch.allclose(out[1, 0], torch.tensor([-3.0, 2, 1, 4, 5, 6, 7, 8], dtype=torch.float64))
    out, _ = paged_more_model.rotate(x, [(0, 0), (0, 1), None], 1, 8, f, interleaved=True, magnitude=2.0)
    assert torch.allclose(out[1, 0], torch.tensor([-4.0, 2, 6, 8, 5, 6, 7, 8], dtype=torch.float64))
    out, _ = paged_more_model.rotate(x, [(0, 0)] * 3, 2, 4, f[1:], norm=torch.tensor([1.0, 1, 1, 2]))
    assert torch.allclose(out[0, 0], torch.tensor([1.0, 2, 3, 8], dtype=torch.float64) / math.sqrt(7.5))


def test_the_plain_attention_with_sinks():
    """Without sinks, or with all of a window's reach, the attention of paged_model; with, softmax over the mask."""
    torch.manual_seed(1)
    keys, values = (torch.randn(3, 2, 32, 64, dtype=torch.float64) for _ in range(2))
    rows = torch.randn(70, 256, dtype=torch.float64)
    call = lambda model, **kw: model.attention(rows, keys, values, [[2, 0, 1]], [3], [0, 70], 4, 64, 32, **kw)[0]
    assert torch.allclose(call(paged_more_model, window=9), call(paged_model, window=9), rtol=1e-12)
    assert torch.allclose(call(paged_more_model, window=9, sinks=200), call(paged_model), rtol=1e-12)
    k, v = (x[[2, 0, 1]].transpose(0, 1).reshape(2, 96, 64)[:, :73].repeat_interleave(2, 0) for x in (keys, values))
    scores = rows.view(70, 4, 64).transpose(0, 1) @ k.transpose(1, 2) / 8
    i, j = torch.arange(3, 73)[:, None], torch.arange(73)
    hidden = (j > i) | ((j <= i - 9) & (j >= 5))
    want = (torch.softmax(scores.masked_fill(hidden, float("-inf")), -1) @ v).transpose(0, 1).reshape(70, 256)
    assert torch.allclose(call(paged_more_model, window=9, sinks=5), want, rtol=1e-10, atol=1e-12)


def test_the_plain_forks_and_releases_by_hand():
    table, lengths = [[5, 6, -1], [7, 8, -1], [9, -1, -1]], [40, 64, 0]
    rows, out, sources, targets, counts = paged_more_model.fork(table, lengths, [0, 1, 0, 1, -1, 2, 0, 0], [20, 21], 32)
    assert rows == [[5, 6, -1], [7, 8, -1], [5, 20, -1], [7, 8, -1], [-1] * 3, [-1] * 3, [5, 21, -1], [5, -1, -1]] and out == [40, 64, 40, 64, 0, 0, 40, 40]
    assert sources == [-1, -1, 6, -1, -1, -1, 6, -1] and targets == [-1, -1, 20, -1, -1, -1, 21, -1] and counts == [2, 1]
    assert paged_more_model.release(rows, out, 32, 9) == ([[5, 6, -1], [7, 8, -1], [5, -1, -1], [7, 8, -1], [-1] * 3, [-1] * 3, [5, -1, -1], [5, -1, -1]], [0, 1, 2, 3, 4, -1, -1, -1, -1], [5, 4])
    # the token at 100 sees 91 .. 100 and, with a sink, token 0
    assert paged_more_model.release([[3, 2, 1, 0]], [100], 32, 4, window=10) == ([[-1, -1, 1, 0]], [2, 3, -1, -1], [2, 2])
    assert paged_more_model.release([[3, 2, 1, 0]], [100], 32, 4, window=10, sinks=1) == ([[3, -1, 1, 0]], [2, -1, -1, -1], [1, 3])
