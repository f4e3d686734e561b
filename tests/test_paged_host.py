"""What the paged cache's C entries refuse, and what they answer without a GPU: the checks come before anything is launched, so
these calls never reach one.  The pointers are numbers that nothing looks behind."""
import pytest
import torch

import paged_model

OK, INVALID, UNSUPPORTED = 0, 1, 3
SOMEWHERE = 1 << 20                                                # aligned, and not null


@pytest.fixture(scope="module")
def capi():
    import os

    from ttmi import capi

    if not os.path.exists(capi.LIB_PATH):
        pytest.skip("libttmi.so not built in this checkout (python tt-metal_amd/build.py)")
    return capi


def call(capi, name, defaults, **changes):
    arguments = {**defaults, **changes}
    status = getattr(capi.lib(), name)(*arguments.values())
    return status, capi.lib().ttmi_last_error().decode()


TABLES = dict(cached=SOMEWHERE, added=SOMEWHERE, requests=3, page_size=64, page_table=SOMEWHERE, max_pages=4, free_pages=SOMEWHERE, free_count=5, tokens=7, page_table_out=SOMEWHERE,
              slots=SOMEWHERE, row_starts=SOMEWHERE, counts=SOMEWHERE, stream=None)
WRITE = dict(rows=SOMEWHERE, layout=0, tokens=5, width=512, key_column=128, value_column=256, slots=SOMEWHERE, key_cache=SOMEWHERE, value_cache=2 * SOMEWHERE, cache_dtype=0, pages=3, kv_heads=2,
             page_size=32, head_dim=64, stream=None)
ATTEND = dict(rows=SOMEWHERE, layout=0, tokens=5, width=512, query_column=0, key_cache=SOMEWHERE, value_cache=SOMEWHERE, cache_dtype=0, pages=3, kv_heads=2, page_size=32, head_dim=64,
              page_table=SOMEWHERE, requests=2, max_pages=2, cached=SOMEWHERE, row_starts=SOMEWHERE, heads=4, scale=0.125, window=0, out=SOMEWHERE, workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize("change", [dict(requests=4097), dict(page_size=48), dict(page_size=0), dict(cached=None), dict(added=None), dict(page_table=None), dict(free_pages=None), dict(page_table_out=None),
                                    dict(slots=None), dict(row_starts=None), dict(counts=None), dict(cached=SOMEWHERE + 2), dict(slots=SOMEWHERE + 1)])
def test_tables_refuse(capi, change):
    status, message = call(capi, "ttmi_paged_tables", TABLES, **change)
    assert status in (INVALID, UNSUPPORTED) and "paged" in message


CACHES = [dict(cache_dtype=4), dict(cache_dtype=1), dict(cache_dtype=17), dict(pages=0), dict(kv_heads=0), dict(page_size=40), dict(page_size=0), dict(head_dim=48), dict(head_dim=0),
          dict(pages=1 << 27), dict(layout=9), dict(width=516), dict(tokens=0x7fffffff), dict(key_cache=None), dict(value_cache=None), dict(key_cache=SOMEWHERE + 8), dict(rows=None)]


@pytest.mark.parametrize("change", CACHES + [dict(key_column=16), dict(value_column=480), dict(key_column=0xffffffe0), dict(slots=None), dict(slots=SOMEWHERE + 2), dict(layout=1, width=504)])
def test_writes_refuse(capi, change):
    status, message = call(capi, "ttmi_paged_write", WRITE, **change)
    assert status in (INVALID, UNSUPPORTED) and "paged" in message


@pytest.mark.parametrize("change", CACHES + [dict(head_dim=32), dict(head_dim=160), dict(heads=3), dict(heads=0), dict(heads=16), dict(heads=0xfffffffe), dict(query_column=288), dict(query_column=1), dict(requests=4097),
                                             dict(max_pages=1 << 27), dict(scale=float("nan")), dict(scale=float("inf")), dict(page_table=None), dict(cached=None), dict(row_starts=None), dict(out=None),
                                             dict(out=SOMEWHERE + 8), dict(row_starts=SOMEWHERE + 2), dict(workspace=SOMEWHERE, workspace_bytes=16), dict(workspace=SOMEWHERE + 16, workspace_bytes=1 << 30)])
def test_attention_refuses(capi, change):
    status, message = call(capi, "ttmi_paged_attention", ATTEND, **change)
    assert status in (INVALID, UNSUPPORTED) and "paged" in message


def test_workspace_sizes(capi):
    """Nothing to do, or a call that is refused: 0.  Otherwise 16 KB of counters and two partial results for each resident workgroup,
    however long the requests are."""
    size = capi.lib().ttmi_paged_attention_workspace_bytes
    assert size(0, 1, 4, 0, 2, 64) == 0 and size(5, 0, 4, 0, 2, 64) == 0 and size(5, 1, 3, 0, 2, 64) == 0 and size(5, 1, 4, 0, 0, 64) == 0
    row_tile = lambda dim: (dim // 16 + 1) * 1024
    assert size(32, 32, 32, 0, 8, 128) == 16384 + 2 * 512 * row_tile(128)
    assert size(32, 32, 32, 3, 8, 128) == 16384 + 2 * 512 * row_tile(128)
    assert size(1, 1, 16, 0, 2, 256) == 16384 + 2 * 256 * row_tile(256)
    assert size(512, 1, 32, 0, 8, 128) == 16384 + 2 * 256 * 8 * (4 * 4 + 1) * 1024


# ---- the plain forms that the kernels are compared with ---------------------------------------------------------------------------------
def test_the_plain_tables_by_hand():
    table, slots, starts, counts = paged_model.tables([31, 0, 64], [2, 0, 1], [[5, -1, -1], [-1, -1, -1], [2, 3, -1]], [9, 8, 7], 32, 5)
    assert table == [[5, 9, -1], [-1, -1, -1], [2, 3, 8]]
    assert slots == [5 * 32 + 31, 9 * 32, 8 * 32, -1, -1] and starts == [0, 2, 2, 3] and counts == [2, 0]


def test_the_plain_attention_is_softmax_attention():
    """Over pages in order, against torch's softmax over the whole sequence."""
    torch.manual_seed(1)
    heads, kv_heads, dim, n, window = 4, 2, 64, 70, 9
    keys, values = (torch.randn(3, kv_heads, 32, dim, dtype=torch.float64) for _ in range(2))
    rows = torch.randn(n, heads * dim, dtype=torch.float64)
    got, _ = paged_model.attention(rows, keys, values, [[2, 0, 1]], [0], [0, n], heads, dim, 32, window=window)
    k, v = (x[[2, 0, 1]].transpose(0, 1).reshape(kv_heads, 96, dim)[:, :n].repeat_interleave(2, 0) for x in (keys, values))
    scores = rows.view(n, heads, dim).transpose(0, 1) @ k.transpose(1, 2) * dim ** -0.5
    i, j = torch.arange(n)[:, None], torch.arange(n)
    want = torch.softmax(scores.masked_fill((j > i) | (j <= i - window), float("-inf")), -1) @ v
    assert torch.allclose(got.view(n, heads, dim).transpose(0, 1), want, rtol=1e-12, atol=1e-12)
