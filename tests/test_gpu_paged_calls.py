"""Calls of the paged cache's attention that a server makes besides its ordinary steps: a step without requests, calls captured into
graphs, row starts that are not those of a plain step, lengths near the end of an int32.

Where a value is computed, the tolerance is that of tests/paged_model.py plus 2^-9 of the result (bf16 has 8 significant bits: the result's own
rounding takes up to 2^-8, of which the bound there holds half)."""
import pytest
import torch

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
