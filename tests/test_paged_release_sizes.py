"""Which releases are one launch, whose every workgroup reads the whole table, and which are three with a byte for every page in a workspace: tables of few long rows and
of many short ones, on both sides of the rule."""
import os

import pytest
import torch

import paged_more_model as model
from ttmi import capi


pytestmark = pytest.mark.skipif(not os.path.exists(capi.LIB_PATH), reason="libttmi.so not built in this checkout (python tt-metal_amd/build.py)")


def workspace(requests, width, pages):
    return capi.lib().ttmi_paged_release_workspace_bytes(requests, width, pages)


@pytest.mark.parametrize("requests,width", [(1, 16384), (1, 4096), (4, 4096), (16, 1024), (1024, 16), (4096, 4)])
def test_a_wavefront_does_not_walk_a_long_table_alone(requests, width):
    """A turn is four rows of 64 entries, behind loads of its own: rows are dealt out to wavefronts, columns are not, so entries alone do not bound the turns.  With 16,384
    entries or fewer, and few pages, these took up to 54 us in one launch where three take 8."""
    assert workspace(requests, width, 4096) > 0


@pytest.mark.parametrize("requests,width", [(1, 1), (1, 512), (4, 512), (32, 64), (32, 512), (64, 256), (128, 128), (256, 64), (512, 32), (0, 0), (64, 0)])
def test_small_tables_are_one_launch(requests, width):
    assert workspace(requests, width, 4096) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("requests,width,pages", [(1, 512, 5000), (1, 513, 5000), (3, 511, 2048), (5, 512, 65536), (31, 513, 4000), (64, 256, 4096), (65, 250, 4096), (66, 64, 300), (512, 32, 900), (513, 31, 900),
                                                  (129, 100, 30000), (1, 16384, 20000)])
def test_both_ways_on_either_side(requests, width, pages):
    """Table in place and behind a window with sinks; the workspace is rubbish."""
    g = torch.Generator().manual_seed(requests + width)
    table = torch.randint(-3, pages + 3, (requests, width), generator=g, dtype=torch.int32)
    lengths = torch.randint(-5, width * 32 + 40, (requests,), generator=g, dtype=torch.int32)
    want, want_free, want_counts = model.release(table.tolist(), lengths.tolist(), 32, pages, 700, 40)
    at, n = table.cuda(), lengths.cuda()
    free, counts = torch.full((pages + 1,), 7, dtype=torch.int32, device="cuda"), torch.full((3,), 7, dtype=torch.int32, device="cuda")
    size = workspace(requests, width, pages)
    space = torch.full((size + 256,), 1, dtype=torch.uint8, device="cuda")
    capi.check(capi.lib().ttmi_paged_release(at.data_ptr(), n.data_ptr(), requests, width, 32, 700, 40, pages, at.data_ptr(), free.data_ptr(), counts.data_ptr(), space.data_ptr() if size else None,
                                             size, capi._stream()))
    assert at.tolist() == want and free.tolist() == want_free + [7] and counts.tolist() == want_counts + [7]
    assert (space[size:] == 1).all()
