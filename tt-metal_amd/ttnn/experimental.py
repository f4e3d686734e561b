"""``ttnn.experimental``: entry points that tt-metal does not have under these names, for callers that want fewer launches."""
from __future__ import annotations

from .matmul import gated_linear  # noqa: F401
from .paged import (allocate_paged_cache, attend_paged_cache, copy_paged_pages, fork_paged_tables, paged_tables, release_paged_pages,  # noqa: F401
                    rotary_frequencies, rotate_heads, rotate_write_paged_cache, write_paged_cache)
