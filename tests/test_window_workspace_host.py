"""What a windowed decode run asks for as scratch memory."""

import pytest

from pagelora_amd import _lib


@pytest.mark.parametrize("batch,pages,heads,page,window,most", [
    (4096, 4096 * 64, (32, 32), 16, 0, 40 << 20),  # (rows that are not cut need none: 1.1 GB with a part for each)
    (4096, 4096 * 64, (32, 8), 16, 1024, 40 << 20),
    (20000, 20000, (32, 32), 16, 0, 40 << 20),
    (64, 64 * 1024, (32, 8), 16, 0, 40 << 20),
    (1, 8192, (32, 8), 16, 0, 40 << 20),
])
def test_decode_workspace_goes_by_the_cuts(batch, pages, heads, page, window, most):
    """2048 workgroups at most are cut, twice as many parts, 16 rows of 130 floats each: 34 MB."""
    nbytes = _lib.load().pl_window_decode_workspace_size(batch, pages, *heads, 128, page, window, 0)
    assert 0 < nbytes <= most
