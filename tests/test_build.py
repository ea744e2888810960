"""What the in-tree build takes for up to date (no GPU, no compiler run)."""

import glob
import os

from wanferenz_b200 import _build


def test_every_source_and_header_of_the_library_is_watched():
    """Headers with inline code count, whatever their suffix: an edit of one alone makes the library stale."""
    here = {os.path.join(_build.CSRC, f) for f in os.listdir(_build.CSRC)}
    device = {f for f in here if f.endswith((".cu", ".cuh", ".h"))}
    assert device and device <= set(_build.deps())
    assert set(glob.glob(os.path.join(_build.ROOT, "include", "*.h"))) <= set(_build.deps())
