"""A kernel whose bounded wait has run out waits for its copies and matrix products on the way before it gives its memory back.  No
wait runs out on purpose on a GPU, so the sources are read: no tensor memory is freed without that step."""
import glob
import os
import re

from tests.conftest import PKG


def source(name):
    with open(os.path.join(PKG, "csrc", name)) as f:
        return f.read()


def test_tensor_memory_is_freed_after_settling():
    found = 0
    for path in glob.glob(os.path.join(PKG, "csrc", "*.cu")):
        text = re.sub(r"\s+", " ", source(os.path.basename(path)))
        frees, settled = text.count("tmem_dealloc("), text.count("settle_after_abort(abort_flag); tc_fence_after(); tmem_dealloc(")
        assert frees == settled, path
        found += frees
    assert found >= 10
