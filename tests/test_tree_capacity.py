"""The largest capacity of a sequence: rows behind it are still counted in 32 bits."""
import pytest

import fa_b200_capi as capi
from tests.test_tree_attention_refusals import params

LIMIT = 2 ** 31 - 1024


@pytest.mark.parametrize("rows,ok", [(LIMIT, True), (LIMIT + 1, False), (2 ** 31 - 256, False), (2 ** 31 - 1, False)])
@pytest.mark.parametrize("num_splits", [0, 1, 7])
def test_capacity(rows, ok, num_splits):
    t = params()
    t.fwd.sk, t.fwd.num_splits = rows, num_splits
    assert capi.lib.fa_tree_fwd_kvcache(t) == (6 if ok else 3)  # 6: the workspace, which comes after all shapes
    assert (b"workspace" if ok else b"rows") in capi.lib.fa_last_error()
    # row numbers that a kernel forms: a token's row, the end of the last tile, the window's last start, the end of a word
    assert LIMIT + 255 < 2 ** 31 and -(-LIMIT // 128) * 128 + 256 < 2 ** 31
