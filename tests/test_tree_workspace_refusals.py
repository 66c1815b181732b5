"""fa_tree_workspace_bytes is asked before any argument has been checked: what the call will refuse needs no workspace."""
import pytest

import fa_b200_capi as capi
from tests.test_tree_attention_refusals import params


@pytest.mark.parametrize("hq,hkv", [(2, 4), (1, 8), (6, 4)])
@pytest.mark.parametrize("num_splits", [0, 3])
def test_heads_that_do_not_divide(hq, hkv, num_splits):
    t = params()
    t.fwd.hq, t.fwd.hkv, t.fwd.num_splits = hq, hkv, num_splits
    assert capi.lib.fa_tree_workspace_bytes(t) == 0
    assert capi.lib.fa_tree_fwd_kvcache(t) == 3 and b"divisible" in capi.lib.fa_last_error()
