"""kvcache_fork compares every row with all rows in front of it: more rows than a second's work are refused."""
import pytest

import fa_b200_capi as capi
from tests.test_kvcache_pages_refusals import params


@pytest.mark.parametrize("n,code,word", [(1 << 20, 6, b"workspace"), ((1 << 20) + 1, 3, b"2^20"), (1 << 24, 3, b"2^20")])
def test_rows_of_a_fork(n, code, word):
    p = params()
    p.n = n
    assert capi.lib.fa_pages_fork(p) == code and word in capi.lib.fa_last_error()     # 6: the workspace, which comes after all shapes
