"""fa_cache_compact moves rows in place: caches that begin at the same place are refused, on the C entry point."""
import pytest

import fa_b200_capi as capi
from tests.test_kvcache_pages_refusals import params


def views(*caches):
    """(address, number of caches, distance) -> params() with these views"""
    p = params()
    p._views = (capi.CacheView * len(caches))(*(capi.CacheView(a, d, 4096, 256, 256, n, 1, 256) for a, n, d in caches))
    p.caches, p.num_caches = capi.C.addressof(p._views), len(caches)
    p.new_seqlens = 0x9000
    p.seqlens = p.new_seqlens                                   # what is refused next: nothing is launched where the caches are apart
    return p


APART = b"new lengths"


@pytest.mark.parametrize("caches,word", [
    (((0x1000, 1, 0),), APART),
    (((0x1000, 1, 0), (0x2000, 1, 0)), APART),
    (((0x1000, 1, 0), (0x2000, 1, 0), (0x1000, 1, 0)), b"once"),
    (((0x10000, 4, 0x1000), (0x13000, 1, 0)), b"once"),
    (((0x10000, 4, 0x1000), (0x14000, 1, 0)), APART),
    (((0x10000, 4, 0x1000), (0x12000, 2, 0x1000)), b"once"),
    (((0x10000, 4, 0x2000), (0x11000, 4, 0x2000)), APART),
    (((0x10000, 2, 0),), b"once"),
    (tuple((0x10000 + 0x1000 * i, 1, 0) for i in range(300)), APART),
    (tuple((0x10000 + 0x1000 * (i % 299), 1, 0) for i in range(300)), b"once"),
])
def test_caches(caches, word):
    assert capi.lib.fa_cache_compact(views(*caches)) == 5 and word in capi.lib.fa_last_error()
