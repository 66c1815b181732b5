"""What the C entry points of the page operations refuse, without a GPU."""
import ctypes

import pytest

import fa_b200_capi as capi

lib = capi.lib


def params():
    p = capi.PagesParams()
    view = capi.CacheView(0x1000, 0, 4096, 256, 256, 1, 1, 256)
    p._view = view
    p.caches, p.num_caches = ctypes.addressof(view), 1
    p.num_pages, p.page_size, p.refs, p.table, p.table_stride, p.b, p.width, p.n = 8, 16, 0x1000, 0x1000, 4, 2, 4, 3
    p.seqlens, p.rows, p.rows2, p.new_table, p.new_seqlens, p.missing = 0x1000, 0x1000, 0x1000, 0x2000, 0x2000, 0x1000
    p.workspace, p.workspace_bytes = 0x1000, 1
    return p


FNS = {"reserve": lib.fa_pages_reserve, "free": lib.fa_pages_free, "fork": lib.fa_pages_fork, "copy": lib.fa_pages_copy, "compact": lib.fa_cache_compact}


@pytest.mark.parametrize("name", list(FNS))
def test_null(name):
    assert FNS[name](None) == 1


@pytest.mark.parametrize("name,change,code", [
    ("reserve", {}, 6), ("fork", {}, 6),
    ("reserve", dict(page_size=0), 3), ("reserve", dict(b=-1), 3), ("reserve", dict(num_pages=0), 3), ("reserve", dict(num_pages=1 << 25), 3),
    ("reserve", dict(refs=None), 1), ("reserve", dict(table=None), 1), ("reserve", dict(seqlens=None), 1), ("reserve", dict(missing=None), 1),
    ("reserve", dict(width=1 << 28), 3), ("reserve", dict(b=1 << 20, width=1 << 12), 3), ("reserve", dict(workspace=0x1008, workspace_bytes=1 << 20), 4),
    ("free", dict(page_size=-1), 3), ("free", dict(refs=None), 1), ("free", dict(table=None), 1),
    ("fork", dict(rows=None), 1), ("fork", dict(new_table=None), 1), ("fork", dict(new_table=0x1000), 5), ("fork", dict(caches=None), 1), ("fork", dict(n=-1), 3),
    ("copy", dict(rows=None), 1), ("copy", dict(rows2=None), 1), ("copy", dict(num_pages=0), 3), ("copy", dict(n=-1), 3),
    ("compact", dict(seqlens=None), 1), ("compact", dict(rows=None), 1), ("compact", dict(new_seqlens=None), 1), ("compact", dict(new_seqlens=0x1000), 5),
    ("compact", dict(cache_batch_idx=0x1000), 5), ("compact", dict(num_caches=0), 3), ("compact", dict(page_size=0), 3),
])
def test_refusals(name, change, code):
    p = params()
    for k, v in change.items():
        setattr(p, k, v)
    assert FNS[name](p) == code


def test_a_bad_cache_is_refused():
    for field, value, code in (("ptr", None, 1), ("heads", 0, 3), ("segment_bytes", 0, 3), ("segment_bytes", 1 << 29, 3), ("caches", -1, 3)):
        p = params()
        setattr(p._view, field, value)
        for name in ("fork", "copy", "compact"):
            assert FNS[name](p) == code


def test_nothing_to_do_launches_nothing():
    for name, change in (("free", dict(b=0)), ("free", dict(width=0)), ("copy", dict(n=0)), ("copy", dict(num_caches=0)), ("compact", dict(b=0))):
        p = params()
        for k, v in change.items():
            setattr(p, k, v)
        assert FNS[name](p) == 0
    assert lib.fa_pages_workspace_bytes(-1, 4) == 0 and lib.fa_pages_workspace_bytes(3, 5000) >= 2 * 12 + 8 + 8192 * 4
