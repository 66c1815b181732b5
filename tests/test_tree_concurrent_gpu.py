"""Calls of the tree attention and of the page operations at once: on two streams, from two threads, as graphs that replay side by
side.  Every result has the bits of the same call by itself."""
import threading

import pytest
import torch

import fa_b200_capi as capi
import flash_attn_npu_3 as fa
from tests.test_tree_attention_gpu import make

pytestmark = pytest.mark.gpu

SHAPES = [(128, 8, 2, [900, 5, 300], 16, 0.0), (64, 8, 8, [1500], 33, 0.0), (256, 4, 2, [700, 90], 9, 0.0), (128, 6, 2, [640, 33], 20, 20.0)]


def calls():
    out = []
    for i, (d, hq, hkv, lens, t, cap) in enumerate(SHAPES):
        c = make(torch.bfloat16, d, hq, hkv, lens, t, 64, seed=i, rotary="half")
        dev = {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}

        def one(dev=dev, cap=cap):
            return fa.flash_attn_tree_with_kvcache(dev["q"], dev["kc"], dev["vc"], dev["k"], dev["v"], dev["parents"], cache_seqlens=dev["lens"],
                                                   page_table=dev["table"], rotary_cos=dev["cos"], rotary_sin=dev["sin"], softcap=cap,
                                                   rotary_interleaved=False, return_softmax_lse=True)
        out.append(one)
    return out


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_streams():
    fs = calls()
    want = [f() for f in fs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for r in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                k = (r + 2 * s) % len(fs)
                got[s].append((k, fs[k]()))
    torch.cuda.synchronize()
    assert capi.lib.fa_debug_get(2) == 0
    assert all(same(o, want[k]) for g in got for k, o in g)


def test_two_threads():
    fs = calls()
    want = [f() for f in fs]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(s):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for r in range(20):
                    k = (r + 2 * s) % len(fs)
                    got[s].append((k, fs[k]()))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(s,)) for s in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and capi.lib.fa_debug_get(2) == 0
    assert len(got[0]) == len(got[1]) == 20 and all(same(o, want[k]) for g in got for k, o in g)


def test_graphs_side_by_side():
    fs = calls()
    want = [f() for f in fs]
    torch.cuda.synchronize()
    graphs = []
    for f in fs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in fs]
    for _ in range(10):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert capi.lib.fa_debug_get(2) == 0
    assert all(same(o, w) for (_, o), w in zip(graphs, want))


def test_pools_on_two_streams():
    """Pools of their own; small ones (one block) and one that takes several launches."""
    def state(pages, b, width):
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
        lens = torch.randint(1, 16 * width, (b,), generator=torch.Generator(device="cuda").manual_seed(pages), device="cuda", dtype=torch.int32)
        caches = torch.randn(3, pages, 16, 2, 64, generator=torch.Generator(device="cuda").manual_seed(b), device="cuda").bfloat16()
        return refs, table, lens, caches

    def step(refs, table, lens, caches):
        missing = fa.kvcache_reserve(refs, table, lens, 16)
        parents = torch.arange(len(lens), device="cuda", dtype=torch.int32).repeat(2)
        new, nl, m2 = fa.kvcache_fork(caches, refs, table, lens, parents)
        fa.kvcache_free(refs, new, nl // 2, 16)
        return [missing, m2, new, nl, refs.clone(), caches.clone()]
    sizes = [(500, 5, 20), (9000, 90, 40)]
    want = [step(*state(*s)) for s in sizes]
    torch.cuda.synchronize()
    states = [[state(*s) for s in sizes] for _ in range(6)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    got = []
    for pair in states:
        for i, st in enumerate(pair):
            with torch.cuda.stream(streams[i]):
                got.append((i, step(*st)))
    torch.cuda.synchronize()
    assert all(same(o, want[i]) for i, o in got)
