"""The operators around drafted tokens as a serving loop uses them together: pages reserved for a draft, attention of the tree
with append and rotary, the accepted path moved behind the prefix, surplus pages returned, sequences forked, the next step on
the children.  A plain model of it - dense lists of rows a sequence, float64 attention - goes along."""
import random

import pytest
import torch

import flash_attn_npu_3 as fa
from flash_attn_npu import flash_attn_with_kvcache
from tests.tree_reference import depths, out_bound, tree_attention

pytestmark = pytest.mark.gpu

PAGE, HQ, HKV, D, T = 16, 8, 2, 64, 9


def path_of(parents, leaf):
    out = []
    while leaf >= 0:
        out.append(leaf)
        leaf = parents[leaf]
    return out[::-1]


class Plain:
    """Rows of every sequence, in order, for each of the layers."""

    def __init__(self, rows):
        self.rows = rows                                         # [seq][layer] -> (k rows, v rows)


def check_rows(plain, k_caches, v_caches, table, lens):
    table, lens = table.tolist(), lens.tolist()
    for b, n in enumerate(lens):
        for layer, (kc, vc) in enumerate(zip(k_caches, v_caches)):
            ks, vs = plain.rows[b][layer]
            assert len(ks) == n
            for cache, want in ((kc, ks), (vc, vs)):
                got = torch.stack([cache[table[b][j // PAGE], j % PAGE] for j in range(n)]).cpu() if n else torch.empty(0)
                assert n == 0 or torch.equal(got.view(torch.int16), torch.stack(want).view(torch.int16)), (b, layer)


@pytest.mark.parametrize("graph", [False, True])
def test_drafting_steps_with_forks(graph):
    rng = random.Random(5)
    layers, b, pages, width = 3, 4, 200, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    k_caches = [torch.randn(pages, PAGE, HKV, D, generator=g, device="cuda").bfloat16() for _ in range(layers)]
    v_caches = [torch.randn(pages, PAGE, HKV, D, generator=g, device="cuda").bfloat16() for _ in range(layers)]
    caches = k_caches + v_caches
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    start = [37, 0, 16, 90]
    lens = torch.tensor(start, dtype=torch.int32, device="cuda")
    assert fa.kvcache_reserve(refs, table, lens, PAGE).item() == 0
    plain = Plain([])
    for i, n in enumerate(start):
        t = table[i].tolist()
        plain.rows.append([([kc[t[j // PAGE], j % PAGE].cpu() for j in range(n)], [vc[t[j // PAGE], j % PAGE].cpu() for j in range(n)])
                           for kc, vc in zip(k_caches, v_caches)])
    ang = torch.arange(400, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    cos, sin = ang.cos().bfloat16(), ang.sin().bfloat16()
    cos_d, sin_d = cos.cuda(), sin.cuda()
    trees = torch.zeros(b, T, dtype=torch.int32, device="cuda")
    kept = torch.zeros(b, T, dtype=torch.int32, device="cuda")
    counts = torch.zeros(b, dtype=torch.int32, device="cuda")
    fork_of = torch.arange(b, dtype=torch.int32, device="cuda")
    q = [torch.zeros(b, T, HQ, D, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]
    k = [torch.zeros(b, T, HKV, D, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]
    v = [torch.zeros(b, T, HKV, D, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]

    def draft():
        missing = fa.kvcache_reserve(refs, table, lens, PAGE, extra=T)
        outs = [fa.flash_attn_tree_with_kvcache(q[i], k_caches[i], v_caches[i], k[i], v[i], trees, cache_seqlens=lens, page_table=table,
                                                rotary_cos=cos_d, rotary_sin=sin_d, rotary_interleaved=False) for i in range(layers)]
        return outs, missing

    def accept():
        lens.copy_(fa.kvcache_compact(caches, lens, kept, counts, page_table=table))
        fa.kvcache_free(refs, table, lens, PAGE)
        new_table, new_lens, missing = fa.kvcache_fork(caches, refs, table, lens, fork_of)
        table.copy_(new_table)
        lens.copy_(new_lens)
        return missing

    run_draft, run_accept = draft, accept
    if graph:                                                    # captured without running: nothing has moved yet
        saved = [x.clone() for x in caches + [refs, table, lens]]
        draft(), accept()                                        # loads what the first call of each kernel loads
        for x, y in zip(caches + [refs, table, lens], saved):
            x.copy_(y)
        torch.cuda.synchronize()
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1):
            drafted = draft()
        with torch.cuda.graph(g2):
            accepted = accept()

        def run_draft():
            g1.replay()
            return drafted

        def run_accept():
            g2.replay()
            return accepted
    for step in range(5):
        par = [[rng.randint(-1, i - 1) if i < T - rng.randint(0, 2) else -2 for i in range(T)] for _ in range(b)]
        trees.copy_(torch.tensor(par, dtype=torch.int32))
        for x in q + k + v:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        outs, missing = run_draft()
        torch.cuda.synchronize()
        assert missing.item() == 0
        host_lens = lens.tolist()
        for layer in range(layers):                              # against the plain rows, dense
            top = max(host_lens) + T
            kd, vd = torch.zeros(b, top, HKV, D).bfloat16(), torch.zeros(b, top, HKV, D).bfloat16()
            for i, n in enumerate(host_lens):
                if n:
                    kd[i, :n], vd[i, :n] = torch.stack(plain.rows[i][layer][0]), torch.stack(plain.rows[i][layer][1])
            want, _, mag = tree_attention(q[layer].cpu(), kd, vd, k[layer].cpu(), v[layer].cpu(), torch.tensor(par), host_lens, cos=cos, sin=sin,
                                          interleaved=False)
            assert ((outs[layer].cpu().double() - want).abs() <= out_bound(want, mag, torch.bfloat16)).all()
            for i, n in enumerate(host_lens):                    # drafted rows, as they stand in the plain cache now
                plain.rows[i][layer] = (plain.rows[i][layer][0] + [kd[i, n + t] for t in range(T)], plain.rows[i][layer][1] + [vd[i, n + t] for t in range(T)])
        keep, count, sons = [], [], []
        for i in range(b):
            there = [t for t, d in enumerate(depths(par[i])) if d >= 0]
            path = path_of(par[i], rng.choice(there)) if there and rng.random() < 0.9 else []
            keep.append(path + [-1] * (T - len(path)))
            count.append(len(path))
            sons.append(rng.randrange(b))
        kept.copy_(torch.tensor(keep, dtype=torch.int32)), counts.copy_(torch.tensor(count, dtype=torch.int32))
        fork_of.copy_(torch.tensor(sons, dtype=torch.int32))
        missing = run_accept()
        torch.cuda.synchronize()
        assert missing.item() == 0
        for i, n in enumerate(host_lens):
            plain.rows[i] = [tuple(r[:n] + [r[n + t] for t in keep[i][:count[i]]] for r in pair) for pair in plain.rows[i]]
        plain.rows = [[(list(kk), list(vv)) for kk, vv in plain.rows[s]] for s in sons]
        check_rows(plain, k_caches, v_caches, table, lens)
        held = [0] * pages
        for row in table.tolist():
            for x in row:
                if x >= 0:
                    held[x] += 1
        assert refs.tolist() == held
    # an ordinary decode step goes on from there
    fa.kvcache_reserve(refs, table, lens, PAGE, extra=1)
    n = lens.tolist()
    out = flash_attn_with_kvcache(q[0][:, :1], k_caches[0], v_caches[0], k[0][:, :1], v[0][:, :1], cache_seqlens=lens, block_table=table.clamp_min(0))
    for i in range(b):
        kk = torch.stack(plain.rows[i][0][0] + [k[0][i, 0].cpu()]).double()
        vv = torch.stack(plain.rows[i][0][1] + [v[0][i, 0].cpu()]).double()
        s = torch.einsum("hgd,nhd->hgn", q[0][i, 0].cpu().double().reshape(HKV, HQ // HKV, D), kk) * D ** -0.5
        p = torch.softmax(s, -1)
        want, mag = torch.einsum("hgn,nhd->hgd", p, vv).reshape(HQ, D), torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(HQ, D)
        assert ((out[i, 0].cpu().double() - want).abs() <= out_bound(want, mag, torch.bfloat16)).all()
    fa.kvcache_free(refs, table)
    assert refs.sum().item() == 0
    assert n == [len(plain.rows[i][0][0]) for i in range(b)]
