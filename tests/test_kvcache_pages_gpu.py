"""Page operations against the sequential definitions (tests/pages_reference.py): everything is whole numbers or copied bits, so
everything is compared exactly."""
import random

import pytest
import torch

import flash_attn_npu_3 as fa
from tests import pages_reference as ref

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(rng, b, width, page, pages, hi, share=0.0):
    """Tables as a server has them after a while: some rows share full pages of an earlier row."""
    order = list(range(pages))
    rng.shuffle(order)
    table, lens = [], []
    for i in range(b):
        n = rng.randint(0, min(hi, width * page))
        row = []
        if table and rng.random() < share:
            j = rng.randrange(len(table))
            row = table[j][:min(n // page, lens[j] // page)]
            row = [x for x in row if x >= 0]
        while len(row) < ref.used(n, page, width) and order:
            row.append(order.pop())
        n = min(n, len(row) * page)
        table.append(row + [-1] * (width - len(row)))
        lens.append(n)
    refs = [0] * pages
    for row in table:
        for x in row:
            if x >= 0:
                refs[x] += 1
    return refs, table, lens


def bits(x):
    return x.contiguous().reshape(x.shape or (1,)).view(torch.uint8).cpu()


SHAPES = [(1, 1, 1, 1, 1), (3, 7, 16, 30, 100), (40, 33, 16, 900, 500), (17, 130, 64, 5000, 8000), (300, 20, 32, 9001, 600)]


@pytest.mark.parametrize("b,width,page,pages,hi", SHAPES)
@pytest.mark.parametrize("extra", [0, 1, 77])
@pytest.mark.parametrize("tight", [False, True])
def test_reserve_and_free(b, width, page, pages, hi, extra, tight):
    rng = random.Random(b * 1000 + extra)
    refs, table, lens = pool(rng, b, width, page, pages, hi, share=0.3)
    if tight:                                                    # hardly a page is free
        free = [p for p, r in enumerate(refs) if r == 0]
        for p in free[min(3, len(free)):]:
            refs[p] = 1
    for row in table:                                            # holes are filled too
        if rng.random() < 0.2 and row[0] >= 0:
            refs[row[0]] -= 1
            row[0] = -1
    r, t, n = i32(refs), i32(table), i32(lens)
    missing = fa.kvcache_reserve(r, t, n, page, extra=extra)
    want = ref.reserve(refs, table, lens, page, extra)
    assert missing.tolist() == [want] and t.tolist() == table and r.tolist() == refs
    fa.kvcache_free(r, t, n, page_size=page, extra=extra // 2)
    ref.free(refs, table, lens, page, extra // 2)
    assert t.tolist() == table and r.tolist() == refs
    fa.kvcache_free(r, t)
    ref.free(refs, table)
    assert t.tolist() == table and r.tolist() == refs


CACHES = {
    "bf16": lambda p, s: [torch.randn(p, s, 2, 64).bfloat16() for _ in range(3)],
    "stack": lambda p, s: [torch.randn(4, p, s, 3, 40).half()],
    "latent": lambda p, s: [torch.randint(-128, 128, (p, s, 512), dtype=torch.int8), torch.randn(p, s), torch.randn(p, s, 64).bfloat16()],
    "odd": lambda p, s: [torch.randint(-128, 128, (p, s, 3, 7), dtype=torch.int8), torch.randn(p, s, 1, 5).half()],
    "many": lambda p, s: [torch.randn(p, s, 1, 8).bfloat16() for _ in range(61)],
}


@pytest.mark.parametrize("kind", list(CACHES))
@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("b,n,page,hi,tight", [(1, 4, 16, 40, False), (5, 9, 16, 100, False), (4, 33, 7, 60, True), (6, 1, 64, 150, False), (3, 8, 1, 9, False)])
def test_fork(kind, keep, b, n, page, hi, tight):
    rng = random.Random(b + 10 * n + 100 * page + keep)
    width = hi // page + 2
    pages = b * (hi // page + 1) + (2 if tight else n + 3)
    refs, table, lens = pool(rng, b, width, page, pages, hi, share=0.5)
    if b > 2 and table[1][0] >= 0:
        refs[table[1][lens[1] // page if lens[1] % page else 0]] += 1   # somebody outside holds a page too
    parents = [rng.choice([rng.randrange(b), rng.randrange(b), 0, -1 if rng.random() < 0.3 else 0, b + 5 if rng.random() < 0.3 else 0]) for _ in range(n)]
    torch.manual_seed(n)
    caches = [c.cuda() for c in CACHES[kind](pages, page)]
    flat = []
    for c in caches:
        stack = c if c.dim() == 5 else c[None]
        for one in stack:
            flat.append([[bits(row).reshape(-1) for row in pg] for pg in one.cpu()])
    r, t, ln = i32(refs), i32(table), i32(lens)
    before = t.clone()
    nt, nl, missing = fa.kvcache_fork(caches[0] if kind == "stack" else caches, r, t, ln, i32(parents), keep_parents=keep)
    wt, wl, wm = ref.fork(flat, refs, table, lens, parents, page, keep)
    assert nt.tolist() == wt and nl.tolist() == wl and missing.tolist() == [wm] and r.tolist() == refs
    assert torch.equal(t, before) and ln.tolist() == lens
    got = []
    for c in caches:
        for one in (c if c.dim() == 5 else c[None]):
            got.append(torch.stack([bits(row).reshape(-1) for pg in one.cpu() for row in pg]))
    for g, w in zip(got, flat):
        assert torch.equal(g, torch.stack([row for pg in w for row in pg]))


def test_beams_keep_their_page_when_nobody_else_wants_it():
    refs, table, lens = [1, 1, 1, 0, 0], [[0, -1], [1, -1], [2, -1]], [5, 6, 7]
    c = torch.randn(5, 16, 1, 8, device="cuda")
    old = c.clone()
    r = i32(refs)
    nt, nl, missing = fa.kvcache_fork(c, r, i32(table), i32(lens), i32([2, 0, 2]))
    # row 0 takes the copy, row 2 keeps page 2; page 1 is let go, and being the lowest free one takes the copy
    assert nt.tolist() == [[1, -1], [0, -1], [2, -1]] and nl.tolist() == [7, 5, 7] and missing.item() == 0
    assert r.tolist() == [1, 1, 1, 0, 0]
    assert torch.equal(c[1, :7], old[2, :7]) and torch.equal(c[1, 7:], old[1, 7:])


@pytest.mark.parametrize("kind", list(CACHES))
def test_copy_pages(kind):
    torch.manual_seed(1)
    caches = [c.cuda() for c in CACHES[kind](40, 9)]
    src, dst = [3, 5, 3, 39, -1, 40, 7], [10, 11, 0, 12, 13, 14, 40]
    want = [c.clone() for c in caches]
    fa.kvcache_copy_pages(caches[0] if kind == "stack" else caches, i32(src), i32(dst))
    for w, c in zip(want, caches):
        v = w if w.dim() == 5 else w[None]
        for s, d in list(zip(src, dst))[:4]:
            v[:, d] = v[:, s]
        assert torch.equal(bits(w), bits(c))


def compact_reference(cache, table, lens, kept, counts, page, idx=None):
    """cache (entries, rows, ..) on the CPU, changed in place -> new lengths."""
    out = []
    width = len(table[0]) if table else 1
    cap = width * page
    for b, n in enumerate(lens):
        n = max(0, min(n, cap))
        def at(row):
            e = table[b][row // page] if table else idx[b] if idx else b
            return (e, row % page) if 0 <= e < cache.shape[0] else None
        done, last = 0, -1
        for i in range(min(max(counts[b], 0), len(kept[b])) if counts else len(kept[b])):
            k = kept[b][i]
            if k <= last or n + k >= cap:
                break
            s, d = at(n + k), at(n + i)
            if s and d and s != d:
                cache[d] = cache[s]
            last, done = k, done + 1
        out.append(n + done)
    return out


@pytest.mark.parametrize("kind", list(CACHES))
@pytest.mark.parametrize("b,t,page,dense", [(1, 1, 16, False), (5, 9, 16, False), (7, 64, 16, False), (3, 100, 64, True), (4, 300, 7, False), (2, 33, 40, True)])
@pytest.mark.parametrize("with_counts", [True, False])
def test_compact(kind, b, t, page, dense, with_counts):
    rng = random.Random(b + t + page)
    lens = [rng.randint(0, 90) for _ in range(b)]
    if b > 3:
        lens[1] = 0
    kept, counts = [], []
    for _ in range(b):
        c = rng.randint(0, t)
        kept.append(sorted(rng.sample(range(t), c)) + [-1] * (t - c))
        counts.append(rng.randint(0, t))
    if b > 2 and t > 5:
        kept[2][:4] = [1, 4, 4, 5]                               # the list ends where it does not grow
    rows = max(lens) + t - (3 if b == 5 else 0)                  # the capacity may end inside the draft
    torch.manual_seed(t)
    if dense:
        idx = list(range(b + 1))
        rng.shuffle(idx)
        idx = idx[:b]
        caches, table = CACHES[kind](b + 1, rows), None
    else:
        width = -(-rows // page)
        order = list(range(b * width + 2))
        rng.shuffle(order)
        table = [order[i * width:(i + 1) * width] for i in range(b)]
        if b == 4:
            table[0][1] = -1                                     # rows without a page do not move
            table[3][2] = 10 ** 6
        caches, idx = CACHES[kind](b * width + 2, page), None
    dev = [c.cuda() for c in caches]
    new = fa.kvcache_compact(dev[0] if kind == "stack" else dev, i32(lens), i32(kept), i32(counts) if with_counts else None,
                             page_table=None if dense else i32(table), cache_batch_idx=i32(idx) if dense else None)
    for c, g in zip(caches, dev):
        for one in (c if c.dim() == 5 else c[None]):
            want = compact_reference(one, table, lens, kept, counts if with_counts else None, one.shape[1], idx)
        assert torch.equal(bits(c), bits(g))
    assert new.tolist() == want


def test_pruning_a_whole_sequence():
    """Long lists of kept rows from row 0 on."""
    rng = random.Random(3)
    n, keep = 5000, 1777
    kept = [sorted(rng.sample(range(n), keep))]
    c = torch.randn(80, 64, 2, 64).bfloat16()
    order = list(range(80))
    rng.shuffle(order)
    g = c.cuda()
    new = fa.kvcache_compact(g, i32([0]), i32(kept), page_table=i32([order]))
    flat = c[torch.tensor(order)].reshape(-1, 2, 64)
    got = g.cpu()[torch.tensor(order)].reshape(-1, 2, 64)
    assert new.tolist() == [keep] and torch.equal(got[:keep], flat[torch.tensor(kept[0])]) and torch.equal(got[keep:], flat[keep:])


def test_strided_caches_and_tables():
    torch.manual_seed(4)
    kv = torch.randn(20, 16, 2, 3, 64, device="cuda").bfloat16()           # k and v of a page side by side
    k, v = kv[:, :, 0], kv[:, :, 1]
    want = kv.clone()
    big = torch.full((4, 50), -1, dtype=torch.int32, device="cuda")
    table = big[:, 10:14]
    table[:2] = i32([[3, 7, -1, -1], [5, 2, 9, -1]])
    refs = torch.zeros(20, dtype=torch.int32, device="cuda")
    refs[[3, 7, 5, 2, 9]] = 1
    nt, nl, missing = fa.kvcache_fork([k, v], refs, table[:2], i32([20, 33]), i32([1, 1, 0]), keep_parents=True)
    assert nt.tolist() == [[5, 2, 0, -1], [5, 2, 1, -1], [3, 4, -1, -1]] and missing.item() == 0
    want[0, :1], want[1, :1], want[4, :4] = want[9, :1], want[9, :1], want[7, :4]
    assert torch.equal(kv, want)
    assert (big[:, :10] == -1).all() and (big[:, 14:] == -1).all()
    fa.kvcache_reserve(refs, table, i32([33, 48, 1, 0]), 16, extra=16)
    assert table.tolist() == [[3, 7, 6, 8], [5, 2, 9, 10], [11, 12, -1, -1], [13, -1, -1, -1]]
    assert (big[:, :10] == -1).all() and (big[:, 14:] == -1).all()


def test_offsets_past_32_bits():
    c = torch.zeros(70000, 64, 8, 64, dtype=torch.bfloat16, device="cuda")
    c[69990] = 1.0
    c[69991, :10] = 2.0
    refs = torch.ones(70000, dtype=torch.int32, device="cuda")
    refs[69999] = 0
    nt, nl, _ = fa.kvcache_fork(c, refs, i32([[69990, 69991]]), i32([74]), i32([0]), keep_parents=True)
    assert nt.tolist() == [[69990, 69999]] and (c[69999, :10] == 2).all() and (c[69999, 10:] == 0).all()
    c[69999, 12] = 3.0
    new = fa.kvcache_compact(c, nl, i32([[2]]), page_table=nt)
    assert new.tolist() == [75] and (c[69999, 10] == 3).all()


def test_graph_with_changing_contents():
    rng = random.Random(9)
    refs, table, lens = pool(rng, 6, 10, 16, 80, 120)
    caches = torch.randn(2, 80, 16, 2, 64, device="cuda").bfloat16()
    r, t, n = i32(refs), i32(table), i32(lens)
    parents = i32([0, 1, 2, 3, 4, 5])

    def step():
        missing = fa.kvcache_reserve(r, t, n, 16, extra=5)
        nt, nl, m2 = fa.kvcache_fork(caches, r, t, n, parents)
        return missing, nt, nl, m2
    saved = r.clone(), t.clone()
    step()
    r.copy_(saved[0]), t.copy_(saved[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    r.copy_(saved[0]), t.copy_(saved[1])
    for trial in range(3):
        refs, table, lens = pool(rng, 6, 10, 16, 80, 120)
        par = [rng.randrange(6) for _ in range(6)]
        r.copy_(i32(refs)), t.copy_(i32(table)), n.copy_(i32(lens)), parents.copy_(i32(par))
        g.replay()
        torch.cuda.synchronize()
        want = ref.reserve(refs, table, lens, 16, 5)
        wt, wl, wm = ref.fork([], refs, table, lens, par, 16)
        assert out[0].item() == want and out[1].tolist() == wt and out[2].tolist() == wl and out[3].item() == wm and r.tolist() == refs


def test_empty():
    refs = torch.zeros(4, dtype=torch.int32, device="cuda")
    c = torch.zeros(4, 16, 1, 8, device="cuda")
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    assert fa.kvcache_reserve(refs, none, none[:, 0], 16).tolist() == [0]
    fa.kvcache_free(refs, none)
    t, n, m = fa.kvcache_fork(c, refs, i32([[0, -1]]), i32([3]), none[:, 0], keep_parents=True)
    assert t.shape == (0, 2) and n.shape == (0,) and m.tolist() == [0]
    fa.kvcache_copy_pages(c, none[:, 0], none[:, 0])
    assert fa.kvcache_compact(c, i32([3, 4]), torch.zeros(2, 0, dtype=torch.int32, device="cuda")).tolist() == [3, 4]
    wide = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    assert fa.kvcache_reserve(refs, wide, i32([5, 6]), 16).tolist() == [0]


def test_refusals():
    refs, table, lens = torch.zeros(4, dtype=torch.int32, device="cuda"), i32([[0, -1]]), i32([3])
    c = torch.zeros(4, 16, 1, 8, device="cuda")
    for call, word in [
        (lambda: fa.kvcache_reserve(refs.long(), table, lens, 16), "int32"),
        (lambda: fa.kvcache_reserve(refs, table, lens, 0), "page_size"),
        (lambda: fa.kvcache_reserve(refs, table, lens, 16, extra=-1), "extra"),
        (lambda: fa.kvcache_reserve(refs, table, i32([1, 2]), 16), "shape"),
        (lambda: fa.kvcache_reserve(refs, table.expand(3, 2), i32([1, 2, 3]), 16), "in place"),
        (lambda: fa.kvcache_reserve(refs, table.cpu(), lens, 16), "CUDA"),
        (lambda: fa.kvcache_reserve(refs, i32([[0, 1, 2, 3]])[:, ::2], lens, 16), "in place"),
        (lambda: fa.kvcache_free(refs, table, lens), "page_size"),
        (lambda: fa.kvcache_fork(c, refs[:3], table, lens, i32([0])), "page_refs"),
        (lambda: fa.kvcache_fork([], refs, table, lens, i32([0])), "at least one"),
        (lambda: fa.kvcache_fork([c, c[:, :8]], refs, table, lens, i32([0])), "same number"),
        (lambda: fa.kvcache_fork(c.cpu(), refs, table, lens, i32([0])), "CUDA"),
        (lambda: fa.kvcache_fork(c[:1].expand(4, 16, 1, 8), refs, table, lens, i32([0])), "expanded"),
        (lambda: fa.kvcache_fork(c.transpose(2, 3), refs, table, lens, i32([0])), "contiguous"),
        (lambda: fa.kvcache_copy_pages(c, i32([0, 1]), i32([2])), "shape"),
        (lambda: fa.kvcache_compact(c, lens, i32([[0]]), page_table=table, cache_batch_idx=lens), "paged"),
        (lambda: fa.kvcache_compact(c, lens, i32([0])), "shape"),
        (lambda: fa.kvcache_compact(c, i32([1] * 5), i32([[0]] * 5)), "fewer"),
    ]:
        with pytest.raises(RuntimeError, match=word):
            call()
