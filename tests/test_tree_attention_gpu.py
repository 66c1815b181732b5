"""flash_attn_tree_with_kvcache against the plain float64 form (tests/tree_reference.py): trees, cache layouts, windows, caps,
rotary axes, drafts with missing tokens, capacities and pages that end early.  Cache rows that hold nothing are NaN, and every
cache row that the call may not touch is compared bit for bit."""
import random

import pytest
import torch

import fa_b200_capi as capi
import flash_attn_npu_3 as fa
from tests.tree_reference import depths, out_bound, tree_attention

pytestmark = pytest.mark.gpu


def random_tree(rng, n, total, holes=0.0):
    par = [rng.randint(-1, i - 1) if rng.random() < 0.6 else i - 1 for i in range(n)]
    par = [-2 if rng.random() < holes else p for p in par]
    return par + [-2] * (total - n)


def make(dtype, d, hq, hkv, lens, t, page, seed, holes=0.0, ragged=False, rotary=None, axes=1, extra_pages=2):
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    c = dict(q=torch.randn(b, t, hq, d, generator=g).to(dtype), k=torch.randn(b, t, hkv, d, generator=g).to(dtype),
             v=torch.randn(b, t, hkv, d, generator=g).to(dtype), lens=torch.tensor(lens, dtype=torch.int32))
    c["parents"] = torch.tensor([random_tree(rng, rng.randint(1, t) if ragged else t, t, holes) for _ in range(b)], dtype=torch.int32)
    if page:
        per = [-(-(n + t) // page) for n in lens]
        pages = sum(per) + extra_pages
        order = list(range(pages))
        rng.shuffle(order)
        width = max(per) + 1
        table, at = torch.full((b, width), -1, dtype=torch.int32), 0
        for i, n in enumerate(per):
            table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        kc, vc = torch.full((pages, page, hkv, d), float("nan"), dtype=dtype), torch.full((pages, page, hkv, d), float("nan"), dtype=dtype)
        for i, n in enumerate(lens):
            for j in range(n):
                at2 = (int(table[i, j // page]), j % page)
                kc[at2], vc[at2] = torch.randn(hkv, d, generator=g).to(dtype), torch.randn(hkv, d, generator=g).to(dtype)
        c["table"] = table
    else:
        kc = torch.full((b, max(lens) + t + 5, hkv, d), float("nan"), dtype=dtype)
        vc = kc.clone()
        for i, n in enumerate(lens):
            kc[i, :n], vc[i, :n] = torch.randn(n, hkv, d, generator=g).to(dtype), torch.randn(n, hkv, d, generator=g).to(dtype)
        c["table"] = None
    c.update(kc=kc, vc=vc, cos=None, sin=None, positions=None, sections=None, axis=None, interleaved=rotary == "interleaved")
    if rotary:
        rd = d if rotary != "partial" else d // 2 + 8
        pairs, rows = rd // 2, max(lens) + t
        ang = torch.rand(rows, pairs, generator=g) * 6.28
        c["cos"], c["sin"] = ang.cos().to(dtype), ang.sin().to(dtype)
        if axes > 1:
            c["positions"] = torch.randint(-2, rows + 2, (axes, b, t), generator=g).int()
            rest = [pairs // (axes + 1)] * (axes - 1)
            c["sections"] = [pairs - sum(rest)] + rest
            c["axis"] = [a for a, s in enumerate(c["sections"]) for _ in range(s)]
    return c


def call(c, left=-1, softcap=0.0, num_splits=0, **kw):
    dev = {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    out, lse = fa.flash_attn_tree_with_kvcache(
        dev["q"], dev["kc"], dev["vc"], dev["k"], dev["v"], dev["parents"], cache_seqlens=dev["lens"], page_table=dev["table"],
        rotary_cos=dev["cos"], rotary_sin=dev["sin"], rotary_positions=dev["positions"], rotary_sections=dev["sections"],
        rotary_interleaved=dev["interleaved"], window_size=(left, -1), softcap=softcap, num_splits=num_splits,
        return_softmax_lse=True, **kw)
    torch.cuda.synchronize()
    assert capi.lib.fa_debug_get(2) == 0
    return out.cpu(), lse.cpu(), dev["kc"].cpu(), dev["vc"].cpu()


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def check(c, left=-1, softcap=0.0, num_splits=0, **kw):
    out, lse, kc, vc = call(c, left, softcap, num_splits, **kw)
    kr, vr = c["kc"].clone(), c["vc"].clone()
    ro, rl, mag = tree_attention(c["q"], kr, vr, c["k"], c["v"], c["parents"], c["lens"], c["table"], None, c["cos"], c["sin"],
                                 c["positions"], c["axis"], c["interleaved"], None, left, softcap)
    assert same_bits(kc, kr) and same_bits(vc, vr), "cache rows differ"
    assert torch.isfinite(out.float()).all()
    err, tol = (out.double() - ro).abs(), out_bound(ro, mag, out.dtype)
    assert (err <= tol).all(), f"out: {(err / tol).max().item():.2f} of its bound"
    fin = torch.isfinite(rl)
    assert torch.equal(fin, torch.isfinite(lse)) and (lse[~fin] > 0).all()
    assert ((lse.double() - rl)[fin].abs() <= 4e-5 * rl[fin].abs().clamp_min(1)).all()


LAYOUTS = [  # dtype, d, hq, hkv, lens, t, page
    ("bf16", 128, 8, 2, [300, 1, 77], 9, 64),
    ("fp16", 64, 4, 4, [129, 128, 127], 5, 16),
    ("bf16", 128, 14, 2, [500, 255], 33, 128),
    ("fp16", 128, 16, 2, [640, 33], 64, 64),
    ("bf16", 64, 6, 2, [1000, 3, 250, 511], 13, 0),
    ("bf16", 256, 4, 2, [270, 19], 12, 64),
    ("fp16", 192, 8, 1, [200, 129], 40, 256),
    ("bf16", 96, 4, 2, [150, 40], 7, 32),
    ("bf16", 40, 3, 1, [90, 17], 6, 48),
    ("fp16", 128, 8, 8, [260], 100, 192),
    ("bf16", 128, 16, 1, [333, 12], 256, 64),
]
_T = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y).replace(" ", "") for y in x))
@pytest.mark.parametrize("num_splits", [0, 1, 3])
def test_layouts(layout, num_splits):
    dt, d, hq, hkv, lens, t, page = layout
    check(make(_T[dt], d, hq, hkv, lens, t, page, seed=d + t), num_splits=num_splits)


@pytest.mark.parametrize("layout", LAYOUTS[:8], ids=lambda x: "-".join(str(y).replace(" ", "") for y in x))
@pytest.mark.parametrize("left,softcap", [(37, 0.0), (0, 0.0), (130, 20.0), (-1, 5.0)])
def test_windows_and_caps(layout, left, softcap):
    dt, d, hq, hkv, lens, t, page = layout
    check(make(_T[dt], d, hq, hkv, lens, t, page, seed=3 * d + t, ragged=True), left=left, softcap=softcap)


@pytest.mark.parametrize("rotary,axes", [("half", 1), ("interleaved", 1), ("half", 3), ("interleaved", 4), ("partial", 1), ("partial", 2)])
@pytest.mark.parametrize("layout", LAYOUTS[:8:2], ids=lambda x: "-".join(str(y).replace(" ", "") for y in x))
def test_rotary(layout, rotary, axes):
    dt, d, hq, hkv, lens, t, page = layout
    check(make(_T[dt], d, hq, hkv, lens, t, page, seed=5 * d + t, rotary=rotary, axes=axes))


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y).replace(" ", "") for y in x))
def test_missing_tokens_are_neither_written_nor_seen(layout):
    dt, d, hq, hkv, lens, t, page = layout
    c = make(_T[dt], d, hq, hkv, lens, t, page, seed=7 * d + t, holes=0.25, ragged=True, rotary="half")
    c["k"][c["parents"] < -1], c["v"][c["parents"] < -1] = float("nan"), float("inf")
    check(c)
    c["q"][c["parents"] < -1] = float("nan")
    check(c)
    check(c, softcap=8.0)
    check(c, num_splits=2)


@pytest.mark.parametrize("t", [1, 2, 31, 32, 33, 65])
@pytest.mark.parametrize("lens", [[0, 1, 0], [127, 128, 129], [95, 96, 97]])
def test_short_prefixes_and_word_edges(t, lens):
    check(make(torch.bfloat16, 64, 4, 2, lens, t, 64, seed=t))


def test_all_missing():
    c = make(torch.bfloat16, 128, 8, 2, [100, 50], 6, 64, seed=1)
    c["parents"][0] = -2
    check(c)


@pytest.mark.parametrize("bad", [5, 6, -7, 2 ** 31 - 1, -2 ** 31])
def test_parents_outside_the_tree_mean_no_token(bad):
    c = make(torch.bfloat16, 64, 4, 2, [70], 6, 64, seed=2)
    c["parents"] = torch.tensor([[-1, 0, bad, 2, 1, 3]], dtype=torch.int32)
    check(c)


def test_chain_is_the_causal_call():
    c = make(torch.bfloat16, 128, 8, 2, [300, 77], 16, 64, seed=11)
    c["parents"] = torch.arange(-1, 15, dtype=torch.int32)[None].repeat(2, 1)
    out, lse, kc, vc = call(c)
    dev = {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    ref = fa.flash_attn_with_kvcache(dev["q"], dev["kc"], dev["vc"], dev["k"], dev["v"], cache_seqlens=dev["lens"], page_table=dev["table"], causal=True)
    # two results with the bound of out_bound each, |o| and sum p |v| at most max |v| = 4.5 here
    assert (out.float() - ref.cpu().float()).abs().max().item() <= 2 * (2 * 2.0 ** -8 + 2.0 ** -12) * 4.5
    assert same_bits(kc, dev["kc"].cpu())


@pytest.mark.parametrize("page", [0, 64, 16])
def test_capacity_ends_inside_the_draft(page):
    c = make(torch.bfloat16, 128, 8, 2, [60, 120], 20, page, seed=4)
    if page:
        c["table"] = c["table"][:, :max(1, 128 // page)].contiguous()
    else:
        c["kc"], c["vc"] = c["kc"][:, :128].contiguous(), c["vc"][:, :128].contiguous()
    check(c)
    c["lens"] = torch.tensor([60, 128], dtype=torch.int32)      # full: the draft sees the prefix only
    c["kc"], c["vc"] = c["kc"].nan_to_num(0.5), c["vc"].nan_to_num(0.5)
    check(c)
    c["lens"] = torch.tensor([-5, 10 ** 9], dtype=torch.int32)  # stale lengths are truncated
    check(c)


@pytest.mark.parametrize("page,d", [(64, 128), (16, 64), (32, 96), (64, 256)])
def test_pages_outside_the_cache(page, d):
    c = make(torch.bfloat16, d, 4, 2, [200, 150], 12, page, seed=6)
    last = (200 + 11) // page
    c["table"][0, last] = -1                                    # part of the draft has no page
    c["table"][1, 1] = c["kc"].shape[0] + 3                     # a prefix page that does not exist reads as zeros
    check(c)


def test_keys_already_in_the_cache_and_shared_tree():
    c = make(torch.float16, 128, 8, 2, [100, 222], 10, 64, seed=8)
    out, lse, kc, vc = call(c)
    c2 = dict(c, kc=kc, vc=vc, k=None, v=None)
    out2, lse2, kc2, _ = call(c2)
    assert same_bits(out, out2) and torch.equal(lse, lse2) and same_bits(kc, kc2)
    c3 = dict(c, parents=c["parents"][0].contiguous())
    out3, _, _, _ = call(c3)
    assert same_bits(out3[0], out[0])


def test_strided_inputs_and_batch_index():
    c = make(torch.bfloat16, 64, 8, 2, [70, 33], 9, 0, seed=9)
    want, lse, _, _ = call(c)
    dev = {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    qkv = torch.zeros(2, 9, 12, 72, dtype=torch.bfloat16, device="cuda")
    qkv[:, :, :8, :64], qkv[:, :, 8:10, :64], qkv[:, :, 10:, :64] = dev["q"], dev["k"], dev["v"]
    big = torch.full((5,) + c["kc"].shape[1:], float("nan"), dtype=torch.bfloat16, device="cuda")
    kc, vc = big.clone(), big.clone()
    idx = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    kc[idx.long()], vc[idx.long()] = dev["kc"], dev["vc"]
    out = fa.flash_attn_tree_with_kvcache(qkv[:, :, :8, :64], kc, vc, qkv[:, :, 8:10, :64], qkv[:, :, 10:, :64], dev["parents"],
                                          cache_seqlens=dev["lens"], cache_batch_idx=idx)
    assert same_bits(out.cpu(), want)
    odd = torch.zeros(2, 9, 8, 65, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = dev["q"]
    out = fa.flash_attn_tree_with_kvcache(odd[..., 1:], kc, vc, qkv[:, :, 8:10, :64], qkv[:, :, 10:, :64], dev["parents"],
                                          cache_seqlens=dev["lens"], cache_batch_idx=idx)
    assert same_bits(out.cpu(), want)


def test_graph_replays_with_new_lengths_and_trees():
    c = make(torch.bfloat16, 128, 8, 2, [300, 40], 12, 64, seed=10, extra_pages=40)
    dev = {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}

    def step():
        return fa.flash_attn_tree_with_kvcache(dev["q"], dev["kc"], dev["vc"], dev["k"], dev["v"], dev["parents"],
                                               cache_seqlens=dev["lens"], page_table=dev["table"], return_softmax_lse=True)
    step()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = step()
    with torch.cuda.graph(g2):
        out2, lse2 = step()
    for seed in (20, 21):
        n = make(torch.bfloat16, 128, 8, 2, [200 + seed, 30], 12, 64, seed=seed, ragged=True, extra_pages=40)
        for key in ("q", "k", "v", "parents", "lens"):
            dev[key].copy_(n[key])
        c2 = dict(c, q=n["q"], k=n["k"], v=n["v"], parents=n["parents"], lens=n["lens"], kc=dev["kc"].cpu(), vc=dev["vc"].cpu())
        g.replay()
        g2.replay()
        torch.cuda.synchronize()
        kr, vr = c2["kc"].clone(), c2["vc"].clone()
        ro, rl, mag = tree_attention(c2["q"], kr, vr, c2["k"], c2["v"], c2["parents"], c2["lens"], c2["table"])
        for o in (out, out2):
            assert ((o.cpu().double() - ro).abs() <= out_bound(ro, mag, torch.bfloat16)).all()


def test_long_cache_and_bitwise_repeats():
    c = make(torch.bfloat16, 64, 8, 1, [5000], 20, 64, seed=12)
    check(c)
    a, b = call(c), call(c)
    assert same_bits(a[0], b[0]) and torch.equal(a[1], b[1])


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements; the sequence stands in its last pages."""
    pages, page, h, d = 36000, 64, 8, 128
    kc = torch.zeros(pages, page, h, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    c = make(torch.bfloat16, d, 16, h, [100], 7, page, seed=13)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32)
    small = c["kc"][c["table"][0, :2].long()], c["vc"][c["table"][0, :2].long()]
    kc[table[0].long().cuda()], vc[table[0].long().cuda()] = small[0].cuda(), small[1].cuda()
    out = fa.flash_attn_tree_with_kvcache(c["q"].cuda(), kc, vc, c["k"].cuda(), c["v"].cuda(), c["parents"].cuda(),
                                          cache_seqlens=c["lens"].cuda(), page_table=table.cuda())
    kr, vr = c["kc"].clone(), c["vc"].clone()
    ro, _, mag = tree_attention(c["q"], kr, vr, c["k"], c["v"], c["parents"], c["lens"], c["table"])
    assert ((out.cpu().double() - ro).abs() <= out_bound(ro, mag, torch.bfloat16)).all()
    assert same_bits(kc[table[0].long().cuda()].cpu(), kr[c["table"][0, :2].long()])


def test_empty_calls():
    c = make(torch.bfloat16, 64, 4, 2, [70], 6, 64, seed=2)
    dev = {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    for b, t in ((0, 6), (1, 0)):
        out, lse = fa.flash_attn_tree_with_kvcache(dev["q"][:b, :t], dev["kc"], dev["vc"], dev["k"][:b, :t], dev["v"][:b, :t],
                                                   dev["parents"][:b, :t], cache_seqlens=dev["lens"][:b], page_table=dev["table"][:b],
                                                   return_softmax_lse=True)
        assert out.shape == (b, t, 4, 64) and lse.shape == (b, 4, t)


def test_depths_of_the_reference():
    assert depths([-1, 0, 0, 2, -2, 4, 5, 7]) == [0, 1, 1, 2, -1, -1, -1, -1]


@pytest.mark.parametrize("d,softcap,page,hq,t,name,form", [
    (128, 0.0, 64, 8, 16, "sm100_tcgen05_tree", 1), (64, 0.0, 16, 14, 40, "sm100_tcgen05_tree", 0), (128, 20.0, 0, 6, 9, "sm100_tcgen05_2q", 2),
    (256, 0.0, 32, 4, 9, "sm100_tcgen05_wide", 0), (192, 5.0, 128, 4, 9, "sm100_tcgen05_wide", 0), (96, 0.0, 64, 4, 9, "sm100_tcgen05_tree", 1), (224, 0.0, 64, 4, 9, "sm100_tcgen05_wide", 0),
    (40, 9.0, 16, 8, 20, "sm100_tcgen05_2q", 2),
    (128, 0.0, 48, 8, 16, "sm100_tcgen05_tree", 1), (128, 0.0, 40, 8, 16, "sm100_tcgen05_tree", 1), (128, 0.0, 36, 8, 16, "generic_mma", 0), (72, 0.0, 1, 8, 16, "generic_mma", 0)])
def test_which_kernel_runs(d, softcap, page, hq, t, name, form):
    check(make(torch.bfloat16, d, hq, 2, [150, 300], t, page, seed=d + page), softcap=softcap)
    assert capi.last_kernel() == name and capi.lib.fa_debug_get(8) == form


def test_the_general_kernels_agree():
    c = make(torch.bfloat16, 128, 14, 2, [400, 77], 30, 64, seed=31, ragged=True, rotary="half", axes=3)
    capi.lib.fa_set_kernel_policy(1)
    try:
        check(c)
        assert capi.last_kernel() == "generic_mma"
    finally:
        capi.lib.fa_set_kernel_policy(0)
    check(c)


@pytest.mark.parametrize("hq,hkv,t,lens", [
    (8, 2, 16, [900, 5, 0, 130, 2000, 64, 300]),          # shares that end inside sequences, sequences inside a share
    (8, 8, 33, [1] * 40),                                 # more units than CTAs, a tile each
    (32, 1, 20, [3000, 1, 1, 1]),                         # several row blocks of a KV head
    (4, 1, 200, [700, 90]),
    (2, 2, 3, [12000]),                                   # one sequence over many CTAs
    (16, 16, 2, [40, 700] * 20),                          # 640 units
    (8, 1, 16, [20000]),                                  # ... an SM each: pieces shared out to the warps that join them
    (8, 1, 31, [9000, 11, 7000]),
])
@pytest.mark.parametrize("left", [-1, 100])
def test_shares_of_the_key_tiles(hq, hkv, t, lens, left):
    check(make(torch.bfloat16, 64, hq, hkv, lens, t, 64, seed=t + len(lens)), left=left)
    assert capi.last_kernel() == "sm100_tcgen05_tree"


def test_many_sequences():
    """More sequences than one step of the search for a CTA's first one looks at."""
    check(make(torch.bfloat16, 64, 2, 1, [(37 * i) % 300 for i in range(1100)], 2, 64, seed=3))


@pytest.mark.parametrize("d", [40, 72, 96, 120])
def test_workspace_has_room_for_padded_head_dims(d):
    """The pieces of cut sequences have the kernel's head dim, 64 or 128, whatever the call's is."""
    def need(dim):
        t = capi.TreeParams()
        p = t.fwd
        p.dtype, p.b, p.sq, p.sk, p.hq, p.hkv, p.d, p.dv, p.scale, p.kv_entries, p.page_size = 1, 16, 26, 8192, 32, 8, dim, dim, 0.1, 999, 64
        p.block_table, p.window_left = 0x1000, -1
        for x in (p.k, p.v):
            x.stride_b, x.stride_s, x.stride_h = 1 << 20, 8 * dim, dim
        return capi.lib.fa_tree_workspace_bytes(t), 16 * 26 * 32 * dim * 2
    full, queries = need(64 if d <= 64 else 128)
    got, fewer = need(d)
    assert got - fewer >= full - queries - 256


def test_padded_head_dim_over_many_pieces():
    check(make(torch.bfloat16, 96, 8, 4, [3000, 1700, 40, 2500], 26, 64, seed=17))
    check(make(torch.float16, 40, 16, 2, [2600, 900], 30, 16, seed=18))
