"""Row blocks times splits past what a grid's second dimension holds."""
import pytest
import torch

import fa_b200_capi as capi
import flash_attn_npu_3 as fa
from tests.test_tree_attention_refusals import params
from tests.tree_reference import out_bound


@pytest.mark.gpu
@pytest.mark.parametrize("d,softcap,name", [(64, 20.0, "sm100_tcgen05_2q"), (136, 0.0, "sm100_tcgen05_wide"), (64, 0.0, "sm100_tcgen05_tree")])
def test_256_row_blocks_in_256_splits(d, softcap, name):
    g = torch.Generator(device="cuda").manual_seed(2)
    t, hq, n = 256, 128, 300
    kc, vc = (torch.full((1, 131072, 1, d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kc[:, :n + t] = torch.randn(1, n + t, 1, d, generator=g, device="cuda").bfloat16()
    vc[:, :n + t] = torch.randn(1, n + t, 1, d, generator=g, device="cuda").bfloat16()
    q = torch.randn(1, t, hq, d, generator=g, device="cuda").bfloat16()
    parents = torch.arange(-1, t - 1, dtype=torch.int32, device="cuda")
    out, lse = fa.flash_attn_tree_with_kvcache(q, kc, vc, None, None, parents, cache_seqlens=n, softcap=softcap, num_splits=256, return_softmax_lse=True)
    assert capi.last_kernel() == name and capi.lib.fa_debug_get(2) == 0
    s = torch.einsum("thd,nd->htn", q[0].double(), kc[0, :n + t, 0].double()) * d ** -0.5
    s = softcap * torch.tanh(s / softcap) if softcap else s
    s = s.masked_fill(torch.arange(n + t, device="cuda") > n + torch.arange(t, device="cuda")[:, None], float("-inf"))
    p, v = torch.softmax(s, -1), vc[0, :n + t, 0].double()
    want, mag = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
    assert ((out[0].double() - want).abs() <= out_bound(want, mag, torch.bfloat16)).all()
    ref = torch.logsumexp(s, -1)
    assert ((lse[0].double() - ref).abs() <= 4e-5 * ref.abs().clamp_min(1)).all()


@pytest.mark.parametrize("sq,hq,hkv,ok", [(256, 32767, 1, True), (256, 32768, 1, False), (256, 1 << 19, 1 << 13, False), (1, 65535 * 128, 1, True), (1, 65535 * 128 + 1, 1, False),
                                            (1, 65530, 32765, True), (16, 1 << 22, 1 << 21, False), (128, 65535 * 15, 65535, False), (128, 65535 * 14, 65535, True)])
def test_more_heads_than_a_grid_holds(sq, hq, hkv, ok):
    t = params()
    t.fwd.sq, t.fwd.hq, t.fwd.hkv = sq, hq, hkv
    assert capi.lib.fa_tree_fwd_kvcache(t) == (6 if ok else 3)  # 6: the workspace, which comes after all shapes
    assert (b"workspace" if ok else b"heads") in capi.lib.fa_last_error()
