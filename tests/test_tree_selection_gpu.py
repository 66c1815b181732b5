"""flash_attn_tree_with_kvcache at the border where the list of key tiles no longer fits its counters: the same result on the
kernel that takes over."""
import pytest
import torch

import fa_b200_capi as capi
import flash_attn_npu_3 as fa
from tests.tree_reference import out_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,name", [(32767, "sm100_tcgen05_tree"), (32768, "generic_mma")])
def test_sequences_times_capacity(b, name):
    """One dense cache entry of 2^22 rows that all sequences read: 32768 of them make 2^30 key tiles, whatever their lengths."""
    g = torch.Generator(device="cuda").manual_seed(1)
    kc, vc = (torch.zeros(1, 1 << 22, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    kc[:, :64] = torch.randn(1, 64, 1, 64, generator=g, device="cuda").half()
    vc[:, :64] = torch.randn(1, 64, 1, 64, generator=g, device="cuda").half()
    q = torch.randn(b, 2, 1, 64, generator=g, device="cuda").half()
    lens = torch.randint(0, 60, (b,), generator=g, device="cuda", dtype=torch.int32)
    parents = torch.tensor([-1, 0], dtype=torch.int32, device="cuda")
    idx = torch.zeros(b, dtype=torch.int32, device="cuda")
    out, lse = fa.flash_attn_tree_with_kvcache(q, kc, vc, None, None, parents, cache_seqlens=lens, cache_batch_idx=idx, return_softmax_lse=True)
    assert capi.last_kernel() == name and capi.lib.fa_debug_get(2) == 0
    s = (q.double()[:, :, 0] @ kc[0, :64, 0].double().T) / 8
    seen = torch.arange(64, device="cuda") <= lens[:, None, None] + torch.arange(2, device="cuda")[:, None]
    s = s.masked_fill(~seen, float("-inf"))
    p, v = torch.softmax(s, -1), vc[0, :64, 0].double()
    want, mag = p @ v, p @ v.abs()
    assert ((out[:, :, 0].double() - want).abs() <= out_bound(want, mag, torch.float16)).all()
    ref = torch.logsumexp(s, -1)
    assert ((lse[:, 0].double() - ref).abs() <= 4e-5 * ref.abs().clamp_min(1)).all()
