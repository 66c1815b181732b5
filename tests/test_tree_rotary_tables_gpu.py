"""fp32 tables of angles: the tree call turns keys to the same bits as rotary_axes_func does."""
import pytest
import torch

import flash_attn_npu_3 as fa
from tests.test_tree_attention_gpu import check, make, same_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotary,axes", [("half", 1), ("interleaved", 3), ("partial", 2), ("partial", 1)])
@pytest.mark.parametrize("dtype,d,page", [(torch.bfloat16, 128, 64), (torch.float16, 64, 0), (torch.bfloat16, 256, 16), (torch.float16, 40, 12)])
def test_against_the_plain_form(rotary, axes, dtype, d, page):
    c = make(dtype, d, 4, 2, [150, 3, 77], 9, page, seed=d + axes, rotary=rotary, axes=axes, ragged=True)
    g = torch.Generator().manual_seed(d)
    ang = torch.rand(c["cos"].shape, generator=g) * 6.28
    c["cos"], c["sin"] = ang.cos(), ang.sin()
    check(c)


def test_the_same_bits_as_the_rotary_call():
    c = make(torch.bfloat16, 128, 8, 2, [100, 33], 7, 64, seed=3, rotary="half", axes=3)
    ang = torch.rand(c["cos"].shape) * 6.28
    dev = {k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in c.items()}
    cos, sin = ang.cos().cuda(), ang.sin().cuda()
    kw = dict(cache_seqlens=dev["lens"], page_table=dev["table"])
    caches = [(dev["kc"].clone(), dev["vc"].clone()) for _ in range(2)]
    a = fa.flash_attn_tree_with_kvcache(dev["q"], *caches[0], dev["k"], dev["v"], dev["parents"], rotary_cos=cos, rotary_sin=sin,
                                        rotary_positions=dev["positions"], rotary_sections=dev["sections"], rotary_interleaved=False, **kw)
    q, k = fa.rotary_axes_func(dev["q"], dev["k"], cos, sin, dev["positions"], sections=dev["sections"])
    b = fa.flash_attn_tree_with_kvcache(q, *caches[1], k, dev["v"], dev["parents"], **kw)
    assert same_bits(a, b) and same_bits(caches[0][0], caches[1][0])


def test_one_table_in_fp32():
    """Tables of two types are both taken in q's."""
    c = make(torch.bfloat16, 128, 8, 2, [100, 33], 7, 64, seed=3, rotary="half")
    want = dict(c)
    c["cos"] = c["cos"].float()
    check(c)
    check(want)
