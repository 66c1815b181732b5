"""Lazily negated tensors (torch's neg bit, as .imag of a conjugate has it) are read with their sign."""
import pytest
import torch

import flash_attn_npu_3 as fa
from tests.test_rotary_axes_gpu import inputs
from tests.test_tree_attention_gpu import make

pytestmark = pytest.mark.gpu


def test_rotary_tables_in_place():
    q, k, cos, sin, pos = inputs(torch.bfloat16, (2, 4), 4, 2, 64, 64, 1, torch.float32)
    z = torch.complex(cos, sin).conj()
    for tables, plain in (((z.real, z.imag), (cos, -sin)), ((cos, torch._neg_view(sin)), (cos, -sin)), ((torch._neg_view(cos), sin), (-cos, sin))):
        want = fa.rotary_axes_func(q, k, *plain, pos)
        here = fa.rotary_axes_func(q.clone(), k.clone(), *tables, pos, inplace=True)
        assert all(torch.equal(x, y) for x, y in zip(want, here))


@pytest.mark.parametrize("table", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["q", "k", "v", "cos", "sin"])
def test_tree_attention(name, table):
    c = make(torch.bfloat16, 128, 8, 2, [100, 33], 7, 64, seed=3, rotary="half")
    dev = {key: (x.cuda() if isinstance(x, torch.Tensor) else x) for key, x in c.items()}
    dev["cos"], dev["sin"] = dev["cos"].to(table), dev["sin"].to(table)

    def run(c):
        kc, vc = c["kc"].clone(), c["vc"].clone()
        out = fa.flash_attn_tree_with_kvcache(c["q"], kc, vc, c["k"], c["v"], c["parents"], cache_seqlens=c["lens"], page_table=c["table"],
                                              rotary_cos=c["cos"], rotary_sin=c["sin"], rotary_interleaved=False)
        return [x.contiguous().view(torch.int16) for x in (out, kc, vc)]
    want = run(dict(dev, **{name: -dev[name]}))
    got = run(dict(dev, **{name: torch._neg_view(dev[name])}))
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("name", ["kc", "vc"])
def test_a_negated_cache_is_refused(name):
    c = make(torch.bfloat16, 128, 8, 2, [100, 33], 7, 64, seed=3)
    dev = {key: (x.cuda() if isinstance(x, torch.Tensor) else x) for key, x in c.items()}
    dev[name] = torch._neg_view(dev[name])
    with pytest.raises(RuntimeError, match="negated"):
        fa.flash_attn_tree_with_kvcache(dev["q"], dev["kc"], dev["vc"], dev["k"], dev["v"], dev["parents"], cache_seqlens=dev["lens"], page_table=dev["table"])


def test_rotary_in_place_on_negated_q_and_k():
    """The memory is turned: the negative of the turned is the turned negative, bit for bit."""
    q, k, cos, sin, pos = inputs(torch.bfloat16, (2, 4), 4, 2, 64, 48, 1, torch.float32)
    want = fa.rotary_axes_func(-q, -k, cos, sin, pos)
    a, b = q.clone(), k.clone()
    here = fa.rotary_axes_func(torch._neg_view(a), torch._neg_view(b), cos, sin, pos, inplace=True)
    assert all(torch.equal(x, y) for x, y in zip(want, here)) and torch.equal(-a, want[0]) and torch.equal(-b, want[1])
