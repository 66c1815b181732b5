"""rotary_axes_func: forward and gradients against the formula, in place, layouts, streams, graphs, refusals.

The kernels compute a c - b s and a s + b c in fp32 with separately rounded products and round once to the element type: the
same steps in torch give the same bits.  Against float64 an element is off by half a step of its type (eps / 2 of its value) and
by three fp32 roundings of terms of at most |a c| + |b s|."""
import pytest
import torch

import fa_b200_capi as capi
import flash_attn_npu_3 as fa

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def axes_of(pairs, sections, cyclic):
    if sections is None:
        return torch.zeros(pairs, dtype=torch.long)
    n = len(sections)
    if cyclic:
        return torch.tensor([i % n if i < n * sections[i % n] else 0 for i in range(pairs)])
    return torch.tensor([a for a, s in enumerate(sections) for _ in range(s)])


def plain(x, cos, sin, positions, axis, interleaved, back=False, dtype=torch.float32):
    pairs = cos.shape[1]
    i = torch.arange(pairs, device=x.device)
    rows = positions.long().clamp(0, cos.shape[0] - 1)[axis.to(x.device)].movedim(0, -1)
    c, s = cos.to(dtype)[rows, i][..., None, :], sin.to(dtype)[rows, i][..., None, :] * (-1 if back else 1)
    y = x.to(dtype).clone()
    lo, hi = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = x.to(dtype)[..., lo], x.to(dtype)[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    mag = torch.zeros_like(y)
    mag[..., lo], mag[..., hi] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, mag


def inputs(dtype, lead, hq, hk, d, rd, axes, table, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(*lead, hq, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(*lead, hk, d, generator=g, device="cuda").to(dtype)
    rows = 50
    ang = torch.rand(rows, rd // 2, generator=g, device="cuda", dtype=torch.float64) * 6.3
    cos, sin = ang.cos().to(table), ang.sin().to(table)
    pos = torch.randint(-3, rows + 3, (axes, *lead), generator=g, device="cuda", dtype=torch.int32)
    return q, k, cos, sin, pos


def sections_of(axes, pairs):
    if axes == 1:
        return None
    rest = [pairs // (axes + 1)] * (axes - 1)
    return [pairs - sum(rest)] + rest


CASES = [  # dtype, lead, hq, hk, d, rd, axes, cyclic, interleaved, fp32 tables
    ("bf16", (2, 5), 8, 2, 128, 128, 3, False, False, True),
    ("fp16", (17,), 4, 4, 64, 64, 3, True, False, False),
    ("bf16", (1, 1), 32, 8, 128, 128, 1, False, True, True),
    ("bf16", (3, 33), 7, 1, 256, 256, 4, True, True, False),
    ("fp16", (2, 9), 5, 3, 96, 48, 2, False, False, True),
    ("bf16", (2, 9), 5, 3, 80, 40, 2, False, False, True),       # rotary dim no multiple of 16: four elements at once
    ("fp16", (31,), 6, 1, 128, 40, 3, False, True, False),
    ("bf16", (3, 5), 8, 2, 256, 72, 2, True, False, True),
    ("fp16", (9,), 4, 2, 60, 24, 3, False, False, False),         # a row ends inside a unit
    ("bf16", (2, 6), 2, 1, 20, 16, 1, False, True, True),
    ("fp16", (5,), 3, 2, 72, 20, 2, False, False, True),         # element by element
    ("fp16", (11,), 3, 2, 72, 22, 3, False, True, False),
    ("bf16", (4, 3), 2, 2, 50, 34, 1, False, False, True),       # head dim no multiple of 8
    ("bf16", (700,), 16, 16, 64, 32, 3, True, True, True),
    ("bf16", (2, 300), 40, 8, 128, 64, 3, False, False, True),
]


def check(got, x, args, back=False):
    same, _ = plain(x, *args, back=back)
    assert torch.equal(got.view(torch.int16), same.to(x.dtype).view(torch.int16)), "not the bits of the same fp32 steps"
    want, mag = plain(x, *args, back=back, dtype=torch.float64)
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + (1 + torch.finfo(x.dtype).eps) * 3 * 2.0 ** -24 * mag + torch.finfo(x.dtype).smallest_normal * 2.0 ** -9
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_forward_backward_and_in_place(case):
    dt, lead, hq, hk, d, rd, axes, cyclic, inter, fp32 = case
    dtype = DT[dt]
    q, k, cos, sin, pos = inputs(dtype, lead, hq, hk, d, rd, axes, torch.float32 if fp32 else dtype)
    sec = sections_of(axes, rd // 2)
    kw = dict(sections=sec, sections_cyclic=cyclic, interleaved=inter)
    args = (cos, sin, pos, axes_of(rd // 2, sec, cyclic), inter)
    q.requires_grad_(True), k.requires_grad_(True)
    qo, ko = fa.rotary_axes_func(q, k, cos, sin, pos, **kw)
    check(qo.detach(), q.detach(), args)
    check(ko.detach(), k.detach(), args)
    dq, dk = torch.randn_like(qo), torch.randn_like(ko)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    check(gq, dq, args, back=True)
    check(gk, dk, args, back=True)
    with torch.no_grad():
        qi, ki = q.detach().clone(), k.detach().clone()
        r = fa.rotary_axes_func(qi, ki, cos, sin, pos, inplace=True, **kw)
        assert r[0] is qi and r[1] is ki and qi._version == 1 and ki._version == 1
        assert torch.equal(qi.view(torch.int16), qo.view(torch.int16)) and torch.equal(ki.view(torch.int16), ko.view(torch.int16))
        alone = fa.rotary_axes_func(q, None, cos, sin, pos, **kw)
        assert torch.equal(alone.view(torch.int16), qo.view(torch.int16))


@pytest.mark.gpu
def test_gradient_against_differences_and_twice():
    """<f(x + h v) - f(x), w> / h = <v, f^T w>: f is linear, so the difference has no error of its own beyond the roundings of
    its two values, eps / 2 of each."""
    q, k, cos, sin, pos = inputs(torch.float16, (2, 6), 3, 1, 64, 64, 3, torch.float32)
    sec = [12, 10, 10]
    f = lambda x: fa.rotary_axes_func(x, None, cos, sin, pos, sections=sec)  # noqa: E731
    v, w = torch.randn_like(q), torch.randn_like(q)
    x = q.clone().requires_grad_(True)
    g, = torch.autograd.grad(f(x), x, w, create_graph=True)
    a, b = f(q + v), f(q)
    step = (q + v) - q                                           # what was added after rounding (exact in fp32)
    step = (q + v).float() - q.float()
    num = ((a.float() - b.float()) * w.float()).sum().item()
    ana = (step * g.detach().float()).sum().item()
    eps = torch.finfo(torch.float16).eps / 2
    tol = eps * ((a.float().abs() + b.float().abs()) * w.float().abs()).sum().item() + eps * (step.abs() * g.detach().float().abs()).sum().item()
    assert abs(num - ana) <= tol
    wv = w.clone().requires_grad_(True)
    y = f(x)
    g, = torch.autograd.grad(y, x, wv, create_graph=True)
    gg, = torch.autograd.grad(g, wv, v)                          # the derivative of the backward is the forward
    assert torch.equal(gg, f(v))


@pytest.mark.gpu
def test_slices_expanded_inputs_and_one_missing_gradient():
    q, k, cos, sin, pos = inputs(torch.bfloat16, (2, 7), 6, 2, 64, 64, 1, torch.bfloat16)
    qkv = torch.cat((q, k, k), 2)
    a, b = fa.rotary_axes_func(qkv[:, :, :6], qkv[:, :, 6:8], cos, sin, pos[0])
    c, d = fa.rotary_axes_func(q, k, cos, sin, pos)
    assert torch.equal(a, c) and torch.equal(b, d)
    one = k[:, :, :1].detach().requires_grad_(True)
    y = fa.rotary_axes_func(one.expand(2, 7, 4, 64), None, cos, sin, pos)
    g, = torch.autograd.grad(y.float().sum(), one)
    full = fa.rotary_axes_func(one.detach().expand(2, 7, 4, 64).contiguous().requires_grad_(True), None, cos, sin, pos)
    assert torch.equal(y, full) and g.shape == one.shape
    qg, kg = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    y, z = fa.rotary_axes_func(qg, kg, cos, sin, pos)
    z.float().sum().backward()
    assert qg.grad is None and kg.grad is not None
    odd = torch.zeros(2, 7, 6, 65, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = q                                             # rows that 16-byte loads cannot read
    assert torch.equal(fa.rotary_axes_func(odd[..., 1:], None, cos, sin, pos), c)
    t = q.transpose(2, 3).contiguous().transpose(2, 3)           # strided last dim
    assert torch.equal(fa.rotary_axes_func(t, None, cos, sin, pos), c)


@pytest.mark.gpu
def test_other_stream_graph_and_compile_op():
    q, k, cos, sin, pos = inputs(torch.bfloat16, (3, 11), 8, 2, 128, 128, 3, torch.float32)
    sec = [24, 20, 20]
    want = fa.rotary_axes_func(q, k, cos, sin, pos, sections=sec)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fa.rotary_axes_func(q, k, cos, sin, pos, sections=sec)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = fa.rotary_axes_func(q, k, cos, sin, pos, sections=sec)
    q.copy_(torch.randn_like(q))
    pos.copy_(pos.flip(-1))
    g.replay()
    want = fa.rotary_axes_func(q, k, cos, sin, pos, sections=sec)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    from flash_attn_npu_3.rotary_axes import _rotary_axes
    torch.library.opcheck(_rotary_axes, (q, k, cos, sin, pos, sec, False, False, False), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(_rotary_axes, (q, None, cos, sin, pos, sec, False, True, True), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_empty_and_special_values():
    q, k, cos, sin, pos = inputs(torch.bfloat16, (2, 4), 4, 2, 64, 32, 1, torch.float32)
    a, b = fa.rotary_axes_func(q[:0], k[:0], cos, sin, pos[:, :0])
    assert a.shape == (0, 4, 4, 64) and b.shape == (0, 4, 2, 64)
    q[0, 0, 0, 40] = float("nan")                                # behind rotary_dim: copied, and nothing else is touched
    q[0, 0, 0, 41] = float("-inf")
    a, _ = fa.rotary_axes_func(q, k, cos, sin, pos)
    assert torch.equal(a[..., 32:].contiguous().view(torch.int16), q[..., 32:].contiguous().view(torch.int16)) and torch.isfinite(a[..., :32]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("change,word", [
    (dict(q=torch.zeros(2, 4, 4, 64)), "FP16"),
    (dict(k=torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16)), "heads"),
    (dict(cos=torch.zeros(9, 33), sin=torch.zeros(9, 33)), "rotary_dim"),
    (dict(cos=torch.zeros(9, 16)), "shape"),
    (dict(cos=torch.zeros(9, 32, dtype=torch.float64), sin=torch.zeros(9, 32, dtype=torch.float64)), "dtype"),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int64)), "int32"),
    (dict(positions=torch.zeros(2, 2, 4, dtype=torch.int32)), "positions"),
    (dict(sections=[16, 15]), "sum"),
    (dict(sections=[32, -16, 16]), "sum"),
    (dict(sections=[10, 11, 11], sections_cyclic=True, positions=torch.zeros(3, 2, 4, dtype=torch.int32)), "cyclic"),
    (dict(inplace=True, q=torch.zeros(2, 4, 4, 64, dtype=torch.bfloat16, requires_grad=True)), "differentiable"),
    (dict(inplace=True, q=torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16).expand(2, 4, 4, 64)), "expanded"),
])
def test_refusals(change, word):
    a = dict(q=torch.zeros(2, 4, 4, 64, dtype=torch.bfloat16), k=torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16), cos=torch.zeros(9, 32),
             sin=torch.zeros(9, 32), positions=torch.zeros(2, 4, dtype=torch.int32))
    a.update(change)
    dev = {}
    for k, x in a.items():
        expanded = isinstance(x, torch.Tensor) and x.dim() == 4 and 0 in x.stride()
        dev[k] = x[:, :, :1].cuda().expand(x.shape) if expanded else x.detach().cuda().requires_grad_(x.requires_grad) if isinstance(x, torch.Tensor) else x
    with pytest.raises(RuntimeError, match=word):
        fa.rotary_axes_func(**dev)


@pytest.mark.gpu
def test_tables_from_complex_numbers():
    """.imag of a conjugate is a lazily negated, strided view: what is read must be the negated values."""
    q, k, cos, sin, pos = inputs(torch.bfloat16, (2, 4), 4, 2, 64, 64, 1, torch.float32)
    z = torch.complex(cos, sin).conj()
    assert z.imag.is_neg()
    want = fa.rotary_axes_func(q, k, cos, -sin, pos)
    for tables in ((z.real, z.imag), (cos, torch._neg_view(sin))):
        got = fa.rotary_axes_func(q, k, *tables, pos)
        assert all(torch.equal(x, y) for x, y in zip(want, got))
    here = fa.rotary_axes_func(q.clone(), k.clone(), z.real, z.imag, pos, inplace=True)
    assert all(torch.equal(x, y) for x, y in zip(want, here))


@pytest.mark.gpu
def test_in_place_on_one_tensor_twice_or_on_what_a_gradient_needs():
    q, _, cos, sin, pos = inputs(torch.bfloat16, (2, 4), 4, 4, 64, 64, 1, torch.float32)
    with pytest.raises(RuntimeError, match="memory of their own"):
        fa.rotary_axes_func(q, q, cos, sin, pos, inplace=True)
    x = torch.randn_like(q).requires_grad_(True)
    y = (x * q).sum()                                            # keeps q for dx
    fa.rotary_axes_func(q, None, cos, sin, pos, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_c_entry_point_refusals():
    def params():
        r = capi.RotaryParams()
        for x in (r.q, r.k, r.q_out, r.k_out):
            x.ptr, x.stride_b, x.stride_s, x.stride_h = 0x1000, 4096, 512, 64
        r.cos = r.sin = r.positions = 0x1000
        r.axes, r.b, r.s, r.hq, r.hk, r.d, r.rotary_dim, r.seqlen_ro, r.dtype, r.table_dtype = 1, 2, 0, 4, 2, 64, 64, 9, 1, 2
        return r
    assert capi.lib.fa_rotary_axes(None) == 1
    assert capi.lib.fa_rotary_axes(params()) == 0                # no tokens: nothing to launch
    for field, value, code in (("dtype", 3, 2), ("table_dtype", 0, 2), ("d", 63, 3), ("d", 258, 3), ("rotary_dim", 66, 3), ("rotary_dim", 31, 3),
                               ("axes", 5, 3), ("axes", 0, 3), ("seqlen_ro", 0, 3), ("cos", None, 1), ("positions", None, 1), ("b", -1, 3), ("hq", -1, 3)):
        r = params()
        setattr(r, field, value)
        assert capi.lib.fa_rotary_axes(r) == code, field
