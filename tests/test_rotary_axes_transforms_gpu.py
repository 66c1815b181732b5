"""rotary_axes_func under forward-mode derivatives and function transforms.  The map is linear: its derivative in a direction is
the same rotation of that direction, bit for bit."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import flash_attn_npu_3 as fa
from tests.test_rotary_axes_gpu import inputs

pytestmark = pytest.mark.gpu


def setup(dtype=torch.float16):
    q, k, cos, sin, pos = inputs(dtype, (2, 5), 4, 2, 64, 48, 3, torch.float32)
    kw = dict(sections=[10, 8, 6])
    return q, k, torch.randn_like(q), torch.randn_like(k), lambda q, k: fa.rotary_axes_func(q, k, cos, sin, pos, **kw)


def test_dual_tensors():
    q, k, tq, tk, f = setup()
    want = f(tq, tk)
    plain = f(q, k)
    for grad in (False, True):                                  # with a gradient wanted as well
        x, y = q.clone().requires_grad_(grad), k.clone().requires_grad_(grad)
        with fwd.dual_level():
            a, b = f(fwd.make_dual(x, tq), fwd.make_dual(y, tk))
            assert torch.equal(a.detach(), plain[0]) and torch.equal(b.detach(), plain[1])
            assert torch.equal(fwd.unpack_dual(a).tangent, want[0]) and torch.equal(fwd.unpack_dual(b).tangent, want[1])
            a, b = f(x, fwd.make_dual(y, tk))
            assert fwd.unpack_dual(a).tangent is None or not fwd.unpack_dual(a).tangent.any()
            assert torch.equal(fwd.unpack_dual(b).tangent, want[1])
            alone = f(fwd.make_dual(x, tq), None)
            assert torch.equal(fwd.unpack_dual(alone).tangent, want[0])
            a, b = f(x, y)                                      # nothing dual
            assert torch.equal(a.detach(), plain[0]) and fwd.unpack_dual(a).tangent is None


def test_jvp_and_jacfwd():
    q, k, tq, tk, f = setup(torch.bfloat16)
    out, tan = torch.func.jvp(f, (q, k), (tq, tk))
    assert all(torch.equal(x, y) for x, y in zip(out, f(q, k)))
    assert all(torch.equal(x, y) for x, y in zip(tan, f(tq, tk)))
    g = lambda x: torch.func.jvp(lambda y: f(y, None), (x,), (tq,))[1]  # noqa: E731
    assert torch.equal(g(q), f(tq, None))
    small = q[:1, :1, :1, :].contiguous()
    _, _, cos, sin, pos = inputs(torch.bfloat16, (1, 1), 1, 1, 64, 48, 3, torch.float32)
    h = lambda x: fa.rotary_axes_func(x, None, cos, sin, pos, sections=[10, 8, 6])  # noqa: E731
    jac = torch.func.jacfwd(h)(small).reshape(64, 64)
    eye = torch.eye(64, dtype=torch.bfloat16, device="cuda").reshape(64, 1, 1, 1, 64)
    assert torch.equal(jac, torch.stack([h(e) for e in eye], -1).reshape(64, 64))


def test_reverse_mode_transforms():
    q, k, tq, tk, f = setup()
    x = q.clone().requires_grad_(True)
    want, = torch.autograd.grad(f(x, None), x, tq)
    got, = torch.func.vjp(lambda y: f(y, None), q)[1](tq)
    assert torch.equal(got, want)
    got = torch.func.grad(lambda y: (f(y, None).float() * tq).sum())(q)
    assert torch.equal(got, want)
    both = torch.stack((q, tq))
    out = torch.vmap(lambda y: f(y, None))(both)
    assert torch.equal(out, torch.stack((f(q, None), f(tq, None))))


def test_a_dual_tensor_is_not_turned_in_place():
    q, k, tq, tk, _ = setup()
    _, _, cos, sin, pos = inputs(torch.float16, (2, 5), 4, 2, 64, 48, 1, torch.float32)
    with fwd.dual_level():
        x = fwd.make_dual(q.clone(), tq)
        for args in ((x, k), (k, x), (x, None)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                fa.rotary_axes_func(*args, cos, sin, pos, inplace=True)
        assert torch.equal(fwd.unpack_dual(x).primal, q)
        y = q.clone()                                           # an ordinary one is, inside a level too
        fa.rotary_axes_func(y, None, cos, sin, pos, inplace=True)
    assert torch.equal(y, fa.rotary_axes_func(q, None, cos, sin, pos))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda a: fa.rotary_axes_func(a, None, cos, sin, pos, inplace=True), (q.clone(),), (tq,))


def test_compiled():
    """Through torch.compile's tracing (whatever it can take into a graph), a call and a training step."""
    q, k, tq, tk, f = setup()
    x, y = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    step = lambda a, b: sum((o.float() * t).sum() for o, t in zip(f(a, b), (tq, tk)))  # noqa: E731
    want = torch.autograd.grad(step(x, y), (x, y))
    torch._dynamo.reset()
    c = torch.compile(f, backend="aot_eager")
    assert all(torch.equal(a, b) for a, b in zip(c(q, k), f(q, k)))
    got = torch.autograd.grad(torch.compile(step, backend="aot_eager")(x, y), (x, y))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
