"""Rotary embedding with several position axes (an addition of this library; the reference rotates inside its cache call only,
flash_attn_npu_3/flash_attn_npu_interface.py:965)."""
import ctypes
import functools
from typing import List, Optional, Tuple

import torch

import fa_b200_capi as capi

MAX_AXES = 4


@functools.lru_cache(maxsize=256)
def axis_table(pairs, sections, cyclic):
    """One byte a pair, its axis, as a host buffer for the library.  sections: pairs of each axis, in consecutive blocks, or
    cyclic: pair i belongs to axis i % n as long as that axis has pairs left, else to axis 0."""
    n = len(sections)
    if not 1 <= n <= MAX_AXES:
        raise RuntimeError(f"rotary sections must name 1 to {MAX_AXES} axes")
    if any(type(s) is not int or s < 0 for s in sections) or sum(sections) != pairs:
        raise RuntimeError(f"rotary sections must be non-negative integers that sum up to rotary_dim / 2 = {pairs}")
    if cyclic:
        axis = [i % n if i < n * sections[i % n] else 0 for i in range(pairs)]
        if any(axis.count(a) != s for a, s in enumerate(sections)):
            raise RuntimeError("cyclic rotary sections: an axis has more pairs than its places in the cycle")
    else:
        axis = [a for a, s in enumerate(sections) for _ in range(s)]
    return ctypes.create_string_buffer(bytes(axis), pairs)


def axis_pointer(pairs, sections, cyclic):
    """-> (buffer to keep alive, its address, number of axes)"""
    if sections is None:
        return None, 0, 1
    table = axis_table(pairs, tuple(sections), bool(cyclic))
    return table, ctypes.addressof(table), len(sections)


def check_positions(positions, axes, lead, index):
    """positions (axes, *lead) int32, or (*lead) for one axis -> (a tensor with a dense last dim, its strides as of (axes, *lead))."""
    if not isinstance(positions, torch.Tensor) or positions.dtype is not torch.int32:
        raise RuntimeError("positions must be an int32 tensor")
    if positions.get_device() != index:
        capi.cuda_index(positions)
        raise RuntimeError("positions must be on the device of the tensors that they belong to")
    shape = positions.shape
    one = axes == 1 and shape == lead
    if not one and shape != (axes, *lead):
        raise RuntimeError(f"positions must have shape {(axes, *lead)}" + (f" or {tuple(lead)}" if axes == 1 else ""))
    st = positions.stride()
    if st[-1] != 1:
        positions = positions.contiguous()
        st = positions.stride()
    return positions, (0,) + st if one else st


_NONE = (0, 0, 0, 0)


def _leaves(t, st):
    """The four leaves of an fa_tensor of (B, S, H, D), or of packed (T, H, D) as one batch entry."""
    return (t.data_ptr(), st[0], st[1], st[2]) if len(st) == 4 else (t.data_ptr(), 0, st[0], st[1])


def _run(q, k, cos, sin, positions, sections, cyclic, interleaved, backward, inplace):
    """The library call; everything has been checked.  positions (axes, *lead), or (*lead) for one axis."""
    rows, pairs = cos.shape
    keep, axis, axes = axis_pointer(pairs, sections, cyclic)
    shape, st = q.shape, q.stride()
    if st[-1] != 1:
        q = q.contiguous()
        st = q.stride()
    packed = len(shape) == 3
    b, s = (1, shape[0]) if packed else (shape[0], shape[1])
    hq, d = shape[-2], shape[-1]
    pos = positions.stride()
    if len(pos) == len(shape) - 2:
        pos = (0,) + pos
    q_out = q if inplace else torch.empty_like(q, memory_format=torch.contiguous_format)
    dense = (s * hq * d, hq * d, d)
    q_in = _leaves(q, st)
    q_to = q_in if inplace else (q_out.data_ptr(),) + dense
    k_out, hk, k_in, k_to = None, 0, _NONE, _NONE
    if k is not None:
        st = k.stride()
        if st[-1] != 1:
            k = k.contiguous()
            st = k.stride()
        hk = k.shape[-2]
        k_out = k if inplace else torch.empty_like(k, memory_format=torch.contiguous_format)
        k_in = _leaves(k, st)
        k_to = k_in if inplace else (k_out.data_ptr(), s * hk * d, hk * d, d)
    if b * s * (hq + hk) > 0:
        index = q.get_device()
        buf = capi.ROTARY_BLOCK.new(
            *q_in, *k_in, *q_to, *k_to, cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), pos[0], 0 if packed else pos[1],
            axis, axes, b, s, hq, hk, d, 2 * pairs, 1 if interleaved else 0, rows, 1 if backward else 0,
            capi.DTYPES[q.dtype], 2 if cos.dtype is torch.float32 else capi.DTYPES[cos.dtype], capi.raw_stream_of(index))
        capi.launch_on(capi._call_rotary, buf, index)
    del keep
    return q_out, k_out


def _out_of_place(q, k, cos, sin, positions, sections, cyclic, interleaved, backward):
    return _run(q, k, cos, sin, positions, sections, cyclic, interleaved, backward, False)


@torch.library.custom_op("flash_attn_npu_3::_rotary_axes", mutates_args=(), device_types="cuda")
def _rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                 sections: Optional[List[int]], cyclic: bool, interleaved: bool, backward: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    q_out, k_out = _out_of_place(q, k, cos, sin, positions, sections, cyclic, interleaved, backward)
    return q_out, torch.empty((0,), dtype=q.dtype, device=q.device) if k is None else k_out


@torch.library.register_fake("flash_attn_npu_3::_rotary_axes")
def _rotary_axes_fake(q, k, cos, sin, positions, sections, cyclic, interleaved, backward):
    return q.new_empty(q.shape), q.new_empty((0,)) if k is None else k.new_empty(k.shape)


def _by_op(q, k, *args):
    q_out, k_out = _rotary_axes(q, k, *args)
    return q_out, None if k is None else k_out


def _forward(q, k, cos, sin, *args):
    if capi.plain(q, k, cos, sin):                             # the op's dispatch would do nothing but call the body
        return _out_of_place(q, k, cos, sin, *args)
    return _by_op(q, k, cos, sin, *args)


def _turn_two(turn, q, k, *args):
    """turn(q, k, *args) for gradients or tangents, each of which may be missing."""
    if q is not None:
        return turn(q, k, *args)
    return (None, None) if k is None else (None, turn(k, None, *args)[0])


class RotaryAxesFunc(torch.autograd.Function):
    """A rotation is linear and orthogonal: its gradient is the rotation back, which is differentiable in the same way."""

    @staticmethod
    def forward(ctx, *inputs):
        ctx.set_materialize_grads(False)
        RotaryAxesFunc.keep(ctx, inputs)
        return _forward(*inputs)

    @staticmethod
    def keep(ctx, inputs):
        _, _, cos, sin, positions, sections, cyclic, interleaved, backward = inputs
        ctx.save_for_backward(cos, sin, positions)
        ctx.args = (sections, cyclic, interleaved)
        ctx.turn_back = not backward

    @staticmethod
    def backward(ctx, dq, dk):
        return _turn_two(_apply, dq, dk, *ctx.saved_tensors, *ctx.args, ctx.turn_back) + (None,) * 7


class RotaryAxesTransformFunc(torch.autograd.Function):
    """The same where a functorch transform or a forward-mode level is active (torch takes 26 us longer to call this kind): the
    derivative in a direction is the rotation of the direction.  Always by the op: what a transform has saved is still wrapped
    when a gradient is asked for after its end.  Missing directions come as zeros: torch takes no None for a tensor's tangent."""
    generate_vmap_rule = True

    @staticmethod
    def forward(q, k, cos, sin, positions, sections, cyclic, interleaved, backward):
        return _by_op(q, k, cos, sin, positions, sections, cyclic, interleaved, backward)

    @staticmethod
    def setup_context(ctx, inputs, output):
        RotaryAxesFunc.keep(ctx, inputs)
        ctx.save_for_forward(*inputs[2:5])

    @staticmethod
    def backward(ctx, dq, dk):
        return _turn_two(RotaryAxesTransformFunc.apply, dq, dk, *ctx.saved_tensors, *ctx.args, ctx.turn_back) + (None,) * 7

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        return _turn_two(RotaryAxesTransformFunc.apply, tq, tk, *ctx.saved_tensors, *ctx.args, not ctx.turn_back)


def _apply(q, k, *args):
    if capi.transforming():
        return RotaryAxesTransformFunc.apply(q, k, *args)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return RotaryAxesFunc.apply(q, k, *args)
    return _forward(q, k, *args)


def rotary_axes_func(q, k, cos, sin, positions, sections=None, sections_cyclic=False, interleaved=False, inplace=False):
    """Rotary embedding of q and k with one to four position axes (time, height, width, ..), differentiable in q and k (in
    reverse and forward mode).

    q (batch, seqlen, nheads, headdim) or packed (total, nheads, headdim), fp16 or bf16; k of the same shape but for its heads,
    or None.  cos / sin (seqlen_ro, rotary_dim / 2) in q's dtype or fp32.  positions int32 (axes, batch, seqlen) or
    (axes, total); without the first dimension for one axis.  Pair i of a head - elements i and i + rotary_dim / 2, or 2 i and
    2 i + 1 when interleaved - is turned by row positions[axis of i] of the tables, column i; columns behind rotary_dim are
    copied.  sections: how many of the rotary_dim / 2 pairs each axis has, in consecutive blocks, or with sections_cyclic pair
    i belongs to axis i % axes while that axis has pairs left, else to axis 0.  None: one axis.  A position outside the tables
    takes the nearest row.  fp32 arithmetic, rounded once; cos, sin and positions get no gradient.

    (Dual tensors given to a function that torch.compile has traced lose their tangent, as in every custom op; torch.func.jvp
    inside or around it does not.)

    inplace writes into q and k instead of new tensors (only where no gradient is needed); q and k must not share memory.
    Returns (q, k), or q alone when k is None."""
    index, dtype, shape = capi.cuda_index(q), q.dtype, q.shape
    if dtype not in capi.DTYPES or (k is not None and k.dtype is not dtype):
        raise RuntimeError("rotary embedding only supports FP16 and BF16 data types, the same for q and k")
    n = len(shape)
    if n != 3 and n != 4:
        raise RuntimeError("q must be (batch, seqlen, nheads, headdim) or (total, nheads, headdim)")
    if k is not None:
        other = k.shape
        if len(other) != n or other[0] != shape[0] or other[-3] != shape[-3] or other[-1] != shape[-1]:
            raise RuntimeError("k must have the shape of q but for its heads")
    if cos.get_device() != index or sin.get_device() != index or (k is not None and k.get_device() != index):
        capi.require_cuda(k, cos, sin)
        raise RuntimeError("q, k, cos and sin must be on one device")
    table = cos.shape
    if len(table) != 2 or sin.shape != table or sin.dtype is not cos.dtype or (cos.dtype is not dtype and cos.dtype is not torch.float32):
        raise RuntimeError("cos and sin must both have shape (seqlen_ro, rotary_dim / 2), in q's dtype or fp32")
    d, (rows, pairs) = shape[-1], table
    if d > 256 or d % 2 or not 0 < 2 * pairs <= d or rows == 0:
        raise RuntimeError("the head dimension must be even and at most 256, rotary_dim positive and at most that, with one table row at least")
    sections_cyclic = bool(sections_cyclic)
    axes = 1
    if sections is not None:
        sections = list(sections)
        axes = len(sections)
        axis_table(pairs, tuple(sections), sections_cyclic)
    positions, _ = check_positions(positions, axes, shape[:-2], index)
    if not cos.is_contiguous() or not sin.is_contiguous():
        cos, sin = cos.contiguous(), sin.contiguous()
    args = (cos, sin, positions, sections, sections_cyclic, bool(interleaved))
    if inplace:
        transforming = capi.transforming()
        for t in (q, k):
            if t is None:
                continue
            if torch.is_grad_enabled() and t.requires_grad:
                raise RuntimeError("inplace rotary embedding is not differentiable: detach q and k, or leave inplace out")
            if transforming and capi.has_tangent(t):
                raise RuntimeError("inplace rotary embedding has no forward-mode derivatives and no function transforms: leave inplace out")
            if t.stride(-1) != 1 or any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
                raise RuntimeError("inplace rotary embedding needs a contiguous last dimension and no expanded dimensions")
        if k is not None and k.data_ptr() == q.data_ptr() and k.numel():
            raise RuntimeError("inplace rotary embedding needs q and k in memory of their own")
        # the op's dispatch reads lazily negated tables with their sign; here nothing stands in front of the kernel.  (q and k may
        # be such views: what is turned is the memory, and the turned negative is the negative of the turned.)
        _run(q, k, cos.resolve_neg(), sin.resolve_neg(), *args[2:], False, True)
        torch.autograd.graph.increment_version(q if k is None else (q, k))
    else:
        q, k = _apply(q, k, *args, False)
    return q if k is None else (q, k)
