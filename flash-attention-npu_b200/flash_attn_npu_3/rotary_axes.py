"""Rotary position axes: which axis (time, height, width, ..) turns which pair of a head."""
import ctypes
import functools

import torch

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


def check_positions(positions, axes, lead, device):
    """positions (axes, *lead) int32, or (*lead) for one axis -> a tensor (axes, *lead)."""
    if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int32:
        raise RuntimeError("positions must be an int32 tensor")
    if positions.device != device:
        raise RuntimeError("positions must be on the device of the tensors that they belong to")
    if axes == 1 and tuple(positions.shape) == tuple(lead):
        positions = positions.unsqueeze(0)
    if tuple(positions.shape) != (axes, *lead):
        raise RuntimeError(f"positions must have shape {(axes, *lead)}" + (f" or {tuple(lead)}" if axes == 1 else ""))
    return positions
