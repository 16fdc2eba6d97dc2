"""AGO (algebraic geometric oscillator) rotary rotations on B200, behind the
reference's signatures (src/attention.py:93-240):

* ``CayleyRotary``               -- the (c, s) table pair, with ``.matrix``
                                   (:93-106)
* ``build_cayley_rotary_matrix`` -- rational Cayley rotation tables without
                                   transcendentals (:156-207)
* ``apply_ago_rotations``        -- rotates q and k by the tables at their
                                   sequence positions (:210-240); the Q/K
                                   prologue of the attention layer
                                   (src/model.py:262-264)

* ``apply_ago_rotations_axes``   -- the rotation with several position axes
                                   (time, height, width), differentiable; no
                                   reference counterpart

All run as CUDA kernels (``afa_ago_table`` / ``afa_ago_rotate`` /
``afa_ago_rotate_axes``): the tables by a per-pair recurrence over positions,
the rotations as one pass over q and k.
"""
from __future__ import annotations

import ctypes
import functools
import operator
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import _lib
from ._tensors import Staged, host_checks_float, refuse_tangents, tangents_exist

__all__ = ["CayleyRotary", "build_cayley_rotary_matrix", "apply_ago_rotations", "apply_ago_rotations_axes"]


class CayleyRotary(NamedTuple):
    """Precomputed Cayley rotary rotation parameters (src/attention.py:93-106).

    Can be unpacked as (c, s), or accessed via .c, .s, or .matrix.
    """
    c: torch.Tensor
    s: torch.Tensor

    @property
    def matrix(self):
        """The 2x2 rotation blocks [[c, -s], [s, c]], shape (..., 2, 2)."""
        row0 = torch.stack([self.c, -self.s], dim=-1)
        row1 = torch.stack([self.s, self.c], dim=-1)
        return torch.stack([row0, row1], dim=-2)


_TORCH_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float64": torch.float64}
_TABLE_DTYPES = frozenset(_TORCH_DTYPES.values())


def _torch_dtype(dtype) -> torch.dtype:
    if isinstance(dtype, torch.dtype):
        return dtype
    name = np.dtype(dtype).name if not isinstance(dtype, str) else dtype
    if name in _TORCH_DTYPES:
        return _TORCH_DTYPES[name]
    raise TypeError(f"unsupported table dtype {dtype!r} (float32, bfloat16 or float64)")


def build_cayley_rotary_matrix(dim: int, max_seq_len: int, freqs=None, base: float = 10000.0,
                               dtype=torch.float32, device=None) -> CayleyRotary:
    """Rational Cayley rotation tables (src/attention.py:156-207).

    Returns CayleyRotary(c, s), each (max_seq_len, dim // 2) in ``dtype`` on the
    GPU: per pair k a frequency w_k (``freqs``, or 1 / (1 + alpha k)^2 with
    alpha = (sqrt(base) - 1) / max(dim/2 - 1, 1)), the step rotation
    ((1 - w^2) / (1 + w^2), 2w / (1 + w^2)), and row m = the m-fold product
    renormalised after every step. Computed in float32 (float64 for float64).
    """
    if dim <= 0 or dim % 2 != 0:
        raise ValueError("dim must be a positive even integer")
    if max_seq_len <= 0:
        raise ValueError("max_seq_len must be a positive integer")
    pairs = dim // 2
    tdt = _torch_dtype(dtype)
    fptr = None
    if freqs is not None:
        w = np.asarray(freqs.detach().cpu() if isinstance(freqs, torch.Tensor) else freqs, dtype=np.float64)
        if w.shape != (pairs,):
            raise ValueError(f"freqs must have shape ({pairs},), got {w.shape}")
        w = np.ascontiguousarray(w)
        fptr = w.ctypes.data_as(ctypes.POINTER(ctypes.c_double))
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    c = torch.empty((max_seq_len, pairs), dtype=tdt, device=dev)
    s = torch.empty((max_seq_len, pairs), dtype=tdt, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().afa_ago_table(c.data_ptr(), s.data_ptr(), dim, max_seq_len, fptr, float(base),
                                       _lib.dtype_code(tdt), _lib.stream_ptr(dev))
    _lib.check(rc, "afa_ago_table")
    return CayleyRotary(c, s)


def _extract_cs(rotary_params):
    """(c, s) from a CayleyRotary, a (c, s) pair, a (..., 2, 2) matrix or a
    (..., 2) stack (src/attention.py:109-119)."""
    if isinstance(rotary_params, (tuple, list)) and len(rotary_params) >= 2:
        return rotary_params[0], rotary_params[1]
    if hasattr(rotary_params, "c") and hasattr(rotary_params, "s"):
        return rotary_params.c, rotary_params.s
    if hasattr(rotary_params, "shape"):
        if rotary_params.ndim >= 4 and tuple(rotary_params.shape[-2:]) == (2, 2):
            return rotary_params[..., 0, 0], rotary_params[..., 1, 0]
        if rotary_params.ndim >= 3 and rotary_params.shape[-1] == 2:
            return rotary_params[..., 0], rotary_params[..., 1]
    raise TypeError(f"Unsupported rotary parameters type: {type(rotary_params)}")


def _default_seq_axis(shape) -> int:
    """src/attention.py:229-230."""
    ndim = len(shape)
    return 0 if ndim == 2 else 1 if ndim == 3 else (1 if shape[1] > shape[2] else 2)


def apply_ago_rotations(q, k, rotary_params=None, seq_axis: Optional[int] = None):
    """AGO Cayley rotations of q and k (src/attention.py:210-240).

    q, k: same shape (..., dim), dim even. Each channel pair (x0, x1) at
    sequence position m becomes (c_m x0 - s_m x1, s_m x0 + c_m x1), with the
    tables cast to the tensors' dtype. ``rotary_params`` defaults to
    ``build_cayley_rotary_matrix(dim, seq_len, dtype=q.dtype)``; ``seq_axis`` to
    the reference's choice (0 for 2-D, 1 for 3-D, for 4-D 1 if shape[1] >
    shape[2] else 2). Returns (q_rot, k_rot) with the input shapes and dtypes.
    """
    if tuple(q.shape) != tuple(k.shape):
        raise ValueError(f"q and k shapes must match, got {tuple(q.shape)} and {tuple(k.shape)}")
    dim = q.shape[-1]
    if dim % 2 != 0:
        raise ValueError(f"Feature dimension must be even, got {dim}")
    host_checks_float(q, k)
    st = Staged(q, k)
    qt, kt = st.tensors
    if qt.dtype != kt.dtype:
        raise TypeError("q and k must share a dtype")
    ndim = qt.ndim
    if ndim < 2:
        raise ValueError("q and k need a sequence axis and a feature axis")
    if seq_axis is None:
        seq_axis = _default_seq_axis(qt.shape)
    if seq_axis < 0:
        seq_axis += ndim
    if not 0 <= seq_axis < ndim - 1:
        raise ValueError(f"seq_axis {seq_axis} must name an axis before the feature axis")
    seq_len = qt.shape[seq_axis]
    if rotary_params is None:
        rotary_params = build_cayley_rotary_matrix(dim, seq_len, dtype=qt.dtype, device=qt.device)
    c, s = _extract_cs(rotary_params)
    c = torch.as_tensor(np.asarray(c)) if isinstance(c, np.ndarray) else c
    s = torch.as_tensor(np.asarray(s)) if isinstance(s, np.ndarray) else s
    c = c.reshape(-1, dim // 2).to(qt.device).contiguous()
    s = s.reshape(-1, dim // 2).to(qt.device).contiguous()
    if c.shape[0] < seq_len or s.shape != c.shape:
        raise ValueError(f"rotary tables hold {c.shape[0]} positions, the sequence needs {seq_len}")
    inner = int(np.prod(qt.shape[seq_axis + 1:-1])) if seq_axis + 1 < ndim - 1 else 1
    rows = qt.numel() // dim
    q_out, k_out = torch.empty_like(qt), torch.empty_like(kt)
    with torch.cuda.device(qt.device):
        rc = _lib.load().afa_ago_rotate(qt.data_ptr(), kt.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                                        c.data_ptr(), s.data_ptr(), _lib.dtype_code(c.dtype), rows, dim, seq_len,
                                        inner, _lib.dtype_code(qt.dtype), _lib.stream_ptr(qt.device))
    _lib.check(rc, "afa_ago_rotate")
    return st.back(q_out), st.back(k_out)


class AxisArguments(NamedTuple):
    """Checked arguments of a rotation with several position axes."""
    c: torch.Tensor          # (positions, dim / 2)
    s: torch.Tensor
    positions: torch.Tensor  # (axes, *shape) int32 or int64, any strides
    sections: ctypes.Array


@functools.lru_cache(maxsize=1024)
def _sections(sections, pairs):
    """Channel pairs of each axis, checked, as a C array."""
    if not 1 <= len(sections) <= 4:
        raise ValueError("between one and four position axes are supported")
    if min(sections) < 0 or sum(sections) > pairs:
        raise ValueError(f"sections must be nonnegative and sum to at most {pairs}, got {sections}")
    return _lib.ints(*sections)


def axis_arguments(rotary_params, positions, sections, dim, shape, device) -> AxisArguments:
    """Tables, positions (axes, *shape) and channel pairs per axis of a rotation, checked, and on ``device`` if one
    is given."""
    if positions is None or sections is None:
        raise ValueError("a rotation needs positions and sections")
    pairs = dim // 2
    sections = _sections(tuple(map(operator.index, sections)), pairs)
    c, s = _extract_cs(rotary_params)
    if isinstance(c, np.ndarray):
        c = torch.from_numpy(np.ascontiguousarray(c))
    if isinstance(s, np.ndarray):
        s = torch.from_numpy(np.ascontiguousarray(s))
    if not isinstance(c, torch.Tensor) or not isinstance(s, torch.Tensor) or c.dtype not in _TABLE_DTYPES \
            or s.dtype is not c.dtype:
        raise TypeError("the rotary tables must share a dtype: float32, bfloat16 or float64")
    rows = c.shape
    if rows != s.shape or len(rows) == 0 or rows[-1] != pairs or c.numel() == 0:
        raise ValueError(f"rotary tables must have shape (positions, {pairs}), got {tuple(c.shape)} and "
                         f"{tuple(s.shape)}")
    if c.requires_grad or s.requires_grad:
        raise ValueError("the rotary tables have no gradient")
    if tangents_exist():
        refuse_tangents("a rotary table", c, s)
    p = positions if isinstance(positions, torch.Tensor) else torch.as_tensor(np.asarray(positions))
    if p.dtype != torch.int32 and p.dtype != torch.int64:
        raise TypeError("positions must be int32 or int64")
    axes = len(sections)
    if p.shape != (axes, *shape):
        raise ValueError(f"positions must have shape {(axes, *shape)}, got {tuple(p.shape)}")
    length = c.numel() // pairs
    if device is None and not p.is_cuda and p.numel() and not (0 <= int(p.min()) and int(p.max()) < length):
        raise ValueError(f"positions must lie in [0, {length}), the tables' rows")
    if device is not None and not c.device == s.device == p.device == device:
        if not p.is_cuda and p.numel() and not (0 <= int(p.min()) and int(p.max()) < length):
            raise ValueError(f"positions must lie in [0, {length}), the tables' rows")
        if any(x.is_cuda and x.device != device for x in (c, s, p)):
            raise ValueError(f"tables and positions must be on {device}")
        c, s, p = c.to(device), s.to(device), p.to(device)
    if c.ndim != 2:
        c, s = c.reshape(length, pairs), s.reshape(length, pairs)
    return AxisArguments(c.contiguous(), s.contiguous(), p, sections)


def _row_strides(t, token_major):
    """Strides (batch, token, head) of the rows of t."""
    st = t.stride()
    return _lib.longs(0, st[0], st[1]) if token_major else _lib.longs(st[0], st[2], st[1])


def _rotate_axes(q, k, axes: AxisArguments, backward: bool):
    """One launch: q and k (or None) turned, backward the other way; contiguous results."""
    token_major = q.ndim == 3
    q = q if q.stride(-1) == 1 else q.contiguous()
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = None
    if k is not None:
        k = k if k.stride(-1) == 1 else k.contiguous()
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    batch, tokens = (1, q.shape[0]) if token_major else (q.shape[0], q.shape[2])
    c, p = axes.c, axes.positions
    pst = p.stride()
    rc = _lib.call(
        q.device, _lib.load().afa_ago_rotate_axes, q.data_ptr(), _row_strides(q, token_major), qo.data_ptr(),
        q.shape[1], *((None, None, None, 0) if k is None else
                      (k.data_ptr(), _row_strides(k, token_major), ko.data_ptr(), k.shape[1])),
        c.data_ptr(), axes.s.data_ptr(), _lib.dtype_code(c.dtype), c.shape[0], p.data_ptr(),
        _lib.longs(pst[0], 0 if len(pst) == 2 else pst[1], pst[-1]), p.dtype == torch.int64,
        axes.sections, p.shape[0], token_major, batch, tokens, q.shape[-1], backward, _lib.dtype_code(q.dtype))
    _lib.check(rc, "afa_ago_rotate_axes")
    return qo, ko


def _on_pairs(t):
    """t, or a copy where a row starts off a channel pair's alignment (the gradient of a concatenation's part does)."""
    if t is None or t.stride(-1) != 1 or (t.data_ptr() % (2 * t.element_size()) == 0 and
                                          not any(s & 1 for s in t.stride()[:-1])):
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _RotateAxes(torch.autograd.Function):
    """A rotation's gradient is the rotation the other way, which is differentiable again."""

    @staticmethod
    def forward(ctx, q, k, c, s, positions, sections, turn_back):
        ctx.save_for_backward(c, s, positions)
        ctx.sections, ctx.turn_back = sections, turn_back
        qo, ko = _rotate_axes(q, k, AxisArguments(c, s, positions, sections), turn_back)
        return qo if k is None else (qo, ko)

    @staticmethod
    def backward(ctx, gq, gk=None):
        c, s, positions = ctx.saved_tensors
        gq, gk = _on_pairs(gq), _on_pairs(gk)
        if torch.is_grad_enabled():  # a gradient of the gradient may follow
            g = _RotateAxes.apply(gq, gk, c, s, positions, ctx.sections, not ctx.turn_back)
            g = (g, None) if gk is None else g
        else:
            g = _rotate_axes(gq, gk, AxisArguments(c, s, positions, ctx.sections), not ctx.turn_back)
        return (*g, None, None, None, None, None)


def apply_ago_rotations_axes(q, k, rotary_params, positions, sections):
    """AGO Cayley rotations with several position axes (time, height, width).

    q (batch, heads, tokens, dim) or, packed, (tokens, heads, dim); k (or None)
    the same with its own number of heads. ``sections`` gives each axis (at most
    four) its channel pairs, in order: pair p of axis a at a token with
    ``positions[a, ..., token]`` = m turns by row m of the tables, pairs behind
    the last section stay as they are. Rows of q and k start on a channel pair
    (views off one are refused; gradients off one are copied). ``positions``:
    (axes, batch, tokens), (axes, tokens) for packed inputs or the same positions
    in every batch row, int32 or int64; one the tables do not hold is an error on
    the host and gives NaN on the device. ``rotary_params`` as in
    ``apply_ago_rotations``, (positions, dim / 2). Unlike there the tables keep
    their dtype: the arithmetic is float32 (float64 for float64 inputs) with one
    rounding, which a bfloat16 table would limit to 2^-9. Differentiable in q and
    k by backward passes (before one is captured into a CUDA graph, release what
    was computed from the same leaves outside of it: PyTorch would wait for those
    leaves' stream). Returns contiguous (q_rot, k_rot).
    """
    if q.ndim not in (3, 4):
        raise ValueError(f"q must have shape (batch, heads, tokens, dim) or (tokens, heads, dim), got {tuple(q.shape)}")
    dim = q.shape[-1]
    if dim % 2 != 0 or dim == 0:
        raise ValueError(f"Feature dimension must be even, got {dim}")
    head = 1
    if k is not None and (k.ndim != q.ndim or [n for i, n in enumerate(k.shape) if i != head] !=
                          [n for i, n in enumerate(q.shape) if i != head]):
        raise ValueError(f"q and k must differ in their heads only, got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.shape[head] == 0 or (k is not None and k.shape[head] == 0):
        raise ValueError("q and k need at least one head")
    host_checks_float(*(t for t in (q, k) if t is not None))
    if tangents_exist():
        refuse_tangents("apply_ago_rotations_axes", q, k)
    if k is not None and k.dtype != q.dtype:
        raise TypeError("q and k must share a dtype")
    on_gpu = all(t is None or (isinstance(t, torch.Tensor) and t.is_cuda) for t in (q, k))
    if on_gpu:
        st, qt, kt = None, q, k
        if k is not None and k.device != q.device:
            raise ValueError(f"tensors on different devices: {q.device} and {k.device}")
    else:
        if any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k)):
            raise ValueError("a differentiable rotation needs CUDA tensors")
        axis_arguments(rotary_params, positions, sections, dim, _axis_shape(q, positions), None)  # before any copy
        st = Staged(*(t for t in (q, k) if t is not None))
        qt, kt = st.tensors[0], (st.tensors[1] if k is not None else None)
    if qt.dtype not in _TABLE_DTYPES:
        raise TypeError("q and k must be float32, bfloat16 or float64")
    axes = axis_arguments(rotary_params, positions, sections, dim, _axis_shape(qt, positions), qt.device)
    if not torch.is_grad_enabled() or not (qt.requires_grad or (kt is not None and kt.requires_grad)):
        outs = _rotate_axes(qt, kt, axes, False)
    elif kt is None:
        outs = _RotateAxes.apply(qt, None, *axes, False), None
    elif qt.requires_grad and kt.requires_grad:
        outs = _RotateAxes.apply(qt, kt, *axes, False)
    else:  # together both results would want a gradient
        outs = tuple(_RotateAxes.apply(t, None, *axes, False) if t.requires_grad else
                     _rotate_axes(t, None, axes, False)[0] for t in (qt, kt))
    return tuple(outs) if st is None else (st.back(outs[0]), st.back(outs[1]))


def _axis_shape(q, positions):
    """The shape positions must have behind their axes."""
    if q.ndim == 3:
        return (q.shape[0],)
    if getattr(positions, "ndim", 3) == 2:
        return (q.shape[2],)
    return (q.shape[0], q.shape[2])
