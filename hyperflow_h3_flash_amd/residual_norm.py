"""The norms before and after a block with its gate and residual, in one pass over the rows of packed requests.

`residual_norm` adds a block's branch to the residual stream (its own norm and gate before) and gives the next block's
normed and modulated input; `RowPlan` says which request each row belongs to. `TransformerBlock` runs it between its INT8
linears and attention.

The reference's blocks do these steps one by one (src/hyperflow_h3_flash/transformer.py:339-380, whose norms are its model
library's). As the other operators, forward only: host tensors compute on the CPU, device tensors on the kernels of
``libhf_block.so``."""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch
from torch import Tensor

from . import _native, host_cache
from .block import (_apart, _check_out, _current, _deliver, _differentiable, _forward_only, _lengths, _lib,
                    _plan_device, _DTYPES, _FLOAT_MAX, _Resident, _vector)
from .int8 import _check, _on, _raw_stream, _same_device

#: Kinds of norm and their codes.
NORMS = {None: 0, "rms": 1, "layer": 2}
_args = _native.RESIDUAL_NORM_ARGS.pack


class RowPlan:
    """Which request each row of a packed batch belongs to, for `residual_norm`: ``lengths[i]`` rows of request i, the
    requests one behind the other. Built on the host, once for all blocks and steps of the batch."""

    def __init__(self, lengths: Sequence[int], *, device: torch.device | str = "cuda") -> None:
        self.lengths = _lengths(lengths, "lengths")
        self.requests, self.rows = len(self.lengths), sum(self.lengths)
        if self.rows > 0x7fffffff:
            raise ValueError(f"{self.rows} rows do not fit 32 bits")
        self.device = _plan_device(device)
        self._index = -1 if self.device.index is None else self.device.index
        #: The request of each row, on the host.
        self.groups = torch.repeat_interleave(torch.arange(self.requests, dtype=torch.int32),
                                              torch.tensor(self.lengths, dtype=torch.int64))
        if self.device.type == "cuda":
            with _on(self.device):
                self.data = _Resident(self.groups, self.device)


def _rows(t: Tensor) -> Tensor:
    """``t`` [rows, columns] with columns side by side, row strides in multiples of 8 and a 16-byte boundary at its start."""
    if t.data_ptr() % 16 == 0 and (t.is_contiguous() or (t.stride(1) == 1 and t.stride(0) % 8 == 0)):
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _new_rows(t: Tensor, dtype: torch.dtype) -> Tensor:
    """Contiguous rows like t's, of a type (the quicker call where t is that)."""
    return torch.empty_like(t) if t.dtype is dtype and t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _place(t: Tensor) -> tuple:
    """A place of block.py (in 16-bit units) of a tensor [rows, columns] or [columns]."""
    units = t.element_size() // 2
    width = t.shape[-1] * units
    rows, row = (t.shape[0], t.stride(0) * units) if t.dim() == 2 and t.shape[0] > 1 else (1, width)
    return t.data_ptr(), rows, 1, row, width, width


def _writable(out: Tensor, inputs: list[Tensor], others: list[Tensor]) -> bool:
    """Whether the kernel may write ``out`` itself: rows that do not overlap, none in ``others``, and each of ``inputs`` (of
    which a lane reads what it writes) in the same place or elsewhere."""
    place = _place(out)
    if out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        return False
    return (all(place == p or _apart(place, p) for p in map(_place, inputs))
            and all(_apart(place, p) for p in map(_place, others)))


def _modulation(t: Tensor) -> tuple[Tensor, int, int]:
    """A vector for all rows or one a group, as the kernel reads it: the tensor, its address and its row stride (0: one)."""
    if t.dim() == 1 or t.shape[0] == 1:
        t = _vector(t.reshape(-1))
        return t, t.data_ptr(), 0
    t = _rows(t)
    return t, t.data_ptr(), t.stride(0)


def residual_norm(x: Tensor, y: Tensor | None = None, *, rows: RowPlan | None = None, residual: float = 1.0,
                  gate: Tensor | None = None, post_norm: str | None = None, post_weight: Tensor | None = None,
                  norm: str | None = "rms", weight: Tensor | None = None, scale: Tensor | None = None,
                  shift: Tensor | None = None, eps: float = 1e-6, dtype: torch.dtype | None = None,
                  out: tuple[Tensor | None, Tensor | None] | None = None) -> tuple[Tensor, Tensor | None]:
    """``r = residual * x + gate * P(y)`` and ``n = N(r) * (1 + scale) + shift``: the residual stream after a block, and the
    next block's input. Returns ``(r, n)``.

    ``x`` [T, C] is the residual stream, ``y`` [T, C] the block's output; without y, r is x itself and only n is computed
    (the first norm of a model). P is ``post_norm`` and N ``norm``: ``"rms"``, ``h / sqrt(mean(h ** 2) + eps)``; ``"layer"``,
    ``(h - mean) / sqrt(var + eps)``; None, h itself; then times ``post_weight`` or ``weight`` [C] where given. ``norm=None``
    without weight, scale and shift computes no n and returns None for it (the last block).

    ``gate``, ``scale`` and ``shift`` are [C], or a row for each request of ``rows``, or without ``rows`` a row for each row
    of x. x is bfloat16, float16 or float32, y and n bfloat16 or float16 (``dtype``: n's type where only a float32 x is
    given, bfloat16 by default), r as x; the vectors of y's type or float32. Computed in float32, r and n rounded once each
    (n from the r that is not rounded). ``out`` may name the results' tensors, x and y among them. C is a multiple of 8 up to
    16384."""
    if x.dim() != 2 or (y is not None and y.shape != x.shape):
        raise ValueError(f"residual_norm expects x and y [T, C], got {tuple(x.shape)}"
                         + ("" if y is None else f" and {tuple(y.shape)}"))
    T, C = x.shape
    if C % 8 or not 0 < C <= 16384:
        raise ValueError(f"C must be a multiple of 8 up to 16384, got {C}")
    kind = y.dtype if y is not None else x.dtype if x.dtype in _DTYPES else dtype or torch.bfloat16
    code = _DTYPES.get(kind)
    if code is None or (x.dtype is not kind and x.dtype is not torch.float32) or dtype not in (None, kind):
        raise ValueError(f"residual_norm takes y and n of bfloat16 or float16 and x of that type or float32, got x "
                         f"{x.dtype}, y {None if y is None else y.dtype}, dtype {dtype}")
    if norm not in NORMS or post_norm not in NORMS:
        raise ValueError(f"a norm is one of {tuple(NORMS)}, got {norm!r} and {post_norm!r}")
    if y is None and (gate is not None or post_norm is not None or post_weight is not None or residual != 1.0):
        raise ValueError("gate, post_norm, post_weight and residual need y")
    want = norm is not None or weight is not None or scale is not None or shift is not None
    if y is None and not want:
        raise ValueError("nothing to compute: no y, norm, weight, scale or shift")
    if not (math.isfinite(residual) and abs(residual) <= _FLOAT_MAX):
        raise ValueError(f"residual must be finite in float32, got {residual}")
    if not eps >= 0 or _FLOAT_MAX < eps < math.inf:
        raise ValueError(f"eps must not be negative nor outside of float32, got {eps}")
    if rows is not None and rows.rows != T:
        raise ValueError(f"the plan has {rows.rows} rows, x has {T}")
    groups = T if rows is None else rows.requests
    wide = x.dtype is not kind
    index = x.get_device()
    if y is not None and y.get_device() != index:
        _same_device(x.device, y)
    f32 = False
    for t in (gate, scale, shift, post_weight, weight):
        if t is None:
            continue
        if t.dtype is not kind:
            f32 = True
            if t.dtype is not torch.float32:
                raise ValueError(f"vectors must be {kind} or float32, got {t.dtype}")
        shape = t.shape
        if t is weight or t is post_weight:
            if shape != (C,):
                raise ValueError(f"a weight must be [{C}], got {tuple(shape)}")
        elif shape != (groups, C) and shape != (C,) and shape != (1, C):
            raise ValueError(f"gate, scale and shift must be [{C}] or [{groups}, {C}], got {tuple(shape)}")
        if t.get_device() != index:
            _same_device(x.device, t)
    if rows is not None and rows._index != index:
        raise ValueError(f"tensors on {x.device}, the plan is for {rows.device}")
    r_out = n_out = None
    if out is not None:
        r_out, n_out = out
        if (r_out is None) != (y is None) or (n_out is None) == want:
            raise ValueError("out must name the results that are computed, and None for the others")
        if r_out is not None:
            _check_out(r_out, x, "residual_norm")
        if n_out is not None and (n_out.shape != x.shape or n_out.dtype is not kind or n_out.device != x.device):
            raise ValueError(f"residual_norm: out[1] must be {tuple(x.shape)} {kind} on {x.device}")
        if r_out is not None and n_out is not None and T and not _apart(_place(r_out), _place(n_out)):
            raise ValueError("the two results need places of their own")
    if _differentiable():
        _forward_only("residual_norm", x, y, gate, scale, shift, post_weight, weight, r_out, n_out)
    if not x.is_cuda:
        r, n = host_cache.residual_norm(x, y, rows, residual, gate, post_norm, post_weight, norm, weight, scale, shift, eps,
                                        kind, want)
        if r_out is not None:
            r = r_out.copy_(r)
        if n_out is not None:
            n = n_out.copy_(n)
        return r, n

    device = x.device
    lib = _lib(device)
    if f32:  # float32 is read as it is, and serves any mixture
        gate, scale, shift, post_weight, weight = (
            None if t is None else t.to(torch.float32) for t in (gate, scale, shift, post_weight, weight))
    gate_at = gate_ld = scale_at = scale_ld = shift_at = shift_ld = post_at = weight_at = 0
    y_at = y_ld = r_at = r_ld = n_at = n_ld = 0
    if gate is not None:
        gate, gate_at, gate_ld = _modulation(gate)
    if scale is not None:
        scale, scale_at, scale_ld = _modulation(scale)
    if shift is not None:
        shift, shift_at, shift_ld = _modulation(shift)
    if post_weight is not None:
        post_weight = _vector(post_weight)
        post_at = post_weight.data_ptr()
    if weight is not None:
        weight = _vector(weight)
        weight_at = weight.data_ptr()
    stream_in = x
    x = _rows(x)
    r = n = None
    if y is not None:
        y = _rows(y)
        y_at, y_ld = y.data_ptr(), y.stride(0) if T > 1 else C
        r = _new_rows(x, x.dtype) if r_out is None else _rows(r_out)
    if want:
        n = _new_rows(x if y is None else y, kind) if n_out is None else _rows(n_out)
    if out is not None:
        inputs = [x] if y is None else [x, y]
        vectors = [t for t in (gate, scale, shift, post_weight, weight) if t is not None]
        if r_out is not None and (r is not r_out or not _writable(r, inputs, vectors if n is None else [n, *vectors])):
            r = _new_rows(x, x.dtype)
        if n_out is not None and (n is not n_out or not _writable(n, inputs, vectors if r is None else [r, *vectors])):
            n = _new_rows(x, kind)
    if r is not None:
        r_at, r_ld = r.data_ptr(), r.stride(0) if T > 1 else C
    if n is not None:
        n_at, n_ld = n.data_ptr(), n.stride(0) if T > 1 else C
    stream = _raw_stream(index)
    with _current(index, device):
        status = lib.hf_residual_norm(_args(
            x.data_ptr(), x.stride(0) if T > 1 else C, y_at, y_ld, r_at, r_ld, n_at, n_ld, gate_at, gate_ld, scale_at,
            scale_ld, shift_at, shift_ld, post_at, weight_at, 0 if rows is None else rows.data.on(stream), groups, T, C, NORMS[post_norm],
            NORMS[norm], rows is None, wide, f32, code, residual, eps, stream))
    _check(status, "hf_residual_norm")
    if r_out is not None:
        r = _deliver(r, r_out)
    if n_out is not None:
        n = _deliver(n, n_out)
    return (stream_in if y is None else r), n


__all__ = ["RowPlan", "residual_norm"]
