"""The operators that an attention block runs around its INT8 linears, on the gfx950 kernels of ``libhf_block.so``:

* `qk_norm_rope` with `RotaryAxes`: the RMS norm of each query and key head and the rotation of its channels by the
  token's position on one or several axes (time, height, width), in one pass;
* `packed_attention` with `AttentionPlan`: attention over the sequences of several requests packed one behind the
  other, full or causal, with grouped heads, from single tokens against a cache to whole clips;
* `adapter_add` with `AdapterPlan`: low-rank adapters of many requests beside a shared projection.

`attention_block.py` has the modules that run them between an `Int8RotLinear` q/k/v projection and an output projection.

The reference holds these layers in its model library (the blocks its transformer keeps,
src/hyperflow_h3_flash/transformer.py:339-380, call them between ``to_q``/``to_k``/``to_v`` and ``to_out``); they have
no counterpart in its own files.

As the linears, they compute host tensors on the CPU (``host_block.py``, the same definitions) and device tensors on the
kernels, and raise when the library is missing. They are forward only: this framework's layers are frozen, and a call
that would have to be differentiated is refused. A plan holds what depends on lengths and requests alone (no data), is
built once on the host and serves every layer and step of that batch, on any stream.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
import threading
from collections.abc import Sequence

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _native, host_block
from .int8 import _check, _forget_input, _on, _raw_stream, _same_device

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_FLOAT_MAX = torch.finfo(torch.float32).max
_HERE = contextlib.nullcontext()
_rope_args, _attention_args, _adapter_args = (s.pack for s in (
    _native.ROPE_ARGS, _native.ATTENTION_ARGS, _native.ADAPTER_ARGS))
#: The current device's index.
_device_index = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


# With few rows the host time of a call is as long as its kernels (a kernel of 5 us in a call of 10): the functions below
# read each property once, and leave their straight path only where something is unusual.

def _differentiable() -> bool:
    """Whether gradients or forward-mode tangents may be recorded; ``torch.no_grad`` leaves the latter on."""
    return torch.is_grad_enabled() or forward_ad._current_level >= 0


def _forward_only(what: str, *tensors: Tensor | None) -> None:
    """Refuses tensors that the call would have to be differentiated for (where `_differentiable`)."""
    grads, tangents = torch.is_grad_enabled(), forward_ad._current_level >= 0
    for t in tensors:
        if t is not None and ((grads and t.requires_grad)
                              or (tangents and forward_ad.unpack_dual(t).tangent is not None)):
            raise RuntimeError(f"{what} is forward only: call it under torch.no_grad(), or on tensors that do not "
                               "require a gradient and have no tangent")


def _lib(device: torch.device) -> ctypes.CDLL:
    try:
        return _native.block_library()
    except RuntimeError as exc:
        raise RuntimeError(f"tensors on {device} need the gfx950 HIP library: {exc}") from exc


def _dtype_code(what: str, dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what} takes bfloat16 or float16, got {dtype}")
    return code


def _current(index: int, device: torch.device):
    """A context in which the device of that index is current: nothing to do when it is already."""
    return _HERE if _device_index() == index else torch.cuda.device(device)


def _heads(t: Tensor) -> tuple[Tensor, int, int]:
    """``t`` [tokens, heads, D] with its token and head strides as the kernels take them: channels side by side, 16-byte
    vectors (a copy where it lies otherwise). The stride of a dimension of one is never used."""
    rows, heads, d = t.shape
    if t.is_contiguous() and t.data_ptr() % 16 == 0 and d % 8 == 0:
        return t, heads * d, d
    token, head, channel = t.stride()
    if rows <= 1:
        token = heads * d
    if heads == 1:
        head = d
    if (channel != 1 and d > 1) or token % 8 or head % 8 or t.data_ptr() % 16:
        t = torch.empty((rows, heads, d), dtype=t.dtype, device=t.device).copy_(t)
        token, head = heads * d, d
    return t, token, head


def _new_like(t: Tensor) -> Tensor:
    """A contiguous tensor of t's size, type and device (of a contiguous t's format: the quicker call)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _vector(t: Tensor) -> Tensor:
    """``t`` [n] with its values side by side from a 16-byte boundary."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _check_out(out: Tensor, like: Tensor, what: str) -> None:
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{what}: out is {tuple(out.shape)} {out.dtype} on {out.device}, expected "
                         f"{tuple(like.shape)} {like.dtype} on {like.device}")


# A place: (address, rows, heads, row stride, head stride, width) of a tensor [rows, heads, width] of 16-bit elements.

def _apart(a: tuple, b: tuple) -> bool:
    """Whether no element of place ``a`` lies in place ``b``: separate memory, or slices of one buffer that take different
    parts of a common period (False where that cannot be told)."""
    p, rows_a, heads_a, row_a, head_a, width_a = a
    o, rows_b, heads_b, row_b, head_b, width_b = b
    heads_take_a, heads_take_b = (heads_a - 1) * head_a + width_a, (heads_b - 1) * head_b + width_b
    if (p + 2 * ((rows_a - 1) * row_a + heads_take_a) <= o or o + 2 * ((rows_b - 1) * row_b + heads_take_b) <= p
            or rows_a * heads_a * rows_b * heads_b == 0):
        return True
    ahead = (o - p) // 2
    # What they take of each period: all heads of a row, all rows of a head, or the channels alone.
    if row_a == row_b and row_a and heads_take_a <= ahead % row_a <= row_a - heads_take_b:
        return True
    if head_a == head_b and head_a and (
            (rows_a - 1) * row_a + width_a <= ahead % head_a <= head_a - (rows_b - 1) * row_b - width_b):
        return True
    period = math.gcd(row_a, head_a, row_b, head_b)
    return period > 0 and width_a <= ahead % period <= period - width_b


def _spread(place: tuple) -> bool:
    """Whether no two elements of a place lie in one."""
    _, rows, heads, row, head, width = place
    return (head >= width and row >= (heads - 1) * head + width) or (row >= width and head >= (rows - 1) * row + width)


def _result(out: Tensor, own: tuple, *others: tuple) -> tuple[Tensor, int, int]:
    """Where the kernels write a result that is to be in ``out`` [rows, heads, width], with its strides: out itself, or new
    memory where out's layout is not theirs or some of it lies in ``others``, which other workgroups may still read, or in
    ``own`` other than element by element (there each element is read by the workgroup that writes it)."""
    o, row, head = _heads(out)
    if o is out:
        rows, heads, width = out.shape
        place = (out.data_ptr(), rows, heads, row, head, width)
        if not _spread(place) or not (place == own or _apart(place, own)) or not all(_apart(place, x) for x in others):
            o, row, head = out.new_empty(out.shape), heads * width, width
    return o, row, head


#: Moves the versions of some tensors, as an operation of torch's own on them would.
_increment_versions = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version


def _written(t: Tensor) -> None:
    """A kernel wrote to ``t``, which was there before: torch is told as by an operation of its own. Autograd's check of
    saved tensors and the codes that `Int8RotLinear` layers share go by a tensor's version; inference tensors have none."""
    if t.is_inference():
        _forget_input(t)
    else:
        _increment_versions((t,))


def _deliver(result: Tensor, out: Tensor) -> Tensor:
    """``out`` holding ``result``, which the kernels wrote to ``out`` itself or to memory of its own."""
    if result is out:
        _written(out)
        return out
    return out.copy_(result)


class _Resident:
    """A host buffer and its copy on a device, uploaded once and not changed after. The copy is complete when the upload
    returns, so any stream may read it; `on` keeps its memory from being given out again while another stream than its own
    reads it. Copies of the objects that hold one share it. Pickled, it is the host buffer: what was loaded uploads at its
    first use, on a machine that has the device."""

    _uploading = threading.Lock()

    def __init__(self, host: Tensor, device: torch.device) -> None:
        self.__setstate__({"host": host, "device": device})
        self._upload()

    def _upload(self) -> None:
        with self._uploading:  # one of several threads: another's copy would take this one's memory back
            if self.device_copy is None:
                there = self.host.to(self.device)
                self._ptr, self._stream = there.data_ptr(), _raw_stream(there.get_device())
                self.device_copy = there

    def on(self, stream: int) -> int:
        if self.device_copy is None:
            self._upload()
        if stream != self._stream:
            self.device_copy.record_stream(torch.cuda.current_stream(self.device_copy.device))
        return self._ptr

    def __copy__(self) -> "_Resident":
        return self

    def __deepcopy__(self, memo: dict) -> "_Resident":
        return self

    def __getstate__(self) -> dict:
        return {"host": self.host, "device": self.device}

    def __setstate__(self, state: dict) -> None:
        self.host, self.device, self.device_copy = state["host"], state["device"], None
        self.host_address = self.host.data_ptr()


# ------------------------------------------------------------------------------------------------- norms and rotation

class RotaryAxes:
    """The rotation of channel pairs by positions on one or several axes.

    ``dims`` gives each axis its channels (each even, their sum a multiple of 16): axis a with n channels turns n / 2
    pairs by ``position[a] * theta ** (-2 i / n)``, i = 0 .. n / 2 - 1, the axes' pairs one behind the other.
    ``interleaved`` pairs channels (2p, 2p + 1), otherwise (p, p + sum(dims) / 2). Channels after ``sum(dims)`` are not
    turned. ``device`` uploads the tables at once (otherwise the first call on a device does)."""

    def __init__(self, dims: Sequence[int], *, theta: float = 10000.0, interleaved: bool = True,
                 device: torch.device | str | None = None) -> None:
        dims = tuple(int(n) for n in dims)
        if not dims or any(n <= 0 or n % 2 for n in dims) or sum(dims) % 16 or len(dims) > 16:
            raise ValueError(f"dims must be up to 16 positive even widths whose sum is a multiple of 16, got {dims}")
        if not (theta > 0 and math.isfinite(theta)):
            raise ValueError(f"theta must be positive and finite, got {theta}")
        self.dims, self.theta, self.interleaved = dims, float(theta), bool(interleaved)
        self.pairs = sum(dims) // 2
        rates, axis = [], []
        for a, n in enumerate(dims):
            rates += [self.theta ** (-2.0 * i / n) for i in range(n // 2)]
            axis += [a] * (n // 2)
        #: Angle per position step, and each pair's axis (float64 and int32, on the host).
        self.rates = torch.tensor(rates, dtype=torch.float64)
        self.axis = torch.tensor(axis, dtype=torch.int32)
        self._tables: dict[int, tuple[_Resident, _Resident]] = {}
        if device is not None and torch.device(device).type == "cuda":
            self.tables(torch.empty(0, device=device).device)

    def tables(self, device: torch.device) -> tuple[_Resident, _Resident]:
        """(revolutions per position step, axis of each pair) on ``device``."""
        found = self._tables.get(device.index)
        if found is None:
            with _on(device):
                found = (_Resident(self.rates / (2 * math.pi), device), _Resident(self.axis, device))
            self._tables[device.index] = found
        return found


def qk_norm_rope(q: Tensor, k: Tensor | None, positions: Tensor | None, rotary: RotaryAxes | None, *,
                 q_weight: Tensor | None = None, k_weight: Tensor | None = None, norm: bool = True, eps: float = 1e-6,
                 out: tuple[Tensor, Tensor | None] | None = None) -> tuple[Tensor, Tensor | None]:
    """Norm each head of ``q`` [T, Hq, D] and ``k`` [T, Hk, D] (or None) and rotate its channels by the token's position.

    ``x / sqrt(mean(x ** 2) + eps) * weight`` over the head's channels (``norm=False``: as it is; a weight of None is
    one; weights [D] in the inputs' type or float32), then the rotation of ``rotary`` (None: none) at ``positions``
    [T, axes] (or [T] for one axis; int32, int64 or float32; up to 2^31 either way the angle keeps float32's accuracy,
    beyond it loses a bit with every doubling). Computed in float32, rounded once to the inputs' type
    (bfloat16 or float16). q and k may be views with any token and head strides, such as slices of a fused projection.
    ``out`` may name the results' tensors, the inputs themselves among them (written directly where each is its own
    input's, through new memory where they overlap otherwise). D is a multiple of 16, up to 256."""
    dtype, shape = q.dtype, q.shape
    if len(shape) != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != shape[0] or k.shape[2] != shape[2])):
        raise ValueError("qk_norm_rope expects q [T, Hq, D] and k [T, Hk, D]")
    T, hq, D = shape
    hk = 0 if k is None else k.shape[1]
    if k is not None and k.dtype is not dtype:
        raise ValueError(f"q and k differ in type: {dtype}, {k.dtype}")
    if D % 16 or D == 0 or D > 256:
        raise ValueError(f"the head's width must be a multiple of 16 up to 256, got {D}")
    axes = pairs = 0
    if rotary is not None:
        axes, pairs = len(rotary.dims), rotary.pairs
        if 2 * pairs > D:
            raise ValueError(f"{2 * pairs} rotated channels exceed the head's {D}")
        if positions is None or positions.dtype not in _POSITIONS:
            raise ValueError("positions must be an int32, int64 or float32 tensor")
        if positions.shape != (T, axes) and (axes != 1 or positions.shape != (T,)):
            raise ValueError(f"positions must be [{T}, {axes}], got {tuple(positions.shape)}")
    else:
        positions = None
    for w in (q_weight, k_weight):
        if w is not None and (not norm or w.shape != (D,)):
            raise ValueError(f"a weight must be [{D}] and needs norm=True")
    if not eps >= 0 or _FLOAT_MAX < eps < math.inf:
        raise ValueError(f"eps must not be negative nor outside of float32, got {eps}")
    if out is not None:
        _check_out(out[0], q, "qk_norm_rope")
        if k is not None:
            _check_out(out[1], k, "qk_norm_rope")
    index = q.get_device()
    for t in (k, positions, q_weight, k_weight):
        if t is not None and t.get_device() != index:
            _same_device(q.device, t)
    if _differentiable():
        _forward_only("qk_norm_rope", q, k, positions, q_weight, k_weight, *(out or ()))
    code = _dtype_code("qk_norm_rope", dtype)
    if not q.is_cuda:
        if positions is not None:
            positions = positions.reshape(T, axes)
        result = host_block.qk_norm_rope(q, k, positions, rotary, q_weight, k_weight, norm, eps)
        if out is None:
            return result
        out[0].copy_(result[0])
        if k is not None:
            out[1].copy_(result[1])
        return out

    device = q.device
    lib = _lib(device)
    qw = kw = 0  # addresses: 0 for none
    wide = False
    if norm:
        wide = ((q_weight is not None and q_weight.dtype is not dtype)
                or (k_weight is not None and k_weight.dtype is not dtype))
        if wide:  # float32 is read as it is, and serves any mixture
            q_weight, k_weight = (None if w is None else w.to(torch.float32) for w in (q_weight, k_weight))
        if q_weight is not None:
            q_weight = _vector(q_weight)
            qw = q_weight.data_ptr()
        if k_weight is not None:
            k_weight = _vector(k_weight)
            kw = k_weight.data_ptr()
    q, qt, qh = _heads(q)
    ko = None
    k_ptr = ko_ptr = kt = kh = kot = koh = 0
    if k is not None:
        k, kt, kh = _heads(k)
        k_ptr = k.data_ptr()
    if out is None:
        qo, qot, qoh = _new_like(q), hq * D, D
        if k is not None:
            ko, kot, koh = _new_like(k), hk * D, D
    else:
        places = [(q.data_ptr(), T, hq, qt, qh, D)]
        if k is not None:
            places.append((k_ptr, T, hk, kt, kh, D))
        if out[0] is q and (k is None or out[1] is k) and all(map(_spread, places)):
            qo, qot, qoh = q, qt, qh  # in place: each element is read by the workgroup that writes it
            if k is not None:
                ko, kot, koh = k, kt, kh
        else:
            qo, qot, qoh = _result(out[0], *places)
            if k is not None:
                ko, kot, koh = _result(out[1], *reversed(places))
    if ko is not None:
        ko_ptr = ko.data_ptr()
    stream = _raw_stream(index)
    pos_ptr = turns = axis = pos_type = ld = 0
    if rotary is not None:
        if not positions.is_contiguous() and (positions.stride(0) < axes or (axes > 1 and positions.stride(1) != 1)):
            positions = positions.contiguous()
        pos_ptr, pos_type = positions.data_ptr(), _POSITIONS[positions.dtype]
        ld = positions.stride(0) if T > 1 else axes
        tables = rotary._tables.get(index) or rotary.tables(device)
        turns, axis = tables[0].on(stream), tables[1].on(stream)
    with _current(index, device):
        status = lib.hf_qk_norm_rope_call(_rope_args(
            q.data_ptr(), qt, qh, hq, k_ptr, kt, kh, hk, qo.data_ptr(), qot, qoh, ko_ptr, kot, koh, pos_ptr, pos_type,
            ld, axes, turns, axis, pairs, rotary is not None and rotary.interleaved, norm, qw, kw, wide, eps, T, D,
            code, stream))
    _check(status, "hf_qk_norm_rope")
    if out is None:
        return qo, ko
    _deliver(qo, out[0])
    if ko is not None:
        _deliver(ko, out[1])
    return out


# ---------------------------------------------------------------------------------------------------------- attention

class _Plan:
    """A planner's result on the host, with its copy on the device when that is not the host."""

    def _fill(self, name: str, lib: ctypes.CDLL, device: torch.device, *args) -> None:
        plan = getattr(lib, name)
        size = plan(*args, None, 0)
        _check(min(size, 0), name)
        host = torch.zeros(size, dtype=torch.uint8)
        size = plan(*args, host.data_ptr(), size)
        _check(min(size, 0), name)
        with _on(device):
            self.data = _Resident(host, device)
        self.bytes = size


def _plan_device(device: torch.device | str) -> torch.device:
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return device


def _lengths(values: Sequence[int], what: str) -> list[int]:
    lengths = [int(v) for v in values]
    if any(v < 0 for v in lengths):
        raise ValueError(f"{what} must not be negative")
    return lengths


def _array(ctype, values: Sequence[int]):
    return (ctype * max(len(values), 1))(*values)


class AttentionPlan(_Plan):
    """The work of attention over sequences packed one behind the other, for `packed_attention`.

    Sequence b has ``q_lengths[b]`` queries and ``kv_lengths[b]`` keys (the same when None); ``heads`` query heads share
    ``kv_heads`` key heads in equal groups. ``causal``: query i sees the keys up to i + kv_length - q_length (the last
    query sees all: a prompt, a prompt's last part, or one new token). Built from lengths on the host, once for all
    layers and steps of a batch."""

    def __init__(self, q_lengths: Sequence[int], kv_lengths: Sequence[int] | None = None, *, heads: int,
                 kv_heads: int | None = None, head_dim: int, causal: bool = False,
                 device: torch.device | str = "cuda") -> None:
        self.q_lengths = _lengths(q_lengths, "q_lengths")
        self.kv_lengths = self.q_lengths if kv_lengths is None else _lengths(kv_lengths, "kv_lengths")
        if len(self.q_lengths) != len(self.kv_lengths):
            raise ValueError(f"{len(self.q_lengths)} query lengths and {len(self.kv_lengths)} key lengths")
        self.heads, self.kv_heads = int(heads), int(heads if kv_heads is None else kv_heads)
        if self.heads < 1 or self.kv_heads < 1 or self.heads % self.kv_heads:
            raise ValueError(f"{self.heads} heads cannot share {self.kv_heads} key heads equally")
        self.head_dim, self.causal = int(head_dim), bool(causal)
        if self.head_dim < 16 or self.head_dim % 16 or self.head_dim > 128:
            raise ValueError(f"head_dim must be a multiple of 16 up to 128, got {head_dim}")
        self.q_rows, self.kv_rows = sum(self.q_lengths), sum(self.kv_lengths)
        self._q_shape = (self.q_rows, self.heads, self.head_dim)
        self._kv_shape = (self.kv_rows, self.kv_heads, self.head_dim)
        self.device = _plan_device(device)
        self._index = -1 if self.device.index is None else self.device.index
        if self.device.type != "cuda":
            return
        lib = _lib(self.device)
        q, kv = _array(ctypes.c_int64, self.q_lengths), _array(ctypes.c_int64, self.kv_lengths)
        cus = torch.cuda.get_device_properties(self.device).multi_processor_count
        self._fill("hf_attention_plan", lib, self.device, ctypes.addressof(q), ctypes.addressof(kv),
                   len(self.q_lengths), self.heads, self.kv_heads, self.head_dim, self.causal, cus)
        self.ws_bytes = lib.hf_attention_ws_bytes(self.data.host_address, self.bytes)


def _keys(t: Tensor) -> tuple[Tensor, int, int]:
    """`_heads` for keys and values, whose rows may not overlap nor lie 2^23 elements apart or more."""
    t, token, head = _heads(t)
    if not t.shape[2] <= token < 1 << 23 and t.shape[0] > 1:
        t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
        token, head = t.shape[1] * t.shape[2], t.shape[2]
    return t, token, head


def packed_attention(q: Tensor, k: Tensor, v: Tensor, plan: AttentionPlan, *, scale: float | None = None,
                     out: Tensor | None = None) -> Tensor:
    """Attention of packed sequences: ``softmax(scale q k^T) v`` within each sequence of ``plan``.

    ``q`` [sum q_lengths, heads, head_dim], ``k`` and ``v`` [sum kv_lengths, kv_heads, head_dim], bfloat16 or float16,
    any token and head strides (slices of a fused projection or a cache, whose sequences lie one behind the other without
    gaps); the result is like q. ``scale`` (default
    ``head_dim ** -0.5``) is positive. A query that sees no key gets zeros; what k and v hold at keys that a query does
    not see never reaches it. Scores, weights' sums and outputs are summed in float32, and divided by the weights' sum at the
    end (values of v times the number of keys have to stay in its range); the weights enter the second product in the
    inputs' type. ``out`` may be any tensor like q, the inputs among them (new memory is used where it lies in k or v)."""
    if q.shape != plan._q_shape or k.shape != plan._kv_shape or v.shape != plan._kv_shape:
        raise ValueError(f"the plan is for q {plan._q_shape} and k, v {plan._kv_shape}; got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    dtype = q.dtype
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError(f"q, k and v differ in type: {dtype}, {k.dtype}, {v.dtype}")
    code = _dtype_code("packed_attention", dtype)
    scale = plan.head_dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale <= _FLOAT_MAX:
        raise ValueError(f"scale must be positive and finite in float32, got {scale}")
    if out is not None:
        _check_out(out, q, "packed_attention")
    index = q.get_device()
    if k.get_device() != index or v.get_device() != index or index != plan._index:
        _same_device(q.device, k, v)
        raise ValueError(f"tensors on {q.device}, the plan is for {plan.device}")
    if _differentiable():
        _forward_only("packed_attention", q, k, v, out)
    if not q.is_cuda:
        result = host_block.packed_attention(q, k, v, plan, scale)
        return result if out is None else out.copy_(result)
    device = plan.device
    lib = _lib(device)
    q, qt, qh = _heads(q)
    k, kt, kh = _keys(k)
    v, vt, vh = _keys(v)
    if out is None:
        o, ot, oh = _new_like(q), plan.heads * plan.head_dim, plan.head_dim
    else:
        rows, heads, d = plan._kv_shape
        o, ot, oh = _result(out, (q.data_ptr(), *plan._q_shape[:2], qt, qh, d), (k.data_ptr(), rows, heads, kt, kh, d),
                            (v.data_ptr(), rows, heads, vt, vh, d))
    stream = _raw_stream(index)
    nbytes = plan.ws_bytes
    # Held until its kernels are launched: given back before, it could be handed to another thread's call in between.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    with _current(index, device):
        status = lib.hf_attention_call(_attention_args(
            q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, o.data_ptr(), ot, oh, scale,
            plan.data.host_address, plan.data.on(stream), plan.bytes, 0 if ws is None else ws.data_ptr(), nbytes, code,
            stream))
    _check(status, "hf_attention")
    return o if out is None else _deliver(o, out)


# ----------------------------------------------------------------------------------------------------------- adapters

class AdapterPlan(_Plan):
    """Which adapter each row of a packed batch takes, for `adapter_add`: ``ids[i]`` (-1: none) for the ``lengths[i]``
    rows of request i (None: one row each), the requests one behind the other, out of ``adapters``. Built on the host,
    once for all projections of the batch."""

    def __init__(self, ids: Sequence[int], lengths: Sequence[int] | None = None, *, adapters: int,
                 device: torch.device | str = "cuda") -> None:
        self.ids = [int(i) for i in ids]
        self.lengths = [1] * len(self.ids) if lengths is None else _lengths(lengths, "lengths")
        if len(self.ids) != len(self.lengths):
            raise ValueError(f"{len(self.ids)} requests and {len(self.lengths)} lengths")
        self.adapters = int(adapters)
        if any(not -1 <= i < self.adapters for i in self.ids):
            raise ValueError(f"adapters must be -1 .. {self.adapters - 1}, got {sorted(set(self.ids))}")
        self.rows = sum(self.lengths)
        self.live_rows = sum(n for i, n in zip(self.ids, self.lengths) if i >= 0)
        self.device = _plan_device(device)
        self._index = -1 if self.device.index is None else self.device.index
        self._ws: dict[tuple[int, int, int], int] = {}
        if self.device.type != "cuda":
            return
        ids_c, lens_c = _array(ctypes.c_int32, self.ids), _array(ctypes.c_int64, self.lengths)
        cus = torch.cuda.get_device_properties(self.device).multi_processor_count
        self._fill("hf_adapter_plan", _lib(self.device), self.device, ctypes.addressof(ids_c),
                   ctypes.addressof(lens_c), len(self.ids), self.adapters, cus)

    def _ws_bytes(self, lib: ctypes.CDLL, K: int, r: int, code: int) -> int:
        found = lib.hf_adapter_ws_bytes(self.data.host_address, self.bytes, K, r, code)
        _check(min(found, 0), "hf_adapter_ws_bytes")
        self._ws[K, r, code] = found
        return found


def _rows16(t: Tensor) -> Tensor:
    """``t`` [rows, columns] with columns side by side, row strides in whole 16-byte vectors and such a start."""
    if t.data_ptr() % 16 == 0 and (t.is_contiguous() or (
            (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])):
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _rows2(t: Tensor) -> Tensor:
    if t.is_contiguous() or ((t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])):
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _ld(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


def adapter_add(y: Tensor, x: Tensor, down: Tensor, up: Tensor, plan: AdapterPlan, *, scale: Tensor | None = None,
                out: Tensor | None = None) -> Tensor:
    """``y[m] + scale[a] * (x[m] @ down[a]^T) @ up[a]^T`` for the adapter a of each row (``plan``), ``y[m]`` where it has
    none: the low-rank adapters of many requests beside the projection that gave ``y``.

    ``x`` [M, K], ``y`` [M, N], ``down`` [adapters, r, K], ``up`` [adapters, N, r] in one type (bfloat16 or float16),
    ``scale`` float32 [adapters] (None: ones). Summed in float32, rounded once. ``out`` may be ``y``, which is then
    updated in place. K is a multiple of 8, r of 8 up to 512."""
    rows = plan.rows
    if x.dim() != 2 or y.dim() != 2 or x.shape[0] != rows or y.shape[0] != rows:
        raise ValueError(f"the plan has {rows} rows; got x {tuple(x.shape)}, y {tuple(y.shape)}")
    K, N = x.shape[1], y.shape[1]
    if down.dim() != 3 or down.shape[0] != plan.adapters or down.shape[2] != K:
        raise ValueError(f"down must be [{plan.adapters}, r, {K}], got {tuple(down.shape)}")
    r = down.shape[1]
    if up.shape != (plan.adapters, N, r):
        raise ValueError(f"up must be [{plan.adapters}, {N}, {r}], got {tuple(up.shape)}")
    if K % 8 or K == 0 or r % 8 or not 0 < r <= 512:
        raise ValueError(f"K must be a multiple of 8 and r one up to 512, got K={K}, r={r}")
    dtype = y.dtype
    if x.dtype is not dtype or down.dtype is not dtype or up.dtype is not dtype:
        raise ValueError(f"y, x, down and up differ in type: {dtype}, {x.dtype}, {down.dtype}, {up.dtype}")
    if scale is not None and (scale.shape != (plan.adapters,) or scale.dtype is not torch.float32):
        raise ValueError(f"scale must be float32 [{plan.adapters}]")
    if out is not None:
        _check_out(out, y, "adapter_add")
    code = _dtype_code("adapter_add", dtype)
    index = y.get_device()
    if (x.get_device() != index or down.get_device() != index or up.get_device() != index or index != plan._index
            or (scale is not None and scale.get_device() != index)):
        _same_device(y.device, x, down, up, scale)
        raise ValueError(f"tensors on {y.device}, the plan is for {plan.device}")
    if _differentiable():
        _forward_only("adapter_add", y, x, down, up, scale, out)
    if plan.live_rows == 0:  # no row has an adapter: y itself
        return y.clone() if out is None else out if out is y else out.copy_(y)
    if not y.is_cuda:
        result = host_block.adapter_add(y, x, down, up, plan, scale)
        return result if out is None else out.copy_(result)
    device = plan.device
    lib = _lib(device)
    in_place = out is y
    x, y = _rows16(x), _rows2(y)
    if not down.is_contiguous() or down.data_ptr() % 16:
        down = down.clone(memory_format=torch.contiguous_format)
    if not up.is_contiguous() or up.data_ptr() % 16:
        up = up.clone(memory_format=torch.contiguous_format)
    if scale is not None and not scale.is_contiguous():
        scale = scale.contiguous()
    o = y if in_place else _new_like(y) if out is None else _rows2(out)
    if o is out and not in_place:
        here, there = (o.data_ptr(), rows, 1, _ld(o), N, N), (y.data_ptr(), rows, 1, _ld(y), N, N)
        if here != there and not _apart(here, there):
            o = out.new_empty(out.shape)  # rows of y that other workgroups may still read
    stream = _raw_stream(index)
    with _current(index, device):
        nbytes = plan._ws.get((K, r, code))
        if nbytes is None:
            nbytes = plan._ws_bytes(lib, K, r, code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None  # held, as attention's
        status = lib.hf_adapter_add_call(_adapter_args(
            x.data_ptr(), _ld(x), y.data_ptr(), _ld(y), down.data_ptr(), up.data_ptr(), r,
            0 if scale is None else scale.data_ptr(), o.data_ptr(), _ld(o), N, K, plan.data.host_address,
            plan.data.on(stream), plan.bytes, 0 if ws is None else ws.data_ptr(), nbytes, code, stream))
    _check(status, "hf_adapter_add")
    return o if out is None else _deliver(o, out)
