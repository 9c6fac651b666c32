"""Keys and values of many requests held in 4 bits in pages of one pool, and the operators over them:

* `KVCache`: the pool with its accounts — which pages belong to which request, forks that share pages until they are written,
  truncating, freeing, compacting;
* `cache_append`: new tokens' keys and values written to the pages, `cache_read`: a request's keys and values out of them as
  `packed_attention` takes them;
* `cached_attention`: attention of packed queries over the pages;
* `copy_pages`: pages of all layers copied within a pool.

A value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (4 bits) times a power of two for each 32 channels of a head
(include/hf_cache.h has the layout and the rounding): 17/64 of 16-bit keys and values for heads of 32, 64 and 128, 13/48 of 96;
others are held as if they had the next multiple of 32 channels.

Beside `packed_attention`, whose caches lie one behind the other without gaps, a pool has room for every request to grow. A
`CachePlan` holds the lengths and pages of one step, is built on the host and serves all layers. As the other operators these
are forward only; host tensors compute on the CPU (``host_cache.py``, the same bytes in the pages), device tensors on the
kernels of ``libhf_block.so``. They have no counterpart in the reference, which keeps no cache."""

from __future__ import annotations

import ctypes
import heapq
import math
from array import array
from collections.abc import Sequence

import torch
from torch import Tensor

from . import _native, host_cache
from .block import (_array, _check_out, _current, _deliver, _differentiable, _dtype_code, _FLOAT_MAX, _forward_only, _heads,
                    _lengths, _lib, _new_like, _plan_device, _Resident, _result, _written)
from .int8 import _check, _on, _raw_stream, _same_device

PAGE_SIZES = (32, 64, 128, 256)
_append_args, _read_args, _attend_args, _copy_args = (s.pack for s in (
    _native.CACHE_APPEND_ARGS, _native.CACHE_READ_ARGS, _native.CACHED_ATTENTION_ARGS, _native.COPY_PAGES_ARGS))


class _Request:
    """A request's tokens in the cache and the pages that hold them. ``moved`` counts the changes that made older plans'
    pages or lengths wrong, ``shared`` those after which their tokens must not be written again."""

    __slots__ = ("length", "table", "moved", "shared")

    def __init__(self, length: int = 0, table: Sequence[int] = ()) -> None:
        self.length, self.table, self.moved, self.shared = length, array("i", table), 0, 0


class CachePlan:
    """One step of a batch over a `KVCache`, for its operators in every layer (`KVCache.plan` builds it): ``q_lengths``
    queries, ``kv_lengths`` tokens in the cache and ``new_lengths`` of them written in this step, by request.

    A plan stays good while its requests keep their pages and tokens: longer requests do no harm, `KVCache.truncate`, `free`
    and a `compact` that moves their pages end it, and after a `fork` it writes no more. What was ended is refused."""

    def __init__(self, cache: "KVCache", requests: Sequence[_Request], tables: list[array], q_lengths: list[int],
                 kv_lengths: list[int], new_lengths: list[int], heads: int, causal: bool) -> None:
        self.cache, self.device, self._index = cache, cache.device, cache._index
        self.q_lengths, self.kv_lengths, self.new_lengths, self.tables = q_lengths, kv_lengths, new_lengths, tables
        self.heads, self.kv_heads, self.head_dim, self.causal = heads, cache.kv_heads, cache.head_dim, causal
        self.q_rows, self.kv_rows, self.new_rows = sum(q_lengths), sum(kv_lengths), sum(new_lengths)
        self._q_shape = (self.q_rows, heads, self.head_dim)
        self._new_shape = (self.new_rows, self.kv_heads, self.head_dim)
        self._kv_shape = (self.kv_rows, self.kv_heads, self.head_dim)
        self._requests = requests
        if self.device.type == "cuda":
            lib = _lib(self.device)
            cus = torch.cuda.get_device_properties(self.device).multi_processor_count
            self._lay_out(lib, cus)

    def _lay_out(self, lib: ctypes.CDLL, cus: int) -> None:
        cache = self.cache
        q, kv, new = (_array(ctypes.c_int64, n) for n in (self.q_lengths, self.kv_lengths, self.new_lengths))
        pages = array("i", b"".join(map(bytes, self.tables)) or bytes(4))
        args = (ctypes.addressof(q), ctypes.addressof(kv), ctypes.addressof(new), len(self.q_lengths),
                pages.buffer_info()[0], cache.pages, cache.page_size, self.heads, self.kv_heads, self.head_dim, self.causal,
                cus)
        # A plan a step: laid out once into room that is enough (tiles of rows, their parts, pages in two lists of segments
        # and a table), not first for its size.
        tiles = sum(-(-n * self.heads // self.kv_heads // 16) for n in self.q_lengths) * self.kv_heads
        room = 4096 + 96 * (tiles + 4 * cus) + 64 * len(pages)
        host = torch.empty(room, dtype=torch.uint8)
        size = lib.hf_cache_plan(*args, host.data_ptr(), room)
        if size < 0:
            size = lib.hf_cache_plan(*args, None, 0)
            _check(min(size, 0), "hf_cache_plan")
            host = torch.empty(size, dtype=torch.uint8)
            size = lib.hf_cache_plan(*args, host.data_ptr(), size)
            _check(min(size, 0), "hf_cache_plan")
        with _on(self.device):
            self.data = _Resident(host[:size].clone(), self.device)
        self.bytes = size
        self.ws_bytes = lib.hf_cache_ws_bytes(self.data.host_address, self.bytes)

    def _start(self) -> None:
        """The state of the requests that the plan was built for (after the step's tokens are counted)."""
        self._moved = [r.moved for r in self._requests]
        self._shared = [r.shared for r in self._requests]
        self._good = self._writes = self.cache._changes

    def _check_good(self, cache: "KVCache", writes: bool) -> None:
        if cache is not self.cache:
            raise ValueError("the plan is of another cache")
        if (self._writes if writes else self._good) == cache._changes:
            return
        if any(r.moved != n for r, n in zip(self._requests, self._moved)):
            raise ValueError("the plan's pages were given back or moved: build a new one")
        self._good = cache._changes
        if writes:
            if any(r.shared != n for r, n, new in zip(self._requests, self._shared, self.new_lengths) if new):
                raise ValueError("a request of the plan was forked after it was built: its tokens are written before that")
            self._writes = cache._changes

    def __copy__(self) -> "CachePlan":
        return self

    def __deepcopy__(self, memo: dict) -> "CachePlan":
        return self

    def __reduce__(self):
        raise TypeError("a CachePlan belongs to its cache's pool and is not pickled")


class KVCache:
    """A pool of ``pages`` pages in each of ``layers`` layers, for keys and values of ``kv_heads`` heads of ``head_dim``
    channels (a multiple of 16 up to 128) in 4 bits, and the accounts of the requests in it. A page holds ``page_size``
    tokens (32, 64, 128 or 256); ``dtype`` (bfloat16 or float16) is the type of keys, values and queries. ``data`` is the
    pool, uint8 [layers, pages, bytes of a page].

    Requests are numbers that `new` and `fork` give. `plan` counts a step's new tokens and finds pages for them. The accounts
    are the host's and the device's work on one stream follows them in order; a plan's upload waits for what the current stream
    has been given before. Not for use by several threads at once."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, *, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda") -> None:
        if layers < 1 or kv_heads < 1 or pages < 0:
            raise ValueError(f"layers and kv_heads must be positive, got {layers}, {kv_heads} and {pages} pages")
        if head_dim < 16 or head_dim % 16 or head_dim > 128:
            raise ValueError(f"head_dim must be a multiple of 16 up to 128, got {head_dim}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if pages * page_size > 0x7fffffff or kv_heads > 65535 or layers > 65535:
            raise ValueError(f"{pages} pages of {page_size} tokens, {kv_heads} heads, {layers} layers exceed the indexes")
        self._code = _dtype_code("KVCache", dtype)
        self.layers, self.kv_heads, self.head_dim, self.pages = int(layers), int(kv_heads), int(head_dim), int(pages)
        self.page_size, self.dtype = int(page_size), dtype
        self.device = _plan_device(device)
        self._index = -1 if self.device.index is None else self.device.index
        #: Groups of 32 channels of a head and the bytes of a token's scales.
        self.groups = -(-self.head_dim // host_cache.GROUP)
        self.page_bytes = self.kv_heads * host_cache.slab_bytes(self.groups, self.page_size)
        self.data = torch.zeros(self.layers, self.pages, self.page_bytes, dtype=torch.uint8, device=self.device)
        self._sample = torch.empty(0, dtype=dtype, device=self.device)  # new tensors are made like it
        self._uses = [0] * self.pages
        self._unused = list(range(self.pages))  # a heap: the lowest page first
        self._requests: dict[int, _Request] = {}
        self._next = 0
        self._changes = 0

    @property
    def free_pages(self) -> int:
        return len(self._unused)

    def _request(self, request: int) -> _Request:
        found = self._requests.get(request)
        if found is None:
            raise ValueError(f"no request {request} in this cache")
        return found

    def length(self, request: int) -> int:
        """Tokens of a request, those of planned steps among them."""
        return self._request(request).length

    def table(self, request: int) -> list[int]:
        """The pages of a request, in its tokens' order."""
        return list(self._request(request).table)

    def _add(self, request: _Request) -> int:
        self._requests[self._next] = request
        self._next += 1
        return self._next - 1

    def new(self) -> int:
        """A request without tokens."""
        return self._add(_Request())

    def fork(self, request: int) -> int:
        """A second request with the tokens of one. They share its pages; a page that either writes to is copied first."""
        found = self._request(request)
        for page in found.table:
            self._uses[page] += 1
        found.shared += 1
        self._changes += 1
        return self._add(_Request(found.length, found.table))

    def _release(self, pages: Sequence[int]) -> None:
        for page in pages:
            self._uses[page] -= 1
            if self._uses[page] == 0:
                heapq.heappush(self._unused, page)

    def truncate(self, request: int, length: int) -> None:
        """Forget a request's tokens from ``length`` on; pages that no request needs any more are free again."""
        found = self._request(request)
        if not 0 <= length <= found.length:
            raise ValueError(f"the request has {found.length} tokens, cannot keep {length}")
        if length == found.length:
            return
        keep = -(-length // self.page_size)
        self._release(found.table[keep:])
        del found.table[keep:]
        found.length = length
        found.moved += 1
        self._changes += 1

    def free(self, request: int) -> None:
        """Forget a request."""
        self.truncate(request, 0)
        self._request(request).moved += 1
        self._changes += 1
        del self._requests[request]

    def compact(self) -> int:
        """Move the pages in use to the front of the pool, copying those behind to free ones; returns how many are in use.
        On the current stream, in every layer."""
        used = [p for p in range(self.pages) if self._uses[p]]
        n = len(used)
        src = [p for p in used if p >= n]
        dst = [p for p in range(n) if not self._uses[p]]
        if src:
            copy_pages(self.data, src, dst)
            to = dict(zip(src, dst))
            for request in self._requests.values():
                if any(p in to for p in request.table):
                    request.table = array("i", [to.get(p, p) for p in request.table])
                    request.moved += 1
            for a, b in to.items():
                self._uses[b], self._uses[a] = self._uses[a], 0
            self._unused = list(range(n, self.pages))
            self._changes += 1
        return n

    def plan(self, requests: Sequence[int], q_lengths: Sequence[int], *, new_lengths: Sequence[int] | None = None,
             heads: int | None = None, causal: bool = False) -> CachePlan:
        """The next step of some requests: ``q_lengths[i]`` queries of request i, ``new_lengths[i]`` tokens (default: as many)
        that `cache_append` writes behind those it has. A request without new tokens may be named several times. ``heads``
        query heads (default: kv_heads) share the key heads in equal groups. ``causal``: the last query sees every key, each one
        before it one key less.

        The new tokens are counted at once and get their pages; a shared page that they begin in is copied, on the current
        stream. RuntimeError, and nothing changed, when too few pages are free."""
        requests = list(requests)
        found = [self._request(r) for r in requests]
        q = _lengths(q_lengths, "q_lengths")
        new = list(q) if new_lengths is None else _lengths(new_lengths, "new_lengths")
        if not len(found) == len(q) == len(new):
            raise ValueError(f"{len(found)} requests, {len(q)} query lengths, {len(new)} new lengths")
        if len(set(requests)) != len(found):  # a request may be read several times, unless it gets tokens
            if any(n and requests.count(r) > 1 for r, n in zip(requests, new)):
                raise ValueError("a request that gets tokens is named twice")
        heads = self.kv_heads if heads is None else int(heads)
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} heads cannot share {self.kv_heads} key heads equally")
        P = self.page_size
        given: dict[int, int] = {}  # uses that the step takes from shared pages
        tables, copies, need = [], [], 0
        for r, n in zip(found, new):
            table = r.table[:]
            if n and r.length % P:
                page = table[-1]
                if self._uses[page] - given.get(page, 0) > 1:
                    given[page] = given.get(page, 0) + 1
                    copies.append((len(tables), len(table) - 1))
                    need += 1
            grow = -(-(r.length + n) // P) - len(table)
            need += grow
            tables.append((table, grow))
        if need > len(self._unused):
            raise RuntimeError(f"the step needs {need} pages, {len(self._unused)} of {self.pages} are free")
        fresh = [heapq.heappop(self._unused) for _ in range(need)]
        at = 0
        src, dst = [], []
        for i, j in copies:
            src.append(tables[i][0][j])
            dst.append(fresh[at])
            tables[i][0][j] = fresh[at]
            at += 1
        for table, grow in tables:
            table.extend(fresh[at:at + grow])
            at += grow
        try:
            plan = CachePlan(self, found, [table for table, _ in tables], q, [r.length + n for r, n in zip(found, new)], new,
                             heads, bool(causal))
            if src:
                copy_pages(self.data, src, dst)
        except BaseException:
            for page in fresh:
                heapq.heappush(self._unused, page)
            raise
        for page in fresh:
            self._uses[page] = 1
        for page, n in given.items():
            self._uses[page] -= n
        for i, _ in copies:
            found[i].moved += 1
        if src:
            self._changes += 1
        for r, n, (table, _) in zip(found, new, tables):
            if n:
                r.table, r.length = table[:], r.length + n
        plan._start()
        return plan


def _layer(cache: KVCache, layer: int) -> int:
    """The address of a layer's first page."""
    if not 0 <= layer < cache.layers:
        raise ValueError(f"layer {layer} of {cache.layers}")
    return cache.data.data_ptr() + layer * cache.pages * cache.page_bytes


def cache_append(cache: KVCache, layer: int, k: Tensor, v: Tensor, plan: CachePlan) -> None:
    """Write a step's new keys and values, ``k`` and ``v`` [sum new_lengths, kv_heads, head_dim] of the cache's type, to one
    layer's pages. Any token and head strides (slices of a fused projection).

    Each 32 channels of a head become 4-bit values times a power of two, the least that is a seventh of their largest
    magnitude or more; a value lies half a step of its codes away from what it is read as, at most, up to the largest
    magnitudes that a type's scales reach (57344 in float16, 7 * 2^125 in bfloat16: what is above is read as six sevenths of
    that). A group with a value that is not finite is read as NaN. Pages are written where their request's tokens lie and
    nowhere else."""
    if k.shape != plan._new_shape or v.shape != plan._new_shape:
        raise ValueError(f"the plan is for k, v {plan._new_shape}; got {tuple(k.shape)}, {tuple(v.shape)}")
    dtype = cache.dtype
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError(f"the cache holds {dtype}, got k {k.dtype} and v {v.dtype}")
    plan._check_good(cache, True)
    address = _layer(cache, layer)
    if k.get_device() != cache._index or v.get_device() != cache._index:
        _same_device(cache.device, k, v)
    if _differentiable():
        _forward_only("cache_append", k, v)
    if plan.new_rows == 0:
        return
    if not k.is_cuda:
        host_cache.append(cache, layer, k, v, plan)
        return
    device = cache.device
    lib = _lib(device)
    k, kt, kh = _heads(k)
    v, vt, vh = _heads(v)
    stream = _raw_stream(cache._index)
    with _current(cache._index, device):
        status = lib.hf_cache_append(_append_args(
            k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, address, plan.data.host_address, plan.data.on(stream), plan.bytes,
            cache._code, stream))
    _check(status, "hf_cache_append")
    _written(cache.data)


def cache_read(cache: KVCache, layer: int, plan: CachePlan) -> tuple[Tensor, Tensor]:
    """The keys and values of a plan's requests in one layer, ``k`` and ``v`` [sum kv_lengths, kv_heads, head_dim], one
    request behind the other: what `packed_attention` takes, and what `cached_attention` computes with."""
    plan._check_good(cache, False)
    address = _layer(cache, layer)
    shape = plan._kv_shape
    k, v = cache._sample.new_empty(shape), cache._sample.new_empty(shape)
    if plan.kv_rows == 0:
        return k, v
    if cache._index < 0:
        host_cache.read(cache, layer, plan, k, v)
        return k, v
    device = cache.device
    lib = _lib(device)
    stream = _raw_stream(cache._index)
    with _current(cache._index, device):
        status = lib.hf_cache_read(_read_args(
            address, k.data_ptr(), v.data_ptr(), plan.data.host_address, plan.data.on(stream), plan.bytes,
            cache._code, stream))
    _check(status, "hf_cache_read")
    return k, v


def cached_attention(q: Tensor, cache: KVCache, layer: int, plan: CachePlan, *, scale: float | None = None,
                     out: Tensor | None = None) -> Tensor:
    """Attention of packed queries over a plan's requests in one layer of the cache: ``softmax(scale q k^T) v`` with the keys
    and values that `cache_read` gives.

    ``q`` [sum q_lengths, heads, head_dim] of the cache's type, any token and head strides; the result is like q. ``scale``
    (default ``head_dim ** -0.5``) is positive. As in `packed_attention` a query that sees no key gets zeros, keys that a
    query does not see never reach it, and scores, sums and outputs are float32 with weights in the inputs' type (values of v
    times 256 times the number of keys have to stay in float32's range). ``out`` may be any tensor like q, q among them."""
    if q.shape != plan._q_shape:
        raise ValueError(f"the plan is for q {plan._q_shape}, got {tuple(q.shape)}")
    dtype = cache.dtype
    if q.dtype is not dtype:
        raise ValueError(f"the cache holds {dtype}, got q {q.dtype}")
    scale = plan.head_dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale <= _FLOAT_MAX:
        raise ValueError(f"scale must be positive and finite in float32, got {scale}")
    if out is not None:
        _check_out(out, q, "cached_attention")
    plan._check_good(cache, False)
    address = _layer(cache, layer)
    index = cache._index
    if q.get_device() != index:
        _same_device(cache.device, q)
    if _differentiable():
        _forward_only("cached_attention", q, out)
    if not q.is_cuda:
        result = host_cache.attention(q, cache, layer, plan, scale)
        return result if out is None else out.copy_(result)
    device = cache.device
    lib = _lib(device)
    q, qt, qh = _heads(q)
    if out is None:
        o, ot, oh = _new_like(q), plan.heads * plan.head_dim, plan.head_dim
    else:
        o, ot, oh = _result(out, (q.data_ptr(), *plan._q_shape[:2], qt, qh, plan.head_dim))
    stream = _raw_stream(index)
    nbytes = plan.ws_bytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None  # held, as packed_attention's
    with _current(index, device):
        status = lib.hf_cached_attention(_attend_args(
            q.data_ptr(), qt, qh, address, o.data_ptr(), ot, oh, scale, plan.data.host_address, plan.data.on(stream),
            plan.bytes, 0 if ws is None else ws.data_ptr(), nbytes, cache._code, stream))
    _check(status, "hf_cached_attention")
    return o if out is None else _deliver(o, out)


def _check_pairs(src: Sequence[int], dst: Sequence[int], pages: int) -> None:
    if any(not 0 <= p < pages for p in (*src, *dst)):
        raise ValueError(f"pages must be 0 .. {pages - 1}")
    if len(set(dst)) != len(dst) or not set(dst).isdisjoint(src):
        raise ValueError("a page is copied to once, and not from and to")


def copy_pages(pool: Tensor, src: Sequence[int], dst: Sequence[int]) -> Tensor:
    """Page ``src[i]`` of every layer copied to page ``dst[i]``, within ``pool`` [layers, pages, ...] of any type, whose pages
    lie one behind the other and hold a multiple of 16 bytes. No page twice in ``dst``, and none in both. Returns pool."""
    if pool.dim() < 3:
        raise ValueError(f"a pool is [layers, pages, ...], got {tuple(pool.shape)}")
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} pages to copy from, {len(dst)} to copy to")
    layers, pages = pool.shape[:2]
    size = math.prod(pool.shape[2:])
    if size and pages and layers and (not pool[0].is_contiguous() or (layers > 1 and pool.stride(0) < pages * size)):
        raise ValueError("a pool's pages must lie one behind the other")
    if size * pool.element_size() % 16 or (layers > 1 and pool.stride(0) * pool.element_size() % 16) or pool.data_ptr() % 16:
        raise ValueError("pages must hold a multiple of 16 bytes, and the pool start on one")
    if _differentiable():
        _forward_only("copy_pages", pool)
    if not pool.is_cuda:
        _check_pairs(src, dst, pages)
        if len(src) and pool.numel():
            pool[:, list(dst)] = pool[:, list(src)]
        return pool
    n = len(src)
    if n and not (0 <= min(src) and max(src) < pages and 0 <= min(dst) and max(dst) < pages):
        raise ValueError(f"pages must be 0 .. {pages - 1}")
    try:
        a, b = (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst)
    except TypeError as exc:
        raise ValueError(f"pages are numbers: {exc}") from None
    device, index = pool.device, pool.get_device()
    lib = _lib(device)
    with _current(index, device):
        status = lib.hf_copy_pages(_copy_args(
            pool.data_ptr(), layers, pool.stride(0) * pool.element_size() if layers > 1 else 0, pages,
            size * pool.element_size(), ctypes.addressof(a), ctypes.addressof(b), n, _raw_stream(index)))
    if status == -1:
        _check_pairs(src, dst, pages)
    _check(status, "hf_copy_pages")
    if n:
        _written(pool)
    return pool


__all__ = ["CachePlan", "KVCache", "cache_append", "cache_read", "cached_attention", "copy_pages"]
