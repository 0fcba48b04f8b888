"""Masked attention over packed clips and streamed attention over a paged cache.

``mass_bias_attention`` serves one clip whose frames are all there: every query sees every merged key.  Here are the
operators for what lies next to that:

* ``masked_attention``   several clips in one call (a document mask), frames in causal order, prefixes of special
  tokens, windows, scores capped by a tanh, a bias that depends on distance, shared key heads;
* ``attention_ranges``   the key interval of every row for those masks;
* ``PagedCache``         the merged keys, values and log-masses of past frames of many streams, in pages: append,
  fork, free and compact them on the device without host synchronisation;
* ``paged_attention``    a chunk of new tokens per stream (a frame, or one token) over that cache.

They have no derivatives: tensors that require a gradient are refused while gradients are recorded, and so are the dual tensors
of forward-mode differentiation.  The reference has no counterpart (its inference is one clip, batch one).
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _clib as C
from .ops import _tma_ready

__all__ = ["PagedCache", "attention_ranges", "masked_attention", "paged_attention"]

_PAGES = (16, 32, 64, 128)
_WIDE = (torch.int64, torch.uint32, torch.uint64)
_Two = ctypes.c_int64 * 2
_HERE = contextlib.nullcontext()
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # without the check that CUDA is up


def _on(device: torch.device):
    """The device made current for a call, where it is not already."""
    return _HERE if _current_device() == device.index else torch.cuda.device(device)


def _refuse_gradients(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad() or detach its inputs")
    if forward_ad._current_level >= 0:  # inside dual_level(); tangents are carried under no_grad() too
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative: its inputs must not be dual tensors")


def _same_device(what: str, device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors are on {device} and {t.device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a packed copy where the kernels cannot read it: a channel stride, rows that are not 16-byte aligned (a
    packed tensor at an odd offset too), broadcast dimensions."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        stride, per = t.stride(), 16 // t.element_size()
        if stride[-1] == 1 and not any([s % per or not s for s in stride[:-1]]):
            return t
        if _tma_ready(t) and 0 not in stride:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _runs(t: torch.Tensor) -> tuple[int, list[tuple[int, int]]]:
    """Bytes of the contiguous runs that a tensor consists of, and the (byte stride, count) of the dimensions that place them."""
    es = t.element_size()
    run, outer = es, []
    for s, n in sorted((s * es, n) for s, n in zip(t.stride(), t.shape) if n > 1 and s):
        if s <= run and not outer:
            run += s * (n - 1)
        else:
            outer.append((s, n))
    return run, outer


def _extent(t: torch.Tensor) -> tuple[int, int]:
    """The addresses from a tensor's first byte to behind its last."""
    at, n = t.data_ptr(), t.numel()
    if n and not t.is_contiguous():
        n = 1 + sum([s * (n - 1) for s, n in zip(t.stride(), t.shape)])
    return at, at + n * t.element_size()


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors have a byte in common.  Views of one buffer may interleave without that."""
    (at, ae), (bt, be) = _extent(a), _extent(b)
    if ae <= bt or be <= at or at == ae or bt == be or a.device != b.device:
        return False
    (ra, oa), (rb, ob) = _runs(a), _runs(b)
    pitch = math.gcd(*(s for s, _ in oa + ob))
    if pitch and ra <= (bt - at) % pitch <= pitch - rb:  # runs at different places of one pitch
        return False

    def starts(t, outer):
        x = torch.tensor([t - min(at, bt)])
        for s, n in outer:
            x = (x[:, None] + s * torch.arange(n)).flatten()
        return x.sort().values

    xa, xb = starts(at, oa), starts(bt, ob)
    before = torch.searchsorted(xa, xb + rb) - 1  # the last run of a that starts before a run of b ends
    return bool(((before >= 0) & (xa[before.clamp(min=0)] + ra > xb)).any())


def _check_out(q: torch.Tensor, out: torch.Tensor, *inputs: torch.Tensor | None, apart: tuple[tuple[int, int], ...] = ()) -> None:
    """``apart``: extents of contiguous inputs on out's device."""
    if out.shape != q.shape or out.dtype != q.dtype or not _tma_ready(out):
        raise ValueError("out must have q's shape and dtype, a unit channel stride and 16-byte aligned rows")
    if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError("out must not be a broadcast tensor")
    first, last = _extent(out)
    shared = any([a < last and first < b for a, b in apart]) and first < last
    for t in (q, *inputs):  # most inputs start behind the output's last byte or end before its first
        if not shared and isinstance(t, torch.Tensor) and t.data_ptr() < last:
            shared = _share_memory(out, t)
    if shared:
        raise ValueError("out must not share memory with the inputs")


def _scratch(size: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _floats(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _float_row(what: str, t: torch.Tensor, batch: int, n: int) -> tuple[torch.Tensor, int]:
    """A [n] or [batch, n] tensor as fp32 with its batch stride."""
    if t.shape != (n,) and t.shape != (batch, n):
        raise ValueError(f"{what} must be [{n}] or [{batch}, {n}], got {list(t.shape)}")
    t = _floats(t)
    return t, n if t.ndim == 2 else 0


def _positive(what: str, value: float | None) -> float:
    if value is None:
        return 0.0
    value = float(value)
    if not (math.isfinite(value) and value > 0):
        raise ValueError(f"{what} must be positive and finite")
    return value


def _int_vector(what: str, t, device: torch.device, n: int | None = None) -> torch.Tensor:
    """A 1-D int32 device tensor; lists and other integer tensors are converted (16 us of a call for int64 on the device, 8 of them
    for the values below; int32 is taken as it is).  Values beyond int32 are refused on the host and
    become its ends on the device, which are out of every range, so that none of them turns into another slot or row."""
    if isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == device and t.ndim == 1 and t.is_contiguous() and (
            n is None or t.numel() == n):
        return t
    if not isinstance(t, torch.Tensor):
        t = torch.tensor(t, dtype=None if len(t) else torch.int32)
    if t.ndim != 1 or t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool or (n is not None and t.numel() != n):
        raise ValueError(f"{what} must be a 1-D integer tensor" + ("" if n is None else f" of {n} entries"))
    if t.dtype in _WIDE:
        t = t.to(torch.int64)  # an unsigned value beyond int64 becomes a negative one
        if t.is_cuda:
            t = t.clamp(-2 ** 31, 2 ** 31 - 1)
        elif t.numel() and not (-2 ** 31 <= int(t.min()) and int(t.max()) < 2 ** 31):
            raise ValueError(f"{what} has values that int32 does not hold")
    return t.to(device=device, dtype=torch.int32).contiguous()


def attention_ranges(queries: int, keys: int | None = None, *, documents: torch.Tensor | None = None, step: int | None = None,
                     prefix: int = 0, window: int | None = None, device=None) -> torch.Tensor:
    """[queries, 2] int32 key intervals (begin, end) for ``masked_attention``; the queries are the last tokens of the keys.

    ``documents``  ascending offsets [n + 1] from 0 to ``keys`` (packed clips): a row sees its own document only.
    ``step``       causal order in blocks of this many tokens from the document's start: 1 is token by token, the tokens
                   of a frame make frames that see themselves and earlier ones.  None: the whole document.
    ``prefix``     the first tokens of a document that every row of it sees (camera and register tokens), besides the above.
    ``window``     no more than this many tokens back (the row's own counts), prefix tokens too: a row's keys are one interval.

    Everything is computed on the device of ``documents`` (else ``device``), without host synchronisation."""
    keys = queries if keys is None else keys
    if queries < 0 or keys < queries or keys >= 2 ** 31:
        raise ValueError("attention_ranges: 0 <= queries <= keys < 2^31 is required")
    if (step is not None and step < 1) or (window is not None and window < 1) or prefix < 0:
        raise ValueError("attention_ranges: step and window are at least 1, prefix at least 0")
    if documents is not None:
        if documents.ndim != 1 or documents.numel() < 2 or documents.dtype.is_floating_point:
            raise ValueError("attention_ranges: documents are at least two integer offsets")
        device = documents.device
    token = torch.arange(keys - queries, keys, device=device)
    if documents is None:
        begin, end = torch.zeros_like(token), torch.full_like(token, keys)
    else:
        cut = documents.to(torch.int64)
        at = torch.searchsorted(cut[1:].contiguous(), token, right=True).clamp(max=documents.numel() - 2)
        begin, end = cut[at], cut[at + 1]
    stop, start = end, begin
    if step is not None:
        end = torch.minimum(stop, start + ((token - start) // step + 1) * step)
    if prefix:
        end = torch.maximum(end, torch.minimum(stop, start + prefix))
    if window is not None:
        begin = torch.maximum(start, token - (window - 1))
    return torch.stack([begin, end], 1).to(torch.int32)


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_key_mass: torch.Tensor | None = None, *,
                     key_range: torch.Tensor | None = None, softcap: float | None = None,
                     distance_slope: torch.Tensor | None = None, query_position: torch.Tensor | None = None,
                     key_position: torch.Tensor | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(softcap * tanh(scale q k^T / softcap) + log_key_mass - slope |distance|) v over each row's key interval.

    q [B, H, Nq, 64], k and v [B, Hkv, Nk, 64] with H a multiple of Hkv (query head h reads key head h // (H // Hkv)),
    one type (fp32, bf16 or fp16), any strides.  ``log_key_mass`` [Nk] or [B, Nk] is added in fp32 (it is not
    rounded to q's type as in ``mass_bias_attention``).  ``key_range`` int32 [Nq, 2] or [B, Nq, 2]: the row sees keys
    [begin, end) (``attention_ranges`` makes them); None: all.  A row without keys gives zeros; what hidden
    keys hold never reaches a row (in 16 bits, infinite or NaN values near a row's keys cost a thousand times its time: keep a
    buffer behind its valid keys finite).  Capped 16-bit scores are fastest within half the cap.  ``distance_slope`` [H] with positions [Nq] / [Nk] (or per batch entry), by default
    token indices with the queries last.  Returns [B, H, Nq, 64] as a view of a token-major buffer, or writes ``out``, which must not share memory with the inputs."""
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k and v must be [batch, heads, tokens, channels]")
    B, H, Nq, D = q.shape
    _, Hkv, Nk, _ = k.shape
    if D != 64 or k.shape[3] != 64 or v.shape[3] != 64:
        raise ValueError("masked_attention supports head_dim=64 only")
    if k.shape != v.shape or k.shape[0] != B or Hkv == 0 or H % Hkv:
        raise ValueError("incompatible q/k/v shapes")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have one dtype")
    dt = C.dtype_code(q.dtype)
    softcap = _positive("softcap", softcap)
    scale = 0.125 if scale is None else _positive("scale", scale)
    if distance_slope is None and (query_position is not None or key_position is not None):
        raise ValueError("positions are used with distance_slope only")
    if distance_slope is not None and distance_slope.shape != (H,):
        raise ValueError(f"distance_slope must be [{H}]")
    if key_range is not None and (key_range.dtype != torch.int32 or key_range.shape not in ((Nq, 2), (B, Nq, 2))):
        raise ValueError(f"key_range must be int32 [{Nq}, 2] or [{B}, {Nq}, 2]")
    if out is not None:
        _check_out(q, out, k, v, log_key_mass, key_range, distance_slope, query_position, key_position)
    C.require_cuda(q, "masked_attention")
    _same_device("masked_attention", q.device, k, v, log_key_mass, key_range, distance_slope, query_position, key_position, out)
    _refuse_gradients("masked_attention", q, k, v, log_key_mass, distance_slope, query_position, key_position, out)
    with _on(q.device):
        if out is None:
            out = q.new_empty(B, Nq, H, D).transpose(1, 2)
        if B == 0 or H == 0 or Nq == 0:
            return out
        if Nk == 0:
            return out.zero_()
        q, k, v = _rows(q), _rows(k), _rows(v)
        mods = C.ScoreMods(scale=scale, softcap=softcap)
        if log_key_mass is not None:
            log_key_mass, mods.key_bias_sb = _float_row("log_key_mass", log_key_mass, B, Nk)
            mods.key_bias = log_key_mass.data_ptr()
        if key_range is not None:
            key_range = key_range.contiguous()
            mods.key_range, mods.key_range_sb = key_range.data_ptr(), 2 * Nq if key_range.ndim == 3 else 0
        if distance_slope is not None:
            distance_slope = _floats(distance_slope)
            mods.slope = distance_slope.data_ptr()
            if query_position is not None:
                query_position, mods.q_position_sb = _float_row("query_position", query_position, B, Nq)
                mods.q_position = query_position.data_ptr()
            if key_position is not None:
                key_position, mods.k_position_sb = _float_row("key_position", key_position, B, Nk)
                mods.k_position = key_position.data_ptr()
        lib = C.lib()
        size, ws = 0, None
        if dt != C.F32:  # fp32 needs none
            size = lib.vb200_masked_attention_workspace_size(dt, B, H, Hkv, Nq, Nk)
            ws = _scratch(size, q.device)
        rc = lib.vb200_masked_attention(dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, Hkv, Nq, Nk, D,
                                        C.strides3(q), C.strides3(k), C.strides3(v), C.strides3(out), mods, C.ptr(ws), size,
                                        C.stream_of(q.device))
        C.check(rc, "masked_attention")
    return out


@dataclass(frozen=True, eq=False)
class PagedCache:
    """Keys, values and log-masses of streams, in pages of 16, 32, 64 or 128 tokens; all state is on the device.

    ``k``, ``v`` [pages, page, kv heads, 64]; ``log_mass`` fp32 [pages, page] or None; ``table`` int32 [slots, max pages]
    of page numbers, -1 where there is none; ``length`` int32 [slots]; ``references`` int32 [pages], 0 for a free page.
    ``PagedCache.empty`` makes one.  The methods enqueue work on the current stream and read nothing back: a step of
    appends and attentions records into a CUDA graph.  What a kernel finds wrong (a slot out of range, a full pool) shows in
    ``device_error_flags()``."""

    k: torch.Tensor
    v: torch.Tensor
    log_mass: torch.Tensor | None
    table: torch.Tensor
    length: torch.Tensor
    references: torch.Tensor

    def __post_init__(self) -> None:
        k = self.k
        if k.ndim != 4 or k.shape[-1] != 64 or k.shape[1] not in _PAGES:
            raise ValueError("cache pools are [pages, 16 | 32 | 64 | 128, kv heads, 64]")
        if self.v.shape != k.shape or self.v.dtype != k.dtype:
            raise ValueError("k and v pools must have one shape and dtype")
        dtype = C.dtype_code(k.dtype)
        pages, page, heads, _ = k.shape
        if pages == 0 or heads == 0:
            raise ValueError("a cache has at least one page and one head")
        if self.log_mass is not None and (self.log_mass.shape != (pages, page) or self.log_mass.dtype != torch.float32):
            raise ValueError(f"log_mass must be fp32 [{pages}, {page}]")
        ints = (self.table, self.length, self.references)
        if self.table.ndim != 2 or 0 in self.table.shape or self.length.shape != self.table.shape[:1] or self.references.shape != (pages,):
            raise ValueError("table must be [slots, max pages], length [slots] and references [pages]")
        if any(t.dtype != torch.int32 for t in ints):
            raise ValueError("table, length and references must be int32")
        every = [t for t in (k, self.v, self.log_mass, *ints) if t is not None]
        if not all(t.is_contiguous() for t in every) or k.data_ptr() % 16 or self.v.data_ptr() % 16:
            raise ValueError("cache tensors must be contiguous, the pools 16-byte aligned")
        C.require_cuda(k, "PagedCache")
        _same_device("PagedCache", k.device, *every)
        # The fields stay what they are, so what every call needs of them is worked out once.  The bookkeeping calls of one cache
        # follow one another in any case, so they share one workspace.
        handle = C.CacheHandle(*(C.ptr(t) for t in (k, self.v, self.log_mass, *ints)), pages, page, heads, *self.table.shape)
        slots = self.table.shape[0]
        size = max(C.lib().vb200_cache_append_workspace_size(slots, slots, pages), C.lib().vb200_cache_compact_workspace_size(pages))
        self.__dict__.update(_extents=tuple(_extent(t) for t in every if t is not self.references), _device=k.device, _heads=heads, _dtype=dtype, _row=k.shape[2:], _slots=slots, _handle=handle, _sizes={},
                             _workspace=torch.empty(size, dtype=torch.uint8, device=k.device), _workspace_bytes=size)

    def _scratch(self, size: int) -> torch.Tensor:
        """The cache's workspace, or a larger one for this call."""
        return self._workspace if size <= self._workspace_bytes else torch.empty(size, dtype=torch.uint8, device=self._device)

    def __reduce__(self):  # copies and pickles carry the tensors, not the addresses
        return type(self), (self.k, self.v, self.log_mass, self.table, self.length, self.references)

    @classmethod
    def empty(cls, slots: int, pages: int, max_pages: int, *, page_size: int = 64, heads: int = 16, dtype=torch.bfloat16,
              masses: bool = True, device="cuda") -> "PagedCache":
        """An empty cache: ``slots`` streams of at most ``max_pages`` pages each from a pool of ``pages``."""
        if min(slots, pages, max_pages, heads) < 1 or page_size not in _PAGES:
            raise ValueError("slots, pages, max_pages and heads are at least 1, pages hold 16, 32, 64 or 128 tokens")
        shape = (pages, page_size, heads, 64)
        make = lambda size, dt: torch.zeros(size, dtype=dt, device=device)  # noqa: E731
        return cls(make(shape, dtype), make(shape, dtype), make(shape[:2], torch.float32) if masses else None,
                   torch.full((slots, max_pages), -1, dtype=torch.int32, device=device), make((slots,), torch.int32),
                   make((pages,), torch.int32))

    @property
    def page_size(self) -> int:
        return self.k.shape[1]

    @property
    def heads(self) -> int:
        return self._heads

    @property
    def device(self) -> torch.device:
        return self._device

    def append(self, sequence, offsets, k: torch.Tensor, v: torch.Tensor, log_mass: torch.Tensor | None = None) -> None:
        """Rows offsets[i] .. offsets[i + 1] of k, v [tokens, kv heads, 64] and log_mass [tokens] go behind the tokens of slot
        sequence[i].  Pages are taken lowest number first; a shared, partly filled last page is copied before it is written.
        All or nothing: a pool or a table row that is too short leaves the cache as it was (error bit 2).  A slot named
        twice in one call takes its first chunk only (error bit 1).  Without log_mass the tokens have mass 1."""
        dev = self._device
        shape = k.shape
        if len(shape) != 3 or shape[1:] != self._row or v.shape != shape:
            raise ValueError(f"append: k and v must be [tokens, {self.heads}, 64]")
        if k.dtype != self.k.dtype or v.dtype != self.k.dtype:
            raise ValueError(f"append: the cache holds {self.k.dtype}")
        if log_mass is not None:
            if self.log_mass is None:
                raise ValueError("append: the cache holds no log-masses")
            if log_mass.shape != shape[:1]:
                raise ValueError(f"append: log_mass must be [{shape[0]}]")
        _same_device("append", dev, k, v, log_mass)
        _refuse_gradients("append", k, v, log_mass, self.k, self.v, self.log_mass)
        with _on(dev):
            sequence = _int_vector("sequence", sequence, dev)
            n = sequence.numel()
            offsets = _int_vector("offsets", offsets, dev, n + 1)
            k, v = _rows(k), _rows(v)
            if log_mass is not None:
                log_mass = _floats(log_mass)
            lib = C.lib()
            size = self._workspace_bytes  # enough for one chunk per slot
            if n > self._slots:
                size = lib.vb200_cache_append_workspace_size(n, self._slots, self.k.shape[0])
            ks, vs = k.stride(), v.stride()
            ws = self._scratch(size)
            rc = lib.vb200_cache_append(self._handle, self._dtype, sequence.data_ptr(), offsets.data_ptr(), n, k.data_ptr(),
                                        v.data_ptr(), C.ptr(log_mass), shape[0], _Two(ks[0], ks[1]), _Two(vs[0], vs[1]),
                                        ws.data_ptr(), size, C.stream_of(dev))
            C.check(rc, "PagedCache.append")

    def fork(self, source, target) -> None:
        """Slot target[i] gets the tokens of slot source[i] by sharing its pages, and gives back what it held.  All
        sources are read before any target is written; of several pairs with one target the last counts."""
        dev = self._device
        with _on(dev):
            source = _int_vector("source", source, dev)
            target = _int_vector("target", target, dev, source.numel())
            lib = C.lib()
            size = lib.vb200_cache_fork_workspace_size(source.numel(), *self.table.shape)
            ws = self._scratch(size)
            rc = lib.vb200_cache_fork(self._handle, self._dtype, source.data_ptr(), target.data_ptr(), source.numel(),
                                      ws.data_ptr(), size, C.stream_of(dev))
            C.check(rc, "PagedCache.fork")

    def free(self, sequence) -> None:
        """Empties slots; pages that no other slot shares become free."""
        dev = self._device
        with _on(dev):
            sequence = _int_vector("sequence", sequence, dev)
            rc = C.lib().vb200_cache_free(self._handle, self._dtype, sequence.data_ptr(), sequence.numel(), C.stream_of(dev))
            C.check(rc, "PagedCache.free")

    def compact(self) -> torch.Tensor:
        """Moves the pages in use to the front of the pool and returns their number (int32 [1], on the device)."""
        dev = self._device
        with _on(dev):
            used = torch.empty(1, dtype=torch.int32, device=dev)
            rc = C.lib().vb200_cache_compact(self._handle, self._dtype, used.data_ptr(), self._workspace.data_ptr(),
                                             self._workspace_bytes, C.stream_of(dev))
            C.check(rc, "PagedCache.compact")
        return used


def paged_attention(q: torch.Tensor, cache: PagedCache, sequence, offsets, *, causal: bool = True,
                    key_range: torch.Tensor | None = None, softcap: float | None = None,
                    distance_slope: torch.Tensor | None = None, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ragged chunks of new tokens over the cache, one token per stream included.

    Rows offsets[i] .. offsets[i + 1] of q [rows, H, 64] are the last tokens of slot sequence[i] and are in the cache
    already (``PagedCache.append``); H is a multiple of the cache's heads.  A row sees the keys up to its own (``causal``) or
    all of its slot, or the keys [begin, end) of ``key_range`` int32 [rows, 2] (frames in causal order).  The cache's log-masses
    are added to the scores; softcap, distance_slope and scale as in ``masked_attention``, positions are token indices.  One call
    takes one kernel by its mean chunk, so single tokens and long chunks are better given in calls of their own.
    Returns [rows, H, 64] or writes ``out``, which must not share memory with q, the cache or another input; rows outside every chunk
    are not written."""
    shape = q.shape
    if len(shape) != 3 or shape[2] != 64:
        raise ValueError("q must be [rows, heads, 64]")
    rows, H, D = shape
    if H == 0 or H % cache._heads:
        raise ValueError(f"{H} query heads are no multiple of the cache's {cache._heads}")
    if q.dtype != cache.k.dtype:
        raise ValueError(f"the cache holds {cache.k.dtype}, q is {q.dtype}")
    softcap = _positive("softcap", softcap)
    scale = 0.125 if scale is None else _positive("scale", scale)
    if distance_slope is not None and distance_slope.shape != (H,):
        raise ValueError(f"distance_slope must be [{H}]")
    if key_range is not None and (key_range.dtype != torch.int32 or key_range.shape != (rows, 2)):
        raise ValueError(f"key_range must be int32 [{rows}, 2]")
    if out is not None:
        _check_out(q, out, key_range, distance_slope, sequence, offsets, apart=cache._extents if out.device == cache._device else ())
    dev = cache._device
    if q.device != dev:
        C.require_cuda(q, "paged_attention")
    _same_device("paged_attention", dev, q, key_range, distance_slope, out)
    _refuse_gradients("paged_attention", q, distance_slope, out, cache.k, cache.v, cache.log_mass)
    with _on(dev):
        sequence = _int_vector("sequence", sequence, dev)
        n = sequence.numel()
        offsets = _int_vector("offsets", offsets, dev, n + 1)
        if out is None:
            out = q.new_empty(rows, H, D)
        q = _rows(q)
        mods = C.ScoreMods(scale=scale, softcap=softcap)
        if key_range is not None:
            key_range = key_range.contiguous()
            mods.key_range = key_range.data_ptr()
        if distance_slope is not None:
            distance_slope = _floats(distance_slope)
            mods.slope = distance_slope.data_ptr()
        lib = C.lib()
        size = cache._sizes.get((rows, H, n))  # a function of these and of the cache's shape
        if size is None:
            size = lib.vb200_paged_attention_workspace_size(cache._dtype, rows, H, cache._handle, n)
            if len(cache._sizes) < 4096:
                cache._sizes[rows, H, n] = size
        ws = _scratch(size, dev)
        rc = lib.vb200_paged_attention(cache._dtype, q.data_ptr(), out.data_ptr(), rows, H, D, _Two(q.stride(1), q.stride(0)),
                                       _Two(out.stride(1), out.stride(0)), cache._handle, sequence.data_ptr(), offsets.data_ptr(),
                                       n, int(causal), mods, C.ptr(ws), size, C.stream_of(dev))
        C.check(rc, "paged_attention")
    return out
