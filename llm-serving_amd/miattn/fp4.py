"""The paged KV cache in 4 bits: the pool, what writes and reads it, and the attention over it.

:class:`Fp4PagedPool` is a :class:`~miattn.paged.PagedPool` whose K and V rows are held in 4 bits: the same
constructor, block tables, slots, writes and containers (``PagedKV``, ``PagedPrefill``'s sinks,
the decoders of ``miattn.qwen3`` and ``miattn.serve`` run on it unchanged), 17/64 of a 16-bit pool's bytes.

* ``pool.write_slots`` / ``write_prefill*`` -- K/V rows rounded to 4 bits on the way in;
* ``pool.read_slots(layer, slots)`` -- the rows that the pool holds, in its dtype;
* ``pool.write_qk_norm_rope`` -- a layer's q/k norm, RoPE and K/V write in one launch;
* :func:`paged_decode_fp4`, :func:`paged_decode_fp4_plan` -- one query token per row against such a pool, the
  counterparts of ``paged_decode`` and ``paged_decode_plan``.

Format. ``pool.keys[layer]`` and ``pool.values[layer]`` are uint8 ``(n_blocks, n_kv_head, page_bytes)``. A row of
``head_dim`` elements is held in groups of 32 that share a scale ``2**e``; an element is a sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 times it (E2M1, the element and scale types of the OCP MX formats). ``e`` is
the smallest integer with ``max|x| <= 7 * 2**e``, held to [-120, 125]; ``x * 2**-e`` goes to the nearest
level, ties to the even code, past 6 to 6. So an element is off by at most ``2**e``, which is less than
``max|x| / 3.5`` of its group (``0.25 * 2**e`` where ``|x| <= 2 * 2**e``; a group whose largest is below
``2**-120`` by at most ``2**-122``, one past ``1.5 * 2**127`` comes out as that). A group with a value that is
not finite reads back as NaN, all 32 of it. A page of one KV head is ``block_size * head_dim / 2`` code bytes, token
by token (element ``2i`` in the low half of byte ``i``), then ``head_dim / 32`` rows of ``block_size`` bytes
``e + 127`` (255: NaN).

Limits: HIP devices only (a 4-bit pool on the host is refused); ``head_dim`` 64, 128 or 256;
``block_size`` a power of two of at least 16; fp16, bf16 or fp32 on the 16/32-bit side. The attention takes pages
below 2^31 bytes per KV head (``block_size`` below 2^24 at ``head_dim`` 256, 2^25 at 128, 2^26 at 64).
"""

from __future__ import annotations

import ctypes
import math
from types import SimpleNamespace

import torch

from . import _lib
from ._contract import Rule, enforce, is_pow2
from .decode import _INDEXING, _PLAN_INPUTS, _SEQLEN_WATCH, DecodeGeometry, _require_backend, _require_device_tensors
from .paged import PagedPool

__all__ = ["GROUP", "Fp4PagedPool", "Fp4DecodePlan", "page_bytes", "paged_decode_fp4", "paged_decode_fp4_plan"]

#: elements that share a scale
GROUP = 32
_HEAD_DIMS = (64, 128, 256)
_MIN_BLOCK = 16
#: the attention's offsets inside a page of one KV head are 32 bits
_MOST_PAGE_BYTES = 2**31 - 1
_ELEMENT_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_SLOT_TYPES = (torch.int32, torch.int64)


def page_bytes(block_size: int, head_dim: int) -> int:
    """Bytes of one page (``block_size`` tokens) of one KV head, K or V."""
    return block_size * (head_dim // 2 + head_dim // GROUP)


_POOL = (
    Rule(lambda a: a.head_dim not in _HEAD_DIMS, ValueError,
         lambda a: f"the 4-bit cache takes head_dim 64, 128 or 256, got {a.head_dim}"),
    Rule(lambda a: not is_pow2(a.block_size) or a.block_size < _MIN_BLOCK, ValueError,
         lambda a: f"the 4-bit cache needs a power of two block_size of at least {_MIN_BLOCK}, got {a.block_size}"),
    Rule(lambda a: a.dtype not in _ELEMENT_TYPES, ValueError,
         lambda a: f"dtype must be fp16, bf16 or fp32, got {a.dtype}"),
    Rule(lambda a: a.device.type != "cuda", RuntimeError,
         lambda a: f"the 4-bit cache is held and read by HIP kernels and needs a CUDA (HIP) device, got {a.device}"),
)

_READ_SLOTS = (
    Rule(lambda a: a.slots.dim() != 1, ValueError,
         lambda a: f"slot_ids must be 1-D, got {tuple(a.slots.shape)}"),
    Rule(lambda a: a.slots.dtype not in _SLOT_TYPES, ValueError,
         lambda a: f"slot_ids must be an integer tensor (int32 or int64), got {a.slots.dtype}"),
    Rule(lambda a: a.slots.device != a.pool._home, ValueError,
         lambda a: f"slot_ids are on {a.slots.device} but the pool is on {a.pool._home}"),
)


class Fp4PagedPool(PagedPool):
    """Physical KV blocks in 4 bits: uint8 ``(n_blocks, n_kv_head, page_bytes)`` K and V per layer (the
    module docstring has the format). ``dtype`` is what writes take, reads return and queries are.
    ``write_qk_norm_rope`` keeps norm and rotation in fp32 and rounds q and k to ``dtype`` once (the 16-bit
    pool's rounds after every op); the pool holds the 4-bit form of that k, as a write of ``k_out`` would."""

    def _check_storage(self) -> None:
        enforce(_POOL, self)
        _lib.require_library("Fp4PagedPool")

    def _store_layout(self) -> tuple[tuple[int, ...], torch.dtype]:
        return (self.n_blocks, self.n_kv_head, page_bytes(self.block_size, self.head_dim)), torch.uint8

    def __init__(self, *args, **kw) -> None:
        super().__init__(*args, **kw)
        # with its index: "cuda" alone would name whichever device is current at a later call
        self.device = self._home = self._write_error.device
        self._row = torch.Size((self.n_kv_head, self.head_dim))
        self._sizes = (self.n_kv_head, self.head_dim, self.n_blocks, self.block_size)
        row = self.n_kv_head * self.head_dim
        self._dense = _lib.int64_array((row, self.head_dim, 1) * 2)  # strides of contiguous k and v
        self._code = _lib.dtype_code(self.dtype)

    def write_slots(self, layer: int, slot_ids: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
        """``pool_flat[slot_ids[i]] = k[i]`` and the same for ``v``, rounded to 4 bits (``PagedPool.write_slots``).
        Distinct slots: a slot named twice may end up with one row's codes under the other's scales."""
        shape, dtype, home = k.shape, self.dtype, self._home
        if (len(shape) != 3 or shape[1:] != self._row or v.shape != shape or slot_ids.shape != shape[:1]
                or k.dtype != dtype or v.dtype != dtype or slot_ids.dtype not in _SLOT_TYPES
                or k.device != home or v.device != home or slot_ids.device != home):
            super().write_slots(layer, slot_ids, k, v)  # raises what is wrong, or converts k and v
            return
        self._scatter_hip(self._layer(layer), slot_ids, k, v)

    def _scatter_hip(self, layer: int, slot_ids, k, v) -> None:
        if k.device != self._home or v.device != self._home:
            raise RuntimeError(f"the pool is on {self._home} and takes k/v there; got {k.device}/{v.device}")
        n = k.shape[0]
        if n == 0:
            return
        slot_ids = slot_ids.contiguous()
        strides = self._dense if k.is_contiguous() and v.is_contiguous() else \
            _lib.int64_array((*k.stride(), *v.stride()))
        with _lib.on_device(self._home):
            rc = _lib.lib.mi_kv_slot_write_fp4(
                k.data_ptr(), v.data_ptr(), slot_ids.data_ptr(), 8 * slot_ids.element_size(),
                self.keys[layer].data_ptr(), self.values[layer].data_ptr(), n, *self._sizes, strides, self._code,
                self._write_error.data_ptr(), _lib.current_stream(self._home))
        _lib.check(rc, "Fp4PagedPool.write_slots")
        if self.strict_writes:
            self.check_writes()

    def read_slots(self, layer: int, slot_ids: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The K and V rows at ``slot_ids`` (int32 or int64, repeats allowed), each ``(n, n_kv_head,
        head_dim)`` in the pool's dtype (exact in bf16 and fp32; in fp16 rounded, past its largest value that).
        A slot outside the pool reads as zeros and is reported by :meth:`check_writes`."""
        layer = self._layer(layer)
        if slot_ids.dim() != 1 or slot_ids.dtype not in _SLOT_TYPES or slot_ids.device != self._home:
            enforce(_READ_SLOTS, SimpleNamespace(pool=self, slots=slot_ids))
        n = slot_ids.shape[0]
        k = torch.empty((n, *self._row), dtype=self.dtype, device=self._home)
        v = torch.empty_like(k)
        if n == 0:
            return k, v
        slot_ids = slot_ids.contiguous()
        with _lib.on_device(self._home):
            rc = _lib.lib.mi_kv_slot_read_fp4(
                self.keys[layer].data_ptr(), self.values[layer].data_ptr(), slot_ids.data_ptr(),
                8 * slot_ids.element_size(), k.data_ptr(), v.data_ptr(), n, *self._sizes, self._code,
                self._write_error.data_ptr(), _lib.current_stream(self._home))
        _lib.check(rc, "Fp4PagedPool.read_slots")
        if self.strict_writes:
            self.check_writes()
        return k, v

    def _refusal(self, token: int) -> str:
        return (f"token {token} of a write or read had a slot (or position) outside the pool's {self.n_slots} slots "
                f"({self.n_blocks} blocks x {self.block_size}): a write left it out, a read returned zeros for it")

    def _launch_epilogue(self, layer, source, row_stride, n_parts, q_norm_w, k_norm_w, cos, sin, rotary, pos, slot_ids,
                         q, k_out, v_out, eps, zero_centred_norm) -> int:
        B, H, D = q.shape
        tensors = (source, q_norm_w, k_norm_w, cos, sin, pos, slot_ids, q)
        tensors += tuple(t for t in (k_out, v_out) if t is not None)
        if any(t.device != self._home for t in tensors):
            raise RuntimeError(f"the pool is on {self._home} and takes every tensor of the epilogue there")
        with _lib.on_device(self._home):
            return _lib.lib.mi_qk_norm_rope_write_fp4(
                source.data_ptr(), row_stride, n_parts, q_norm_w.data_ptr(), k_norm_w.data_ptr(), cos.data_ptr(),
                sin.data_ptr(), cos.shape[0], rotary, pos.data_ptr(), slot_ids.data_ptr(),
                8 * slot_ids.element_size(), q.data_ptr(), self.keys[layer].data_ptr(), self.values[layer].data_ptr(),
                None if k_out is None else k_out.data_ptr(), None if v_out is None else v_out.data_ptr(),
                B, H, *self._sizes, float(eps), int(bool(zero_centred_norm)), self._code, self._write_error.data_ptr(),
                _lib.current_stream(self._home))

    def decode_plan(self, q, block_table, seqlen, *, scale=None, window: int | None = None,
                    sinks: int = 0) -> "Fp4DecodePlan":
        if window is not None or sinks:
            raise ValueError("the attention over a 4-bit pool has no window: it sees whole rows")
        return paged_decode_fp4_plan(q, self.keys, self.values, block_table, seqlen, scale=scale)

    def bytes(self) -> int:
        return 2 * self.n_layer * self.n_blocks * self.n_kv_head * page_bytes(self.block_size, self.head_dim)


# -- the attention's contract, in the order a caller learns about mistakes ------------
_LAYOUT = (
    Rule(lambda a: a.q.dim() != 3, ValueError,
         lambda a: f"q must be (B, H, D), got shape {tuple(a.q.shape)}"),
    Rule(lambda a: a.k.dim() != 3 or a.v.dim() != 3, ValueError,
         lambda a: "4-bit k_cache/v_cache must be (n_blocks, H_kv, page_bytes), got "
                   f"{tuple(a.k.shape)} / {tuple(a.v.shape)}"),
    Rule(lambda a: a.k.shape != a.v.shape, ValueError,
         lambda a: f"k_cache/v_cache shapes differ: {tuple(a.k.shape)} vs {tuple(a.v.shape)}"),
    Rule(lambda a: a.q.dtype not in _ELEMENT_TYPES, ValueError,
         lambda a: f"q dtype must be fp16, bf16 or fp32, got {a.q.dtype}"),
    Rule(lambda a: a.k.dtype != torch.uint8 or a.v.dtype != torch.uint8, ValueError,
         lambda a: f"4-bit k_cache/v_cache must be uint8 pages, got {a.k.dtype}, {a.v.dtype}"),
    Rule(lambda a: a.q.shape[2] not in _HEAD_DIMS, ValueError,
         lambda a: f"the 4-bit cache takes head_dim 64, 128 or 256, got {a.q.shape[2]}"),
    Rule(lambda a: a.k.shape[1] < 1 or a.q.shape[1] < 1 or a.q.shape[1] % a.k.shape[1] != 0, ValueError,
         lambda a: f"n_head ({a.q.shape[1]}) must be a multiple of n_kv_head ({a.k.shape[1]})"),
    Rule(lambda a: _block_size(a.k, a.q.shape[2]) < _MIN_BLOCK, ValueError,
         lambda a: f"pages of {a.k.shape[2]} bytes at head_dim {a.q.shape[2]} hold no power of two block_size of at "
                   f"least {_MIN_BLOCK} tokens ({page_bytes(1, a.q.shape[2])} bytes each)"),
    Rule(lambda a: a.k.shape[2] > _MOST_PAGE_BYTES, ValueError,
         lambda a: f"the 4-bit decode reads pages below 2^31 bytes per KV head, got {a.k.shape[2]}"),
)

_PAGES = (
    Rule(lambda a: a.k.stride(2) != 1 or a.v.stride(2) != 1, ValueError,
         lambda a: f"the 4-bit decode reads contiguous pages; got strides {a.k.stride()} / {a.v.stride()}"),
    Rule(lambda a: (a.k.data_ptr() | a.v.data_ptr()) % 16 != 0 or any(_odd_stride(t, i) for t in (a.k, a.v) for i in (0, 1)),
         ValueError, lambda a: "the 4-bit decode needs 16-byte aligned pages"),
)


def _odd_stride(pages, dim: int) -> bool:
    """Whether a step along ``dim`` leaves the 16-byte grid (no launch steps along the heads of a single one)."""
    return pages.stride(dim) % 16 != 0 and (dim == 0 or pages.shape[dim] > 1)


def _block_size(k_cache, head_dim: int) -> int:
    """Tokens per page, from the page's bytes (0 where no power of two fits)."""
    tokens, rest = divmod(int(k_cache.shape[2]), page_bytes(1, head_dim))
    return tokens if rest == 0 and is_pow2(tokens) else 0


def _check(q, k_cache, v_cache, block_table, seqlen) -> DecodeGeometry:
    a = SimpleNamespace(q=q, k=k_cache, v=v_cache, table=block_table, seqlen=seqlen)
    enforce(_LAYOUT, a)
    enforce(_INDEXING, a)
    g = DecodeGeometry(int(q.shape[0]), int(q.shape[1]), int(k_cache.shape[1]), int(q.shape[2]),
                       _block_size(k_cache, int(q.shape[2])), int(block_table.shape[1]))
    if g.rows:
        _SEQLEN_WATCH.confirm(seqlen, g.capacity)
    return g


def _workspace_bytes(g: DecodeGeometry, dtype: torch.dtype) -> int:
    return int(_lib.lib.mi_paged_decode_fp4_workspace_size(*g.dims(), _lib.dtype_code(dtype)))


def _strides(q, k, v, out, table):
    return _lib.int64_array((*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *out.stride()[:2], table.stride(0)))


def paged_decode_fp4(q, k_cache, v_cache, block_table, seqlen, *, scale: float | None = None) -> torch.Tensor:
    """Decode one query token per row against a 4-bit paged pool: ``softmax(scale q K^T) V`` over each
    row's first ``seqlen`` tokens, zeros for a row of none. ``q`` ``(B, H, D)`` fp16, bf16 or fp32;
    ``k_cache``/``v_cache`` uint8 ``(n_blocks, H_kv, page_bytes)``; ``block_table`` ``(B, width)`` int32 (ids trusted,
    as in ``paged_decode``); ``seqlen`` ``(B,)`` int32 or int64. Sums are fp32, the output is rounded once; in fp16 what is past
    its largest value (pages may hold more, written from bf16 or fp32; an fp32 sum's infinity too) comes out as that, as
    ``Fp4PagedPool.read_slots`` returns it."""
    _require_backend()
    _require_device_tensors((("q", q), ("k_cache", k_cache), ("v_cache", v_cache),
                             ("block_table", block_table), ("seqlen", seqlen)))
    g = _check(q, k_cache, v_cache, block_table, seqlen)
    if g.rows == 0:
        return torch.empty_like(q)
    enforce(_PAGES, SimpleNamespace(k=k_cache, v=v_cache))
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    table = block_table if block_table.stride(1) == 1 else block_table.contiguous()
    lens = seqlen.to(torch.int32).contiguous()
    with _lib.on_device(q.device):
        out = torch.empty_like(q)
        n_ws = _workspace_bytes(g, q.dtype)
        ws = torch.zeros(n_ws, dtype=torch.uint8, device=q.device) if n_ws else None
        rc = _lib.lib.mi_paged_decode_fp4(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lens.data_ptr(), out.data_ptr(),
            *g.dims(), _strides(q, k_cache, v_cache, out, table),
            float(1.0 / math.sqrt(g.head_dim) if scale is None else scale), _lib.dtype_code(q.dtype),
            None if ws is None else ws.data_ptr(), n_ws, _lib.current_stream(q.device))
    _lib.check(rc, "paged_decode_fp4")
    return out


class Fp4DecodePlan:
    """Checked-once launch state for the decode calls of one container over a 4-bit pool: the counterpart of
    :class:`~miattn.decode.PagedDecodePlan`, with the same contract (pools, table and ``seqlen`` by
    reference, ``seqlen`` updates in place seen; one workspace, so its runs stay ordered on one stream). Built
    outside a capture: the workspace is cleared once, here, and the host waits for that."""

    __slots__ = ("n_layer", "geometry", "q_signature", "_k_ptrs", "_v_ptrs", "_pools", "_table", "_seqlen", "_ws",
                 "_strides", "_frozen", "_shape", "_stride", "_dtype", "_device", "_index", "_table_ptr", "_seqlen_ptr")

    def __init__(self, q, k_caches, v_caches, block_table, seqlen, *, scale=None) -> None:
        _require_backend()
        _require_device_tensors((("q", q), ("block_table", block_table), ("seqlen", seqlen)))
        ks, vs = list(k_caches), list(v_caches)
        enforce(_PLAN_INPUTS, SimpleNamespace(q=q, ks=ks, vs=vs, table=block_table, seqlen=seqlen))
        first = (tuple(ks[0].shape), ks[0].stride(), vs[0].stride())
        for layer, (k, v) in enumerate(zip(ks, vs)):
            _require_device_tensors(((f"k_cache[{layer}]", k), (f"v_cache[{layer}]", v)))
            g = _check(q, k, v, block_table, seqlen)
            enforce(_PAGES, SimpleNamespace(k=k, v=v))
            if (tuple(k.shape), k.stride(), v.stride()) != first:
                raise ValueError("paged_decode_fp4_plan needs one pool shape and layout for every layer "
                                 f"(layer {layer} differs from layer 0)")
        self.n_layer = len(ks)
        self.geometry = g
        self.q_signature = (tuple(q.shape), q.dtype, q.device, q.stride())
        self._shape, self._stride, self._dtype, self._device = q.shape, q.stride(), q.dtype, q.device
        self._pools = (ks, vs)  # keeps the pool tensors alive
        # every argument that no run changes, as the C call takes it (a run's call 1.8 -> 1.5 us)
        self._k_ptrs = [ctypes.c_void_p(k.data_ptr()) for k in ks]
        self._v_ptrs = [ctypes.c_void_p(v.data_ptr()) for v in vs]
        self._table, self._seqlen = block_table, seqlen  # kept alive; read in place at every run
        self._table_ptr, self._seqlen_ptr = ctypes.c_void_p(block_table.data_ptr()), ctypes.c_void_p(seqlen.data_ptr())
        self._index = q.device.index
        self._strides = _strides(q, ks[0], vs[0], q, block_table)
        n_ws = _workspace_bytes(g, q.dtype)
        with _lib.on_device(q.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("paged_decode_fp4_plan clears its workspace once, which a capture would only "
                                   "record: build the plan before the capture")
            self._ws = torch.zeros(n_ws, dtype=torch.uint8, device=q.device) if n_ws else None
            torch.cuda.current_stream().synchronize()  # runs may be on any stream
        self._frozen = (*map(ctypes.c_int, g.dims()), self._strides,
                        ctypes.c_float(1.0 / math.sqrt(g.head_dim) if scale is None else scale),
                        ctypes.c_int(_lib.dtype_code(q.dtype)),
                        ctypes.c_void_p(None if self._ws is None else self._ws.data_ptr()), ctypes.c_size_t(n_ws))

    def run(self, layer: int, q) -> torch.Tensor:
        """Launch one layer; ``q`` must have the layout the plan was built with."""
        layer = int(layer)
        if not 0 <= layer < self.n_layer:
            raise IndexError(f"layer {layer} is outside the plan's {self.n_layer} layers")
        if (q.shape != self._shape or q.dtype != self._dtype or q.get_device() != self._index
                or q.stride() != self._stride):
            raise ValueError(
                "paged_decode_fp4_plan.run: the query does not match the validated layout (built for "
                f"shape/dtype/device/strides {self.q_signature}, got "
                f"{(tuple(q.shape), q.dtype, q.device, q.stride())}); build a new plan for a new layout"
            )
        if self._index != _lib._current_device():
            with torch.cuda.device(self._index):
                return self._launch(layer, q)
        return self._launch(layer, q)

    def _launch(self, layer: int, q) -> torch.Tensor:
        out = torch.empty_like(q)
        rc = _lib.lib.mi_paged_decode_fp4(q.data_ptr(), self._k_ptrs[layer], self._v_ptrs[layer], self._table_ptr,
                                          self._seqlen_ptr, out.data_ptr(), *self._frozen,
                                          _lib.current_stream(self._device))
        if rc:
            _lib.check(rc, "paged_decode_fp4_plan.run")
        return out

    def fused_supported(self, dtype: torch.dtype, rotary_dim: int, zero_centred_norm: bool = False) -> bool:
        """No fused epilogue here: a step calls ``Fp4PagedPool.write_qk_norm_rope`` and :meth:`run`."""
        return False


def paged_decode_fp4_plan(q, k_caches, v_caches, block_table, seqlen, *, scale=None) -> Fp4DecodePlan:
    """Check one container's 4-bit decode tensors once and freeze their launch arguments."""
    return Fp4DecodePlan(q, k_caches, v_caches, block_table, seqlen, scale=scale)
