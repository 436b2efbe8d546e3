"""Quantised slot records and attention over them.

Records in the OCP microscaling formats: blocks of 32 elements along head_dim of
one (token, head) with one power-of-two scale; ``mxint8`` holds int8 / 64 (8.25 bits
an element), ``mxfp4`` e2m1 (4.25 bits). A store of such records holds 1.94 or 3.76
times as many chunks as one of 16-bit records, and its file and PCIe transfers, the
slow part of every save and load, are as much shorter.

:func:`gather` / :func:`scatter` and :func:`gather_slots` / :func:`scatter_slots` are
``daser_amd.ops``' functions of the same names for such records: the same tables,
checks and streams, with an :class:`MXFormat`. :func:`attend` is attention over
records where they lie. Layout, rounding and limits: include/daser_kv.h.

The reference keeps records in the cache's own type only
(daser/connector/daser_connector.py:625-632).
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from daser_amd import _lib, ops
from daser_amd.position import _current

FORMATS = {"mxint8": _lib.DSR_MX_INT8, "mxfp4": _lib.DSR_MX_FP4}
_DTYPES = {torch.bfloat16: _lib.DSR_DTYPE_BF16, torch.float16: _lib.DSR_DTYPE_FP16}


@dataclass(frozen=True)
class MXFormat:
    """The records of one set of caches in an MX format."""

    name: str  # "mxint8" or "mxfp4"
    num_layers: int
    block_size: int
    num_heads: int
    head_dim: int

    def __post_init__(self) -> None:
        if self.name not in FORMATS:
            raise ValueError(f"unknown record format {self.name!r}: 'mxint8' or 'mxfp4'")
        n = _lib.lib().dsr_mx_layer_bytes(self.code, self.block_size, self.num_heads,
                                          self.head_dim)
        if n < 0:
            raise ValueError("quantised records need a known block size and heads, a head_dim "
                             f"that is a multiple of 32 and pages under 2 GiB: got {self}")
        object.__setattr__(self, "_layer_bytes", n)

    @staticmethod
    def of(layout: ops.PagedKVLayout, name: str) -> "MXFormat":
        """The format of the records of caches of this layout."""
        if layout.dtype not in _DTYPES:
            raise TypeError(f"quantised records are made from bfloat16 or float16 caches, not "
                            f"{layout.dtype}")
        if layout.k_layout == "kx":
            raise ValueError("quantised records do not support split-x (3-D) caches")
        return MXFormat(name, layout.num_layers, layout.block_size, layout.num_heads,
                        layout.head_dim)

    @property
    def code(self) -> int:
        return FORMATS[self.name]

    @property
    def layer_bytes(self) -> int:
        """Bytes of one layer of a record."""
        return self._layer_bytes

    @property
    def slot_bytes(self) -> int:
        """Bytes of a record: one block over all layers."""
        return self._layer_bytes * self.num_layers


def _check_format(lay: ops.PagedKVLayout, fmt: MXFormat) -> None:
    if (fmt.num_layers, fmt.block_size, fmt.num_heads, fmt.head_dim) != \
            (lay.num_layers, lay.block_size, lay.num_heads, lay.head_dim) or \
            lay.dtype not in _DTYPES or lay.k_layout == "kx":
        MXFormat.of(lay, fmt.name)  # says what such caches lack
        raise ValueError(f"{fmt} is not the format of these caches' records")


def _check_staging(lay: ops.PagedKVLayout, staging: torch.Tensor) -> int:
    if staging.dtype != torch.uint8:
        raise ValueError("quantised records lie in a uint8 tensor")
    return ops._check_staging(lay, staging)


def _args(table: ops.LayerTable, fmt: MXFormat, staging: torch.Tensor, nbytes: int,
          layer0: int) -> _lib.MxArgs:
    lay = table.layout
    return _lib.MxArgs(table.ptr(), lay.kv_stride, lay.page_stride, lay.num_blocks,
                       staging.data_ptr(), nbytes, fmt.layer_bytes, lay.num_layers, layer0,
                       lay.block_size, lay.num_heads, lay.head_dim, _DTYPES[lay.dtype],
                       ops._K_LAYOUTS[lay.k_layout], fmt.code)


def _prepare(table: ops.LayerTable, fmt: MXFormat, staging: torch.Tensor, layer0: int, layers):
    """(first, count, staging bytes) of a call, its format and buffers checked."""
    _check_format(table.layout, fmt)
    if layer0 < 0:
        raise IndexError("layer0 must not be negative")
    first, count = ops._layer_range(table.layout, layers)
    return first, count, _check_staging(table.layout, staging)


def _device_pair(lay, a, b, dtype_a, dtype_b, names):
    """Checked device tables of a call."""
    a = ops._as_device_table(a, dtype_a, lay.device, names[0])
    b = ops._as_device_table(b, dtype_b, lay.device, names[1])
    if a.numel() != b.numel():
        raise ValueError(f"{names[0]} and {names[1]} differ in length")
    return a, b


def _host_pair(a, b, names):
    """Both tables as host vectors, or None if they are on the device."""
    on = ops._on_device(a)
    if on != ops._on_device(b):
        raise ValueError(f"{names[0]} and {names[1]} must both be host data or device tensors")
    if on:
        return None
    a, b = ops._host_list(a), ops._host_list(b)
    if a is None or b is None or a.size != b.size:
        raise ValueError(f"{names[0]} and {names[1]} must be vectors of one length")
    return a, b


def _host_rope(host, rope_idx, name: str) -> Optional[np.ndarray]:
    """rope_idx as a host vector where the other tables are; checked device tables are
    made of it elsewhere."""
    if rope_idx is None:
        return None
    if (host is None) != ops._on_device(rope_idx):
        raise ValueError(f"rope_idx and {name} must both be host data or device tensors")
    if host is None:
        return None
    ridx = ops._host_list(rope_idx)
    if ridx is None or ridx.size != host[0].size:
        raise ValueError(f"rope_idx and {name} differ in length")
    return ridx


_PAGES = ("page_ids", "slot_offsets")
_SLOTS = ("slot_mapping", "record_rows")


class PreparedGather:
    """A save of fixed page tables into fixed records, checked and uploaded once; each
    call launches it for a layer range (see :class:`daser_amd.ops.PreparedGather`)."""

    def __init__(self, table: ops.LayerTable, fmt: MXFormat, page_ids, slot_offsets,
                 staging: torch.Tensor, *, layer0: int = 0,
                 layers: Optional[tuple[int, int]] = None) -> None:
        lay = table.layout
        first, count, nbytes = _prepare(table, fmt, staging, layer0, layers)
        host = _host_pair(page_ids, slot_offsets, _PAGES)
        self._plan = self._tables = None
        if host is None:
            self._tables = _device_pair(lay, page_ids, slot_offsets, torch.int32, torch.int64,
                                        _PAGES)
            self._tail = (self._tables[0].data_ptr(), self._tables[1].data_ptr(),
                          self._tables[0].numel())
        elif not host[0].size:
            self._tail = (None, None, 0)
        else:
            ids, offs = host
            lib, span = _lib.lib(), count * fmt.layer_bytes

            def fill(out: int, size: int, at: int) -> None:
                ops._plan_check("dsr_plan_gather", lib.dsr_plan_gather(
                    ops._addr(ids), ops._addr(offs), ids.size, lay.num_blocks,
                    span + (layer0 + first) * fmt.layer_bytes, span, nbytes, out, size, at),
                    lay.num_blocks)

            self._plan = plan = ops._HostPlan(ids.size, lay.device, fill)
            self._tail = (plan.ids, plan.offsets, ids.size)
        self._keep = (table, staging)
        self._args = _args(table, fmt, staging, nbytes, layer0)
        self._args_ptr = ctypes.addressof(self._args)
        self._range = (first, first + count)
        self._device = lay.device
        self._fn = _lib.lib().dsr_gather_mx

    @property
    def tables(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(page_ids, slot_offsets) as device tensors."""
        if self._tables is None:
            n, dev = self._tail[2], self._device
            self._tables = (torch.empty(0, dtype=torch.int32, device=dev),
                            torch.empty(0, dtype=torch.int64, device=dev)) if not n else (
                self._plan.table(self._plan.plan.off_ids, n, torch.int32),
                self._plan.table(0, n, torch.int64))
        return self._tables

    def __call__(self, first: int, count: int, stream: int) -> None:
        """Saves table layers [first, first + count) on ``stream`` (a HIP stream handle)."""
        if count < 0 or first < self._range[0] or first + count > self._range[1]:
            raise IndexError("layer range outside the registered caches")
        with _current(self._device):
            _lib.check("dsr_gather_mx", self._fn(self._args_ptr, first, count, *self._tail, stream))


def gather(table: ops.LayerTable, fmt: MXFormat, page_ids, slot_offsets, staging: torch.Tensor, *,
           layer0: int = 0, layers: Optional[tuple[int, int]] = None) -> None:
    """Packs pages into quantised slot records (``ops.gather`` for ``fmt``)."""
    save = PreparedGather(table, fmt, page_ids, slot_offsets, staging, layer0=layer0,
                          layers=layers)
    save(save._range[0], save._range[1] - save._range[0],
         ops._stream_handle(table.layout.device))


def _rope(lay: ops.PagedKVLayout, cos_sin, rope_idx, rot_dim, style: str, layer0: int,
          layer_group):
    """(MxRope without its rope_idx, what it points to) or None, checked."""
    if cos_sin is None:
        if rope_idx is not None or layer_group is not None:
            raise ValueError("rope_idx and layer_group need cos_sin")
        return None
    if rope_idx is None:
        raise ValueError("cos_sin needs rope_idx")
    if style not in ops.ROPE_STYLES:
        raise ValueError(f"unknown rope style {style!r}")
    rot_dim, n_tables, n_groups, lg, _ = ops._rope_args(lay, cos_sin, rope_idx, rot_dim, None,
                                                        layer0, layer_group)
    _check_rot_dim(rot_dim, lay.head_dim, style)
    return _lib.MxRope(cos_sin.data_ptr(), None, None if lg is None else lg.data_ptr(), n_tables,
                       n_groups, rot_dim, ops.ROPE_STYLES[style]), (cos_sin, lg)


def _check_rot_dim(rot_dim: int, head_dim: int, style: str) -> None:
    step = 16 if style == "neox" else 8
    if rot_dim <= 0 or rot_dim > head_dim or rot_dim % step:
        raise ValueError(f"quantised records rotate widths of a multiple of {step} elements up "
                         f"to head_dim ({style}): got {rot_dim}")


def scatter(table: ops.LayerTable, fmt: MXFormat, page_ids, slot_offsets, staging: torch.Tensor,
            cos_sin: Optional[torch.Tensor] = None, rope_idx=None, *,
            rot_dim: Optional[int] = None, style: str = "neox", layer0: int = 0,
            layers: Optional[tuple[int, int]] = None, layer_group=None) -> None:
    """Unpacks quantised records into pages (``ops.scatter``) and, with ``cos_sin`` and
    ``rope_idx``, re-rotates K on the way (``ops.scatter_rerotate``): a row is decoded,
    rotated in fp32 and rounded to the cache's type once."""
    lay = table.layout
    first, count, nbytes = _prepare(table, fmt, staging, layer0, layers)
    host = _host_pair(page_ids, slot_offsets, _PAGES)
    ridx = _host_rope(host, rope_idx, "page_ids")
    n = page_ids.numel() if host is None else host[0].size
    rope = _rope(lay, cos_sin, rope_idx, rot_dim, style, layer0, layer_group)
    if not n:
        return
    keep, r = None, None if rope is None else rope[0]
    if host is not None:
        lib = _lib.lib()

        def fill(out: int, size: int, at: int) -> None:
            ops._plan_check("dsr_plan_load", lib.dsr_plan_load(
                ops._addr(host[0]), ops._addr(host[1]), ops._addr(ridx), n, lay.num_blocks,
                (layer0 + first + count) * fmt.layer_bytes, nbytes, 0 if r is None else r.n_tables,
                0, out, size, at), lay.num_blocks)

        keep = ops._HostPlan(n, lay.device, fill)
        tables = (keep.ids, keep.offsets, keep.plan.n_pages)
        if r is not None:
            r.rope_idx = keep.rope
    else:
        keep = [*_device_pair(lay, page_ids, slot_offsets, torch.int32, torch.int64, _PAGES)]
        tables = (keep[0].data_ptr(), keep[1].data_ptr(), n)
        if r is not None:
            keep.append(ops._as_device_table(rope_idx, torch.int32, lay.device, "rope_idx"))
            if keep[2].numel() != n:
                raise ValueError("rope_idx and page_ids differ in length")
            r.rope_idx = keep[2].data_ptr()
    args = _args(table, fmt, staging, nbytes, layer0)
    with _current(lay.device):
        _lib.check("dsr_scatter_mx", _lib.lib().dsr_scatter_mx(
            ctypes.addressof(args), first, count, *tables,
            None if r is None else ctypes.addressof(r), ops._stream_handle(lay.device)))


def record_rows(req_tokens: Sequence[int], fmt: MXFormat, base: int = 0) -> np.ndarray:
    """The record row of each token for requests whose records are packed back to back
    from ``base``: token t of a request lies in its record t // block_size at row t %
    block_size, and a row is named record offset * block_size + row."""
    return np.concatenate([np.zeros(0, np.int64)] + [
        (first + t // fmt.block_size * fmt.slot_bytes) * fmt.block_size + t % fmt.block_size
        for first, t in _requests(req_tokens, fmt, base)])


def _requests(req_tokens, fmt: MXFormat, base: int):
    for n in req_tokens:
        yield base, np.arange(int(n), dtype=np.int64)
        base += -(-int(n) // fmt.block_size) * fmt.slot_bytes


def _slot_tables(lay, fmt: MXFormat, slot_mapping, record_rows, rope_idx, n_tables: int,
                 nbytes: int, last: int, written: bool):
    """Addresses of a token-form call's device tables (slots, rows, rope) with the number of
    tokens, and what holds them. Host tables are planned by the library: of a record row
    (``written``) or cache slot listed more than once the last entry stays, as sequential
    copies would leave it."""
    host = _host_pair(slot_mapping, record_rows, _SLOTS)
    ridx = _host_rope(host, rope_idx, "slot_mapping")
    if host is None:
        tables = [*_device_pair(lay, slot_mapping, record_rows, torch.int64, torch.int64, _SLOTS)]
        if rope_idx is not None:
            tables.append(ops._as_device_table(rope_idx, torch.int32, lay.device, "rope_idx"))
        if any(t.numel() != tables[0].numel() for t in tables):
            raise ValueError("rope_idx and slot_mapping differ in length")
        at = [t.data_ptr() for t in tables] + [None]
        return (at[0], at[1], at[2], tables[0].numel()), tables
    slots, rows = host
    if not slots.size:
        return (None, None, None, 0), None
    lib = _lib.lib()

    def fill(out: int, size: int, at: int) -> None:
        ops._plan_check("dsr_plan_slots_mx", lib.dsr_plan_slots_mx(
            ops._addr(slots), ops._addr(rows), ops._addr(ridx), slots.size, lay.num_blocks,
            lay.block_size, last, nbytes, n_tables, int(written), out, size, at), lay.num_blocks)

    plan = ops._HostPlan(slots.size, lay.device, fill)
    return (plan.offsets, plan.ids, plan.rope, plan.plan.n_pages), plan


def gather_slots(table: ops.LayerTable, fmt: MXFormat, slot_mapping, record_rows,
                 staging: torch.Tensor, *, layer0: int = 0,
                 layers: Optional[tuple[int, int]] = None) -> None:
    """Token-granular save (``ops.gather_slots`` for ``fmt``): each valid token's K and V
    rows (slot -1: padding) go to its record row (see :func:`record_rows`); the record's
    other rows stay as they are."""
    lay = table.layout
    first, count, nbytes = _prepare(table, fmt, staging, layer0, layers)
    (slots, rows, _, n), _keep = _slot_tables(
        lay, fmt, slot_mapping, record_rows, None, 0, nbytes,
        (layer0 + first + count) * fmt.layer_bytes, True)
    args = _args(table, fmt, staging, nbytes, layer0)
    with _current(lay.device):
        _lib.check("dsr_gather_slots_mx", _lib.lib().dsr_gather_slots_mx(
            ctypes.addressof(args), first, count, slots, rows, n,
            ops._stream_handle(lay.device)))


def scatter_slots(table: ops.LayerTable, fmt: MXFormat, slot_mapping, record_rows,
                  staging: torch.Tensor, cos_sin: Optional[torch.Tensor] = None, rope_idx=None, *,
                  rot_dim: Optional[int] = None, style: str = "neox", layer0: int = 0,
                  layers: Optional[tuple[int, int]] = None, layer_group=None) -> None:
    """Inverse of :func:`gather_slots`; with ``cos_sin`` and ``rope_idx`` (per token, -1:
    not) K is re-rotated as :func:`scatter` does."""
    lay = table.layout
    first, count, nbytes = _prepare(table, fmt, staging, layer0, layers)
    rope = _rope(lay, cos_sin, rope_idx, rot_dim, style, layer0, layer_group)
    r = None if rope is None else rope[0]
    (slots, rows, ridx, n), _keep = _slot_tables(
        lay, fmt, slot_mapping, record_rows, rope_idx, 0 if r is None else r.n_tables, nbytes,
        (layer0 + first + count) * fmt.layer_bytes, False)
    if not n:
        return
    if r is not None:
        r.rope_idx = ridx
    args = _args(table, fmt, staging, nbytes, layer0)
    with _current(lay.device):
        _lib.check("dsr_scatter_slots_mx", _lib.lib().dsr_scatter_slots_mx(
            ctypes.addressof(args), first, count, slots, rows, n, None if r is None else ctypes.addressof(r),
            ops._stream_handle(lay.device)))


def _vector(x, dtype: torch.dtype, device: torch.device, name: str, size: Optional[int] = None):
    if isinstance(x, torch.Tensor) and x.dtype == dtype and x.device == device and \
            x.dim() == 1 and x.is_contiguous() and (size is None or x.shape[0] == size):
        return x
    if ops._on_device(x) and x.device != device:
        raise ValueError(f"{name} must live on q's device")
    t = ops._as_device_table(x, dtype, device, name)
    if t.dim() != 1 or (size is not None and t.numel() != size):
        raise ValueError(f"{name} must be a vector" + (f" of {size}" if size is not None else ""))
    return t


def _check_host_tables(fmt, q, staging, q_start, page_start, slot_offsets, context, last):
    """Errors of the attention's tables, as far as they are on the host."""
    def starts(x, n, name):
        a = ops._host_list(x)
        if a is not None and a.size and (a[0] < 0 or (np.diff(a) < 0).any() or a[-1] > n):
            raise IndexError(f"{name} must not decrease and stay in [0, {n}]")
        return a

    n_pages = slot_offsets.numel() if ops._on_device(slot_offsets) else np.size(slot_offsets)
    starts(q_start, q.shape[0], "q_start")
    ps = starts(page_start, n_pages, "page_start")
    offs = ops._host_list(slot_offsets)
    if offs is not None and offs.size:
        if offs.min() < 0 or offs.max() + last > staging.numel():
            raise IndexError("slot record outside the staging buffer")
        if (offs % 16).any():
            raise ValueError("slot offsets must be multiples of 16 bytes")
    ctx = ops._host_list(context)
    if ctx is not None and ctx.size:
        if ctx.min() < 0:
            raise IndexError("context must not be negative")
        if ps is not None and ps.size == ctx.size + 1 and \
                (ctx > np.diff(ps) * fmt.block_size).any():
            raise IndexError("context reaches past its request's pages")


def attend(q: torch.Tensor, fmt: MXFormat, staging: torch.Tensor, q_start, page_start,
           slot_offsets, context, *, layer: int, scale: Optional[float] = None,
           max_queries: Optional[int] = None, max_context: Optional[int] = None, limits=None,
           cos_sin: Optional[torch.Tensor] = None, rope_idx=None, rot_dim: Optional[int] = None,
           style: str = "neox", prior: Optional[tuple[torch.Tensor, torch.Tensor]] = None,
           out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of ``q`` [n, q_heads, head_dim] over records, in place of a load.

    Request r's queries are rows ``q_start[r]`` to ``q_start[r + 1] - 1``; its tokens lie
    in order in the records ``slot_offsets[page_start[r]:page_start[r + 1]]``, block_size
    to each, ``context[r]`` of them. Query i sees the first ``limits[i]`` of them (None:
    all). Returns (out [n, q_heads, head_dim] of q's type, lse float32 [n, q_heads]:
    the natural logarithm of the sum of exponentials); a query that sees no token gets
    zeros and -inf. ``scale`` defaults to head_dim ** -0.5.

    ``rope_idx[page]`` names the table of ``cos_sin`` [n_tables, rot_dim / 2, 2] by which
    the page's K is moved (-1: not), as for :func:`scatter`: a layer's own tables where
    layers differ. ``prior`` = (out, lse) is the same queries' attention over other keys
    (the request's own pages, say); the result is then over both sets.

    Tables may be host data, checked here, or device tensors, used as they are.
    ``max_queries`` / ``max_context`` are the largest request's, for the launch's
    shape; None: from host tables, or bounds that hold for any. Results are right
    whatever they say; how the tokens are split, and so the last bit of a sum, follows
    them. Rows of ``out`` that belong to no request are left as they were, and their
    lse is not set."""
    if q.dim() != 3 or q.dtype not in _DTYPES:
        raise ValueError("q must be bfloat16 or float16 [n, q_heads, head_dim]")
    n, heads, dim = q.shape
    if dim != fmt.head_dim or heads % fmt.num_heads or not heads:
        raise ValueError(f"q of {heads} heads of {dim} does not fit {fmt}")
    if dim not in (32, 64, 96, 128, 256) or fmt.block_size % 16:
        raise ValueError("attention over records needs a head_dim of 32, 64, 96, 128 or 256 and "
                         "blocks of a multiple of 16 tokens")
    if q.numel() and (q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or
                      q.data_ptr() % 16):
        raise ValueError("q's rows of head_dim must be contiguous and 16-byte aligned")
    if staging.device != q.device or staging.dtype != torch.uint8 or not staging.is_contiguous():
        raise ValueError("staging must be a contiguous uint8 tensor on q's device")
    if not 0 <= layer < fmt.num_layers:
        raise IndexError("layer outside the records")
    dev = q.device
    tables = (q_start, page_start, slot_offsets, context)
    if not all(isinstance(x, torch.Tensor) and x.is_cuda for x in tables):
        _check_host_tables(fmt, q, staging, *tables, (layer + 1) * fmt.layer_bytes)
    if not q.is_cuda:
        raise ValueError("q must live on a GPU")
    if max_queries is None:
        h = ops._host_list(q_start)
        max_queries = n if h is None else int(np.diff(h).max(initial=0))
    ctx_host = ops._host_list(context)
    qs = _vector(q_start, torch.int32, dev, "q_start")
    n_req = qs.numel() - 1
    if n_req < 0:
        raise ValueError("q_start holds one entry more than there are requests")
    ps = _vector(page_start, torch.int32, dev, "page_start", n_req + 1)
    offs = _vector(slot_offsets, torch.int64, dev, "slot_offsets")
    ctx = _vector(context, torch.int32, dev, "context", n_req)
    if max_context is None:
        max_context = offs.numel() * fmt.block_size if ctx_host is None else \
            int(ctx_host.max(initial=0))
    lim = None if limits is None else _vector(limits, torch.int32, dev, "limits", n)
    ridx = None
    if cos_sin is not None:
        if rope_idx is None:
            raise ValueError("cos_sin needs rope_idx")
        if style not in ops.ROPE_STYLES:
            raise ValueError(f"unknown rope style {style!r}")
        rot_dim = dim if rot_dim is None else rot_dim
        _check_rot_dim(rot_dim, dim, style)
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 3 or cos_sin.device != dev or \
                cos_sin.shape[1:] != (rot_dim // 2, 2) or not cos_sin.is_contiguous():
            raise ValueError(f"cos_sin must be contiguous float32 [n, {rot_dim // 2}, 2] on q's "
                             "device")
        host = ops._host_list(rope_idx)
        if host is not None and host.size and (host.max() >= len(cos_sin) or host.min() < -1):
            raise IndexError("rope_idx outside [-1, n_tables)")
        ridx = _vector(rope_idx, torch.int32, dev, "rope_idx", offs.numel())
    elif rope_idx is not None:
        raise ValueError("rope_idx needs cos_sin")
    if prior is not None:
        po, pl = prior
        if po.shape != q.shape or po.dtype != q.dtype or po.device != dev or \
                not po.is_contiguous() or pl.shape != (n, heads) or pl.device != dev or \
                pl.dtype != torch.float32 or not pl.is_contiguous():
            raise ValueError("prior must be contiguous (out, lse) as attend returns them")
    if out is None:
        out = torch.empty((n, heads, dim), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or \
            not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, type and device")
    lse = torch.empty((n, heads), dtype=torch.float32, device=dev)
    a = _lib.AttendArgs(
        q.data_ptr(), 2 * q.stride(0), 2 * q.stride(1), out.data_ptr(), lse.data_ptr(),
        None if prior is None else prior[0].data_ptr(),
        None if prior is None else prior[1].data_ptr(), qs.data_ptr(), ps.data_ptr(),
        offs.data_ptr(), ctx.data_ptr(), None if lim is None else lim.data_ptr(),
        None if ridx is None else ridx.data_ptr(),
        None if cos_sin is None else cos_sin.data_ptr(), staging.data_ptr(), staging.numel(),
        fmt.layer_bytes, None, 0, dim ** -0.5 if scale is None else float(scale), n_req, n,
        offs.numel(), max_queries, max_context, heads, fmt.num_heads, dim, fmt.block_size, layer,
        0 if cos_sin is None else len(cos_sin), rot_dim or 0, ops.ROPE_STYLES.get(style, 0),
        _DTYPES[q.dtype], fmt.code)
    at = ctypes.addressof(a)
    with _current(dev):
        need = _lib.lib().dsr_attend_workspace(at)
        if need > 0:
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = work.data_ptr(), need
        _lib.check("dsr_attend_mx", _lib.lib().dsr_attend_mx(at, ops._stream_handle(dev)))
    return out, lse
