"""Quantised records: format arithmetic, tables and refusals, without a GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from daser_amd import _lib, mx, ops
from tests import mx_reference as ref


def caches(layers=2, blocks=4, bs=16, heads=2, dim=64, dtype=torch.bfloat16):
    return [torch.zeros(2, blocks, bs, heads, dim, dtype=dtype) for _ in range(layers)]


@pytest.mark.parametrize("name", ["mxint8", "mxfp4"])
@pytest.mark.parametrize("bs,heads,dim", [(16, 8, 128), (1, 1, 32), (16, 2, 64), (7, 3, 96)])
def test_format_sizes(name, bs, heads, dim):
    fmt = mx.MXFormat(name, 3, bs, heads, dim)
    codes, scales = ref.sections(fmt)
    assert fmt.layer_bytes == 2 * (codes + scales) and fmt.layer_bytes % 16 == 0
    assert fmt.slot_bytes == 3 * fmt.layer_bytes


def test_store_ratio():
    lay = ops.PagedKVLayout.from_caches(caches(heads=8, dim=128))
    assert lay.slot_bytes / mx.MXFormat.of(lay, "mxint8").slot_bytes == pytest.approx(64 / 33)
    assert lay.slot_bytes / mx.MXFormat.of(lay, "mxfp4").slot_bytes == pytest.approx(64 / 17)


def test_format_refusals():
    with pytest.raises(ValueError, match="unknown record format"):
        mx.MXFormat("int4", 1, 16, 8, 128)
    for bad in ((0, 8, 128), (16, 0, 128), (16, 8, 80), (16, 8, 0), (1 << 16, 1 << 8, 128)):
        with pytest.raises(ValueError, match="multiple of 32"):
            mx.MXFormat("mxfp4", 1, *bad)
    lay = ops.PagedKVLayout.from_caches(caches(dtype=torch.float8_e4m3fn))
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        mx.MXFormat.of(lay, "mxint8")
    flat = [torch.zeros(2, 4, 16 * 2 * 64, dtype=torch.bfloat16)]
    lay = ops.PagedKVLayout.from_caches(flat, block_size=16, head_dim=64)
    with pytest.raises(ValueError, match="split-x"):
        mx.MXFormat.of(lay, "mxint8")


def test_record_rows():
    fmt = mx.MXFormat("mxfp4", 2, 16, 2, 64)
    rows = mx.record_rows([17, 0, 3], fmt, base=32)
    want = [(32 + t // 16 * fmt.slot_bytes) * 16 + t % 16 for t in range(17)] + \
        [(32 + 2 * fmt.slot_bytes) * 16 + t for t in range(3)]
    assert rows.tolist() == want
    assert mx.record_rows([], fmt).size == 0


def test_reference_rounding_is_half_a_step():
    """The plain statement itself: no element is off by more than half a step of the
    scale that the format's largest value allows, and ties go to even."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 32)) * 10.0 ** rng.integers(-6, 6, (500, 1))
    for name, step in (("mxint8", 1 / 64), ("mxfp4", 2.0)):
        q, s = ref.quantise(x, name)
        scale = 2.0 ** (s - 127.0)
        assert (np.abs(ref.dequantise(q, s, name) - x) <= step / 2 * scale).all()
        a = np.abs(x).max(-1, keepdims=True)
        assert (a > (127.5 / 64 if name == "mxint8" else 7.0) * scale / 2).all()
    mid = (ref.E2M1[1:] + ref.E2M1[:-1]) / 2
    assert ref.nearest_even(mid, "mxfp4").tolist() == [0, 2, 2, 4, 4, 6, 6]


@pytest.mark.parametrize("fn", [mx.gather, mx.scatter])
def test_page_form_refusals(fn):
    kv = caches()
    table = ops.LayerTable(kv)
    fmt = mx.MXFormat.of(table.layout, "mxfp4")
    rec = torch.zeros(4 * fmt.slot_bytes, dtype=torch.uint8)
    with pytest.raises(ValueError, match="not the format"):
        fn(table, mx.MXFormat("mxfp4", 3, 16, 2, 64), [0], [0], rec)
    with pytest.raises(ValueError, match="uint8"):
        fn(table, fmt, [0], [0], rec.view(torch.int16))
    with pytest.raises(ValueError, match="contiguous"):
        fn(table, fmt, [0], [0], torch.zeros(2 * fmt.slot_bytes, 2, dtype=torch.uint8).T[0])
    with pytest.raises(IndexError, match="block id"):
        fn(table, fmt, [4], [0], rec)
    with pytest.raises(IndexError, match="outside the staging"):
        fn(table, fmt, [0], [4 * fmt.slot_bytes], rec)
    with pytest.raises(IndexError, match="outside the staging"):
        fn(table, fmt, [0], [3 * fmt.slot_bytes + 16], rec)
    with pytest.raises(ValueError, match="multiples of 16"):
        fn(table, fmt, [0], [8], rec)
    with pytest.raises(ValueError, match="one length"):
        fn(table, fmt, [0, 1], [0], rec)
    with pytest.raises(IndexError, match="layer range"):
        fn(table, fmt, [0], [0], rec, layers=(1, 2))
    with pytest.raises(IndexError, match="layer0"):
        fn(table, fmt, [0], [0], rec, layer0=-1)
    if fn is mx.gather:
        with pytest.raises(ValueError, match="overlap"):
            fn(table, fmt, [0, 1], [0, 16], rec)


def test_rope_refusals():
    table = ops.LayerTable(caches())
    fmt = mx.MXFormat.of(table.layout, "mxint8")
    rec = torch.zeros(fmt.slot_bytes, dtype=torch.uint8)
    cs = torch.zeros(1, 32, 2)
    for kw, err, text in (
            (dict(cos_sin=cs), ValueError, "needs rope_idx"),
            (dict(rope_idx=[0]), ValueError, "need cos_sin"),
            (dict(cos_sin=cs, rope_idx=[0, 0]), ValueError, "differ in length"),
            (dict(cos_sin=cs, rope_idx=[1]), IndexError, "rope_idx outside"),
            (dict(cos_sin=cs, rope_idx=[0], style="glm"), ValueError, "style"),
            (dict(cos_sin=cs[:, :12].contiguous(), rope_idx=[0], rot_dim=24), ValueError,
             "multiple of 16"),
            (dict(cos_sin=cs[:, :16].contiguous(), rope_idx=[0]), ValueError, "cos_sin must be"),
            (dict(cos_sin=cs, rope_idx=[0], layer_group=[0]), ValueError, "cos_sin must be")):
        with pytest.raises(err, match=text):
            mx.scatter(table, fmt, [0], [0], rec, **kw)


@pytest.mark.parametrize("fn", [mx.gather_slots, mx.scatter_slots])
def test_token_form_refusals(fn):
    table = ops.LayerTable(caches())
    fmt = mx.MXFormat.of(table.layout, "mxfp4")
    rec = torch.zeros(2 * fmt.slot_bytes, dtype=torch.uint8)
    row = lambda off, t: off * 16 + t  # noqa: E731
    with pytest.raises(IndexError, match="slot outside"):
        fn(table, fmt, [64], [0], rec)
    with pytest.raises(IndexError, match="outside the staging"):
        fn(table, fmt, [0], [row(2 * fmt.slot_bytes, 0)], rec)
    with pytest.raises(IndexError, match="outside the staging"):
        fn(table, fmt, [0], [-1], rec)
    with pytest.raises(ValueError, match="multiples of 16"):
        fn(table, fmt, [0], [row(8, 0)], rec)
    with pytest.raises(ValueError, match="one length"):
        fn(table, fmt, [0, 1], [0], rec)


class OnDevice(torch.Tensor):
    """A tensor that says it is not in host memory."""

    is_cpu = False


def test_tables_are_of_one_kind():
    """Host tables are checked and ordered, device tables used as they are: not both in
    one call."""
    table = ops.LayerTable(caches())
    fmt = mx.MXFormat.of(table.layout, "mxint8")
    rec = torch.zeros(fmt.slot_bytes, dtype=torch.uint8)
    there = torch.zeros(1, dtype=torch.int64).as_subclass(OnDevice)
    for fn in (mx.gather, mx.scatter, mx.gather_slots, mx.scatter_slots):
        with pytest.raises(ValueError, match="both be host data"):
            fn(table, fmt, [0], there, rec)
        with pytest.raises(ValueError, match="both be host data"):
            fn(table, fmt, there, [0], rec)
    cs = torch.zeros(1, 32, 2)
    for fn in (mx.scatter, mx.scatter_slots):
        with pytest.raises(ValueError, match="both be host data"):
            fn(table, fmt, [0], [0], rec, cs, there.int())


def attend_args(**kw):
    fmt = mx.MXFormat("mxfp4", 2, 16, 2, 64)
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), fmt=fmt,
             staging=torch.zeros(4 * fmt.slot_bytes, dtype=torch.uint8), q_start=[0, 1, 3],
             page_start=[0, 2, 3], slot_offsets=[0, fmt.slot_bytes, 2 * fmt.slot_bytes],
             context=[20, 16], layer=1)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "live on a GPU"),
    (dict(q=torch.zeros(3, 4, 64)), ValueError, "bfloat16 or float16"),
    (dict(q=torch.zeros(3, 3, 64, dtype=torch.float16)), ValueError, "does not fit"),
    (dict(q=torch.zeros(3, 4, 32, dtype=torch.float16)), ValueError, "does not fit"),
    (dict(q=torch.zeros(3, 64, 4, dtype=torch.float16).transpose(1, 2)), ValueError,
     "contiguous"),
    (dict(fmt=mx.MXFormat("mxfp4", 2, 8, 2, 64)), ValueError, "multiple of 16 tokens"),
    (dict(layer=2), IndexError, "layer"),
    (dict(layer=-1), IndexError, "layer"),
    (dict(q_start=[0, 2, 1]), IndexError, "q_start"),
    (dict(q_start=[0, 1, 4]), IndexError, "q_start"),
    (dict(page_start=[0, 2, 4]), IndexError, "page_start"),
    (dict(slot_offsets=[0, 8, 16]), ValueError, "multiples of 16"),
    (dict(slot_offsets=[0, 16, 1 << 30]), IndexError, "outside the staging"),
    (dict(context=[33, 16]), IndexError, "past its request"),
    (dict(context=[-1, 16]), IndexError, "negative"),
    (dict(staging=torch.zeros(64, dtype=torch.int32)), ValueError, "uint8"),
])
def test_attend_refusals(kw, err, text):
    with pytest.raises(err, match=text):
        mx.attend(**attend_args(**kw))


def c_attend(**kw):
    a = dict(q=16, q_row_stride=512, q_head_stride=128, out=16, lse=16, q_start=16, page_start=16,
             slot_offsets=16, context=16, staging=16, staging_bytes=1 << 20,
             layer_bytes=1 << 14, workspace=16, workspace_bytes=1 << 40, scale=1.0, n_req=1,
             n_q=1, n_pages=1, max_queries=1, max_context=16, q_heads=4, kv_heads=2, head_dim=64,
             block_size=16, format=1)
    a.update(kw)
    s = _lib.AttendArgs(**a)
    return _lib.lib().dsr_attend_mx(ctypes.addressof(s), None)


def test_c_attend_refusals():
    lib = _lib.lib()
    assert lib.dsr_attend_mx(None, None) == _lib.DSR_ERR_ARG
    assert c_attend(n_q=0) == _lib.DSR_OK and c_attend(n_req=0) == _lib.DSR_OK
    for kw in (dict(n_req=-1), dict(n_pages=-1), dict(layer=-1), dict(format=2), dict(dtype=2),
               dict(q=None), dict(lse=None), dict(slot_offsets=None), dict(prior_out=16),
               dict(rope_idx=16, rot_dim=64, n_tables=1), dict(rope_idx=16, rot_dim=64, style=3)):
        assert c_attend(**kw) == _lib.DSR_ERR_ARG, kw
    for kw in (dict(head_dim=80), dict(head_dim=160), dict(block_size=24), dict(q_heads=3),
               dict(q_heads=0), dict(layer_bytes=1024), dict(rope_idx=16, rot_dim=24),
               dict(rope_idx=16, rot_dim=128), dict(kv_heads=0)):
        assert c_attend(**kw) == _lib.DSR_ERR_SHAPE, kw
    for kw in (dict(q=24), dict(q_row_stride=8), dict(out=8), dict(staging=8),
               dict(layer_bytes=16392)):
        assert c_attend(**kw) == _lib.DSR_ERR_ALIGN, kw


def c_pages(first=0, count=1, n=1, ids=16, offs=16, rope=None, fn="dsr_scatter_mx", **kw):
    a = dict(layer_base=16, kv_stride=4096, page_stride=4096, num_blocks=4, staging=16,
             staging_bytes=1 << 20, layer_bytes=1 << 14, n_layers=2, block_size=16, num_heads=2,
             head_dim=64, format=0)
    a.update(kw)
    s = _lib.MxArgs(**a)
    r = [] if "gather" in fn else [None if rope is None else ctypes.addressof(rope)]
    return getattr(_lib.lib(), fn)(ctypes.addressof(s), first, count, ids, offs, n, *r, None)


@pytest.mark.parametrize("fn", ["dsr_gather_mx", "dsr_scatter_mx", "dsr_gather_slots_mx",
                                "dsr_scatter_slots_mx"])
def test_c_page_and_token_refusals(fn):
    assert c_pages(fn=fn, n=0) == _lib.DSR_OK and c_pages(fn=fn, count=0) == _lib.DSR_OK
    for kw in (dict(n=-1), dict(first=-1), dict(first=2), dict(count=3), dict(ids=None),
               dict(offs=None), dict(format=5), dict(dtype=2), dict(k_layout=9), dict(layer0=-1),
               dict(staging=None), dict(layer_base=None)):
        assert c_pages(fn=fn, **kw) == _lib.DSR_ERR_ARG, kw
    for kw in (dict(k_layout=1), dict(head_dim=40), dict(block_size=0), dict(layer_bytes=64)):
        assert c_pages(fn=fn, **kw) == _lib.DSR_ERR_SHAPE, kw
    for kw in (dict(kv_stride=4100), dict(page_stride=8), dict(staging=24),
               dict(layer_bytes=16392)):
        assert c_pages(fn=fn, **kw) == _lib.DSR_ERR_ALIGN, kw


def test_c_rope_refusals():
    rope = lambda **kw: _lib.MxRope(**{**dict(cos_sin=16, rope_idx=16, n_tables=1,  # noqa: E731
                                              rot_dim=64), **kw})
    for fn in ("dsr_scatter_mx", "dsr_scatter_slots_mx"):
        for kw in (dict(rope_idx=None), dict(cos_sin=None), dict(style=2), dict(n_tables=-1),
                   dict(layer_group=16)):
            assert c_pages(fn=fn, rope=rope(**kw)) == _lib.DSR_ERR_ARG, kw
        for kw in (dict(rot_dim=24), dict(rot_dim=0), dict(rot_dim=128),
                   dict(style=1, rot_dim=20)):
            assert c_pages(fn=fn, rope=rope(**kw)) == _lib.DSR_ERR_SHAPE, kw
