"""Quantised records on the GPU against their plain statement in 64 bits: codes byte for
byte, values read back bit for bit, rotated K within its rounding."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from daser_amd import mx, ops, position
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

FORMATS = ["mxint8", "mxfp4"]
DTYPES = ["bf16", "fp16"]
THETA = 10000.0


def make_caches(dev, dt, layout, layers, blocks, bs, heads, dim, seed, block_major=False):
    """Caches [2, NB, bs, H, D] in token- or head-major pages, with rows from quiet to loud,
    zeros, and a few blocks that hold infinities or NaN."""
    g = torch.Generator().manual_seed(seed)
    shape = (2, blocks, heads, bs, dim) if layout == "hnd" else (2, blocks, bs, heads, dim)
    out = []
    for _ in range(layers):
        x = torch.randn(shape, generator=g, dtype=torch.float64)
        x *= 10.0 ** torch.randint(-4, 4, (*shape[:-1], 1), generator=g)
        x[..., :1] *= 20
        x.view(-1, 32)[::7] = 0
        x = x.to(ref.TORCH[dt])
        x.view(-1)[::997] = float("inf")
        x.view(-1)[::1409] = float("nan")
        if block_major:
            x = x.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
        else:
            x = x.to(dev)
        out.append(x.transpose(2, 3) if layout == "hnd" else x)
    return out


def pages64(cache, half, block):
    """A page as [H, bs, D] float64 on the host."""
    return cache[half, block].transpose(0, 1).double().cpu().numpy()


def want_layer(fmt, cache, block):
    out = np.zeros(fmt.layer_bytes, np.uint8)
    ref.pack(fmt, pages64(cache, 0, block), pages64(cache, 1, block), out)
    return out


def same_bits(got: torch.Tensor, want: np.ndarray, dt: str):
    """got holds want (float64 values of the type, NaN as the canonical one)."""
    w = torch.from_numpy(np.ascontiguousarray(want)).float().to(ref.TORCH[dt])
    w = w.view(torch.int16)
    nan = torch.from_numpy(np.isnan(want))
    w[nan] = 0x7FC0 if dt == "bf16" else 0x7E00
    got = got.cpu().contiguous().view(torch.int16)
    assert torch.equal(got, w), (got != w).nonzero()[:5]


SHAPES = [  # layout, layers, bs, heads, dim, pages, block_major
    ("nhd", 3, 16, 8, 128, 9, False),
    ("nhd", 2, 16, 2, 64, 5, True),
    ("hnd", 2, 16, 4, 128, 7, False),
    ("nhd", 2, 5, 3, 96, 6, False),
    ("nhd", 1, 1, 1, 32, 3, False),
    ("hnd", 2, 32, 3, 256, 4, False),
    ("nhd", 2, 128, 1, 160, 3, False),
]


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_pages_round_trip(gpu, name, dt, shape):
    layout, layers, bs, heads, dim, pages, block_major = shape
    blocks = pages + 3
    src = make_caches(gpu, dt, layout, layers, blocks, bs, heads, dim, 1, block_major)
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, name)
    rng = np.random.default_rng(0)
    ids = rng.permutation(blocks)[:pages].astype(np.int32)
    offs = rng.permutation(pages + 2)[:pages].astype(np.int64) * fmt.slot_bytes + 32
    rec = torch.full((32 + (pages + 2) * fmt.slot_bytes,), 0xA5, dtype=torch.uint8, device=gpu)
    mx.gather(table, fmt, ids, offs, rec)
    host = rec.cpu().numpy()
    want = np.full_like(host, 0xA5)
    codes, scales = ref.sections(fmt)
    for b, o in zip(ids, offs):
        for l in range(layers):
            at = o + l * fmt.layer_bytes
            want[at:at + fmt.layer_bytes] = want_layer(fmt, src[l], b)
            # padding of the sections is not written
            elems = bs * heads * dim
            used = elems // (2 if name == "mxfp4" else 1)
            for lo, hi in ((at + used, at + codes), (at + codes + used, at + 2 * codes),
                           (at + 2 * codes + elems // 32, at + 2 * codes + scales),
                           (at + 2 * codes + scales + elems // 32, at + fmt.layer_bytes)):
                want[lo:hi] = 0xA5
    assert np.array_equal(host, want), np.nonzero(host != want)[0][:8]
    # and back, into caches that hold something else
    dst = make_caches(gpu, dt, layout, layers, blocks, bs, heads, dim, 2, block_major)
    before = [d.clone() for d in dst]
    mx.scatter(ops.LayerTable(dst), fmt, ids, offs, rec)
    for l in range(layers):
        others = [b for b in range(blocks) if b not in set(ids.tolist())]
        assert torch.equal(dst[l][:, others].view(torch.int16),
                           before[l][:, others].view(torch.int16))
        for b, o in zip(ids, offs):
            at = o + l * fmt.layer_bytes
            for half in (0, 1):
                v = ref.unpack(fmt, host[at:at + fmt.layer_bytes], half)
                same_bits(dst[l][half, b].transpose(0, 1), ref.in_type(v, dt), dt)


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("dt", DTYPES)
def test_every_value_of_the_type(gpu, name, dt):
    """All 65,536 bit patterns, each in blocks led by magnitudes of its own binade and by
    ones up to 9 binades above: every rounding, tie, clip and subnormal."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    rows = []
    for up in range(0, 10):
        x = bits.view(ref.TORCH[dt])
        lead = (x.double().abs() * 2.0 ** up * 1.37).clamp(max=ref.TOP[dt])
        lead = torch.where(torch.isfinite(x), lead, torch.ones_like(lead))
        # a leader, fractions of the pattern, and the pattern
        block = torch.zeros(1 << 16, 32, dtype=ref.TORCH[dt])
        block[:, 0] = lead.to(ref.TORCH[dt])
        for j in range(1, 8):
            block[:, j] = (x.double() * (1 - j / 9)).to(ref.TORCH[dt])
        block[:, 17] = x
        rows.append(block)
    x = torch.cat(rows).view(1, -1, 16, 1, 32)
    src = torch.cat([x, -x]).to(gpu)
    table = ops.LayerTable([src])
    fmt = mx.MXFormat.of(table.layout, name)
    n = src.shape[1]
    rec = torch.zeros(n * fmt.slot_bytes, dtype=torch.uint8, device=gpu)
    offs = np.arange(n, dtype=np.int64) * fmt.slot_bytes
    mx.gather(table, fmt, np.arange(n), offs, rec)
    host = rec.cpu().numpy().reshape(n, -1)
    nc, ns = ref.sections(fmt)
    for half in (0, 1):
        q, s = ref.quantise(src[half].double().cpu().numpy().reshape(n, 16, 32), name)
        want = np.zeros((n, fmt.layer_bytes), np.uint8)
        c = q.reshape(n, -1)
        c = c[:, 0::2] | (c[:, 1::2] << 4) if name == "mxfp4" else c
        assert np.array_equal(host[:, 2 * nc + half * ns:][:, :16], s.reshape(n, 16))
        assert np.array_equal(host[:, half * nc:][:, :c.shape[1]], c)
    dst = torch.zeros_like(src)
    mx.scatter(ops.LayerTable([dst]), fmt, np.arange(n), offs, rec)
    q, s = ref.quantise(src.double().cpu().numpy().reshape(2, n, 16, 1, 32), name)
    v = ref.in_type(ref.dequantise(q, s, name), dt)
    same_bits(dst, v.reshape(dst.shape), dt)


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("dt", DTYPES)
def test_every_code_reads_back(gpu, name, dt):
    """All element codes under all scale codes, subnormal and saturated results too."""
    n_codes = 16 if name == "mxfp4" else 256
    per = max(1, n_codes // 32)  # blocks that show every code
    q = np.tile(np.arange(max(32, n_codes)) % n_codes, 256).reshape(-1, 32)
    s = np.repeat(np.arange(256), per)
    blocks = len(s) // 16
    fmt = mx.MXFormat(name, 1, 16, 1, 32)
    rec = np.zeros((blocks, fmt.layer_bytes), np.uint8)
    for b in range(blocks):
        for half in (0, 1):
            sl = slice(b * 16, b * 16 + 16)
            ref.pack_codes(fmt, q[sl], s[sl], half, rec[b])
    dst = torch.zeros(2, blocks, 16, 1, 32, dtype=ref.TORCH[dt], device=gpu)
    mx.scatter(ops.LayerTable([dst]), fmt, np.arange(blocks),
               np.arange(blocks) * fmt.slot_bytes, torch.from_numpy(rec.reshape(-1)).to(gpu))
    v = ref.in_type(ref.dequantise(q, s[:, None], name), dt).reshape(1, blocks, 16, 1, 32)
    same_bits(dst, np.concatenate([v, v]), dt)


ROPE = [  # layout, bs, heads, dim, rot_dim, style
    ("nhd", 16, 8, 128, 128, "neox"),
    ("hnd", 16, 2, 64, 64, "gptj"),
    ("nhd", 16, 3, 96, 96, "neox"),
    ("nhd", 16, 2, 96, 48, "neox"),
    ("nhd", 4, 1, 256, 64, "gptj"),
    ("nhd", 16, 2, 64, 8, "gptj"),
    ("hnd", 32, 2, 256, 256, "neox"),
]


def rope_inputs(gpu, name, dt, layout, bs, heads, dim, layers=2, pages=6, seed=3):
    g = torch.Generator().manual_seed(seed)
    shape = (2, pages, heads, bs, dim) if layout == "hnd" else (2, pages, bs, heads, dim)
    src = [torch.randn(shape, generator=g).to(ref.TORCH[dt]).to(gpu) for _ in range(layers)]
    if layout == "hnd":
        src = [x.transpose(2, 3) for x in src]
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, name)
    rec = torch.zeros(pages * fmt.slot_bytes, dtype=torch.uint8, device=gpu)
    offs = np.arange(pages, dtype=np.int64)[::-1] * fmt.slot_bytes
    mx.gather(table, fmt, np.arange(pages), offs, rec)
    return table, fmt, rec, offs, [torch.full_like(x, 7) for x in src]


def check_rotated(got, x, want, dt):
    """Rotated K: the result's rounding (half a step, or half of the smallest subnormal) and
    the arithmetic's: the table's two entries and the two products in fp32, 2^-24 of
    either term each."""
    terms = np.abs(x).max(-1, keepdims=True) * 2
    tiny = 2.0 ** -134 if dt == "bf16" else 2.0 ** -25
    tol = ref.HALF_STEP[dt] * np.abs(want) + 2.0 ** -22 * terms + tiny
    assert (np.abs(got - want) <= tol * (1 + 2.0 ** -10)).all()


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", ROPE, ids=str)
@pytest.mark.parametrize("by_token", [False, True])
def test_rerotation(gpu, name, dt, shape, by_token):
    layout, bs, heads, dim, rot, style = shape
    table, fmt, rec, offs, dst = rope_inputs(gpu, name, dt, layout, bs, heads, dim)
    deltas = [5, -3000, 29000]
    inv = [position.rope_inv_freq(rot, THETA), position.rope_inv_freq(rot, 500.0)]
    tabs = torch.stack([position.delta_tables(deltas, rot, inv_freq=i, device=gpu) for i in inv])
    ridx = np.array([0, -1, 2, 1, 0, 2])
    group = [1, 0]
    to = ops.LayerTable(dst)
    how = dict(rot_dim=rot, style=style, layer_group=group)
    if by_token:
        slots = np.arange(6 * bs, dtype=np.int64)
        rows = offs.repeat(bs) * bs + np.tile(np.arange(bs), 6)
        mx.scatter_slots(to, fmt, slots, rows, rec, tabs, ridx.repeat(bs), **how)
    else:
        mx.scatter(to, fmt, np.arange(6), offs, rec, tabs, ridx, **how)
    host = rec.cpu().numpy()
    for l in range(2):
        for p in range(6):
            layer = host[offs[p] + l * fmt.layer_bytes:][:fmt.layer_bytes]
            same_bits(dst[l][1, p].transpose(0, 1), ref.in_type(ref.unpack(fmt, layer, 1), dt), dt)
            k = ref.unpack(fmt, layer, 0)
            got = dst[l][0, p].transpose(0, 1)
            if ridx[p] < 0:
                same_bits(got, ref.in_type(k, dt), dt)
                continue
            want = ref.rotate(k, deltas[ridx[p]], inv[group[l]], style)
            check_rotated(got.double().cpu().numpy(), k, want, dt)


def test_rerotation_of_layers_without_rope(gpu):
    table, fmt, rec, offs, dst = rope_inputs(gpu, "mxfp4", "bf16", "nhd", 16, 2, 64)
    plain = [torch.zeros_like(d) for d in dst]
    mx.scatter(ops.LayerTable(plain), fmt, np.arange(6), offs, rec)
    tabs = position.delta_tables([77], 64, THETA, device=gpu)[None]
    mx.scatter(ops.LayerTable(dst), fmt, np.arange(6), offs, rec, tabs.contiguous(),
               np.zeros(6, np.int32), layer_group=[-1, 0])
    assert torch.equal(dst[0], plain[0])
    assert not torch.equal(dst[1][0], plain[1][0]) and torch.equal(dst[1][1], plain[1][1])


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("layout,bs,heads,dim", [("nhd", 16, 2, 64), ("hnd", 16, 8, 128),
                                                 ("nhd", 5, 3, 96), ("nhd", 16, 1, 32)])
def test_tokens_match_pages(gpu, name, layout, bs, heads, dim):
    """Single tokens write the page form's rows, with padding, a part page, and repeated
    record rows or slots, of which the last entry stays."""
    src = make_caches(gpu, "bf16", layout, 2, 6, bs, heads, dim, 5)
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, name)
    tokens = 2 * bs + max(1, bs // 3)
    blocks = [4, 1, 3]
    slots = ops.slot_mapping_for([blocks], [tokens], bs)
    rows = mx.record_rows([tokens], fmt)
    whole = torch.zeros(3 * fmt.slot_bytes, dtype=torch.uint8, device=gpu)
    mx.gather(table, fmt, blocks, np.arange(3) * fmt.slot_bytes, whole)
    # a padding entry, and an early entry for row 0 that a later one replaces
    s = np.concatenate([[-1, 5 * bs], slots])
    r = np.concatenate([[0, rows[0]], rows])
    rec = torch.zeros_like(whole)
    mx.gather_slots(table, fmt, s, r, rec)
    a, b = rec.cpu().numpy(), whole.cpu().numpy()
    last = np.zeros((heads, bs), bool)
    last[:, :tokens - 2 * bs] = True
    for p in range(3):
        for l in range(2):
            at = p * fmt.slot_bytes + l * fmt.layer_bytes
            for half in (0, 1):
                got, want = (ref.unpack(fmt, x[at:at + fmt.layer_bytes], half) for x in (a, b))
                seen = last if p == 2 else np.ones((heads, bs), bool)
                assert np.array_equal(got[seen], want[seen], equal_nan=True)
                # the rows behind the last token were left as they were: zero codes, scale 0
                assert not got[~seen].any()
    dst = [torch.zeros_like(x) for x in src]
    page = [torch.zeros_like(x) for x in src]
    mx.scatter(ops.LayerTable(page), fmt, blocks, np.arange(3) * fmt.slot_bytes, whole)
    s2 = np.concatenate([[slots[3], -7], slots])
    r2 = np.concatenate([[rows[5], 0], rows])
    mx.scatter_slots(ops.LayerTable(dst), fmt, s2, r2, whole)
    for l in range(2):
        d, w = dst[l].view(torch.int16), page[l].view(torch.int16)
        assert torch.equal(d[:, [4, 1]], w[:, [4, 1]])
        left = tokens - 2 * bs
        assert torch.equal(d[:, 3, :left], w[:, 3, :left])
        assert not d[:, 3, left:].any() and not d[:, [0, 2, 5]].any()


def test_device_tables_skip_what_is_out_of_bounds(gpu):
    """Device tables are not checked by the host: bad entries move nothing."""
    src = make_caches(gpu, "bf16", "nhd", 2, 4, 16, 2, 64, 6)
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, "mxfp4")
    rec = torch.full((3 * fmt.slot_bytes,), 9, dtype=torch.uint8, device=gpu)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=gpu)  # noqa: E731
    big = 1 << 40
    mx.gather(table, fmt, i32([4, -1, 0, 1, 2]),
              i64([0, 0, -16, 3 * fmt.slot_bytes - 16, big]), rec)
    mx.gather_slots(table, fmt, i64([-1, 64, 0, 0, 1 << 50]),
                    i64([0, 0, -16, (3 * fmt.slot_bytes) * 16, 0]), rec)
    assert (rec == 9).all()
    dst = [torch.zeros_like(x) for x in src]
    to = ops.LayerTable(dst)
    mx.scatter(to, fmt, i32([4, -1, 0, 1, 2]),
               i64([0, 0, -16, 3 * fmt.slot_bytes - 16, big]), rec)
    mx.scatter_slots(to, fmt, i64([-1, 64, 0, 0, 1 << 50]),
                     i64([0, 0, -16, (3 * fmt.slot_bytes) * 16, 0]), rec)
    assert all(not d.view(torch.int16).any() for d in dst)
    # a table index out of range is no rotation
    mx.gather(table, fmt, [0], [0], rec)
    cs = position.delta_tables([9], 64, THETA, device=gpu)
    mx.scatter(to, fmt, i32([0, 1]), i64([0, 0]), rec, cs, i32([5, -9]))
    assert torch.equal(dst[0][:, 0].view(torch.int16), dst[0][:, 1].view(torch.int16))


def test_layer_ranges_and_split_launches(gpu, tuning):
    """Layers one by one, records of another layer stride start, and launches cut by the
    workgroup limit write what one launch does."""
    src = make_caches(gpu, "fp16", "nhd", 4, 5, 16, 4, 64, 8)
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, "mxint8")
    ids, offs = [3, 0, 4], np.arange(3, dtype=np.int64) * (fmt.slot_bytes + fmt.layer_bytes)
    size = 3 * (fmt.slot_bytes + fmt.layer_bytes)
    one, many, cut = (torch.zeros(size, dtype=torch.uint8, device=gpu) for _ in range(3))
    mx.gather(table, fmt, ids, offs, one, layer0=1)
    save = mx.PreparedGather(table, fmt, ids, offs, many, layer0=1)
    stream = torch.cuda.current_stream().cuda_stream
    for l in range(4):
        save(l, 1, stream)
    with pytest.raises(IndexError):
        save(3, 2, stream)
    tuning("max_wg_per_launch", 16)
    mx.gather(table, fmt, ids, offs, cut, layer0=1)
    assert torch.equal(one, many) and torch.equal(one, cut)
    rows = (offs[:, None] * 16 + np.arange(16)).reshape(-1)
    slots = (np.array(ids)[:, None] * 16 + np.arange(16)).reshape(-1)
    cut.zero_()
    mx.gather_slots(table, fmt, slots, rows, cut, layer0=1)
    assert torch.equal(one, cut)
    back, byt = ([torch.zeros_like(x) for x in src] for _ in range(2))
    cs = position.delta_tables([40, 2], 64, THETA, device=gpu)
    mx.scatter(ops.LayerTable(back), fmt, ids, offs, one, cs, [0, 1, 0], layer0=1)
    mx.scatter_slots(ops.LayerTable(byt), fmt, slots, rows, one, cs, np.repeat([0, 1, 0], 16),
                     layer0=1)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(back, byt))
    tuning("max_wg_per_launch", 0)
    whole = [torch.zeros_like(x) for x in src]
    mx.scatter(ops.LayerTable(whole), fmt, ids, offs, one, cs, [0, 1, 0], layer0=1)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(back, whole))
    part = [torch.zeros_like(x) for x in src]
    mx.scatter(ops.LayerTable(part), fmt, ids, offs, one, cs, [0, 1, 0], layer0=1, layers=(1, 2))
    assert all(torch.equal(part[l].view(torch.int16), whole[l].view(torch.int16)) for l in (1, 2))
    assert not part[0].any() and not part[3].any()


def test_empty_calls(gpu):
    src = make_caches(gpu, "bf16", "nhd", 2, 4, 16, 2, 64, 6)
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, "mxfp4")
    rec = torch.full((fmt.slot_bytes,), 9, dtype=torch.uint8, device=gpu)
    mx.gather(table, fmt, [], [], rec)
    mx.gather_slots(table, fmt, [-1, -1], [0, 0], rec)
    mx.scatter(table, fmt, [], [], rec)
    mx.scatter_slots(table, fmt, [], [], rec)
    mx.gather(table, fmt, [0], [0], rec, layers=(1, 0))
    assert (rec == 9).all()


def test_graph_replays(gpu):
    """A captured save and load (device tables), replayed with new contents and eager work
    between."""
    src = make_caches(gpu, "bf16", "nhd", 2, 5, 16, 2, 128, 6)
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, "mxint8")
    rec = torch.zeros(3 * fmt.slot_bytes, dtype=torch.uint8, device=gpu)
    dst = [torch.zeros_like(x) for x in src]
    to = ops.LayerTable(dst)
    ids = torch.tensor([4, 0, 2], dtype=torch.int32, device=gpu)
    offs = torch.arange(3, device=gpu) * fmt.slot_bytes
    cs = position.delta_tables([40, 2], 128, THETA, device=gpu)
    ridx = torch.tensor([0, -1, 1], dtype=torch.int32, device=gpu)
    slots = torch.tensor([17, -1, 3], device=gpu)
    rows = torch.tensor([5, 0, fmt.slot_bytes * 16 + 2], device=gpu)

    def step(records, table_to):
        mx.gather(table, fmt, ids, offs, records)
        mx.gather_slots(table, fmt, slots, rows, records)
        mx.scatter(table_to, fmt, ids, offs, records, cs, ridx)
        mx.scatter_slots(table_to, fmt, slots, rows, records)

    step(rec, to)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(rec, to)
    for i in range(3):
        for x in src:
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        r2, d2 = torch.zeros_like(rec), [torch.zeros_like(x) for x in src]
        step(r2, ops.LayerTable(d2))
        assert torch.equal(rec, r2)
        for a, b in zip(dst, d2):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), i
    with pytest.raises(ValueError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            mx.gather(table, fmt, [0], [0], rec)


def test_on_another_stream(gpu):
    src = make_caches(gpu, "bf16", "nhd", 2, 5, 16, 2, 128, 6)
    table = ops.LayerTable(src)
    fmt = mx.MXFormat.of(table.layout, "mxfp4")
    rec = torch.zeros(2 * fmt.slot_bytes, dtype=torch.uint8, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mx.gather(table, fmt, [1, 2], [0, fmt.slot_bytes], rec)
    side.synchronize()
    assert np.array_equal(rec[:fmt.layer_bytes].cpu().numpy(), want_layer(fmt, src[0], 1))


@pytest.mark.parametrize("name,dt,layout,bs,heads,dim,pages", [
    ("mxint8", "bf16", "nhd", 16, 8, 128, 1700), ("mxfp4", "fp16", "hnd", 16, 8, 128, 1700),
    ("mxfp4", "bf16", "nhd", 5, 3, 96, 19000)])
def test_large_launches_match_small_ones(gpu, name, dt, layout, bs, heads, dim, pages):
    """Launches over 200 MiB (other pieces, stores and orders) against the same work in
    slices of a layer and some pages, which the tests above hold to the definition."""
    g = torch.Generator(gpu).manual_seed(3)
    shape = (2, pages, heads, bs, dim) if layout == "hnd" else (2, pages, bs, heads, dim)
    src = [torch.randn(shape, generator=g, device=gpu).to(ref.TORCH[dt]) for _ in range(2)]
    view = (lambda x: x.transpose(2, 3)) if layout == "hnd" else (lambda x: x)
    table = ops.LayerTable([view(x) for x in src])
    fmt = mx.MXFormat.of(table.layout, name)
    assert 2 * table.layout.page_bytes * 2 * pages > 200 << 20
    rng = np.random.default_rng(1)
    ids, offs = rng.permutation(pages), rng.permutation(pages) * fmt.slot_bytes
    rec, part = (torch.zeros(pages * fmt.slot_bytes, dtype=torch.uint8, device=gpu)
                 for _ in range(2))
    mx.gather(table, fmt, ids, offs, rec)
    cuts = [(l, slice(i, i + pages // 4 + 1)) for l in (0, 1)
            for i in range(0, pages, pages // 4 + 1)]
    for l, s in cuts:
        mx.gather(table, fmt, ids[s], offs[s], part, layers=(l, 1))
    assert torch.equal(rec, part)
    for rot, style in ((0, "neox"), (dim, "neox"), (dim // 2 // 16 * 16, "neox"), (dim, "gptj")):
        rope, ridx = {}, np.zeros(pages, np.int64)
        if rot:
            rope = dict(cos_sin=position.delta_tables([977, -5], rot, THETA, device=gpu),
                        rot_dim=rot, style=style)
            ridx = rng.integers(-1, 2, pages)
        res = [[torch.zeros_like(x) for x in src] for _ in range(2)]
        to = [ops.LayerTable([view(x) for x in r]) for r in res]
        mx.scatter(to[0], fmt, ids, offs, rec, **rope, **(dict(rope_idx=ridx) if rot else {}))
        for l, s in cuts:
            mx.scatter(to[1], fmt, ids[s], offs[s], rec, layers=(l, 1), **rope,
                       **(dict(rope_idx=ridx[s]) if rot else {}))
        for a, b in zip(*res):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), (rot, style)
