"""Attention over quantised records against softmax attention in 64 bits over the records'
values, at the lengths, groups and masks where it can go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from daser_amd import mx, ops, position
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

THETA = 500000.0


class Case:
    """Requests over random records of 3 layers, and what attention over layer 1 gives."""

    def __init__(self, gpu, name="mxfp4", dt="bf16", bs=16, heads=2, group=4, dim=128,
                 contexts=(37,), queries=(1,), moved=False, style="neox", rot=None, limits=False,
                 seed=0, loud=1.0):
        rng = np.random.default_rng(seed)
        self.fmt = fmt = mx.MXFormat(name, 3, bs, heads, dim)
        self.dt, self.gpu, self.layer = dt, gpu, 1
        self.contexts, self.queries = list(contexts), list(queries)
        pages = [-(-c // bs) for c in contexts]
        total = sum(pages)
        self.page_start = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
        self.q_start = np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)
        self.offsets = rng.permutation(total).astype(np.int64) * fmt.slot_bytes
        host = np.zeros(max(1, total) * fmt.slot_bytes, np.uint8)
        # bytes of the other layers are NaN scales: reading one would show
        host[:] = 255
        k = rng.standard_normal((total, heads, bs, dim)) * loud
        k[..., 3] *= 5
        v = rng.standard_normal((total, heads, bs, dim))
        self.k, self.v = np.zeros_like(k), np.zeros_like(v)
        for p in range(total):
            at = self.offsets[p] + fmt.layer_bytes
            layer = host[at:at + fmt.layer_bytes]
            ref.pack(fmt, k[p], v[p], layer)
            self.k[p] = ref.in_type(ref.unpack(fmt, layer, 0), dt)
            self.v[p] = ref.in_type(ref.unpack(fmt, layer, 1), dt)
        self.host = host
        self.staging = torch.from_numpy(host).to(gpu)
        n = int(self.q_start[-1])
        self.q = torch.from_numpy(rng.standard_normal((n, heads * group, dim))) \
            .to(ref.TORCH[dt]).to(gpu)
        self.scale = dim ** -0.5
        self.rope = {}
        if moved:
            rot = rot or dim
            inv = position.rope_inv_freq(rot, THETA)
            deltas = [700, -31000, 3]
            ridx = rng.integers(-1, 3, total) if total else np.zeros(0, np.int64)
            for p in range(total):
                if ridx[p] >= 0:
                    self.k[p] = ref.rotate(self.k[p], deltas[ridx[p]], inv, style)
            self.rope = dict(cos_sin=position.delta_tables(deltas, rot, inv_freq=inv, device=gpu),
                             rope_idx=ridx.astype(np.int32), rot_dim=rot, style=style)
        self.limits = None
        if limits:
            self.limits = np.concatenate([rng.integers(0, c + 2, q) for c, q in
                                          zip(contexts, queries)] or [[]]).astype(np.int32)

    def args(self):
        return dict(q=self.q, fmt=self.fmt, staging=self.staging, q_start=self.q_start,
                    page_start=self.page_start, slot_offsets=self.offsets,
                    context=np.array(self.contexts, np.int32), layer=self.layer,
                    limits=self.limits, **self.rope)

    def want(self):
        q = self.q.double().cpu().numpy()
        res = []
        for r, c in enumerate(self.contexts):
            a, b = self.page_start[r], self.page_start[r + 1]
            k, v = (x[a:b].transpose(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])
                    for x in (self.k, self.v))
            rows = slice(self.q_start[r], self.q_start[r + 1])
            seen = np.full(self.queries[r], c)
            if self.limits is not None:
                seen = np.clip(self.limits[rows], 0, c)
            res.append(ref.attend(q[rows], k, v, seen, self.scale))
        return [np.concatenate(x) for x in zip(*res)]

    def check(self, out, lse, want=None):
        """Tolerances, from the formula: a score sums head_dim products (2^-24 of the largest
        partial sum for each step, twice that with a rotated query held as two halves of
        16 bits in all: 2^-16 of it), so p is off by e^(2 ds) - 1 <= 4 ds and by its rounding
        to q's type (half a step); out by that times sum p |v| and by its own rounding. A sum
        over T tokens in fp32 adds T 2^-24, an exponential 2^-21."""
        o, l, mag, width = want or self.want()
        dim = self.fmt.head_dim
        ds = width * ((dim + 8) * 2.0 ** -24 + (2.0 ** -15 if self.rope else 0))
        t = max(self.contexts, default=0) * 2.0 ** -24 + 2.0 ** -20
        half = ref.HALF_STEP[self.dt]
        got = out.double().cpu().numpy()
        tol = mag * (half * 1.05 + 4 * ds + t)[..., None] + half * np.abs(o) + 1e-30
        empty = np.isneginf(l)
        assert np.array_equal(np.isneginf(lse.cpu().numpy()), empty)
        assert not got[empty].any()
        bad = np.abs(got - o) > tol
        assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], o[bad][:4], tol[bad][:4])
        fine = ~empty
        d = np.abs(lse.double().cpu().numpy()[fine] - l[fine])
        assert (d <= (2 * ds + t + 2.0 ** -21 * (1 + np.abs(np.where(empty, 0, l))))[fine]).all()

    def run_and_check(self, **kw):
        out, lse = mx.attend(**{**self.args(), **kw})
        self.check(out, lse)
        return out, lse


@pytest.mark.parametrize("name", ["mxint8", "mxfp4"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
def test_types_and_widths(gpu, name, dt, dim):
    Case(gpu, name, dt, dim=dim, contexts=(50, 16, 1), queries=(1, 3, 2)).run_and_check()


@pytest.mark.parametrize("heads,group", [(1, 1), (1, 8), (2, 7), (8, 1), (3, 16), (1, 71), (4, 33)])
def test_head_groups(gpu, heads, group):
    Case(gpu, heads=heads, group=group, dim=64, contexts=(33, 100), queries=(2, 1),
         seed=group).run_and_check()


@pytest.mark.parametrize("context", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 511,
                                     1000, 2049])
def test_lengths(gpu, context):
    Case(gpu, heads=1, group=2, dim=64, contexts=(context,), queries=(1,),
         seed=context).run_and_check()


@pytest.mark.parametrize("bs", [16, 32, 48, 128])
def test_block_sizes(gpu, bs):
    Case(gpu, "mxint8", bs=bs, contexts=(1, bs - 1, bs, bs + 1, 5 * bs + 3),
         queries=(1, 2, 1, 1, 3)).run_and_check()


def test_ragged_batch_with_empty_requests(gpu):
    """Requests without tokens give 0 and -inf; requests without queries give nothing."""
    c = Case(gpu, contexts=(0, 40, 300, 0, 17, 5), queries=(2, 0, 5, 1, 33, 0))
    c.run_and_check()
    Case(gpu, contexts=(0,), queries=(3,)).run_and_check()
    Case(gpu, contexts=(0, 0), queries=(0, 1)).run_and_check()


def test_no_queries(gpu):
    out, lse = mx.attend(**Case(gpu, contexts=(20, 4), queries=(0, 0)).args())
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_limits(gpu, dt):
    """Each query sees a length of its own, none and more than there is among them."""
    Case(gpu, dt=dt, contexts=(90, 33, 300), queries=(40, 3, 70), limits=True,
         seed=4).run_and_check()


@pytest.mark.parametrize("name,dt,dim,rot,style", [
    ("mxfp4", "bf16", 128, None, "neox"), ("mxint8", "fp16", 64, None, "gptj"),
    ("mxint8", "bf16", 96, 48, "neox"), ("mxfp4", "fp16", 256, 64, "gptj"),
    ("mxfp4", "bf16", 64, 16, "neox"), ("mxint8", "bf16", 32, 8, "gptj")])
def test_moved_chunks(gpu, name, dt, dim, rot, style):
    Case(gpu, name, dt, dim=dim, contexts=(200, 77, 16), queries=(2, 1, 20), moved=True, rot=rot,
         style=style, limits=True, seed=dim).run_and_check()


def test_many_queries(gpu):
    Case(gpu, "mxint8", heads=2, group=4, dim=64, contexts=(150, 700), queries=(70, 33),
         limits=True, moved=True).run_and_check()


def test_long_context_and_wide_split(gpu):
    """Few rows over a long context: the work is split along it and joined."""
    Case(gpu, heads=1, group=2, dim=64, contexts=(20000, 3), queries=(1, 1)).run_and_check()
    Case(gpu, "mxint8", heads=2, group=1, dim=128, contexts=(9001,), queries=(2,), moved=True,
         limits=True).run_and_check()


@pytest.mark.parametrize("heads,requests,kw", [
    (4, 8, dict()), (4, 8, dict(moved=True, limits=True)), (8, 4, dict(name="mxint8", dt="fp16")),
    (2, 16, dict()), (6, 6, dict(limits=True)), (3, 11, dict(moved=True, style="gptj"))])
def test_large_launches(gpu, heads, requests, kw):
    """Where requests, heads and the longest context make a large launch, each wave takes a
    head of its own (4 or 2 to a workgroup), short and empty requests beside the long one."""
    contexts = [8200] + [(7 * i * i) % 90 for i in range(requests - 1)]
    assert requests * heads * 8200 >= 1 << 18
    Case(gpu, heads=heads, group=2, dim=64, contexts=contexts, queries=[1, 3] * (requests // 2) +
         [2] * (requests % 2), seed=heads, **kw).run_and_check()


def test_many_short_requests(gpu):
    """A large launch that is not split: the waves write the results themselves."""
    contexts = [1 + (5 * i) % 32 for i in range(2060)]
    contexts[7] = 0
    c = Case(gpu, heads=4, group=1, dim=32, contexts=contexts, queries=[1] * 2060, seed=1)
    out, lse = c.run_and_check()
    prior = (torch.randn_like(out), torch.randn_like(lse))
    both, both_lse = mx.attend(**c.args(), prior=prior)
    share = torch.sigmoid(prior[1].double() - lse.double())[..., None]
    o, l, mag, width = c.want()
    own = torch.from_numpy(o).to(gpu)
    want = own * (1 - share) + prior[0].double() * share
    want_lse = torch.logaddexp(torch.from_numpy(l).to(gpu), prior[1].double())
    # the share is off by what the lse is (some 2^-18), the result by half a step more
    far = (both.double() - want).abs()
    half = ref.HALF_STEP["bf16"]
    tol = torch.from_numpy(mag).to(gpu) * (half * 1.05 + 2.0 ** -16) + half * want.abs() + \
        2.0 ** -16 * (own.abs() + prior[0].double().abs())
    assert (far <= tol).all()
    assert ((both_lse.double() - want_lse).abs() <= 2.0 ** -16 * (1 + want_lse.abs())).all()


def test_loud_scores(gpu):
    """Scores of hundreds: the running maximum carries the sum."""
    Case(gpu, contexts=(500, 64), queries=(3, 1), loud=60.0, seed=9).run_and_check()


def test_scale_and_strided_queries(gpu):
    c = Case(gpu, contexts=(100, 9), queries=(2, 3))
    c.scale = 0.31
    wide = torch.randn(5, 24, 128, device=gpu).to(torch.bfloat16)
    wide[:, 8:16] = c.q
    out, lse = mx.attend(**{**c.args(), "q": wide[:, 8:16], "scale": 0.31})
    c.check(out, lse)
    heads_first = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    again, _ = mx.attend(**{**c.args(), "q": heads_first, "scale": 0.31})
    assert torch.equal(again, out)


def test_prior(gpu):
    """Joined with attention over other keys: as over both sets at once."""
    whole = Case(gpu, contexts=(96, 0, 64), queries=(4, 2, 1), seed=3)
    q = whole.args()
    first, second = dict(q), dict(q)
    first["context"] = np.array([48, 0, 64], np.int32)
    out1, lse1 = mx.attend(**first)
    # request 0's other three pages as a request of its own
    second.update(page_start=np.array([3, 6, 6, 6], np.int32), context=[48, 0, 0])
    second["slot_offsets"] = whole.offsets
    out, lse = mx.attend(**second, prior=(out1, lse1))
    want = list(whole.want())
    # the prior's own rounding to q's type joins the result's
    want[2] = want[2] * 2.2
    whole.check(out, lse, want)
    assert torch.equal(out[4:6], torch.zeros_like(out[4:6])) and torch.isneginf(lse[4:6]).all()
    assert torch.equal(out[6:], out1[6:]) and torch.equal(lse[6:], lse1[6:])


def test_nan_stays_where_it_is_seen(gpu):
    """A NaN block that is seen makes its head's queries NaN; one behind the context or
    behind a query's limit does nothing, in K or in V."""
    c = Case(gpu, heads=2, group=2, dim=64, contexts=(40,), queries=(2,))
    nc, ns = ref.sections(c.fmt)
    clean, clean_lse = c.run_and_check()
    for half in (0, 1):
        at = int(c.offsets[2]) + c.fmt.layer_bytes + 2 * nc + half * ns
        hidden = c.staging.clone()
        hidden[at + 8 * 2:at + 16 * 2] = 255  # head 0 from row 8 of the last page: token 40 on
        hidden[at + 24 * 2:at + 32 * 2] = 255  # head 1 likewise
        out, lse = mx.attend(**{**c.args(), "staging": hidden})
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
        seen = c.staging.clone()
        seen[at + 7 * 2] = 255  # head 0, token 39
        out, lse = mx.attend(**{**c.args(), "staging": seen, "limits": np.array([39, 40])})
        lim = mx.attend(**{**c.args(), "limits": np.array([39, 40])})[0]
        assert torch.equal(out[0], lim[0]) and torch.equal(out[1, 2:], lim[1, 2:])
        assert torch.isnan(out[1, :2, :32]).all()
        if half == 0:
            assert torch.isnan(out[1, :2]).all() and torch.isnan(lse[1, :2]).all()


def test_device_tables_and_hints(gpu):
    """Device tables give the same bits, whatever the launch's hints say, and entries out
    of bounds are not seen."""
    c = Case(gpu, contexts=(200, 77, 30), queries=(2, 1, 20), moved=True, limits=True)
    out, lse = c.run_and_check()
    d = {k: torch.from_numpy(np.ascontiguousarray(v)).to(gpu) if isinstance(v, np.ndarray) else v
         for k, v in c.args().items()}
    for hints in (dict(), dict(max_queries=20, max_context=200)):
        o2, l2 = mx.attend(**d, **hints)
        c.check(o2, l2)
    o3, l3 = mx.attend(**d, max_queries=1, max_context=1)
    c.check(o3, l3)
    # a context past the request's pages ends with them; a page outside is not seen
    far = dict(d)
    far["context"] = torch.tensor([200, 1 << 30, 30], dtype=torch.int32, device=gpu)
    c.contexts[1] = 80
    o4, l4 = mx.attend(**far)
    c.check(o4, l4)
    off = d["slot_offsets"].clone()
    off[[0, 12]] = torch.tensor([-16, c.staging.numel() - 16], device=gpu)
    assert torch.isfinite(mx.attend(**{**d, "slot_offsets": off})[0].float()).all()
    start = torch.tensor([-5, 2, 3, 99], dtype=torch.int32, device=gpu)
    o5, l5 = mx.attend(**{**d, "q_start": start})
    assert torch.isfinite(o5.float()).all()


def test_pages_outside_are_not_seen(gpu):
    c = Case(gpu, heads=1, group=1, dim=64, contexts=(64,), queries=(1,))
    d = {k: torch.from_numpy(np.ascontiguousarray(v)).to(gpu) if isinstance(v, np.ndarray) else v
         for k, v in c.args().items()}
    off = c.offsets.copy()
    off[1], off[2] = -16, c.staging.numel() - 16
    out, lse = mx.attend(**{**d, "slot_offsets": torch.from_numpy(off).to(gpu)})
    keep = [0, 3]
    k, v = (x[keep].transpose(1, 0, 2, 3).reshape(1, 32, 64) for x in (c.k, c.v))
    q = c.q.double().cpu().numpy()
    c.check(out, lse, ref.attend(q, k, v, [32], c.scale))


def test_rows_of_no_request_stay(gpu):
    c = Case(gpu, contexts=(50, 20), queries=(2, 3))
    args = c.args()
    args["q_start"] = np.array([0, 2, 4], np.int32)
    out = torch.full_like(c.q, 5)
    got, lse = mx.attend(**args, out=out)
    assert got is out and (out[4] == 5).all()
    full, _ = mx.attend(**c.args())
    assert torch.equal(out[:4], full[:4])


def test_same_bits_every_time(gpu):
    c = Case(gpu, heads=2, group=4, contexts=(3000, 100), queries=(1, 9), moved=True)
    first = mx.attend(**c.args())
    for _ in range(3):
        again = mx.attend(**c.args())
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_past_32_bits(gpu):
    """Records beyond 4 GiB of staging."""
    c = Case(gpu, heads=1, group=2, dim=64, contexts=(48,), queries=(1,))
    want = mx.attend(**c.args())
    base = (1 << 32) + (1 << 20)
    big = torch.empty(base + c.staging.numel(), dtype=torch.uint8, device=gpu)
    big[base:] = c.staging
    args = {**c.args(), "staging": big, "slot_offsets": c.offsets + base}
    got = mx.attend(**args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_graphs_and_streams(gpu):
    """Captured calls keep workspaces of their own: two graphs replayed on two streams at
    once, eager work between, give the eager results each time."""
    cases = [Case(gpu, contexts=(4000, 10), queries=(1, 2), seed=s) for s in (1, 2)]
    held = []
    for c in cases:
        d = {k: torch.from_numpy(np.ascontiguousarray(v)).to(gpu) if isinstance(v, np.ndarray)
             else v for k, v in c.args().items()}
        d.update(max_queries=2, max_context=4000)
        mx.attend(**d)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = mx.attend(**d)
        held.append((graph, d, res, torch.cuda.Stream()))
    for i in range(3):
        for graph, d, _, s in held:
            d["q"].normal_()
        torch.cuda.synchronize()
        for graph, d, _, s in held:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, d, res, _), c in zip(held, cases):
            eager = mx.attend(**d)
            assert torch.equal(res[0], eager[0]) and torch.equal(res[1], eager[1]), i
            c.check(*res)


def test_save_attend_load(gpu):
    """The operators together: prompts saved from the caches, a few tokens appended by slot,
    attended in place, and loaded into pages whose attention is the same."""
    heads, group, dim, bs = 2, 4, 128, 16
    g = torch.Generator().manual_seed(1)
    cache = [torch.randn(2, 12, bs, heads, dim, generator=g).to(torch.bfloat16).to(gpu)
             for _ in range(2)]
    table = ops.LayerTable(cache)
    fmt = mx.MXFormat.of(table.layout, "mxfp4")
    blocks, tokens = [[3, 7, 1], [10, 2]], [45, 20]
    rec = torch.zeros(5 * fmt.slot_bytes, dtype=torch.uint8, device=gpu)
    ids = [3, 7, 10]  # the whole pages; the rest by slot
    offs = np.array([0, 1, 3]) * fmt.slot_bytes
    mx.gather(table, fmt, ids, offs, rec)
    slots = ops.slot_mapping_for(blocks, tokens, bs)
    rows = mx.record_rows(tokens, fmt)
    late = np.array([t for t in range(65) if (t % 45 if t < 45 else t - 45) >= (32 if t < 45 else 16)])
    for t in late:  # one decode step each
        mx.gather_slots(table, fmt, slots[t:t + 1], rows[t:t + 1], rec)
    q = torch.randn(2, heads * group, dim, generator=g).to(torch.bfloat16).to(gpu)
    loaded = [torch.zeros_like(c) for c in cache]
    mx.scatter_slots(ops.LayerTable(loaded), fmt, slots, rows, rec)
    for layer in (0, 1):
        out, lse = mx.attend(q, fmt, rec, [0, 1, 2], [0, 3, 5], np.arange(5) * fmt.slot_bytes,
                             tokens, layer=layer)
        for r in (0, 1):
            b = torch.tensor(blocks[r])
            k, v = (loaded[layer][h, b].reshape(-1, heads, dim)[:tokens[r]].transpose(0, 1)
                    .double().cpu().numpy() for h in (0, 1))
            want = ref.attend(q[r:r + 1].double().cpu().numpy(), k, v, [tokens[r]], dim ** -0.5)
            c = Case.__new__(Case)
            c.fmt, c.rope, c.contexts, c.dt = fmt, {}, tokens, "bf16"
            c.check(out[r:r + 1], lse[r:r + 1], want)
