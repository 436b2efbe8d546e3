"""Timed cases of the quantised records: written from the caches, read back, attended.

What a serving process does with records in the OCP microscaling formats (blocks
of 32 elements along head_dim with one power-of-two scale; ``mxint8``: int8 / 64,
``mxfp4``: e2m1): it saves pages or single tokens of the paged caches in them,
loads them into pages, K re-rotated where a chunk moves, and attends records in
place. Shapes are those of this repository's workloads and benchmark. What is held
in 8 or 4 bits is returned as the values it stands for, so a save is timed with
its reading back into other caches.

``own`` False: plain torch operations. True: the calls of ``daser_amd.mx``.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

THETA = 500000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# layers, KV heads, head_dim, block_size, query heads
SHAPES = {
    "qwen2-0.5b": (24, 2, 64, 16, 14),
    "llama-3.2-1b": (16, 8, 64, 16, 32),
    "qwen2.5-7b": (28, 4, 128, 16, 28),
    "llama-3-8b": (32, 8, 128, 16, 32),
    "llama-3-8b-block32": (32, 8, 128, 32, 32),
    "gemma-2-9b": (42, 8, 256, 16, 16),
    "phi-3-mini": (32, 32, 96, 16, 32),
    "llama-3-70b": (80, 8, 128, 16, 64),
    "llama-3-70b-tp8": (80, 1, 128, 16, 8),
}
ATTEND_LAYERS = 4  # records of an attended case hold this many layers, the third is read
CHUNK = 256        # tokens of a cached chunk


def _case(op, shape, fmt, dtype="bf16", layout="nhd", requests=1, low=CHUNK, high=CHUNK, moved=0,
          style="neox", rot_dim=0, queries=0, limits=False, prior=False):
    """op: save_step (a gather per layer), save, load, tokens (saved and read back by
    slot), append (one token per request, likewise), attend. Requests of ``low`` to
    ``high`` tokens; ``moved``: tokens of a chunk, each chunk at another position than it
    was stored at (0: none moves); ``queries``: query tokens of a request, the last
    of them seeing one token less each with ``limits``; ``prior``: joined with the
    attention over other keys."""
    return dict(op=op, shape=shape, fmt=fmt, dtype=dtype, layout=layout, requests=requests,
                low=low, high=high, moved=moved, style=style, rot_dim=rot_dim, queries=queries,
                limits=limits, prior=prior)


def listed():
    return [
        # one chunk of a small model: nothing but latency
        dict(_case("save", "qwen2-0.5b", "mxint8"), name="save-chunk"),
        # a prefill step as the connector saves it, layer by layer
        dict(_case("save_step", "llama-3-8b", "mxfp4", requests=8), name="save-step"),
        # long prompts saved at once
        dict(_case("save", "llama-3-8b", "mxint8", requests=16, low=512, high=8192),
             name="save-prompts"),
        # one chunk hit at another position
        dict(_case("load", "llama-3-8b", "mxfp4", moved=256), name="load-chunk-moved"),
        # prompts assembled from ten chunks each
        dict(_case("load", "llama-3-8b", "mxint8", requests=16, low=5120, high=5120, moved=512),
             name="load-rag-moved"),
        # prefix hits of a model with head-major pages in half precision
        dict(_case("load", "qwen2.5-7b", "mxfp4", dtype="fp16", layout="hnd", requests=8, low=256,
                   high=4096), name="load-hnd"),
        # a decode step's tokens, appended to resident records
        dict(_case("append", "llama-3-8b", "mxfp4", requests=64, low=1, high=64),
             name="append-step"),
        # prompts of any length by slot_mapping
        dict(_case("tokens", "qwen2-0.5b", "mxint8", requests=64, low=100, high=2000),
             name="tokens-prompts"),
        # one new token over one short context: latency
        dict(_case("attend", "llama-3-8b", "mxfp4", low=500, high=500, queries=1),
             name="attend-one"),
        # a decode batch over long contexts
        dict(_case("attend", "llama-3-8b", "mxfp4", requests=64, low=2048, high=16384, queries=1),
             name="attend-decode"),
        # questions over eight retrieved chunks each, moved to their places
        dict(_case("attend", "llama-3-8b", "mxint8", requests=4, low=4096, high=4096, moved=512,
                   queries=64, prior=True), name="attend-question"),
        # one rank's head of a large model, long moved contexts, a few draft tokens
        dict(_case("attend", "llama-3-70b-tp8", "mxfp4", requests=16, low=8192, high=32768,
                   moved=512, queries=3, limits=True), name="attend-tp8-moved"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["save_step", "save", "load", "load", "tokens", "append", "attend", "attend",
                     "attend"])
    shape = rng.choice(sorted(SHAPES))
    layers, heads, dim, block, q_heads = SHAPES[shape]
    case = _case(op, shape, rng.choice(["mxint8", "mxfp4"]), rng.choice(["bf16", "bf16", "fp16"]))
    case["requests"] = _log(rng, 1, 64)
    # tokens in all: up to 8 GB of cache moved, or 500,000 attended
    most = (1 << 33) // (4 * layers * heads * dim)
    if op == "attend":
        most = 500000 * 8 * 128 // (heads * dim)
        case["queries"] = _log(rng, 1, 48) if rng.random() < 0.5 else 1
        case["limits"] = rng.random() < 0.3
        case["prior"] = rng.random() < 0.3
        most = min(most, (1 << 30) // (case["queries"] * q_heads))
    elif op != "append":
        case["layout"] = rng.choice(["nhd", "nhd", "hnd"]) if op != "tokens" else "nhd"
    top = max(64, min(20000, most // case["requests"]))
    case["high"] = _log(rng, 40, 64 if op == "append" else top)
    case["low"] = _log(rng, 1, case["high"])
    if op in ("load", "attend") and rng.random() < 0.5:
        case["moved"] = block * rng.randint(1, 40)
        case["style"] = rng.choice(["neox", "neox", "gptj"])
        case["rot_dim"] = rng.choice([0, 0, dim // 2])
    return case


# The format: a case's sizes and its records' layout ------------------------------------


class _Step:
    def __init__(self, case, seed):
        self.case, self.seed = case, seed
        self.layers, self.heads, self.dim, self.block, self.q_heads = SHAPES[case["shape"]]
        if case["op"] == "attend":
            self.layers = ATTEND_LAYERS
        self.dtype, self.four = DTYPES[case["dtype"]], case["fmt"] == "mxfp4"
        self.rot_dim = case["rot_dim"] or self.dim
        rng = np.random.default_rng(7)  # lengths belong to the case, not to the seed
        self.tokens = rng.integers(case["low"], case["high"] + 1, case["requests"]).tolist()
        self.pages = [-(-t // self.block) for t in self.tokens]
        self.total = sum(self.pages)
        self.elems = self.block * self.heads * self.dim  # of a K (or V) page
        pad = lambda n: -(-n // 16) * 16  # noqa: E731
        self.codes = pad(self.elems // (2 if self.four else 1))
        self.scales = pad(self.elems // 32)
        self.layer_bytes = 2 * (self.codes + self.scales)
        self.slot_bytes = self.layers * self.layer_bytes
        rng = np.random.default_rng(seed)
        self.num_blocks = self.total + self.total // 20 + 1
        self.page_ids = rng.permutation(self.num_blocks)[:self.total].astype(np.int32)
        self.records = rng.permutation(self.total)  # slot record of each page
        self.offsets = self.records.astype(np.int64) * self.slot_bytes
        self.page_start = np.concatenate([[0], np.cumsum(self.pages)]).astype(np.int32)
        self.rope = np.full(self.total, -1, np.int32)
        self.deltas = []
        if case["moved"]:
            per = max(1, case["moved"] // self.block)
            for a, b in zip(self.page_start[:-1], self.page_start[1:]):
                for p in range(a, b, per):
                    self.rope[p:min(p + per, b)] = len(self.deltas)
                    self.deltas.append(int(rng.integers(-8192, 32768)) or 1)
        self.slots = np.concatenate([
            self.page_ids[a:b].astype(np.int64).repeat(self.block)[:n] * self.block +
            np.arange(n) % self.block
            for a, b, n in zip(self.page_start[:-1], self.page_start[1:], self.tokens)])
        self.rows = np.concatenate([
            self.offsets[a:b].repeat(self.block)[:n] * self.block + np.arange(n) % self.block
            for a, b, n in zip(self.page_start[:-1], self.page_start[1:], self.tokens)])
        if case["op"] == "append":  # the last token of each request
            last = np.cumsum(self.tokens) - 1
            self.slots, self.rows = self.slots[last], self.rows[last]


def _block_scales(x, four):
    """E8M0 codes of blocks x [..., 32] (float32): the smallest power of two that leaves at
    most half a step over the largest element."""
    bits = x.abs().amax(-1).view(torch.int32)
    add, sub = (0x1FFFFF, 2) if four else (0x00FFFF, 0)
    code = ((bits + add) >> 23) - sub
    return torch.where(bits >= 0x7F800000, 255, code.clamp(min=0))


def _round(y, four):
    """Elements y (float64, scaled) rounded to the format's, ties to even."""
    if not four:
        return (y * 64).round().clamp(-127, 127) / 64
    a = y.abs()
    r = torch.where(a < 2, (a * 2).round() / 2, torch.where(a < 4, a.round(), (a / 2).round() * 2))
    return torch.copysign(r.clamp(max=6), y)


def _power(code):
    return torch.exp2(code.double() - 127)


def _quantise(x, four):
    """x [..., D] of the caches' type -> (element values float32 [..., D/32, 32], E8M0 codes)."""
    b = x.float().unflatten(-1, (-1, 32))
    s = _block_scales(b, four)
    q = _round(b.double() / _power(s.clamp(max=254))[..., None], four)
    return q.float(), s


def _values(q, s):
    """What elements and codes stand for, in float32 (exact but for its own limits)."""
    v = (q.double() * _power(s)[..., None]).float().flatten(-2)
    return torch.where((s == 255)[..., None].expand(q.shape).flatten(-2), torch.nan, v)


def _read_back(v, dtype):
    top = torch.finfo(dtype).max
    return v.clamp(-top, top).to(dtype)


def _pack(q, s, step, out):
    """Elements [n, H, bs, D/32, 32] of K or V and their codes -> out = (codes, scales) bytes."""
    if step.four:
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=q.device)
        c = torch.bucketize(q.abs(), grid) | (torch.signbit(q).long() << 3)
        c = c.to(torch.uint8).reshape(len(q), -1, 2)
        c = c[..., 0] | (c[..., 1] << 4)
    else:
        c = (q * 64).to(torch.int8).view(torch.uint8).reshape(len(q), -1)
    out[0][:, :c.shape[1]] = c
    out[1][:, :step.elems // 32] = s.to(torch.uint8).reshape(len(q), -1)


def _unpack(rec, step, half):
    """K (half 0) or V pages of records [n, layer_bytes] -> float32 [n, H, bs, D]."""
    n, c, e = len(rec), step.codes, step.elems
    codes = rec[:, half * c:half * c + e // (2 if step.four else 1)]
    at = 2 * c + half * step.scales
    s = rec[:, at:at + e // 32].reshape(n, step.heads, step.block, -1).int()
    if step.four:
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=rec.device)
        grid = torch.cat([grid, -grid])
        q = grid[torch.stack([codes & 15, codes >> 4], -1).long()]
    else:
        q = codes.view(torch.int8).float() / 64
    return _values(q.reshape(n, step.heads, step.block, -1, 32), s)


def _tables(step, device):
    """(cos, sin) of each delta, as daser_amd.position.delta_tables lays them out."""
    half = step.rot_dim // 2
    inv = THETA ** (-2.0 * torch.arange(half, dtype=torch.float64) / step.rot_dim)
    ang = torch.tensor(step.deltas, dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().to(device)


def _rotate(x, cs, step, sign=1.0):
    """x [n, ..., D] with row i rotated by table cs[i] [half, 2]."""
    r = step.rot_dim
    cs = cs.reshape(len(x), *([1] * (x.dim() - 2)), r // 2, 2)
    c, s = cs[..., 0], cs[..., 1] * sign
    y = x.clone()
    if step.case["style"] == "neox":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    return y


# Inputs ---------------------------------------------------------------------------------


def _fill(out, gen):
    """Activations: N(0, 1) with a few louder channels, as keys have."""
    out.normal_(generator=gen)
    out.mul_(1 + 3 * (torch.arange(out.shape[-1], device=out.device) % 29 == 5).to(out.dtype))


def prepare(case, seed):
    dev = torch.device("cuda")
    step = _Step(case, seed)
    gen = torch.Generator(dev).manual_seed(seed)
    state = dict(case=case, step=step)
    state["records"] = rec = torch.zeros((step.total, step.layers, step.layer_bytes),
                                         dtype=torch.uint8, device=dev)
    if case["op"] in ("load", "attend"):
        k, e = step.codes, step.scales
        for l in range(step.layers):
            for a in range(0, step.total, 2048):
                part = rec[a:a + 2048, l]
                x = torch.empty((len(part), step.heads, step.block, step.dim), dtype=step.dtype,
                                device=dev)
                for half in (0, 1):
                    _fill(x, gen)
                    q, s = _quantise(x, step.four)
                    _pack(q, s, step, (part[:, half * k:half * k + k],
                                       part[:, 2 * k + half * e:2 * k + half * e + e]))
    state["cos_sin"] = _tables(step, dev) if step.deltas else None
    if case["op"] == "attend":
        _prepare_attend(state, step, dev, gen)
        return state
    # caches as vLLM holds them; those that a pass writes are others than it reads
    shape = (step.layers, 2, step.num_blocks)
    shape += (step.heads, step.block) if case["layout"] == "hnd" else (step.block, step.heads)
    view = (lambda t: t.transpose(3, 4)) if case["layout"] == "hnd" else (lambda t: t)
    if case["op"] != "load":
        source = torch.empty(*shape, step.dim, dtype=step.dtype, device=dev)
        _fill(source, gen)
        state["source"] = view(source)
    state["target"] = view(torch.zeros(*shape, step.dim, dtype=step.dtype, device=dev))
    if own:
        from daser_amd import mx, ops

        state["to"] = ops.LayerTable(list(state["target"].unbind(0)))
        if "source" in state:
            state["from"] = ops.LayerTable(list(state["source"].unbind(0)))
        state["fmt"] = mx.MXFormat.of(state["to"].layout, case["fmt"])
    return state


def _prepare_attend(state, step, dev, gen):
    case, n = state["case"], state["case"]["requests"]
    per = case["queries"]
    on = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    state["q"] = torch.empty((n * per, step.q_heads, step.dim), dtype=step.dtype, device=dev)
    state["q"].normal_(generator=gen)
    state["q_start"] = on(np.arange(n + 1, dtype=np.int32) * per)
    state["page_start"] = on(step.page_start)
    state["offsets"] = on(step.offsets)
    state["context"] = on(np.array(step.tokens, np.int32))
    state["rope"] = on(step.rope) if step.deltas else None
    state["max_context"] = max(step.tokens)
    state["limits"] = None
    if case["limits"]:  # token i of a request's last ones sees what is before it
        seen = np.array(step.tokens)[:, None] - np.arange(per)[::-1]
        state["limits"] = on(np.maximum(seen, 0).reshape(-1).astype(np.int32))
    state["prior"] = None
    if case["prior"]:
        out = torch.empty_like(state["q"]).normal_(generator=gen)
        lse = torch.empty(out.shape[:2], device=dev).normal_(generator=gen) + 5
        state["prior"] = (out, lse)
    if own:
        from daser_amd import mx

        state["fmt"] = mx.MXFormat(case["fmt"], step.layers, step.block, step.heads, step.dim)


# One pass -------------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from daser_amd import mx

    case, step, rec = s["case"], s["step"], s["records"]
    op, fmt = case["op"], s["fmt"]
    rope = {}
    if step.deltas:
        rope = dict(cos_sin=s["cos_sin"], rot_dim=step.rot_dim, style=case["style"],
                    rope_idx=step.rope if op != "attend" else s["rope"])
    if op == "attend":
        return mx.attend(s["q"], fmt, rec, s["q_start"], s["page_start"], s["offsets"],
                         s["context"], layer=2, max_queries=case["queries"],
                         max_context=s["max_context"], limits=s["limits"], prior=s["prior"],
                         **rope)
    if op in ("append", "tokens"):
        mx.gather_slots(s["from"], fmt, step.slots, step.rows, rec)
        mx.scatter_slots(s["to"], fmt, step.slots, step.rows, rec)
        return s["target"]
    if op == "save":
        mx.gather(s["from"], fmt, step.page_ids, step.offsets, rec)
    elif op == "save_step":
        gather = mx.PreparedGather(s["from"], fmt, step.page_ids, step.offsets, rec)
        stream = torch.cuda.current_stream().cuda_stream
        for layer in range(step.layers):
            gather(layer, 1, stream)
    mx.scatter(s["to"], fmt, step.page_ids, step.offsets, rec, **rope)
    return s["target"]


def _index(state):
    step, dev = state["step"], state["records"].device
    return {k: torch.from_numpy(np.ascontiguousarray(v)).to(dev).long()
            for k, v in dict(ids=step.page_ids, records=step.records, rope=step.rope,
                             slots=step.slots).items()}


def _run_plain(s):
    case, step = s["case"], s["step"]
    if case["op"] == "attend":
        return _attend_plain(s)
    at = _index(s)
    for l in range(step.layers):
        for half in (0, 1):
            cache = s["target"][l, half]  # [NB, bs, H, D]
            if case["op"] in ("append", "tokens"):
                b, t = at["slots"] // step.block, at["slots"] % step.block
                v = _values(*_quantise(s["source"][l, half][b, t], step.four))
                cache[b, t] = _read_back(v, step.dtype)
                continue
            if case["op"] == "load":
                v = _unpack(s["records"][at["records"], l], step, half)
                if step.deltas and half == 0:
                    v = _rotate(v, s["cos_sin"][at["rope"]], step)
                v = v.transpose(1, 2)
            else:
                v = _values(*_quantise(s["source"][l, half][at["ids"]], step.four))
            cache[at["ids"]] = _read_back(v, step.dtype)
    return s["target"]


def _attend_plain(s, wide=torch.float32):
    case, step = s["case"], s["step"]
    at, group, per = _index(s), step.q_heads // step.heads, case["queries"]
    out, lse = [], []
    for r, n in enumerate(step.tokens):
        pages = slice(int(step.page_start[r]), int(step.page_start[r + 1]))
        rec = s["records"][at["records"][pages], 2]
        k, v = (_read_back(_unpack(rec, step, h), step.dtype).to(wide) for h in (0, 1))
        if step.deltas:
            k = _rotate(k, s["cos_sin"][at["rope"][pages]].to(wide), step)
        k, v = (x.transpose(0, 1).flatten(1, 2)[:, :n].contiguous() for x in (k, v))  # [H, n, D]
        q = s["q"][r * per:(r + 1) * per].to(wide)
        q = q.view(per, step.heads, group, -1).transpose(0, 1).flatten(1, 2)  # [H, per * group, D]
        w = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(step.dim)
        if s["limits"] is not None:
            seen = s["limits"][r * per:(r + 1) * per].repeat_interleave(group)
            hidden = torch.arange(n, device=w.device) >= seen[:, None]
            w = w.masked_fill(hidden, -math.inf)
        top = w.amax(-1, keepdim=True)
        p = torch.exp(w - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = torch.bmm(p, v) / torch.where(total == 0, 1.0, total)
        out.append(o.view(step.heads, per, group, -1).transpose(0, 1).flatten(1, 2))
        lse.append((top + total.log()).view(step.heads, per, group).transpose(0, 1).flatten(1, 2))
    out, lse = torch.cat(out), torch.cat(lse)
    if s["prior"] is not None:
        o2, l2 = s["prior"][0].to(wide), s["prior"][1].to(wide)
        both = torch.logaddexp(lse, l2)
        out = out * torch.exp(lse - both)[..., None] + o2 * torch.exp(l2 - both)[..., None]
        lse = both
    return (out.to(step.dtype), lse) if wide == torch.float32 else (out, lse)


# What a pass cannot do without -----------------------------------------------------------


def work(case):
    step = _Step(case, 0)
    page = 2 * step.elems  # K and V elements of one layer's page
    if case["op"] == "attend":
        tokens = sum(step.tokens)
        rows = case["queries"] * step.q_heads
        held = 2 * step.heads * step.dim * ((0.5 if step.four else 1.0) + 1 / 32)
        io = case["requests"] * rows * (step.dim * 4 + 4)
        if case["prior"]:
            io += case["requests"] * rows * (step.dim * 2 + 4)
        return {"bytes": tokens * held + io, "flops": 4.0 * tokens * rows * step.dim}
    n = (len(step.slots) if case["op"] in ("append", "tokens") else step.total * step.block)
    elems = float(n) * step.layers * page / step.block
    held = (0.5 if step.four else 1.0) + 1 / 32
    passes = 1 if case["op"] == "load" else 2
    flops = 8.0 * elems
    return {"bytes": passes * elems * (2 + held), "flops": flops}


# The definition in 64 bits ---------------------------------------------------------------


def _e2m1(codes):
    """Values of 4-bit codes: sign, two exponent bits of bias 1, one mantissa bit."""
    e, m = (codes >> 1) & 3, (codes & 1).double()
    v = torch.where(e == 0, m / 2, torch.ldexp(1 + m / 2, e.double() - 1))
    return torch.where(codes >= 8, -v, v)


def _held(x, four):
    """The definition, by search: each block x [..., 32] (float64) is held in the smallest
    scale 2^e >= 2^-127 under which its largest element is at most half a step past the
    largest value, and each element as the nearest value of even code."""
    a = x.abs().amax(-1, keepdim=True)
    limit = 7.0 if four else 127.5 / 64
    e = torch.ceil(torch.log2(a / limit).clamp(min=-127))
    e = torch.where(a > limit * torch.exp2(e), e + 1, e)
    low = a <= limit * torch.exp2(e - 1)
    e = torch.where(low & (e > -127), e - 1, e)
    y = x / torch.exp2(e)
    if four:
        grid = _e2m1(torch.arange(8, device=x.device))
        best, d = torch.zeros_like(y), torch.full_like(y, math.inf)
        for i in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first: they win ties
            new = (y.abs() - grid[i]).abs()
            best, d = torch.where(new < d, grid[i], best), torch.minimum(new, d)
        v = torch.copysign(best, y)
    else:
        f = torch.floor(y * 64)
        r = y * 64 - f
        v = torch.where((r > 0.5) | ((r == 0.5) & (f % 2 != 0)), f + 1, f).clamp(-127, 127) / 64
    return v * torch.exp2(e)


def exact(case, seed):
    step = _Step(case, seed)
    if case["op"] != "attend" and step.total * 2 * step.elems * step.layers > 1 << 29:
        return None
    s = prepare(case, seed)
    step = s["step"]
    if case["op"] == "attend":
        if work(case)["flops"] > 4e11:
            return None
        return _attend_exact(s)
    at = _index(s)
    top = torch.finfo(step.dtype).max
    result = torch.zeros(s["target"].shape, dtype=torch.float64, device=s["target"].device)
    for l in range(step.layers):
        for half in (0, 1):
            if case["op"] == "load":
                v = _decoded(s["records"][at["records"], l], step, half)
                if step.deltas and half == 0:
                    v = _turned(v, step, step.rope)
                v = v.transpose(1, 2)
            elif case["op"] in ("append", "tokens"):
                b, t = at["slots"] // step.block, at["slots"] % step.block
                x = s["source"][l, half][b, t].double()
                result[l, half, b, t] = _held(x.unflatten(-1, (-1, 32)), step.four) \
                    .flatten(-2).clamp(-top, top)
                continue
            else:
                x = s["source"][l, half][at["ids"]].double()
                v = _held(x.unflatten(-1, (-1, 32)), step.four).flatten(-2)
            result[l, half, at["ids"]] = v.clamp(-top, top)
    return result


def _decoded(rec, step, half):
    """K or V of records, float64 [n, H, bs, D], from the bytes' meaning."""
    n, e = len(rec), step.elems
    if step.four:
        b = rec[:, half * step.codes:half * step.codes + e // 2].long()
        v = torch.empty((n, e), dtype=torch.float64, device=rec.device)
        v[:, 0::2], v[:, 1::2] = _e2m1(b & 15), _e2m1(b >> 4)
    else:
        b = rec[:, half * step.codes:half * step.codes + e].double()
        v = torch.where(b >= 128, b - 256, b) / 64
    at = 2 * step.codes + half * step.scales
    s = torch.exp2(rec[:, at:at + e // 32].double() - 127)
    return (v.view(n, -1, 32) * s[..., None]).view(n, step.heads, step.block, step.dim)


def _turned(v, step, rope):
    """Rows of page i turned by its delta's angles, as complex numbers."""
    half = step.rot_dim // 2
    inv = THETA ** (-2.0 * torch.arange(half, dtype=torch.float64) / step.rot_dim)
    ang = (torch.tensor(step.deltas, dtype=torch.float64)[:, None] * inv).to(v.device)
    unit = torch.polar(torch.ones_like(ang), ang)[torch.from_numpy(rope).to(v.device).long()]
    unit = unit[:, None, None]
    out = v.clone()
    if step.case["style"] == "neox":
        z = torch.complex(v[..., :half].contiguous(), v[..., half:2 * half].contiguous()) * unit
        out[..., :half], out[..., half:2 * half] = z.real, z.imag
    else:
        z = torch.view_as_complex(v[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * unit
        out[..., :2 * half] = torch.view_as_real(z).flatten(-2)
    return out


def _attend_exact(s):
    case, step = s["case"], s["step"]
    per, group = case["queries"], step.q_heads // step.heads
    rows = len(s["q"])
    out = torch.zeros((rows, step.q_heads, step.dim), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((rows, step.q_heads), -math.inf, dtype=torch.float64, device=s["q"].device)
    for r, n in enumerate(step.tokens):
        a, b = int(step.page_start[r]), int(step.page_start[r + 1])
        rec = s["records"][torch.from_numpy(step.records[a:b]).to(out.device), 2]
        k, v = _decoded(rec, step, 0), _decoded(rec, step, 1)
        if step.deltas:
            k = _turned(k, step, step.rope[a:b])
        for h in range(step.heads):
            kh, vh = k[:, h].reshape(-1, step.dim)[:n], v[:, h].reshape(-1, step.dim)[:n]
            q = s["q"][r * per:(r + 1) * per, h * group:(h + 1) * group].double()
            w = q.reshape(-1, step.dim) @ kh.T.contiguous() / math.sqrt(step.dim)
            if s["limits"] is not None:
                seen = s["limits"][r * per:(r + 1) * per].repeat_interleave(group)
                w[torch.arange(n, device=w.device)[None] >= seen[:, None]] = -math.inf
            p, z = torch.softmax(w, -1).nan_to_num(0.0), torch.logsumexp(w, -1)
            where = slice(r * per, (r + 1) * per), slice(h * group, (h + 1) * group)
            out[where] = (p @ vh).view(per, group, -1)
            lse[where] = z.view(per, group)
    if s["prior"] is not None:
        o2, l2 = s["prior"][0].double(), s["prior"][1].double()
        share = torch.sigmoid(l2 - lse)[..., None]
        out = out * (1 - share) + o2 * share
        lse = torch.logaddexp(lse, l2)
    return out, lse
