"""Quantised records through the connector: its hooks write the store file in the format,
and load it back into other blocks, moved chunks re-rotated."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from daser_amd import _lib, connector as C, data_plane, mx, ops, position
from daser_amd.config import DaserConfig
from daser_amd.workloads import KVShape
from tests import mx_reference as ref
from tests.helpers import rand_caches

SHAPE = KVShape(3, 2, 64, 16, 2)


def test_record_format_is_checked(tmp_path):
    with pytest.raises(ValueError, match="record_format"):
        data_plane.KVDataPlane(str(tmp_path / "s"), record_format="int4")
    plane = data_plane.KVDataPlane(str(tmp_path / "s"), record_format="mxfp4")
    caches = {"a": torch.zeros(2, 4, 16, 2, 64, dtype=torch.float8_e4m3fn)}
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        plane.register(caches)
    caches = {"a": torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16)}
    with pytest.raises(ValueError, match="slot_size"):
        plane.register(caches, SHAPE.slot_bytes)


def test_config_slot_size():
    c = DaserConfig(num_kv_heads=8, head_dim=128, num_layers=32, record_format="mxint8")
    assert c.resolved_slot_size() == mx.MXFormat("mxint8", 32, 16, 8, 128).slot_bytes
    assert DaserConfig(num_kv_heads=8, head_dim=128, num_layers=32).resolved_slot_size() == 2097152


def plan(slots, rows, bs, mode, ridx=None, blocks=64, rec_end=32, staging=1 << 20):
    slots, rows = (np.ascontiguousarray(x, np.int64) for x in (slots, rows))
    r = None if ridx is None else np.ascontiguousarray(ridx, np.int64)
    out = np.zeros(_lib.plan_bytes(slots.size), np.uint8)
    p = _lib.Plan()
    import ctypes

    rc = _lib.lib().dsr_plan_slots_mx(
        ops._addr(slots), ops._addr(rows), ops._addr(r), slots.size, blocks, bs, rec_end, staging,
        4, mode, ops._addr(out), out.size, ctypes.addressof(p))
    if rc:
        return rc
    n = p.n_pages
    at = lambda o, t: out[o:o + n * np.dtype(t).itemsize].view(t)  # noqa: E731
    return at(0, np.int64), at(p.off_ids, np.int64), None if r is None else at(p.off_rope, np.int32)


@pytest.mark.parametrize("seed", range(30))
def test_token_tables_keep_the_last(seed):
    """Random tokens in runs, with padding and repeats: of what is written twice the last
    entry stays, in the order of the destinations."""
    rng = np.random.default_rng(seed)
    bs = int(rng.choice([1, 4, 16]))
    slots, rows, ridx = [], [], []
    for _ in range(int(rng.integers(1, 20))):
        n = int(rng.integers(1, bs + 1))
        s, r = int(rng.integers(0, 64 * bs - n + 1)), int(rng.integers(0, bs - n + 1))
        off = 16 * int(rng.integers(0, 40))
        slots += list(range(s, s + n))
        rows += [off * bs + r + i for i in range(n)]
        ridx += list(rng.integers(-1, 4, n))
        if rng.random() < 0.3:
            slots.append(-1)
            rows.append(-99)
            ridx.append(0)
    for mode in (0, 1):
        last = {}
        for i, s in enumerate(slots):
            if s >= 0:
                last[rows[i] if mode else s] = i
        want = [last[k] for k in sorted(last)]
        s, r, t = plan(slots, rows, bs, mode, ridx)
        assert s.tolist() == [slots[i] for i in want]
        assert r.tolist() == [rows[i] for i in want]
        assert t.tolist() == [ridx[i] for i in want]


@pytest.mark.parametrize("seed", range(4))
def test_many_token_runs(seed):
    """Enough runs for the ordering by digits, far apart, with and without repeats."""
    rng = np.random.default_rng(seed)
    bs, n = 16, 700
    blocks = rng.permutation(4000)[:n] if seed < 2 else rng.integers(0, 300, n)
    offs = rng.permutation(1 << 20)[:n] * 16 if seed % 2 else rng.integers(0, 500, n) * 16
    part = rng.integers(1, bs + 1, n)
    slots = np.concatenate([b * bs + np.arange(p) for b, p in zip(blocks, part)])
    rows = np.concatenate([o * bs + np.arange(p) for o, p in zip(offs, part)])
    for mode in (0, 1):
        last = {}
        for i, k in enumerate(rows if mode else slots):
            last[int(k)] = i
        want = [last[k] for k in sorted(last)]
        s, r, _ = plan(slots, rows, bs, mode, blocks=4000, staging=1 << 25)
        assert np.array_equal(s, slots[want]) and np.array_equal(r, rows[want])


def test_token_table_refusals():
    ok = plan([3], [16 * 16 + 2], 16, 0)
    assert ok[0].tolist() == [3]
    assert plan([64 * 16], [0], 16, 0) == _lib.DSR_PLAN_ERR_SLOT
    assert plan([3], [-1], 16, 0) == _lib.DSR_PLAN_ERR_ROW
    assert plan([3], [(1 << 20) * 16], 16, 0) == _lib.DSR_PLAN_ERR_ROW
    assert plan([3], [8 * 16], 16, 0) == _lib.DSR_PLAN_ERR_ALIGN
    assert plan([3, 4], [15, 16], 16, 1) == _lib.DSR_PLAN_ERR_ALIGN  # runs into the next name
    assert plan([3], [0], 16, 0, [4]) == _lib.DSR_PLAN_ERR_ROPE
    assert plan([3], [0], 16, 2) == _lib.DSR_ERR_ARG
    s, r, _ = plan([-1, -5], [7, 7], 16, 1)
    assert not s.size and not r.size


class FakeAsyncIPC:
    def __init__(self):
        self.committed = []

    async def commit_chunk(self, key):
        self.committed.append(key)


def worker(tmp_path, **extra):
    cfg = SimpleNamespace(kv_transfer_config=SimpleNamespace(kv_connector_extra_config=dict(
        store_path=str(tmp_path / "daser.store"), io_slot_mb=0.03125, io_slots=3, **extra)))
    return C.DaserConnector(cfg, C.KVConnectorRole.WORKER, ipc_async=FakeAsyncIPC())


def named(caches):
    return {f"model.layers.{i}.self_attn.attn": c for i, c in enumerate(caches)}


@pytest.mark.gpu
@pytest.mark.parametrize("name,dt,mode,asynchronous", [
    ("mxfp4", "bf16", "per_layer", False), ("mxint8", "fp16", "deferred", False),
    ("mxint8", "bf16", "per_layer", True)])
def test_save_and_load_through_the_hooks(gpu, tmp_path, name, dt, mode, asynchronous):
    caches = rand_caches(SHAPE, 16, dt, gpu, seed=31)
    w = worker(tmp_path, record_format=name, save_mode=mode, async_save=asynchronous)
    w.register_kv_caches(named(caches))
    fmt = mx.MXFormat(name, 3, 16, 2, 64)
    slot = fmt.slot_bytes
    assert w._slot_size == slot
    w.bind_connector_metadata(C.DaserConnectorMeta(reqs_to_store={
        "a": C.ReqStoreSpec("ka", 3, 3, [5, 9, 2], 3 * slot, 40),
        "b": C.ReqStoreSpec("kb", 10, 1, [7], 10 * slot, 16)}))
    other = caches[1].clone()  # a tensor that is not the registered cache
    for i, (layer, t) in enumerate(named(caches).items()):
        w.save_kv_layer(layer, other if i == 1 else t, None)
    w.wait_for_save()
    w.clear_connector_metadata()
    w.shutdown()
    data = np.fromfile(tmp_path / "daser.store", np.uint8)
    for start, blocks in ((3, [5, 9, 2]), (10, [7])):
        for i, b in enumerate(blocks):
            for l in range(3):
                at = (start + i) * slot + l * fmt.layer_bytes
                want = np.zeros(fmt.layer_bytes, np.uint8)
                k, v = (caches[l][h, b].transpose(0, 1).double().cpu().numpy() for h in (0, 1))
                ref.pack(fmt, k, v, want)
                assert np.array_equal(data[at:at + fmt.layer_bytes], want)

    r = worker(tmp_path, record_format=name, rope_theta=10000.0)
    fresh = [torch.zeros_like(c) for c in caches]
    r.register_kv_caches(named(fresh))
    r.bind_connector_metadata(C.DaserConnectorMeta(reqs_to_load={
        "x": C.ReqLoadSpec("ka", 3, 3, [1, 12, 4], 3 * slot, 40, pos_offset=0, new_pos=1234),
        "y": C.ReqLoadSpec("kb", 10, 1, [0], 10 * slot, 16)}))
    r.start_load_kv(None)
    torch.cuda.synchronize()
    r.shutdown()
    inv = position.rope_inv_freq(64, 10000.0)
    tiny = 2.0 ** -25
    for l in range(3):
        for start, blocks, delta in ((3, [1, 12, 4], 1234), (10, [0], 0)):
            for i, b in enumerate(blocks):
                at = (start + i) * slot + l * fmt.layer_bytes
                k, v = (ref.unpack(fmt, data[at:at + fmt.layer_bytes], h) for h in (0, 1))
                gk, gv = (fresh[l][h, b].transpose(0, 1).double().cpu().numpy() for h in (0, 1))
                assert np.array_equal(gv, ref.in_type(v, dt))
                want = ref.rotate(k, delta, inv, "neox")
                # the result's rounding, and 2^-24 of either term for the table's entries and
                # the products
                tol = ref.HALF_STEP[dt] * np.abs(want) + 2.0 ** -22 * 2 * \
                    np.abs(k).max(-1, keepdims=True) + tiny
                assert (np.abs(gk - want) <= tol * (1 + 2.0 ** -10)).all()
        assert not fresh[l][:, [2, 3, 5, 6, 7, 8, 9, 10, 11, 13, 14, 15]].any()
