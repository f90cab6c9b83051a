"""Refusals of the adapter, rotary and compaction entry points before any device call, the angles of
scaled rotary positions, and the block manager's plan of a compaction against a model of it."""
import ctypes

import numpy as np
import pytest

import atomflow_amd
from atomflow_amd import (AF_ERR_BAD_SEQUENCE, AF_ERR_INVALID_ARG, AF_ERR_OUT_OF_RANGE, AF_ERR_POOL_EXHAUSTED,
                          AF_ERR_UNSUPPORTED, AF_ERR_WORKSPACE, AF_FP16, AF_FP32, AF_KV_FP16, AF_KV_FP8_E4M3, AF_OK,
                          _abi, kv)
from rows_ref import frequencies

FAKE = 0x10000  # never dereferenced
BAD, NOT, RANGE = AF_ERR_INVALID_ARG, AF_ERR_UNSUPPORTED, AF_ERR_OUT_OF_RANGE


def call(name, args, **changes):
    assert set(changes) <= set(args), changes
    return getattr(atomflow_amd.lib(), name)(*{**args, **changes}.values())


def pool(**changes):
    p = kv.make_pool(FAKE, AF_KV_FP16, 16, 2, 8, 128, 100)
    for k, v in changes.items():
        setattr(p, k, v)
    return ctypes.byref(p)


def lora(**changes):
    p = kv.make_lora(FAKE, FAKE, 4, 16, 64, [32, 48])
    for k, v in changes.items():
        if k == "ends":
            p.slice_end[:len(v)] = v
        else:
            setattr(p, k, v)
    return ctypes.byref(p)


LORA = dict(x=FAKE, xs=64, m=4, ids=FAKE, lora=None, y=FAKE, ys=48, out=FAKE, outs=48, dtype=AF_FP16, ws=FAKE,
            bytes=1 << 20, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(x=None), BAD), (dict(ids=None), BAD), (dict(y=None), BAD), (dict(out=None), BAD), (dict(m=-1), BAD),
    (dict(xs=56), BAD), (dict(xs=68), BAD), (dict(ys=47), BAD), (dict(outs=47), BAD), (dict(x=FAKE + 8), BAD),
    (dict(ids=FAKE + 2), BAD), (dict(y=FAKE + 1), BAD), (dict(out=FAKE + 2, dtype=AF_FP32), BAD),
    (dict(dtype=3), NOT), (dict(outs=64), BAD), (dict(m=(1 << 20) + 1, bytes=1 << 40), NOT),
    (dict(ws=None), AF_ERR_WORKSPACE), (dict(ws=FAKE + 4), AF_ERR_WORKSPACE), (dict(bytes=511), AF_ERR_WORKSPACE),
    (dict(m=0, x=None, ids=None, y=None, out=None, ws=None), AF_OK)])
def test_lora_refusals(changes, status):
    assert call("af_lora_add", {**LORA, "lora": lora()}, **changes) == status


@pytest.mark.parametrize("changes,status", [
    (dict(a=None), BAD), (dict(b=None), BAD), (dict(a=FAKE + 8), BAD), (dict(b=FAKE + 8), BAD),
    (dict(ranks=FAKE + 2), BAD), (dict(scales=FAKE + 2), BAD), (dict(n_adapters=0), BAD), (dict(max_rank=0), BAD),
    (dict(max_rank=12), NOT), (dict(max_rank=136), NOT), (dict(k=60), NOT), (dict(k=0), BAD), (dict(n=0), BAD),
    (dict(n_slices=0), BAD), (dict(n_slices=5), NOT), (dict(ends=[0, 48]), BAD), (dict(ends=[48, 32]), BAD),
    (dict(ends=[32, 47]), BAD), (dict(n=49), BAD), (dict(n_adapters=(1 << 20) + 1), NOT)])
def test_lora_descriptor_refusals(changes, status):
    d = lora(**changes)
    assert call("af_lora_add", {**LORA, "lora": d}) == status
    if not set(changes) & {"a", "b", "ranks", "scales"}:
        assert atomflow_amd.lib().af_lora_workspace_size(d, 4) == 0


def test_lora_null_descriptor_and_workspace():
    assert call("af_lora_add", LORA) == BAD
    assert atomflow_amd.lib().af_lora_workspace_size(None, 4) == 0
    assert atomflow_amd.lib().af_lora_workspace_size(lora(), -1) == 0
    sizes = [atomflow_amd.lib().af_lora_workspace_size(lora(k=4096), m) for m in (0, 1, 2, 77, 256, 257, 8192)]
    assert sizes[0] > 0 and sizes == sorted(sizes)


ROWS = dict(q=FAKE, qs=512, qo=FAKE, qos=512, nq=4, k=FAKE, ks=256, ko=FAKE, kos=256, nk=2, m=4, hd=128, rot=64,
            layout=0, inverse=0, cos=FAKE, sin=FAKE, max_pos=64, pos=FAKE, p0=0, status=None, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(q=None), BAD), (dict(qo=None), BAD), (dict(ko=None), BAD), (dict(k=None, ko=None), AF_OK),
    (dict(nk=-1), BAD), (dict(nq=0), BAD), (dict(m=-1), BAD), (dict(hd=0), BAD), (dict(hd=127), NOT),
    (dict(hd=514, qs=4096, qos=4096, ks=4096, kos=4096), NOT), (dict(rot=0), BAD),
    (dict(rot=63), BAD), (dict(rot=130), BAD), (dict(layout=2), NOT), (dict(inverse=2), BAD), (dict(cos=None), BAD),
    (dict(sin=None), BAD), (dict(cos=FAKE + 4), BAD), (dict(max_pos=0), BAD), (dict(qs=511), BAD),
    (dict(qos=511), BAD), (dict(ks=255), BAD), (dict(kos=255), BAD), (dict(qos=520), BAD), (dict(kos=264), BAD),
    (dict(pos=None, p0=61), RANGE), (dict(pos=None, p0=-1), RANGE), (dict(q=FAKE + 1), BAD),
    (dict(pos=FAKE + 2), BAD), (dict(status=FAKE + 2), BAD), (dict(m=0, q=None, qo=None), AF_OK)])
def test_rope_rows_refusals(changes, status):
    if status == AF_OK:
        changes = {**changes, "m": 0}
    assert call("af_rope_rows", ROWS, **changes) == status


APPEND = dict(x=FAKE, xs=2560, m=4, qo=FAKE, qos=512, nq=4, pool=None, layer=1, slots=FAKE, pos=FAKE, rot=64,
              layout=1, cos=FAKE, sin=FAKE, max_pos=64, status=None, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(x=None), BAD), (dict(qo=None), BAD), (dict(slots=None), BAD), (dict(pos=None), BAD), (dict(m=-1), BAD),
    (dict(xs=2559), BAD), (dict(qos=511), BAD), (dict(nq=0), BAD), (dict(layer=2), BAD), (dict(layer=-1), BAD),
    (dict(rot=130), BAD), (dict(rot=3), BAD), (dict(layout=-1), NOT), (dict(cos=None), BAD), (dict(max_pos=0), BAD),
    (dict(slots=FAKE + 4), BAD), (dict(x=FAKE + 1), BAD), (dict(status=FAKE + 1), BAD), (dict(qos=2560), AF_OK),
    (dict(m=0, x=None), AF_OK)])
def test_append_refusals(changes, status):
    if status == AF_OK:
        changes = {**changes, "m": 0}
    assert call("af_paged_rope_append_rows", {**APPEND, "pool": pool()}, **changes) == status


@pytest.mark.parametrize("changes,status", [
    (dict(base=None), BAD), (dict(base=FAKE + 8), BAD), (dict(block_size=12), NOT), (dict(dtype=2), NOT),
    (dict(flags=2), BAD), (dict(total_blocks=0), BAD), (dict(n_kv_heads=0), BAD), (dict(head_dim=0), BAD),
    (dict(n_kv_heads=1, head_dim=4), NOT)])
def test_pool_refusals(changes, status):
    assert call("af_paged_rope_append_rows", {**APPEND, "pool": pool(**changes)}) == status
    assert call("af_kv_compact", {**COMPACT, "pool": pool(**changes)}) == status


def test_append_refuses_fp8_without_scales():
    assert call("af_paged_rope_append_rows", {**APPEND, "pool": pool(dtype=AF_KV_FP8_E4M3)}) == BAD


COMPACT = dict(pool=None, src=FAKE, dst=FAKE, max_blocks=4, n=2, keep=FAKE, start=FAKE, first=FAKE, max_rows=9,
               rot=64, layout=0, cos=FAKE, sin=FAKE, max_pos=64, factor=1.0, status=None, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(src=None), BAD), (dict(dst=None), BAD), (dict(keep=None), BAD), (dict(start=None), BAD),
    (dict(first=None), BAD), (dict(max_blocks=0), BAD), (dict(n=-1), BAD), (dict(max_rows=-1), BAD),
    (dict(rot=-2), BAD), (dict(rot=3), BAD), (dict(rot=130), BAD), (dict(layout=2), NOT), (dict(cos=None), BAD),
    (dict(sin=FAKE + 8), BAD), (dict(max_pos=0), BAD), (dict(factor=0.0), BAD), (dict(factor=-1.0), BAD),
    (dict(factor=float("nan")), BAD), (dict(factor=float("inf")), BAD), (dict(keep=FAKE + 2), BAD),
    (dict(status=FAKE + 2), BAD), (dict(n=65536), NOT), (dict(n=0), AF_OK), (dict(max_rows=0), AF_OK)])
def test_compact_refusals(changes, status):
    assert call("af_kv_compact", {**COMPACT, "pool": pool()}, **changes) == status


# ---- tables ------------------------------------------------------------------------------------
def test_table_refusals():
    lib = atomflow_amd.lib()
    f = np.ones(64)
    args = dict(cos=FAKE, sin=FAKE, first=0, rows=4, rot=128, f=f.ctypes.data, factor=1.0, stream=None)
    for changes, status in [(dict(f=None), BAD), (dict(first=-1), BAD), (dict(rows=-1), BAD), (dict(rot=0), BAD),
                            (dict(rot=7), BAD), (dict(rot=258), NOT), (dict(first=1 << 31), NOT),
                            (dict(factor=float("nan")), BAD), (dict(cos=None), BAD), (dict(sin=FAKE + 4), BAD),
                            (dict(rows=0, cos=None), AF_OK)]:
        assert lib.af_rope_table_scaled(*{**args, **changes}.values()) == status, changes
    f[3] = np.inf
    assert lib.af_rope_table_scaled(*args.values()) == BAD


@pytest.mark.parametrize("rot", [2, 4, 64, 128, 256])
@pytest.mark.parametrize("kind", ["none", "linear", "ntk", "bands", "yarn"])
def test_frequencies(rot, kind):
    for factor, context, base in ((8.0, 8192, 500000.0), (1.0, 2048, 10000.0), (32.0, 100, 1000.0)):
        got, mult = kv.rope_frequencies(rot, base, kind, factor, context)
        want, m = frequencies(kind, rot, base, factor, context)
        assert np.allclose(got, want, rtol=1e-13, atol=0) and abs(mult - m) < 1e-14
    assert kv.rope_frequencies(rot, 1e4, kind, 2.0, 4096, attention_factor=1.5)[1] == 1.5


def test_frequencies_refusals():
    def scaling(**changes):
        s = _abi.RopeScaling(4, 8192, 5e5, 8.0, 1.0, 4.0, 32.0, 1.0, 0.0)
        for k, v in changes.items():
            setattr(s, k, v)
        return s

    out, mult = np.zeros(128), ctypes.c_double()
    lib = atomflow_amd.lib()

    def status(s, rot=64, f=out.ctypes.data, m=ctypes.byref(mult)):
        return lib.af_rope_frequencies(None if s is None else ctypes.byref(s), rot, f, m)

    nan = float("nan")
    assert status(scaling()) == AF_OK
    assert status(None) == BAD and status(scaling(), f=None) == BAD
    assert status(scaling(), rot=0) == BAD and status(scaling(), rot=3) == BAD and status(scaling(), rot=258) == NOT
    for changes in (dict(base=0.0), dict(base=nan), dict(factor=0.0), dict(factor=-2.0), dict(factor=nan),
                    dict(attention_factor=-1.0), dict(attention_factor=nan), dict(original_max_pos=0),
                    dict(beta_fast=0.0), dict(beta_slow=nan), dict(base=1.0), dict(kind=3, low_freq_factor=0.0),
                    dict(kind=3, high_freq_factor=1.0), dict(kind=3, original_max_pos=-1)):
        assert status(scaling(**changes)) == BAD, changes
    assert status(scaling(kind=5)) == NOT and status(scaling(kind=-1)) == NOT
    with pytest.raises(ValueError):
        kv.rope_frequencies(64, scaling="other")
    with pytest.raises(atomflow_amd.AfError):
        kv.rope_frequencies(7)
    with pytest.raises(ValueError):
        kv.build_rope_table_scaled(FAKE, FAKE, 0, 1, 64, np.ones(31))
    with pytest.raises(ValueError):
        kv.make_lora(FAKE, FAKE, 1, 8, 8, [])


# ---- plan_compact --------------------------------------------------------------------------------
def slots(tables, rows, bs):
    return [int(tables[r // bs]) * bs + r % bs for r in rows]


def test_plan_against_a_model():
    """Random plans over forked sequences: the moves, carried out row by row on the plan's tables with
    every read before every write, leave each sequence its rows and every other sequence its own; blocks
    are neither lost nor handed out twice."""
    r = np.random.default_rng(17)
    for trial in range(150):
        bs = int(r.choice([8, 16]))
        total = 80
        bm = kv.BlockManager(total, bs)
        cache = np.full(total * bs, -1, np.int64)
        rows = {}  # sequence -> the values that its logical rows hold
        stamp = 0
        for _ in range(int(r.integers(1, 5))):
            s, n = bm.seq_create(), int(r.integers(0, 70))
            bm.seq_extend(s, n)
            rows[s] = list(range(stamp, stamp + n))
            cache[slots(bm.seq_table(s)[0], range(n), bs)] = rows[s]
            stamp += n
        for _ in range(int(r.integers(0, 4))):
            src = int(r.choice(list(rows)))
            rows[bm.seq_fork(src)] = list(rows[src])
        for _ in range(3):
            some = [int(s) for s in r.permutation(list(rows))[:int(r.integers(0, len(rows) + 1))]]
            keeps = []
            for s in some:
                n = len(rows[s])
                keep = np.nonzero(r.random(n) < r.choice([0.1, 0.5, 0.95, 1.0]))[0]
                keeps.append(keep[:int(r.integers(0, len(keep) + 1))] if r.random() < 0.3 else keep)
            free = bm.num_free_blocks()
            before = {s: bm.seq_table(s) for s in rows}
            plan = bm.plan_compact(some, keeps)
            if not isinstance(plan, dict):
                assert plan == AF_ERR_POOL_EXHAUSTED
                assert bm.num_free_blocks() == free and {s: bm.seq_table(s) for s in rows} == before
                continue
            old = cache.copy()
            written = []
            for i, s in enumerate(some):
                part = plan["keep"][plan["start"][i]:plan["start"][i + 1]]
                to = plan["first"][i] + np.arange(len(part))
                assert len(part) <= plan["max_rows"] and np.all(part >= to) and np.all(np.diff(part) > 0)
                dst = slots(plan["dst_tables"][i], to, bs)
                cache[dst] = old[slots(plan["src_tables"][i], part, bs)]
                written += dst
                rows[s] = [rows[s][k] for k in keeps[i]]
            assert len(set(written)) == len(written)
            for s in rows:
                assert bm.seq_len(s) == len(rows[s])
                assert list(cache[slots(bm.seq_table(s)[0], range(len(rows[s])), bs)]) == rows[s]
        held = {}
        for s in rows:
            for b in bm.seq_table(s)[0]:
                held[b] = held.get(b, 0) + 1
        assert all(bm.ref_count(b) == held.get(b, 0) for b in range(total))
        assert bm.num_free_blocks() == total - len(held)
        for s in rows:  # appends go on from there
            assert bm.seq_append(s)[0] == len(rows[s]) if bm.num_free_blocks() else True
        bm.close()


def test_plan_leaves_held_blocks():
    """A copy source that is held until its copy has run is not written in place."""
    bm = kv.BlockManager(8, 8)
    s = bm.seq_create()
    bm.seq_extend(s, 20)
    old, _ = bm.seq_table(s)
    bm.hold_copy_source(old[0])
    plan = bm.plan_compact([s], [[3, 4, 19]])
    assert plan["dst_tables"][0][0] not in old and plan["start"][-1] == 3
    assert bm.num_free_blocks() == 8 - 1 - 1  # the new block, and the held one
    bm.release_copy_sources()
    assert bm.num_free_blocks() == 7


def test_plan_refusals():
    bm = kv.BlockManager(6, 8)
    s, t = bm.seq_create(), bm.seq_create()
    bm.seq_extend(s, 20)
    u = bm.seq_fork(s)
    before = bm.seq_table(s)
    assert bm.plan_compact([s, 99], [[0], []]) == AF_ERR_BAD_SEQUENCE
    assert bm.plan_compact([s, s], [[0], [0]]) == AF_ERR_INVALID_ARG
    assert bm.plan_compact([s], [[0, 20]]) == AF_ERR_OUT_OF_RANGE
    assert bm.plan_compact([s], [[-1, 3]]) == AF_ERR_OUT_OF_RANGE
    assert bm.plan_compact([s], [[3, 3]]) == AF_ERR_INVALID_ARG
    assert bm.plan_compact([s], [[4, 3]]) == AF_ERR_INVALID_ARG
    assert bm.plan_compact([s], [[4]], max_blocks=2) == AF_ERR_OUT_OF_RANGE
    assert bm.plan_compact([s, u], [np.arange(1, 20)] * 2) == AF_ERR_POOL_EXHAUSTED  # 6 new blocks of 3
    assert bm.seq_table(s) == before and bm.seq_table(u) == before and bm.num_free_blocks() == 3
    with pytest.raises(ValueError):
        bm.plan_compact([s], [])
    plan = bm.plan_compact([t, s], [[], np.arange(9)])  # cut at the end: nothing moves
    assert plan["max_rows"] == 0 and bm.seq_len(s) == 9 and bm.seq_len(u) == 20 and bm.num_free_blocks() == 3
    assert bm.plan_compact([], [])["max_rows"] == 0
