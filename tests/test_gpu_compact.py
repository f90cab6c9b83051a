"""Rows dropped out of cached sequences on the GPU (af_kv_compact, with BlockManager's
plan_compact) against the same moves in 64 bits (rows_ref): every row of the pool is compared, what does
not turn bit for bit."""
import numpy as np
import pytest

import atomflow_amd
from atomflow_amd import AF_KV_FP16, AF_KV_FP8_E4M3, AF_ROPE_HALF, AF_ROPE_INTERLEAVED
from atomflow_amd import device as dev
from atomflow_amd import kv
from rows_ref import assert_compact, table

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


def up(a):
    return dev.DeviceBuffer.from_array(a)


def values(shape, fp8, seed):
    r = np.random.default_rng(seed)
    if fp8:
        c = r.integers(0, 256, shape).astype(np.uint8)
        return np.where((c & 0x7f) == 0x7f, 0x38, c).astype(np.uint8)  # no NaN
    return r.standard_normal(shape).astype(np.float16)


class Pool:
    def __init__(self, layers, blocks, bs, heads, hd, fp8, seed):
        self.bs, self.fp8 = bs, fp8
        self.host = values((layers, 2, blocks * bs, heads, hd), fp8, seed)
        self.buf = up(self.host)
        self.desc = kv.make_pool(self.buf.ptr, AF_KV_FP8_E4M3 if fp8 else AF_KV_FP16, bs, layers, heads, hd,
                                 blocks)

    def get(self):
        return self.buf.download(self.host.dtype, self.host.shape)


def launch(pool, src, dst, keeps, first, rot, layout, cos, sin, factor=1.0, status=None, max_rows=None,
           stream=None):
    start = np.zeros(len(keeps) + 1, np.int32)
    start[1:] = np.cumsum([len(k) for k in keeps])
    keep = np.concatenate([np.asarray(k, np.int32) for k in keeps] + [np.zeros(1, np.int32)])
    dc, ds = (up(cos), up(sin)) if rot else (None, None)
    bufs = [up(np.ascontiguousarray(t, np.int32)) for t in (src, dst, keep, start, first)]
    kv.kv_compact(pool.desc, bufs[0], bufs[1], np.asarray(src).shape[1], len(keeps), bufs[2], bufs[3], bufs[4],
                  max([len(k) for k in keeps] + [0]) if max_rows is None else max_rows, rot, layout, dc, ds,
                  0 if not rot else cos.shape[0], factor, d_status=status, stream=stream)
    dev.synchronize()


def rows_of(kind, n, r):
    """Logical rows that stay, of n."""
    if kind == "half":
        return np.nonzero(r.random(n) < 0.5)[0]
    if kind == "most":
        return np.nonzero(r.random(n) < 0.97)[0]
    if kind == "few":
        return np.nonzero(r.random(n) < 0.02)[0]
    if kind == "window":
        return np.concatenate([np.arange(min(4, n)), np.arange(max(4, n - n // 3), n)])
    return np.arange(1, n)  # all but the first: every row moves by one


SHAPES = [  # layers, kv heads, head_dim, rot, block size
    (2, 8, 128, 128, 16), (1, 2, 64, 32, 8), (2, 4, 80, 80, 16), (1, 3, 16, 8, 32), (1, 8, 20, 6, 16),
    (1, 1, 512, 256, 8), (2, 5, 96, 48, 16), (1, 8, 2, 2, 8)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layout", [AF_ROPE_HALF, AF_ROPE_INTERLEAVED])
@pytest.mark.parametrize("layers,heads,hd,rot,bs", SHAPES)
@pytest.mark.parametrize("kind", ["half", "most", "few", "window", "one"])
def test_in_place(gpu, fp8, layout, layers, heads, hd, rot, bs, kind):
    say(f"compact in place fp8={fp8} layout={layout} {layers}x{heads}x{hd} rot={rot} keep {kind}")
    if heads * hd * (1 if fp8 else 2) % 16:
        pytest.skip("rows of whole 16 bytes")
    lengths = [1, 700, bs, 0, 333, 2 * bs + 1]
    r = np.random.default_rng(hd + bs)
    pages = [-(-n // bs) for n in lengths]
    blocks = sum(pages) + 4
    pool = Pool(layers, blocks, bs, heads, hd, fp8, hd)
    ids = r.permutation(blocks).astype(np.int32)
    tables = np.zeros((len(lengths), max(pages)), np.int32)
    for i, p in enumerate(pages):
        tables[i, :p] = ids[sum(pages[:i]):sum(pages[:i + 1])]
    keeps = [rows_of(kind, n, r) for n in lengths]
    first = [int(np.argmax(k != np.arange(len(k)))) if len(k) and (k != np.arange(len(k))).any() else len(k)
             for k in keeps]
    moved = [k[f:] for k, f in zip(keeps, first)]
    cos, sin = table(max(lengths), rot)
    launch(pool, tables, tables, moved, first, rot, layout, cos, sin)
    moves = list(zip(tables, tables, first, moved))
    assert_compact(pool.get(), pool.host, moves, bs, rot, layout, cos, sin)


@pytest.mark.parametrize("rot,factor", [(0, 1.0), (128, 1.25), (64, 1.0)])
def test_forms(gpu, rot, factor):
    """Without a turn every bit stays; a table's own factor is taken out; 28 layers."""
    say(f"compact rot={rot} factor={factor}")
    r = np.random.default_rng(rot)
    bs, n = 16, 500
    pool = Pool(28, 40, bs, 8, 128, False, 3)
    tables = r.permutation(40)[None, :32].astype(np.int32)
    keep = rows_of("half", n, r)
    cos, sin = table(n, rot) if rot else (None, None)
    if rot:
        cos, sin = (cos * np.float32(factor)), (sin * np.float32(factor))
    launch(pool, tables, tables, [keep], [0], rot, 0, cos, sin, factor)
    assert_compact(pool.get(), pool.host, [(tables[0], tables[0], 0, keep)], bs, rot, 0, cos, sin, factor)


def test_many_sequences_and_long(gpu):
    """More workgroups than the device holds at once, and one sequence of many chunks, in place."""
    say("compact 40 sequences of up to 3000 rows")
    r = np.random.default_rng(5)
    bs, seqs, most = 16, 40, 3000
    pages = -(-most // bs)
    pool = Pool(1, seqs * pages, bs, 4, 128, True, 9)
    tables = r.permutation(seqs * pages).reshape(seqs, pages).astype(np.int32)
    keeps = [rows_of("most" if i % 2 else "half", int(r.integers(0, most + 1)), r) for i in range(seqs)]
    cos, sin = table(most, 128)
    launch(pool, tables, tables, keeps, [0] * seqs, 128, 0, cos, sin)
    moves = [(tables[i], tables[i], 0, keeps[i]) for i in range(seqs)]
    assert_compact(pool.get(), pool.host, moves, bs, 128, 0, cos, sin)


def test_bad_entries(gpu):
    """Rows past the table, blocks outside the pool, rows that would move down or further than the tables
    reach: left out, with a status; the others move."""
    say("compact, entries out of range")
    bs = 16
    cos, sin = table(40, 64)
    tables = np.array([[3, 1, 2, 0]], np.int32)
    good = [5, 9, 17]
    for keep, bad_table, out in (([5, 9, 64], None, 2), ([5, 9, 2 ** 31 - 1], None, 2), ([0, 0, 1], None, 2),
                                 ([5, 9, 60], None, 2), ([5, 9, 33], 2, 2)):
        for block in ((4, -1, 2 ** 31 - 1, -2 ** 31) if bad_table is not None else (0,)):
            pool = Pool(1, 4, bs, 2, 64, False, 1)
            t = tables.copy()
            if bad_table is not None:
                t[0, bad_table] = block
            st = up(np.zeros(1, np.int32))
            launch(pool, t, t, [keep], [0], 64, 0, cos, sin, status=st)
            assert st.download(np.int32)[0] == atomflow_amd.AF_ERR_OUT_OF_RANGE
            ok = [i for i, k in enumerate(keep) if i != out and k >= i and not (k == 0 and i)]
            want = [(tables[0], tables[0], i, [keep[i]]) for i in ok]
            assert_compact(pool.get(), pool.host, want, bs, 64, 0, cos, sin)
    pool = Pool(1, 4, bs, 2, 64, False, 1)
    st = up(np.zeros(1, np.int32))
    launch(pool, tables, tables, [good], [0], 64, 0, cos, sin, status=st, max_rows=2)
    assert st.download(np.int32)[0] == 0
    assert_compact(pool.get(), pool.host, [(tables[0], tables[0], 0, good[:2])], bs, 64, 0, cos, sin)


def test_captured(gpu):
    """A captured launch reads the rows and tables as they are at each replay."""
    say("compact, captured")
    r = np.random.default_rng(8)
    bs, n = 16, 300
    st = dev.Stream()
    pool = Pool(3, 24, bs, 4, 64, False, 4)
    cos, sin = table(n, 64)
    bufs = [up(np.zeros(s, np.int32)) for s in ((1, 20), (1, 20), (n,), (2,), (1,))]
    dc, ds = up(cos), up(sin)

    def call():
        kv.kv_compact(pool.desc, bufs[0], bufs[1], 20, 1, bufs[2], bufs[3], bufs[4], n, 64, 1, dc, ds, n, stream=st)

    g = dev.Graph.capture(st, call)
    for _ in range(4):
        tables = r.permutation(24)[None, :20].astype(np.int32)
        keep = rows_of("half", int(r.integers(50, n)), r).astype(np.int32)
        for b, a in zip(bufs, (tables, tables, keep, np.array([0, len(keep)], np.int32), np.zeros(1, np.int32))):
            b.upload(a, st)
        before = pool.get()
        g.launch(st)
        st.sync()
        assert_compact(pool.get(), before, [(tables[0], tables[0], 0, keep)], bs, 64, 1, cos, sin)
    g.destroy()
    st.destroy()


def test_plan_in_place_and_forked(gpu):
    """plan_compact over a pool with forks: shared pages stay with the other sequence, and both forks of
    one prompt may be cut in one launch."""
    say("compact, planned")
    bs, hd, heads = 16, 64, 2
    bm = kv.BlockManager(64, bs, 2, heads, hd, AF_KV_FP16)
    pool = Pool(2, 64, bs, heads, hd, False, 12)
    a = bm.seq_create()
    bm.seq_extend(a, 100)
    b = bm.seq_fork(a)
    c = bm.seq_fork(a)
    d = bm.seq_create()
    bm.seq_extend(d, 77)
    r = np.random.default_rng(3)
    logical = {}
    for s, n in ((a, 100), (b, 100), (c, 100), (d, 77)):
        ids, _ = bm.seq_table(s)
        logical[s] = pool.host[:, :, np.array([ids[i // bs] * bs + i % bs for i in range(n)])]
    keeps = {b: rows_of("half", 100, r), c: np.concatenate([np.arange(20), [50, 51, 99]]), d: rows_of("half", 77, r)}
    plan = bm.plan_compact([b, c, d], [keeps[b], keeps[c], keeps[d]])
    bufs = {k: up(np.ascontiguousarray(plan[k])) for k in ("src_tables", "dst_tables", "start", "first")}
    keep = up(plan["keep"])
    kv.kv_compact(pool.desc, bufs["src_tables"], bufs["dst_tables"], plan["src_tables"].shape[1], 3, keep,
                  bufs["start"], bufs["first"], plan["max_rows"])
    got = pool.get()
    for s, rows in [(a, np.arange(100))] + list(keeps.items()):
        assert bm.seq_len(s) == len(rows)
        ids, _ = bm.seq_table(s)
        now = got[:, :, np.array([ids[i // bs] * bs + i % bs for i in range(len(rows))], np.int64)]
        assert np.array_equal(now.view(np.uint16), logical[s][:, :, rows].view(np.uint16))
    bm.close()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layout", [AF_ROPE_HALF, AF_ROPE_INTERLEAVED])
@pytest.mark.parametrize("layers,heads,hd,rot,bs", SHAPES)
def test_new_blocks(gpu, fp8, layout, layers, heads, hd, rot, bs):
    """Into blocks that nobody reads: all of them, or all but the first (then some rows move in place)."""
    say(f"compact into new blocks fp8={fp8} layout={layout} {layers}x{heads}x{hd} rot={rot}")
    if heads * hd * (1 if fp8 else 2) % 16:
        pytest.skip("rows of whole 16 bytes")
    r = np.random.default_rng(hd * 3 + bs)
    lengths = [600, 2 * bs + 1, 350]
    pages = max(-(-n // bs) for n in lengths)
    pool = Pool(layers, 6 * pages, bs, heads, hd, fp8, hd)
    ids = r.permutation(6 * pages).reshape(2, 3, pages).astype(np.int32)
    src, dst = ids[0], ids[1].copy()
    dst[2, 0] = src[2, 0]
    keeps = [rows_of("half", n, r) for n in lengths]
    cos, sin = table(600, rot)
    launch(pool, src, dst, keeps, [0, 0, 0], rot, layout, cos, sin)
    moves = [(src[i], dst[i], 0, keeps[i]) for i in range(3)]
    assert_compact(pool.get(), pool.host, moves, bs, rot, layout, cos, sin)


def test_bound_of_rows_far_above(gpu):
    """max_rows is a bound: far above the sequences' rows, and below a workgroup's share of them."""
    say("compact, max_rows of another order than the rows")
    r = np.random.default_rng(6)
    bs, n = 16, 900
    cos, sin = table(n, 64)
    for kind, most in (("window", 1 << 30), ("half", 1 << 30), ("window", 1 << 20)):
        pool = Pool(1, 60, bs, 2, 64, False, 2)
        tables = r.permutation(60)[None, :57].astype(np.int32)
        keep = rows_of(kind, n, r)
        f = 4 if kind == "window" else 0
        launch(pool, tables, tables, [keep[f:]], [f], 64, 0, cos, sin, max_rows=most)
        assert_compact(pool.get(), pool.host, [(tables[0], tables[0], f, keep[f:])], bs, 64, 0, cos, sin)


def test_far_rows(gpu):
    """Rows whose byte offsets pass 32 bits, of a layer whose slabs do too; in place, and in any order."""
    say("compact, far rows")
    bs, blocks, heads, hd = 16, 70000, 8, 128
    row = heads * hd * 2
    r = np.random.default_rng(1)
    buf = dev.DeviceBuffer(2 * 2 * blocks * bs * row)
    desc = kv.make_pool(buf.ptr, AF_KV_FP16, bs, 2, heads, hd, blocks)
    table_ = np.array([[blocks - 1, 3, blocks - 2, 40000]], np.int32)
    cos, sin = table(64, hd)
    for keep in (np.arange(1, 60), np.arange(40, 62)):
        data = r.standard_normal((2, 2, 64, heads, hd)).astype(np.float16)
        at = lambda w, i: (w * blocks * bs + int(table_[0, i // bs]) * bs + i % bs) * row  # noqa: E731
        for w in range(4):
            for i in range(0, 64, bs):
                buf.upload(data[w // 2, w % 2, i:i + bs], offset=at(w, i))
        launch(type("P", (), {"desc": desc}), table_, table_, [keep], [0], hd, 0, cos, sin)
        got = np.stack([np.stack([buf.download(np.float16, (bs, heads, hd), offset=at(w, i))
                                  for i in range(0, 64, bs)]).reshape(64, heads, hd) for w in range(4)])
        flat = np.arange(4, dtype=np.int32)
        assert_compact(got.reshape(2, 2, 64, heads, hd), data, [(flat, flat, 0, keep)], bs, hd, 0, cos, sin)
