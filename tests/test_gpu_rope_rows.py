"""Rotary positions in other forms on the GPU (af_rope_table_scaled, af_rope_rows,
af_paged_rope_append_rows) against the same operators in 64 bits, within bounds that count each
rounding (rows_ref)."""
import numpy as np
import pytest

import atomflow_amd
import oracle
from atomflow_amd import AF_KV_FP16, AF_KV_FP8_E4M3, AF_ROPE_HALF, AF_ROPE_INTERLEAVED
from atomflow_amd import device as dev
from atomflow_amd import kv
from rows_ref import EPS24, Rows, assert_fp8, e4m3_decode, frequencies, table, turn, turn_bound

pytestmark = pytest.mark.gpu
LAYOUTS = [AF_ROPE_HALF, AF_ROPE_INTERLEAVED]


def say(msg):
    print(f"[case] {msg}", flush=True)


def up(a):
    return dev.DeviceBuffer.from_array(a)


def rows16(m, n, seed):
    return np.random.default_rng(seed).standard_normal((m, n)).astype(np.float16)


def tables(max_pos, rot):
    c, s = table(max_pos, rot)
    return c, s, up(c), up(s)


# ---- the table ---------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["none", "linear", "ntk", "bands", "yarn"])
@pytest.mark.parametrize("rot,first,rows", [(128, 0, 513), (64, 131000, 100), (2, 5, 7), (96, 999983, 33),
                                            (18, 0, 70), (256, 1 << 21, 9), (128, 77, 1)])
def test_table(gpu, kind, rot, first, rows):
    say(f"table {kind} rot={rot} first={first} rows={rows}")
    freq, mult = kv.rope_frequencies(rot, 500000.0, kind, 8.0, 8192)
    want, factor = frequencies(kind, rot, 500000.0, 8.0, 8192)
    assert np.allclose(freq, want, rtol=1e-14, atol=0) and abs(mult - factor) < 1e-15
    c = Rows(up, np.float32, rows, rot // 2)
    s = Rows(up, np.float32, rows, rot // 2)
    kv.build_rope_table_scaled(c.ptr, s.ptr, first, rows, rot, freq, mult)
    angle = (first + np.arange(rows, dtype=np.longdouble))[:, None] * freq.astype(np.longdouble)
    for got, f in ((c.get(), np.cos), (s.get(), np.sin)):
        exact = (f(angle) * mult).astype(np.float64)
        # half a step of fp32, the series' end, and the turns' rounding (angles below 2^22)
        bound = EPS24 * np.abs(exact) + mult * (1e-11 + np.abs(angle.astype(np.float64)) * 2.0 ** -51)
        assert np.all(np.abs(got - exact) <= bound)


def test_table_captured(gpu):
    """A captured launch keeps the angles that it was given; replays after eager work agree."""
    say("table, captured")
    st = dev.Stream()
    freq, mult = kv.rope_frequencies(64, 10000.0, "yarn", 4.0, 4096)
    c, s = up(np.zeros((50, 32), np.float32)), up(np.zeros((50, 32), np.float32))
    kv.build_rope_table_scaled(c, s, 1000, 50, 64, freq, mult, stream=st)
    want = c.download(np.float32, stream=st), s.download(np.float32, stream=st)
    mine = freq.copy()
    g = dev.Graph.capture(st, lambda: kv.build_rope_table_scaled(c, s, 1000, 50, 64, mine, mult, stream=st))
    mine[:] = 0
    for _ in range(3):
        c.fill_u32(0, st), s.fill_u32(0, st)
        g.launch(st)
        assert np.array_equal(c.download(np.float32, stream=st), want[0])
        assert np.array_equal(s.download(np.float32, stream=st), want[1])
    g.destroy()
    st.destroy()


# ---- rows ----------------------------------------------------------------------------------------
SHAPES = [  # q heads, k heads, head_dim, rot_dim
    (24, 8, 128, 128), (4, 1, 64, 32), (3, 3, 80, 32), (5, 2, 96, 40), (2, 1, 20, 6), (1, 0, 8, 8),
    (7, 1, 72, 24), (1, 1, 512, 256), (2, 2, 2, 2), (33, 5, 16, 16), (9, 4, 128, 20)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("nq,nk,hd,rot", SHAPES)
@pytest.mark.parametrize("m,off", [(1, 0), (5, 1), (130, 0), (37, 4)])
def test_rope_rows(gpu, layout, nq, nk, hd, rot, m, off):
    say(f"rope rows layout={layout} {nq}+{nk} heads of {hd}, {rot} turn, m={m}, offset {off}")
    max_pos = 700
    c, s, dc, ds = tables(max_pos, rot)
    pos = np.random.default_rng(m).integers(0, max_pos, m).astype(np.int32)
    xq, xk = rows16(m, nq * hd, m + hd), rows16(m, max(nk, 1) * hd, m + hd + 1)
    pad = off
    q = Rows(up, np.float16, m, nq * hd, nq * hd + pad, off, xq)
    k = Rows(up, np.float16, m, max(nk, 1) * hd, max(nk, 1) * hd + 2 * pad, off, xk)
    qo = Rows(up, np.float16, m, nq * hd, nq * hd + 3 * pad, off)
    ko = Rows(up, np.float16, m, max(nk, 1) * hd, max(nk, 1) * hd, off)
    dp = up(pos)

    def call(q_out, k_out, inverse=False):
        kv.launch_rope_rows(q.ptr, q.stride, q_out.ptr, q_out.stride, nq, k.ptr if nk else None, k.stride,
                            k_out.ptr if nk else None, k_out.stride, nk, m, hd, rot, layout, dc, ds, max_pos,
                            positions=dp, inverse=inverse)

    for inverse in (False, True):
        call(qo, ko, inverse)
        for heads, x, out in ((nq, xq, qo), (nk, xk, ko)):
            if not heads:
                continue
            y, mag = turn(x.reshape(m, heads, hd), c[pos], -s[pos] if inverse else s[pos], rot, layout)
            got = out.get().reshape(m, heads, hd).astype(np.float64)
            assert np.all(np.abs(got - y)[..., :rot] <= turn_bound(y, mag)[..., :rot])
            assert np.array_equal(got[..., rot:], x.reshape(m, heads, hd)[..., rot:].astype(np.float64))
    # in place: the same bits as out of place
    call(qo, ko)
    call(q, k)
    assert np.array_equal(q.get().view(np.uint16), qo.get().view(np.uint16))
    if nk:
        assert np.array_equal(k.get().view(np.uint16), ko.get().view(np.uint16))


def test_rope_rows_is_rope(gpu):
    """Halves over the whole head: af_rope's bits (and p0 is the first row's position)."""
    say("rope rows against af_rope")
    m, nq, nk, hd, max_pos = 70, 24, 8, 128, 256
    c, s, dc, ds = tables(max_pos, hd)
    xq, xk = rows16(m, nq * hd, 1), rows16(m, nk * hd, 2)
    q, k, q2, k2 = up(xq), up(xk), up(xq), up(xk)
    kv.launch_rope(q, k, dc.ptr + 60 * hd // 2 * 4, ds.ptr + 60 * hd // 2 * 4, m, nk, nq, hd)
    kv.launch_rope_rows(q2, nq * hd, q2, nq * hd, nq, k2, nk * hd, k2, nk * hd, nk, m, hd, hd, AF_ROPE_HALF,
                        dc, ds, max_pos, p0=60)
    assert np.array_equal(q.download(np.uint16), q2.download(np.uint16))
    assert np.array_equal(k.download(np.uint16), k2.download(np.uint16))


def test_rope_rows_many(gpu):
    """Enough rows that a thread walks over several heads; 64-bit offsets are exercised elsewhere."""
    say("rope rows, 5000 rows of 40 heads")
    m, nq, nk, hd, rot, max_pos = 5000, 32, 8, 128, 64, 8192
    c, s, dc, ds = tables(max_pos, rot)
    x = rows16(m, (nq + nk) * hd, 3)
    d = up(x)
    for layout in LAYOUTS:
        out = dev.DeviceBuffer(x.nbytes)
        kv.launch_rope_rows(d, (nq + nk) * hd, out, (nq + nk) * hd, nq, d.ptr + nq * hd * 2, (nq + nk) * hd,
                            out.ptr + nq * hd * 2, (nq + nk) * hd, nk, m, hd, rot, layout, dc, ds, max_pos, p0=17)
        y, mag = turn(x.reshape(m, -1, hd), c[17:17 + m], s[17:17 + m], rot, layout)
        got = out.download(np.float16).reshape(m, -1, hd).astype(np.float64)
        assert np.all(np.abs(got - y) <= turn_bound(y, mag))


def test_rope_rows_out_of_range(gpu):
    say("rope rows, positions out of range")
    m, nq, hd, rot, max_pos = 9, 3, 64, 32, 50
    c, s, dc, ds = tables(max_pos, rot)
    pos = np.array([0, 49, 50, -1, 7, 2 ** 31 - 1, -2 ** 31, 3, 4], np.int32)
    x = rows16(m, nq * hd, 4)
    for fill in (0, 1):
        st = up(np.zeros(1, np.int32))
        d, out = up(x), up(np.zeros_like(x))
        p = pos if fill else np.clip(pos, 0, 49).astype(np.int32)
        kv.launch_rope_rows(d, nq * hd, out, nq * hd, nq, None, 0, None, 0, 0, m, hd, rot, AF_ROPE_INTERLEAVED,
                            dc, ds, max_pos, positions=up(p), d_status=st)
        bad = (p < 0) | (p >= max_pos)
        at = np.where(bad, 0, p)
        y, mag = turn(x.reshape(m, nq, hd), c[at], s[at], rot, 1)
        y[bad] = x.reshape(m, nq, hd)[bad]
        got = out.download(np.float16).reshape(m, nq, hd)
        assert np.all(np.abs(got.astype(np.float64) - y) <= turn_bound(y, mag) * ~bad[:, None, None])
        assert st.download(np.int32)[0] == (atomflow_amd.AF_ERR_OUT_OF_RANGE if bad.any() else 0)


def test_rope_rows_not_finite(gpu):
    """A NaN or an infinity stays within its pair."""
    say("rope rows, NaN and infinities")
    m, nq, hd, rot = 6, 2, 32, 16
    c, s, dc, ds = tables(64, rot)
    x = rows16(m, nq * hd, 5).reshape(m, nq, hd)
    x[1, 0, 3], x[2, 1, 9], x[3, 0, 31], x[4, 1, 0] = np.nan, np.inf, np.nan, -np.inf
    for layout in LAYOUTS:
        out = up(np.zeros_like(x))
        kv.launch_rope_rows(up(x), nq * hd, out, nq * hd, nq, None, 0, None, 0, 0, m, hd, rot, layout, dc, ds, 64,
                            p0=20)
        with np.errstate(invalid="ignore"):
            y, _ = turn(x, c[20:26], s[20:26], rot, layout)
        got = out.download(np.float16).reshape(x.shape).astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(y))
        assert np.array_equal(got[np.isinf(y)], y[np.isinf(y)]) and np.isfinite(got[np.isfinite(y)]).all()


# ---- append --------------------------------------------------------------------------------------
POOLS = [  # q heads, kv heads, head_dim, rot_dim, block size
    (24, 8, 128, 128, 16), (4, 2, 64, 32, 8), (3, 1, 80, 80, 16), (5, 4, 20, 6, 32), (2, 2, 24, 8, 8)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("nq,nk,hd,rot,bs", POOLS)
@pytest.mark.parametrize("m", [1, 45, 300])
def test_append(gpu, fp8, layout, nq, nk, hd, rot, bs, m):
    say(f"append fp8={fp8} layout={layout} {nq}+{nk} heads of {hd}, {rot} turn, m={m}")
    if (nk * hd * (1 if fp8 else 2)) % 16:
        pytest.skip("rows of whole 16 bytes")
    max_pos, layers, blocks = 900, 3, -(-m // bs) + 3
    c, s, dc, ds = tables(max_pos, rot)
    r = np.random.default_rng(m + hd)
    pos = r.integers(0, max_pos, m).astype(np.int32)
    slots = r.permutation(blocks * bs)[:m].astype(np.int64)
    if m > 2:
        slots[m // 2] = -1  # padding
    width = (nq + 2 * nk) * hd
    x = rows16(m, width, m + 7)
    qkv = Rows(up, np.float16, m, width, width + 8, 0, x)
    qo = Rows(up, np.float16, m, nq * hd, nq * hd + 8, 0)
    dtype = np.uint8 if fp8 else np.float16
    before = (r.integers(0, 120, (layers, 2, blocks * bs, nk, hd)).astype(np.uint8) if fp8
              else r.standard_normal((layers, 2, blocks * bs, nk, hd)).astype(np.float16))
    scales = (0.004 + 0.02 * r.random((layers, 2, nk))).astype(np.float32)
    d_pool, d_scales, st = up(before), up(scales), up(np.zeros(1, np.int32))
    pool = kv.make_pool(d_pool.ptr, AF_KV_FP8_E4M3 if fp8 else AF_KV_FP16, bs, layers, nk, hd, blocks,
                        scales=d_scales.ptr if fp8 else None)
    kv.launch_paged_rope_append_rows(qkv.ptr, qkv.stride, m, qo.ptr, qo.stride, nq, pool, 1, up(slots), up(pos),
                                     rot, layout, dc, ds, max_pos, d_status=st)
    heads = x.reshape(m, nq + 2 * nk, hd)
    y, mag = turn(heads[:, :nq + nk], c[pos], s[pos], rot, layout)
    got = qo.get().reshape(m, nq, hd).astype(np.float64)
    assert np.all(np.abs(got - y[:, :nq]) <= turn_bound(y, mag)[:, :nq])
    assert np.array_equal(qkv.get().view(np.uint16), x.view(np.uint16)), "the rows are only read"
    after = d_pool.download(dtype, before.shape)
    cached = slots >= 0
    k, ky, kmag = after[1, 0][slots[cached]], y[cached, nq:], mag[cached, nq:]
    v, vx = after[1, 1][slots[cached]], heads[cached, nq + nk:].astype(np.float64)
    if fp8:
        ks, vs = (scales[1, i].astype(np.float64)[:, None] for i in (0, 1))
        assert_fp8(k, ky / ks, 1.01 * EPS24 * (kmag + 2 * np.abs(ky)) / ks)
        assert_fp8(v, vx / vs, 1.01 * EPS24 * np.abs(vx) / vs)
    else:
        assert np.all(np.abs(k.astype(np.float64) - ky) <= turn_bound(ky, kmag))
        assert np.array_equal(v.astype(np.float64), vx)
    want = before.copy()
    want[1, 0][slots[cached]], want[1, 1][slots[cached]] = k, v
    assert after.tobytes() == want.tobytes(), "other rows changed"
    assert st.download(np.int32)[0] == 0
    # in place: Q turned within qkv, K and V left
    kv.launch_paged_rope_append_rows(qkv.ptr, qkv.stride, m, qkv.ptr, qkv.stride, nq, pool, 1, up(slots),
                                     up(pos), rot, layout, dc, ds, max_pos)
    z = qkv.get().reshape(m, -1, hd)
    assert np.array_equal(z[:, :nq].view(np.uint16), qo.get().reshape(m, nq, hd).view(np.uint16))
    assert np.array_equal(z[:, nq:].view(np.uint16), heads[:, nq:].view(np.uint16))
    assert d_pool.download(dtype, before.shape).tobytes() == want.tobytes()


def test_append_is_paged_rope_append(gpu):
    """fp16, halves over the whole head: af_paged_rope_append's rows, bit for bit."""
    say("append against af_paged_rope_append")
    m, nq, nk, hd, bs, blocks = 33, 24, 8, 128, 16, 5
    c, s, dc, ds = tables(128, hd)
    x = rows16(m, (nq + 2 * nk) * hd, 9)
    slots = np.random.default_rng(2).permutation(blocks * bs)[:m].astype(np.int64)
    pos = np.arange(m, dtype=np.int32) + 40
    pools = []
    for own in (False, True):
        buf = up(np.zeros((1, 2, blocks * bs, nk, hd), np.float16))
        pool = kv.make_pool(buf.ptr, AF_KV_FP16, bs, 1, nk, hd, blocks)
        d = up(x)
        if own:
            kv.launch_paged_rope_append_rows(d, x.shape[1], m, d, x.shape[1], nq, pool, 0, up(slots), up(pos), hd,
                                             AF_ROPE_HALF, dc, ds, 128)
        else:
            kv.launch_paged_rope_append(d, m, pool, 0, up(slots), up(pos), dc, ds, 128, nq)
        dev.synchronize()
        pools.append((buf.download(np.uint16), d.download(np.uint16).reshape(m, -1)[:, :nq * hd]))
    assert np.array_equal(pools[0][0], pools[1][0]) and np.array_equal(pools[0][1], pools[1][1])


def test_append_out_of_range(gpu):
    """Slots past the pool and positions past the tables cache nothing and say so; slot -1 alone
    does not."""
    say("append, slots and positions out of range")
    m, nq, nk, hd, bs, blocks, max_pos = 8, 2, 1, 64, 16, 2, 40
    c, s, dc, ds = tables(max_pos, hd)
    x = rows16(m, (nq + 2 * nk) * hd, 11)
    pos = np.arange(m, dtype=np.int32)
    for bad_slot, bad_pos, status in ((-1, 3, 0), (32, 3, -4), (-2, 3, -4), (2 ** 40, 3, -4), (5, 40, -4),
                                      (5, -1, -4), (-1, 99, -4)):
        slots = np.arange(10, 10 + m).astype(np.int64)
        slots[4], pos[4] = bad_slot, bad_pos
        buf = up(np.full((1, 2, blocks * bs, nk, hd), 7.0, np.float16))
        pool = kv.make_pool(buf.ptr, AF_KV_FP16, bs, 1, nk, hd, blocks)
        st, qo = up(np.zeros(1, np.int32)), up(np.zeros((m, nq * hd), np.float16))
        kv.launch_paged_rope_append_rows(up(x), x.shape[1], m, qo, nq * hd, nq, pool, 0, up(slots), up(pos), hd,
                                         AF_ROPE_HALF, dc, ds, max_pos, d_status=st)
        dev.synchronize()
        assert st.download(np.int32)[0] == status
        got = buf.download(np.float16, (2, blocks * bs, nk, hd))
        written = np.zeros(blocks * bs, bool)
        written[np.delete(slots, 4)] = True
        assert np.all(got[:, ~written] == 7.0) and not np.any(got[:, written] == 7.0)
        q = qo.download(np.float16, (m, nq, hd))[4].astype(np.float64)
        ok = 0 <= bad_pos < max_pos
        y, mag = turn(x.reshape(m, -1, hd)[4:5, :nq], c[[bad_pos if ok else 0]], s[[bad_pos if ok else 0]], hd, 0)
        if ok:
            assert np.all(np.abs(q - y[0]) <= turn_bound(y, mag)[0])
        else:
            assert np.array_equal(q, x.reshape(m, -1, hd)[4, :nq].astype(np.float64))


def test_fp8_of_every_half(gpu):
    """V with scale 1: every fp16 value's code is the nearest E4M3 value, ties to even, clamped;
    NaN stays NaN."""
    say("fp8 codes of every fp16 value")
    hd, bs = 128, 16
    x = np.arange(65536, dtype=np.uint32).astype(np.uint16).view(np.float16).reshape(512, hd)
    rows = np.concatenate([np.zeros((512, 2 * hd), np.float16), x], axis=1)
    buf = up(np.zeros((1, 2, 512, 1, hd), np.uint8))
    scales = up(np.ones((1, 2, 1), np.float32))
    pool = kv.make_pool(buf.ptr, AF_KV_FP8_E4M3, bs, 1, 1, hd, 32, scales=scales.ptr)
    c, s, dc, ds = tables(8, hd)
    kv.launch_paged_rope_append_rows(up(rows), 3 * hd, 512, up(np.zeros((512, hd), np.float16)), hd, 1, pool, 0,
                                     up(np.arange(512, dtype=np.int64)), up(np.zeros(512, np.int32)), hd,
                                     AF_ROPE_HALF, dc, ds, 8)
    dev.synchronize()
    codes = buf.download(np.uint8, (2, 512, hd))[1]
    nan = np.isnan(x)
    assert np.all((codes[nan] & 0x7f) == 0x7f)
    clamped = np.clip(x[~nan].astype(np.float32), -448, 448)
    want = oracle.e4m3_encode(clamped)
    assert np.array_equal(e4m3_decode(codes[~nan]), e4m3_decode(np.asarray(want, np.uint8)))


def test_append_far_slots(gpu):
    """A slot whose byte offset passes 32 bits, in a layer whose slab does too."""
    say("append, far slots")
    nk, hd, bs, blocks, layers = 8, 128, 16, 140000, 1
    buf = dev.DeviceBuffer(layers * 2 * blocks * bs * nk * hd * 2)
    pool = kv.make_pool(buf.ptr, AF_KV_FP16, bs, layers, nk, hd, blocks)
    c, s, dc, ds = tables(16, hd)
    x = rows16(2, 3 * nk * hd, 12)
    slots = np.array([blocks * bs - 1, 2 ** 21 + 5], np.int64)
    kv.launch_paged_rope_append_rows(up(x), x.shape[1], 2, up(np.zeros((2, nk * hd), np.float16)), nk * hd, nk,
                                     pool, 0, up(slots), up(np.zeros(2, np.int32)), hd, AF_ROPE_HALF, dc, ds, 16)
    dev.synchronize()
    row = nk * hd * 2
    for i, slot in enumerate(slots):
        for w in (0, 1):
            got = buf.download(np.uint16, (nk * hd,), offset=(w * blocks * bs + int(slot)) * row)
            assert np.array_equal(got, x[i, (1 + w) * nk * hd:(2 + w) * nk * hd].view(np.uint16))
