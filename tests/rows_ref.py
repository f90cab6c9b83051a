"""Adapters, rotary positions and cache compaction in 64 bits, for the tests of their GPU operators."""
import numpy as np

from inputs import _e4m3_positive_values, e4m3_encode_np, fp16_ulp

EPS24 = 2.0 ** -24  # half a step of fp32, relative
HALF, INTERLEAVED = 0, 1


class Rows:
    """A host matrix of m rows, `stride` elements apart, `off` elements into a buffer whose other
    bytes must stay as they were; on the device through `upload` (a DeviceBuffer maker)."""

    def __init__(self, upload, dtype, m, n, stride=None, off=0, data=None):
        self.dtype, self.m, self.n, self.off = np.dtype(dtype), m, n, off
        self.stride = n if stride is None else stride
        total = off + max(m, 1) * self.stride + 8
        host = np.full(total * self.dtype.itemsize, 0x5b, np.uint8).view(self.dtype)
        if data is not None:
            self.view(host)[:] = data
        self.before = host.copy()
        self.buf = upload(host)
        self.ptr = self.buf.ptr + off * self.dtype.itemsize

    def view(self, flat):
        return flat[self.off:self.off + self.m * self.stride].reshape(self.m, self.stride)[:, :self.n]

    def get(self):
        """The rows; asserts that nothing around them changed."""
        flat = self.buf.download(self.dtype, (len(self.before),))
        rows = self.view(flat).copy()
        want = self.before.copy()
        self.view(want)[:] = rows
        assert flat.tobytes() == want.tobytes(), "bytes around the rows changed"
        return rows


# ---- rotary positions --------------------------------------------------------------------------
def turn(x, cos, sin, rot, layout):
    """x [..., heads, dim] in 64 bits turned by cos and sin [..., rot / 2]; and the sum of the
    magnitudes of each result's products."""
    x = np.asarray(x, np.float64)
    c, s = (np.asarray(t, np.float64)[..., None, :] for t in (cos, sin))
    y, mag = x.copy(), np.abs(x)
    first = slice(0, rot // 2) if layout == HALF else slice(0, rot, 2)
    second = slice(rot // 2, rot) if layout == HALF else slice(1, rot, 2)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    mag[..., first] = np.abs(a * c) + np.abs(b * s)
    mag[..., second] = np.abs(a * s) + np.abs(b * c)
    return y, mag


def turn_bound(y, mag):
    """Two products and their sum in fp32 (half a step each, of the products' magnitudes at
    most), then one rounding to fp16; second-order terms within 1 %."""
    off = 1.01 * EPS24 * (mag + np.abs(y))
    return off + 0.5 * fp16_ulp(np.abs(y) + off)


def e4m3_decode(codes):
    vals = np.concatenate([_e4m3_positive_values(), [np.nan]])
    return np.where(codes & 0x80, -1.0, 1.0) * vals[codes & 0x7f]


def e4m3_step(v):
    """Spacing of E4M3 values at |v| (2^-9 below the normal range)."""
    a = np.clip(np.abs(v), 2.0 ** -6, 448.0)
    return 2.0 ** (np.floor(np.log2(a)) - 3)


def assert_fp8(codes, y, off):
    """codes of y (64 bits, unclamped), whose fp32 values are off by at most `off`: half a step."""
    want = np.clip(y, -448.0, 448.0)
    nan = np.isnan(y)
    assert np.array_equal((codes & 0x7f) == 0x7f, nan)
    got = e4m3_decode(codes[~nan])
    off = np.broadcast_to(off, y.shape)[~nan]
    err = np.abs(got - want[~nan])
    assert np.all(err <= off + 0.5 * e4m3_step(np.abs(want[~nan]) + off))


def frequencies(kind, rot, base, factor=1.0, context=0, low=1.0, high=4.0, fast=32.0, slow=1.0):
    """Angles per position and the factor on cos and sin, pair by pair."""
    import math
    mult = 1.0
    out = []
    if kind == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    for i in range(rot // 2):
        f = 1.0 / base ** (2 * i / rot)
        if kind == "linear":
            f = f / factor
        if kind == "bands":
            wave = 2 * math.pi / f
            if wave > context / low:
                f = f / factor
            elif wave >= context / high:
                t = (context / wave - low) / (high - low)
                f = (1 - t) * f / factor + t * f
        if kind == "yarn":
            edge = [rot * math.log(context / (2 * math.pi * b)) / (2 * math.log(base))
                    for b in (fast, slow)]
            lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
            t = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = (1 - t) * f + t * f / factor
            mult = 0.1 * math.log(factor) + 1.0
        out.append(f)
    return np.array(out), mult


def table(rows, rot, base=500000.0):
    """A plain fp32 table [rows, rot / 2] of (cos, sin)."""
    angle = np.arange(rows)[:, None] * frequencies("none", rot, base)[0]
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


# ---- adapters ------------------------------------------------------------------------------------
def lora(x, ids, a, b, ranks, scales, slice_ends, y):
    """(result in 64 bits, bound before the last rounding) of the adapters' addition. The bound
    counts a rounding (half a step of fp32) for each term of both sums, 2^-22 of a token's largest
    v for its two fp16 halves, and three for the scale, the product with a power of 2 and y's
    addition; second-order terms within 1 %."""
    x, y = x.astype(np.float64), y.astype(np.float64)
    out, bound = y.copy(), np.zeros_like(y)
    k = x.shape[1]
    begins = [0] + list(slice_ends[:-1])
    for i, ad in enumerate(ids):
        if not 0 <= ad < a.shape[0] or ranks[ad] <= 0:
            continue
        r = min(int(ranks[ad]), a.shape[2])
        sc = float(scales[ad])
        for s, (c0, c1) in enumerate(zip(begins, slice_ends)):
            down = a[ad, s, :r].astype(np.float64)
            up = b[ad, c0:c1, :r].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                v = down @ x[i]
                ev = EPS24 * (k + 8) * (np.abs(down) @ np.abs(x[i])) + 2.0 ** -22 * np.abs(v).max()
                d = up @ (sc * v)
                mag = np.abs(up) @ (abs(sc) * np.abs(v))
                out[i, c0:c1] += d
                bound[i, c0:c1] = 1.01 * (np.abs(up) @ (abs(sc) * ev) + EPS24 * (r + 4) * mag +
                                          EPS24 * (np.abs(y[i, c0:c1]) + np.abs(d)))
    return out, bound


def assert_lora(got, out, bound):
    if got.dtype == np.float16:
        bound = bound + 0.5 * fp16_ulp(np.abs(out) + bound)
    else:
        bound = bound + 1.01 * EPS24 * np.abs(out) + 2.0 ** -149
    err = np.abs(got.astype(np.float64) - out)
    assert np.all(err <= bound), (float((err / bound).max()), np.unravel_index((err / bound).argmax(), err.shape))


# ---- compaction ----------------------------------------------------------------------------------
def places(tables, rows, bs):
    return tables[rows // bs].astype(np.int64) * bs + rows % bs


def compact(pool, moves, bs, rot, layout, cos, sin, factor=1.0):
    """pool [layer, 2, row, head, dim] (fp16, or E4M3 codes) after the moves of one launch:
    [(src table, dst table, first, keep)]. Returns (V and unturned rows exact) the new pool with
    the moved K rows as 64-bit values beside: {(layer, row): ...} arrays, their bound's parts."""
    new = pool.copy()
    turned = []
    for src_t, dst_t, first, keep in moves:
        keep = np.asarray(keep, np.int64)
        if not len(keep):
            continue
        to = first + np.arange(len(keep))
        src, dst = places(src_t, keep, bs), places(dst_t, to, bs)
        new[:, :, dst] = pool[:, :, src]
        if rot:
            moved = keep - to
            some = moved != 0
            k = pool[:, 0][:, src[some]]
            k = e4m3_decode(k) if pool.dtype == np.uint8 else k.astype(np.float64)
            c, s = cos[moved[some]] / factor, -sin[moved[some]] / factor
            y, mag = turn(k, c, s, rot, layout)
            turned.append((dst[some], y, mag))
    return new, turned


def assert_compact(got, pool, moves, bs, rot, layout, cos, sin, factor=1.0):
    new, turned = compact(pool, moves, bs, rot, layout, cos, sin, factor)
    want = new.copy()
    extra = 3 if factor != 1.0 else 0  # 1 / factor, and its products with cos and sin
    for dst, y, mag in turned:
        k = got[:, 0][:, dst]
        off = 1.01 * EPS24 * (mag * (1 + extra) + np.abs(y))
        if pool.dtype == np.uint8:
            assert_fp8(k[..., :rot], y[..., :rot], off[..., :rot])
        else:
            err = np.abs(k.astype(np.float64) - y)[..., :rot]
            assert np.all(err <= (off + 0.5 * fp16_ulp(np.abs(y) + off))[..., :rot])
        want[:, 0, dst, :, :rot] = k[..., :rot]
    assert got.tobytes() == want.tobytes(), "a row that moves keeps its bits, and no other changes"


def encode(y):
    return e4m3_encode_np(np.clip(y, -448, 448))
