"""GPU parity of the int8 projection path (af_quantize_rows, af_silu_mul_quantize,
af_rmsnorm_quantize, af_w8a8_gemm) against the same operators in 64 bits, alone and as a
layer runs them, with bounds that count each rounding (w8a8_ref)."""
import numpy as np
import pytest

import atomflow_amd
import oracle
from atomflow_amd import AF_FP16, AF_FP32
from atomflow_amd import device as dev
from atomflow_amd import kv
from inputs import HD, fp16_ulp
from w8a8_ref import (EPS24, assert_codes, gemm_bound, gemm_parts, norm_delta, rmsnorm, silu_delta,
                      silu_mul)

pytestmark = pytest.mark.gpu

CANARY8, CANARY16, CANARY32 = 0x5b, 0x7a7a, 0x7a7a7a7a


def say(msg):
    print(f"[case] {msg}", flush=True)


def up(a):
    return dev.DeviceBuffer.from_array(a)


class Rows:
    """A device matrix of m rows, `stride` elements apart, starting `off` elements into its
    buffer, every other byte of which must stay as it was."""

    def __init__(self, dtype, m, n, stride, off=0, data=None):
        self.dtype, self.m, self.n, self.stride, self.off = np.dtype(dtype), m, n, stride, off
        total = off + max(m, 1) * stride + 8
        host = np.full(total * self.dtype.itemsize, CANARY8, np.uint8).view(self.dtype)
        self.before = host.copy()
        if data is not None:
            self._view(host)[:] = data
            self._view(self.before)[:] = data
        self.buf = up(host)
        self.ptr = self.buf.ptr + off * self.dtype.itemsize

    def _view(self, flat):
        return flat[self.off:self.off + self.m * self.stride].reshape(self.m, self.stride)[:, :self.n]

    def get(self):
        """The rows; asserts that nothing around them changed."""
        flat = self.buf.download(self.dtype, (len(self.before),))
        rows = self._view(flat).copy()
        self._view(flat)[:] = 0
        want = self.before.copy()
        self._view(want)[:] = 0
        assert flat.tobytes() == want.tobytes(), "bytes around the rows changed"
        return rows


def activations(m, n, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((m, n)) * np.where(r.random(n) < 0.01, 12.0, 1.0)
    return x.astype(np.float16)


def odd_rows(x):
    """In the last rows: zeros, a NaN, an infinity, the type's extremes, subnormals."""
    x = x.copy()
    kinds = [lambda r: r * 0, lambda r: np.where(np.arange(r.size) == r.size // 2, np.nan, r),
             lambda r: np.where(np.arange(r.size) == r.size - 1, np.inf, r),
             lambda r: np.where(np.arange(r.size) % 2, 65504.0, -65504.0),
             lambda r: np.full(r.size, 6e-8), lambda r: np.where(np.arange(r.size) == 0, -np.inf, 0)]
    for i, f in enumerate(kinds):
        if i + 1 < x.shape[0]:
            x[-1 - i] = f(x[-1 - i].astype(np.float32)).astype(np.float16)
    return x


def check_codes(codes, scales, v, delta, what):
    bad = ~np.isfinite(v).all(axis=1)
    assert np.all(np.isnan(scales[bad])) and np.all(codes[bad] == 0), what
    if (~bad).any():
        assert_codes(codes[~bad], scales[~bad], v[~bad], np.broadcast_to(delta, bad.shape)[~bad], what)


# one wave per row, one to four chunks per thread, workgroups of 1024, rows past the registers
WIDTHS = [1, 7, 8, 64, 511, 512, 513, 2048, 2049, 4096, 5120, 8190, 8200, 14336, 16391, 32768, 40001]


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("m,off", [(1, 0), (9, 1), (70, 0)])
def test_quantize_rows(gpu, n, m, off):
    say(f"quantize rows m={m} n={n} offset {off}")
    x = odd_rows(activations(m, n, m + n))
    xr = Rows(np.float16, m, n, n + 3 * off, off, x)
    c = Rows(np.int8, m, n, n + off, 3 * off)
    s = Rows(np.float32, m, 1, 1)
    kv.launch_quantize_rows(xr.ptr, xr.stride, m, n, c.ptr, c.stride, s.ptr)
    codes, scales = c.get(), s.get()[:, 0]
    check_codes(codes, scales, x.astype(np.float64), 0.0, f"m={m} n={n}")
    good = np.isfinite(scales)
    assert good.any() or m == 1
    top = np.abs(x.astype(np.float32)).max(axis=1)
    want = np.where(top > 0, top / np.float32(127), np.float32(1))
    assert np.array_equal(scales[good], want[good])


def exact_codes(x):
    """Codes of fp16 rows in whole numbers: 127 * v / a to nearest, halves to even."""
    v = np.rint(x.astype(np.float64) * 2.0 ** 24).astype(np.int64)  # (fp16 is a multiple of 2^-24)
    a = np.abs(v).max(axis=1, keepdims=True)
    num, den = 254 * np.abs(v), 2 * np.maximum(a, 1)
    q, rest = num // den, 2 * (num % den)
    return np.sign(v) * (q + ((rest > den) | ((rest == den) & (q % 2 == 1))))


@pytest.mark.parametrize("m,n", [(600, 512), (40, 1024), (300, 4096), (9, 8192), (5, 40000)])
def test_quantize_rows_halves(gpu, m, n):
    """Quotients halfway between two codes are common in fp16 rows: halves, and other odd
    multiples of a / 254, of the row's largest value. Codes are those of exact arithmetic."""
    say(f"quantize rows, halves m={m} n={n}")
    r = np.random.default_rng(m + n)
    top = np.exp2(r.uniform(-22, 15.9, (m, 1))).astype(np.float16)
    odd = 2 * r.integers(-127, 127, (m, n)) + 1
    x = (odd * (top.astype(np.float64) / 254)).astype(np.float16)
    x[:, 1::5] = (r.uniform(-1, 1, x[:, 1::5].shape) * top).astype(np.float16)
    x[:, 2::7] = np.where(odd[:, 2::7] > 0, top / np.float16(2), top / np.float16(-2))
    x[:, :1] = top
    xr = Rows(np.float16, m, n, n, 0, x)
    c, s = Rows(np.int8, m, n, n), Rows(np.float32, m, 1, 1)
    kv.launch_quantize_rows(xr.ptr, xr.stride, m, n, c.ptr, c.stride, s.ptr)
    assert np.array_equal(c.get(), exact_codes(x))


@pytest.mark.parametrize("m,n", [(511, 5120), (512, 4097), (600, 5120), (520, 8190), (1100, 8192)])
def test_quantize_rows_halves_of_large_batches(gpu, m, n):
    """Rows of 4097 to 8192 elements: 1024 threads each up to twice the device's CUs (511 rows), 512
    with two chunks each from there on, the form of a large prompt's attention output."""
    test_quantize_rows_halves(gpu, m, n)


@pytest.mark.parametrize("n", [1000, 4096, 4104, 5120, 7168, 8192, 12000, 40000])
def test_plain_rows_do_not_depend_on_their_number(gpu, n):
    say(f"plain row bits n={n}")
    m = 1100
    x = odd_rows(activations(m, n, n))[::-1]  # (the odd rows in every batch of 40)
    kinds = {}
    for rows in (m, 600, 40, 1):
        xr = Rows(np.float16, rows, n, n, 0, x[:rows])
        c, s = Rows(np.int8, rows, n, n), Rows(np.float32, rows, 1, 1)
        kv.launch_quantize_rows(xr.ptr, n, rows, n, c.ptr, n, s.ptr)
        kinds[rows] = c.get(), s.get()
    check_codes(kinds[m][0], kinds[m][1][:, 0], x.astype(np.float64), 0.0, f"n={n}")
    for rows in (600, 40, 1):
        for whole, got in zip(kinds[m], kinds[rows]):
            assert whole[:rows].tobytes() == got.tobytes(), rows


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("m,off,fused", [(1, 0, True), (9, 1, False), (33, 0, True)])
def test_silu_mul_quantize(gpu, n, m, off, fused):
    say(f"silu mul quantize m={m} n={n} offset {off}")
    r = np.random.default_rng(n + m)
    gate = (4.0 * r.standard_normal((m, n))).astype(np.float16)
    up_ = odd_rows(activations(m, n, 3 * m + n))
    if m > 8:
        gate[0], gate[1], gate[2] = 65504.0, -65504.0, -20.0
        up_[:3] = 1.0
    if fused:
        xr = Rows(np.float16, m, 2 * n, 2 * n + off, off, np.concatenate([gate, up_], axis=1))
        args = (xr.ptr, xr.ptr + 2 * n, xr.stride)
    else:
        gr, ur = (Rows(np.float16, m, n, n + 5, off, a) for a in (gate, up_))
        args = (gr.ptr, ur.ptr, gr.stride)
    c, s = Rows(np.int8, m, n, n + 2 * off, off), Rows(np.float32, m, 1, 1)
    kv.launch_silu_mul_quantize(*args, m, n, c.ptr, c.stride, s.ptr)
    check_codes(c.get(), s.get()[:, 0], silu_mul(gate, up_), silu_delta(gate), f"m={m} n={n}")


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("m,off,res,inplace,out", [
    (1, 0, np.float16, False, "codes"), (9, 1, np.float32, True, "both"),
    (33, 0, np.float16, True, "both"), (2, 1, None, False, "normed"), (8, 0, None, False, "codes"),
    (70, 0, np.float32, False, "codes")])
def test_rmsnorm_quantize(gpu, n, m, off, res, inplace, out):
    say(f"rmsnorm quantize m={m} n={n} residual {res} in place {inplace} out {out}")
    r = np.random.default_rng(5 * n + m)
    x = activations(m, n, 7 * m + n)
    residual = None
    if res is not None:
        residual = (3.0 * r.standard_normal((m, n))).astype(res)
    if m > 6:
        x[-1] = 0
        if residual is not None:
            residual[-1] = 0
        x[-2, n // 2] = np.nan
        x[-3, -1] = np.inf
        x[-4] = np.float16(6e-8)
    w = (1.0 + 0.2 * r.standard_normal(n)).astype(np.float32)
    if n > 8:
        w[3] = 0.0
    eps = 1e-5
    xr = Rows(np.float16, m, n, n + off, off, x)
    c, s = Rows(np.int8, m, n, n + off, off), Rows(np.float32, m, 1, 1)
    nr = Rows(np.float16, m, n, n + 2 * off, off)
    kw = {}
    if res is not None:
        rr = Rows(res, m, n, n + off, off, residual)
        ro = rr if inplace else Rows(res, m, n, n + off, off)
        kw.update(residual=rr.ptr, residual_out=ro.ptr, residual_stride=rr.stride,
                  residual_dtype=AF_FP32 if res == np.float32 else AF_FP16)
    if out != "normed":
        kw.update(codes=c.ptr, codes_stride=c.stride, scales=s.ptr)
    if out != "codes":
        kw.update(normed=nr.ptr, normed_stride=nr.stride)
    kv.launch_rmsnorm_quantize(xr.ptr, xr.stride, up(w), eps, m, n, **kw)
    s64, v = rmsnorm(x, residual, w, eps)
    v[~np.isfinite(s64).all(axis=1)] = np.nan
    bad = np.isnan(v).any(axis=1)
    delta = norm_delta(n)
    if res is not None:
        got = ro.get()
        with np.errstate(invalid="ignore"):
            want = (x.astype(np.float32) + residual.astype(np.float32))
        assert np.array_equal(got, want.astype(res), equal_nan=True)
    if out != "normed":
        check_codes(c.get(), s.get()[:, 0], v, delta, f"m={m} n={n}")
    if out != "codes":
        got = nr.get().astype(np.float64)
        assert np.all(np.isnan(got[bad]))
        err = np.abs(got[~bad] - v[~bad])
        assert np.all(err <= 1.01 * delta * np.abs(v[~bad]) + 0.5 * fp16_ulp(v[~bad])), err.max()


def test_norm_of_rows_past_fp32_squares(gpu):
    """A finite row whose sum of squares is not counts as one that holds a NaN."""
    say("rmsnorm of a huge fp32 residual")
    n = 100
    x, w = np.zeros((2, n), np.float16), np.ones(n, np.float32)
    residual = np.ones((2, n), np.float32)
    residual[1, 5] = 1e25
    c, s = Rows(np.int8, 2, n, n), Rows(np.float32, 2, 1, 1)
    nr, ro = Rows(np.float16, 2, n, n), Rows(np.float32, 2, n, n)
    kv.launch_rmsnorm_quantize(up(x), n, up(w), 1e-5, 2, n, codes=c.ptr, codes_stride=n, scales=s.ptr,
                               residual=up(residual), residual_out=ro.ptr, residual_stride=n,
                               residual_dtype=AF_FP32, normed=nr.ptr, normed_stride=n)
    codes, scales, normed = c.get(), s.get()[:, 0], nr.get()
    assert np.all(codes[0] == 127) and np.isfinite(scales[0]) and np.isfinite(normed[0]).all()
    assert np.all(codes[1] == 0) and np.isnan(scales[1]) and np.isnan(normed[1]).all()
    assert np.array_equal(ro.get(), residual)


def test_more_rows_than_one_launch(gpu):
    """A launch takes 2^21 rows: the rows on both sides of its end, and the last."""
    say("quantise and normalise 2^21 + 37 rows")
    m, n = 2 ** 21 + 37, 24
    r = np.random.default_rng(5)
    x = (r.standard_normal((m, n), np.float32)).astype(np.float16)
    w = np.ones(n, np.float32)
    dx, c, s = up(x), Rows(np.int8, m, n, n), Rows(np.float32, m, 1, 1)
    kv.launch_quantize_rows(dx, n, m, n, c.ptr, n, s.ptr)
    assert_codes(c.get(), s.get()[:, 0], x.astype(np.float64), 0.0)
    kv.launch_rmsnorm_quantize(dx, n, up(w), 1e-5, m, n, codes=c.ptr, codes_stride=n, scales=s.ptr)
    _, v = rmsnorm(x, None, w, 1e-5)
    assert_codes(c.get(), s.get()[:, 0], v, norm_delta(n))


def put_rows(buf, a, stride):
    """Rows of a, `stride` elements apart."""
    for i, row in enumerate(a):
        buf.upload(row, offset=i * stride * a.itemsize)


def get_rows(buf, dtype, m, n, stride):
    size = np.dtype(dtype).itemsize
    return np.stack([buf.download(dtype, (n,), offset=i * stride * size) for i in range(m)])


def test_row_offsets_past_32_bits(gpu):
    say("rows whose offsets pass 2^32 elements")
    m, n, far = 4, 300, (1 << 31) + 40
    x, res = activations(m, n, 1), activations(m, n, 2)
    w = np.ones(n, np.float32)
    bufs = [dev.DeviceBuffer(2 * (far * (m - 1) + n)) for _ in range(4)]
    dx, dr, dro, dn = bufs
    c, s = dev.DeviceBuffer(far * (m - 1) + n), dev.DeviceBuffer(4 * m)
    put_rows(dx, x, far)
    put_rows(dr, res, far)
    kv.launch_quantize_rows(dx, far, m, n, c, far, s)
    assert_codes(get_rows(c, np.int8, m, n, far), s.download(np.float32), x.astype(np.float64), 0.0)
    kv.launch_silu_mul_quantize(dx, dr, far, m, n, c, far, s)
    assert_codes(get_rows(c, np.int8, m, n, far), s.download(np.float32), silu_mul(x, res), silu_delta(x))
    kv.launch_rmsnorm_quantize(dx, far, up(w), 1e-5, m, n, codes=c, codes_stride=far, scales=s,
                               residual=dr, residual_out=dro, residual_stride=far, normed=dn,
                               normed_stride=far)
    s64, v = rmsnorm(x, res, w, 1e-5)
    assert_codes(get_rows(c, np.int8, m, n, far), s.download(np.float32), v, norm_delta(n))
    assert np.array_equal(get_rows(dro, np.float16, m, n, far),
                          (x.astype(np.float32) + res.astype(np.float32)).astype(np.float16))
    normed = get_rows(dn, np.float16, m, n, far).astype(np.float64)
    assert np.all(np.abs(normed - v) <= 1.01 * norm_delta(n) * np.abs(v) + 0.5 * fp16_ulp(v))
    for b in bufs + [c]:
        b.free()


# ---- the product ----------------------------------------------------------------


def product_case(m, n, k, seed):
    r = np.random.default_rng(seed)
    x = r.integers(-128, 128, (m, k)).astype(np.int8)
    w = r.integers(-128, 128, (n, k)).astype(np.int8)
    xs = (0.01 * r.random(m) + 0.001).astype(np.float32)
    ws = (0.01 * r.random(n) + 0.0001).astype(np.float32)
    return x, xs, w, ws, r.standard_normal(n).astype(np.float32)


def product_gpu(x, xs, w, ws, bias=None, dtype=np.float16, xpad=0, wpad=0, ypad=0, off=0):
    (m, k), n = x.shape, w.shape[0]
    xr, wr = Rows(np.int8, m, k, k + xpad, 0, x), Rows(np.int8, n, k, k + wpad, 0, w)
    y = Rows(dtype, m, n, n + ypad, off)
    d = [up(a) for a in (xs, ws)] + [None if bias is None else up(bias)]
    kv.launch_w8a8_gemm(xr.ptr, xr.stride, d[0], m, wr.ptr, wr.stride, d[1], y.ptr, y.stride, n, k,
                        bias=d[2], y_dtype=AF_FP32 if dtype == np.float32 else AF_FP16)
    return y.get()


SHAPES = [(1, 1, 16), (1, 17, 48), (1, 4100, 4096), (2, 16, 64), (3, 1000, 80), (5, 300, 1024),
          (15, 100, 1008), (16, 4100, 528), (17, 33, 144), (31, 1025, 2064), (33, 257, 4112),
          (45, 5121, 1024), (64, 96, 112), (65, 1, 16), (65, 130, 128), (70, 4100, 272),
          (128, 128, 256), (129, 127, 400), (200, 1000, 1040), (257, 513, 640), (300, 2049, 4096),
          (513, 4100, 1040), (1000, 300, 2048), (2100, 1025, 336), (64, 20000, 256),
          (130, 16390, 144), (4100, 8200, 256)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype,bias,pad", [(np.float16, False, 0), (np.float32, True, 1)])
def test_w8a8_gemm(gpu, m, n, k, dtype, bias, pad):
    say(f"w8a8 gemm m={m} n={n} k={k} {np.dtype(dtype).name} bias {bias} pad {pad}")
    x, xs, w, ws, b = product_case(m, n, k, m + n + k)
    if m > 1:
        x[m // 2] = 0
    b = b if bias else None
    got = product_gpu(x, xs, w, ws, b, dtype, 48 * pad, 16 * pad, 3 * pad, pad)
    _, p, y = gemm_parts(x, xs, w, ws, b)
    assert np.isfinite(got).all()
    err = np.abs(got.astype(np.float64) - y)
    assert np.all(err <= gemm_bound(p, y, dtype)), (err - gemm_bound(p, y, dtype)).max()


@pytest.mark.parametrize("n", [1000, 4096, 4104, 5120, 7168, 8192, 12000, 40000])
@pytest.mark.parametrize("res", [None, np.float16, np.float32])
def test_rows_do_not_depend_on_their_number(gpu, n, res):
    """A token's norm, codes and scale have the same bits alone and in any batch."""
    say(f"row bits n={n} residual {res}")
    m = 1100
    r = np.random.default_rng(n)
    x = r.standard_normal((m, n)).astype(np.float16)
    residual = None if res is None else (3.0 * r.standard_normal((m, n))).astype(res)
    w = up((1.0 + 0.2 * r.standard_normal(n)).astype(np.float32))
    kinds = {}
    for rows in (m, 600, 40, 1):
        xr, c = Rows(np.float16, rows, n, n, 0, x[:rows]), Rows(np.int8, rows, n, n)
        s, nr = Rows(np.float32, rows, 1, 1), Rows(np.float16, rows, n, n)
        kw = {}
        if res is not None:
            rr = Rows(res, rows, n, n, 0, residual[:rows])
            kw = dict(residual=rr.ptr, residual_out=rr.ptr, residual_stride=n,
                      residual_dtype=AF_FP32 if res == np.float32 else AF_FP16)
        kv.launch_rmsnorm_quantize(xr.ptr, n, w, 1e-5, rows, n, codes=c.ptr, codes_stride=n,
                                   scales=s.ptr, normed=nr.ptr, normed_stride=n, **kw)
        kinds[rows] = c.get(), s.get(), nr.get()
    for rows in (600, 40, 1):
        for whole, got in zip(kinds[m], kinds[rows]):
            assert np.array_equal(whole[:rows], got), rows


@pytest.mark.parametrize("n", [1000, 5120, 7168, 8192, 12000, 40000])
def test_silu_rows_do_not_depend_on_their_number(gpu, n):
    say(f"silu row bits n={n}")
    m = 1100
    x = (3.0 * np.random.default_rng(n).standard_normal((m, 2 * n))).astype(np.float16)
    kinds = {}
    for rows in (m, 600, 40, 1):
        xr = Rows(np.float16, rows, 2 * n, 2 * n, 0, x[:rows])
        c, s = Rows(np.int8, rows, n, n), Rows(np.float32, rows, 1, 1)
        kv.launch_silu_mul_quantize(xr.ptr, xr.ptr + 2 * n, 2 * n, rows, n, c.ptr, n, s.ptr)
        kinds[rows] = c.get(), s.get()
    for rows in (600, 40, 1):
        for whole, got in zip(kinds[m], kinds[rows]):
            assert np.array_equal(whole[:rows], got), rows


# Every form of the product, by its rule on a device of 256 CUs: one token in pairs of rows, the
# tiles in the order of the table, with partial steps and tiles; for 256 x 256 tiles launches
# of 1 to 13 steps, whole and partial, with one tile for some workgroups and two for others.
FORMS = [(1, 4100, 14352), (1, 33, 4112), (1, 37, 131056), (2, 54, 14352), (33, 4362, 14352),
         (17, 4211, 1024), (18, 4121, 14352), (2, 8210, 128), (18, 8225, 1040), (17, 8457, 400),
         (4395, 65, 400), (33, 5193, 14352), (98, 4259, 528), (34, 8311, 1040), (100, 8560, 1552),
         (67, 8462, 14352), (130, 11086, 1552), (139, 11121, 2080), (129, 11300, 400),
         (4679, 385, 208), (196, 8792, 48), (539, 10659, 528), (266, 13342, 1552),
         (515, 14499, 48), (525, 14634, 144), (586, 13115, 400), (513, 14851, 528),
         (67, 10881, 16), (69, 11088, 400), (4131, 201, 1552), (65, 11432, 1040),
         (259, 13824, 16), (325, 10899, 48), (261, 13611, 400), (385, 11597, 1040),
         (34, 8295, 1024), (33, 8532, 14352), (33, 11148, 400), (71, 11082, 2080),
         (65, 10997, 4096), (135, 11087, 14352), (1283, 12683, 16), (259, 14429, 144),
         (322, 11060, 528), (642, 12292, 16), (513, 13126, 1024), (129, 8507, 14352),
         (4129, 788, 16), (265, 14548, 16), (404, 11022, 400), (2725, 1411, 208),
         (385, 9362, 528), (31, 125003, 1040)]
WIDE = [(986, 11095, 16), (991, 10899, 48), (981, 10949, 128), (812, 13272, 144), (965, 11011, 256),
        (965, 10859, 384), (806, 13146, 400), (777, 13348, 528), (1001, 10996, 1552),
        (3670, 6695, 16), (1818, 13482, 48), (3588, 6882, 128), (2182, 11239, 144),
        (1679, 14555, 256), (5279, 4618, 384), (3607, 6663, 400), (3090, 7818, 528),
        (5006, 4896, 1040)]


def check_product(m, n, k, dtype, bias, pad):
    x, xs, w, ws, b = product_case(m, n, k, m + n + k)
    b = b if bias else None
    got = product_gpu(x, xs, w, ws, b, dtype, 48 * pad, 16 * pad, 3 * pad, pad)
    assert np.isfinite(got).all()
    for lo in range(0, m, 512):  # (bounds the host's arrays)
        part = slice(lo, lo + 512)
        _, p, y = gemm_parts(x[part], xs[part], w, ws, b)
        over = np.abs(got[part].astype(np.float64) - y) - gemm_bound(p, y, dtype)
        assert over.max() <= 0, (lo, over.max())


@pytest.mark.parametrize("m,n,k", FORMS)
@pytest.mark.parametrize("dtype,bias,pad", [(np.float16, True, 1), (np.float32, False, 0)])
def test_w8a8_gemm_forms(gpu, m, n, k, dtype, bias, pad):
    say(f"w8a8 form m={m} n={n} k={k} {np.dtype(dtype).name}")
    check_product(m, n, k, dtype, bias, pad)


@pytest.mark.parametrize("m,n,k", WIDE)
def test_w8a8_gemm_wide(gpu, m, n, k):
    say(f"w8a8 wide m={m} n={n} k={k}")
    check_product(m, n, k, np.float32 if k % 32 else np.float16, n % 2 == 1, m % 2)


# Tiled forms (tokens and weight rows of a tile, parts of K, workgroups per CU) whose one row of
# tiles streams the weights, each workgroup from a k of its own on: loops longer than the stages,
# loops of the stages' number and fewer, and a layer's projections. Partial steps and tiles.
# (That each shape takes its form, and the lists together every form, is asserted on the host.)
STREAMED = {
    (16, 16, 8, 1): [(2, 2194, 5808), (2, 3131, 4080)],
    (16, 32, 4, 2): [(2, 6071, 2080), (2, 9150, 1376), (16, 6144, 4096)],
    (32, 32, 4, 1): [(18, 4526, 2800), (17, 7919, 1600)],
    (32, 64, 2, 2): [(17, 8374, 1504), (2, 16784, 752), (8, 28672, 4096)],
    (64, 32, 4, 1): [(35, 5550, 2320)],
    (64, 64, 1, 2): [(34, 19227, 656), (33, 31696, 400)],
    (64, 64, 2, 1): [(33, 8837, 1440), (33, 13769, 928)],
    (128, 64, 2, 1): [(97, 10120, 1264)],
    (128, 96, 1, 1): [(65, 16475, 1680)],
    (128, 128, 1, 1): [(65, 22560, 560)],
    (192, 128, 1, 1): [(130, 21869, 576), (130, 88084, 144)],
    (192, 256, 1, 1): [(129, 38295, 400), (129, 112474, 112)],
    (64, 128, 1, 2): [(2, 33463, 528), (33, 65625, 192), (45, 28672, 4096)],
    (128, 128, 1, 2): [(98, 32921, 400), (66, 52453, 240)],
    (32, 256, 1, 2): [(4, 49953, 400), (2, 79077, 160)],
}
# Several rows of tiles: a layer's projection, and the form that the lists above lack so.
UNSTREAMED = [(32, 4096, 14336), (6435, 129, 1488)]


@pytest.mark.parametrize("m,n,k", [q for shapes in STREAMED.values() for q in shapes] + UNSTREAMED)
@pytest.mark.parametrize("dtype,bias,pad", [(np.float16, True, 1), (np.float32, False, 0)])
def test_w8a8_gemm_streamed(gpu, m, n, k, dtype, bias, pad):
    say(f"w8a8 streamed m={m} n={n} k={k} {np.dtype(dtype).name} {kv.w8a8_gemm_form(m, n, k)}")
    check_product(m, n, k, dtype, bias, pad)

@pytest.mark.parametrize("m,n", [(1, 1), (20, 3), (70, 40), (300, 129)])
def test_w8a8_gemm_largest_sums(gpu, m, n):
    """The longest k with every code -128: 2^14 * 131056 just fits 32 bits."""
    say(f"w8a8 largest sums m={m} n={n}")
    k = 131056
    x, w = np.full((m, k), -128, np.int8), np.full((n, k), -128, np.int8)
    w[n // 2] = 127
    ones = lambda c: np.ones(c, np.float32)
    got = product_gpu(x, ones(m), w, ones(n), dtype=np.float32)
    want = np.full((m, n), 2 ** 14 * k, np.float64)
    want[:, n // 2] = -128 * 127 * k
    assert np.array_equal(got, want.astype(np.float32))


@pytest.mark.parametrize("n,k", [(1000, 4096), (4100, 144), (130, 1040)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_w8a8_bits_do_not_depend_on_the_launch(gpu, n, k, dtype):
    say(f"w8a8 bits n={n} k={k}")
    x, xs, w, ws, b = product_case(1100, n, k, n)
    whole = product_gpu(x, xs, w, ws, b, dtype)
    for lo, m in ((0, 1), (7, 2), (30, 16), (100, 20), (200, 50), (300, 65), (400, 130), (500, 600)):
        part = product_gpu(x[lo:lo + m], xs[lo:lo + m], w, ws, b, dtype)
        assert part.tobytes() == whole[lo:lo + m].tobytes(), (lo, m)
        rows = slice(n // 3, n // 3 + 40)
        part = product_gpu(x[lo:lo + m], xs[lo:lo + m], w[rows], ws[rows], b[rows], dtype)
        assert part.tobytes() == np.ascontiguousarray(whole[lo:lo + m, rows]).tobytes(), (lo, m)


@pytest.mark.parametrize("m,n,k", [(1818, 13482, 48), (1001, 10996, 1552), (586, 13115, 400)])
def test_w8a8_bits_of_large_launches(gpu, m, n, k):
    """A large launch's rows and columns against small launches of some of them."""
    say(f"w8a8 bits of a large launch m={m} n={n} k={k}")
    x, xs, w, ws, b = product_case(m, n, k, n)
    whole = product_gpu(x, xs, w, ws, b)
    for lo, rows in ((0, 1), (255, 3), (m - 40, 40), (m // 2, 200)):
        for c0, cols in ((0, 70), (250, 300), (n - 33, 33)):
            t, j = slice(lo, lo + rows), slice(c0, c0 + cols)
            part = product_gpu(x[t], xs[t], w[j], ws[j], b[j])
            assert part.tobytes() == np.ascontiguousarray(whole[t, j]).tobytes(), (lo, c0)


@pytest.mark.parametrize("m", [1, 40, 100, 300])
def test_w8a8_odd_scales(gpu, m):
    """Zero, negative, infinite and NaN scales, and overflow of fp16, as IEEE products say."""
    say(f"w8a8 odd scales m={m}")
    n, k = 70, 256
    x, xs, w, ws, _ = product_case(m, n, k, m)
    ws[0], ws[1], ws[2], ws[3], ws[4] = 0.0, -ws[1], np.inf, np.nan, 1e30
    xs[m - 1] = np.nan
    w[5] = 0
    got = product_gpu(x, xs, w, ws).astype(np.float64)
    acc = x.astype(np.float64) @ w.astype(np.float64).T
    with np.errstate(all="ignore"):
        want = (acc.astype(np.float32) * xs[:, None] * ws).astype(np.float16).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want))
    ok = np.isfinite(want)
    assert np.all(np.abs(got[ok] - want[ok]) <= fp16_ulp(want[ok]))


@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_w8a8_fp16_extremes(gpu, m):
    """Subnormal, just overflowing and tied results: the bits of fp32 products rounded once."""
    say(f"w8a8 fp16 extremes m={m}")
    n, k = 400, 64
    x, xs, w, _, _ = product_case(m, n, k, m)
    ws = np.float32(2.0) ** np.random.default_rng(2).integers(-42, 14, n).astype(np.float32)
    xs[:] = np.float32(2.0) ** -4
    got = product_gpu(x, xs, w, ws)
    acc = (x.astype(np.int32) @ w.astype(np.int32).T).astype(np.float32)
    with np.errstate(over="ignore"):
        want = (acc * xs[:, None] * ws).astype(np.float16)
    assert np.isinf(want).any() and (np.abs(want[want != 0]) < 2.0 ** -14).any()
    assert np.array_equal(got == 0, want == 0)
    assert np.array_equal(np.where(got == 0, 0, got.view(np.uint16)),
                          np.where(want == 0, 0, want.view(np.uint16)))


@pytest.mark.parametrize("m,n,k", [(600, 70, 64), (520, 9000, 144)])
def test_w8a8_offsets_past_32_bits(gpu, m, n, k):
    """Rows of x, w and y whose byte offsets pass 2^32."""
    say(f"w8a8 offsets past 32 bits m={m} n={n}")
    xstr, ystr = (1 << 23) - 16, (1 << 22) + 3
    wstr = xstr if n < 2 * m else (1 << 19) + 16
    x, xs, w, ws, b = product_case(m, n, k, m)
    dx, dw = dev.DeviceBuffer(xstr * (m - 1) + k), dev.DeviceBuffer(wstr * (n - 1) + k)
    y = dev.DeviceBuffer(4 * (ystr * (m - 1) + n))
    assert min(xstr * (m - 1), 4 * ystr * (m - 1)) > 2 ** 32
    put_rows(dx, x, xstr)
    put_rows(dw, w, wstr)
    kv.launch_w8a8_gemm(dx, xstr, up(xs), m, dw, wstr, up(ws), y, ystr, n, k, bias=up(b), y_dtype=AF_FP32)
    got = get_rows(y, np.float32, m, n, ystr)
    _, p, want = gemm_parts(x, xs, w, ws, b)
    assert np.all(np.abs(got - want) <= gemm_bound(p, want, np.float32))
    for d in (dx, dw, y):
        d.free()


def test_codes_of_a_row_with_a_nan_make_its_products_nan(gpu):
    say("a NaN through the quantiser and the product")
    m, n, k = 5, 40, 272
    act = activations(m, k, 3)
    act[2, 100] = np.nan
    _, _, w, ws, _ = product_case(m, n, k, 4)
    c, s, y = dev.DeviceBuffer(m * k), dev.DeviceBuffer(4 * m), dev.DeviceBuffer(2 * m * n)
    kv.launch_quantize_rows(up(act), k, m, k, c, k, s)
    kv.launch_w8a8_gemm(c, k, s, m, up(w), k, up(ws), y, n, n, k)
    bad = np.isnan(y.download(np.float16, (m, n)))
    assert bad[2].all() and not bad[[0, 1, 3, 4]].any()


def test_no_rows_launch_nothing(gpu):
    say("m = 0")
    x, xs, w, ws, _ = product_case(2, 30, 64, 1)
    y = Rows(np.float16, 2, 30, 30)
    keep = [up(a) for a in (x, xs, w, ws)]
    kv.launch_w8a8_gemm(keep[0], 64, keep[1], 0, keep[2], 64, keep[3], y.ptr, 30, 30, 64)
    a, c, s = up(activations(1, 64, 1)), Rows(np.int8, 1, 64, 64), Rows(np.float32, 1, 1, 1)
    kv.launch_quantize_rows(a, 64, 0, 64, c.ptr, 64, s.ptr)
    kv.launch_silu_mul_quantize(a, a, 64, 0, 64, c.ptr, 64, s.ptr)
    kv.launch_rmsnorm_quantize(a, 64, up(np.ones(64, np.float32)), 1e-5, 0, 64, codes=c.ptr,
                               codes_stride=64, scales=s.ptr)
    for r in (y, c, s):
        assert r.get().tobytes() == r._view(r.before).tobytes()


# ---- a layer --------------------------------------------------------------------


class Layer:
    """One layer of a serving step over a paged fp16 pool: int8 projections around the
    framework's append and attention, every intermediate kept for checking."""

    nq, nkv, ffn, bs, eps = 8, 2, 1040, 16, 1e-5

    def __init__(self, m, seed):
        self.m, self.d = m, self.nq * HD
        self.kvd = self.nkv * HD
        self.qkv_dim = self.d + 2 * self.kvd
        r = np.random.default_rng(seed)
        lin = lambda n, k: (r.integers(-127, 128, (n, k)).astype(np.int8),
                            ((0.5 + r.random(n)) / (73 * np.sqrt(k))).astype(np.float32))
        self.w = {"qkv": lin(self.qkv_dim, self.d), "o": lin(self.d, self.d),
                  "gate_up": lin(2 * self.ffn, self.d), "down": lin(self.d, self.ffn)}
        self.norms = [(1 + 0.1 * r.standard_normal(self.d)).astype(np.float32) for _ in range(3)]
        self.x = r.standard_normal((m, self.d)).astype(np.float16)
        self.res = (2 * r.standard_normal((m, self.d))).astype(np.float32)
        self.positions = r.integers(0, 90, m).astype(np.int32)
        blocks = 8 * m
        self.tables = r.permutation(blocks).reshape(m, 8).astype(np.int32)
        self.slots = (self.tables[np.arange(m), self.positions // self.bs].astype(np.int64) * self.bs
                      + self.positions % self.bs)
        self.pool0 = (0.5 * r.standard_normal((2, blocks * self.bs, self.kvd))).astype(np.float16)
        self.cos, self.sin = oracle.rope_table(128, HD, 500000.0)
        self.dw = {k: (up(w), up(s)) for k, (w, s) in self.w.items()}
        self.dn = [up(w) for w in self.norms]
        self.dx, self.dpos, self.dslots, self.dt = map(up, (self.x, self.positions, self.slots,
                                                            self.tables))
        self.dlens = up(self.positions + 1)
        self.dc, self.ds = up(self.cos), up(self.sin)
        self.dres, self.pool_mem = up(self.res), up(self.pool0)
        self.pool = kv.make_pool(self.pool_mem, atomflow_amd.AF_KV_FP16, self.bs, 1, self.nkv, HD, blocks)
        self.ws = kv.AttentionWorkspace(m, self.nq, self.nkv, HD)
        b = lambda *s: dev.DeviceBuffer(int(np.prod(s)))
        self.out = {"c1": b(m, self.d), "s1": b(m, 4), "qkv": b(m, self.qkv_dim, 2),
                    "attn": b(m, self.d, 2), "c2": b(m, self.d), "s2": b(m, 4), "o": b(m, self.d, 2),
                    "c3": b(m, self.d), "s3": b(m, 4), "gu": b(m, 2 * self.ffn, 2),
                    "c4": b(m, self.ffn), "s4": b(m, 4), "down": b(m, self.d, 2),
                    "final": b(m, self.d, 2)}

    def reset(self):
        self.dres.upload(self.res)
        self.pool_mem.upload(self.pool0)
        for o in self.out.values():
            o.fill_u32(CANARY32)
        dev.synchronize()

    def norm(self, x, i, stream, codes=None, scales=None, normed=None):
        kv.launch_rmsnorm_quantize(x, self.d, self.dn[i], self.eps, self.m, self.d, codes, self.d,
                                   scales, self.dres, self.dres, self.d, AF_FP32, normed, self.d,
                                   stream)

    def linear(self, name, c, s, y, k, stream):
        w, ws = self.dw[name]
        n = len(self.w[name][1])
        kv.launch_w8a8_gemm(c, k, s, self.m, w, k, ws, y, n, n, k, stream=stream)

    def run(self, stream=None):
        m, o = self.m, self.out
        self.norm(self.dx, 0, stream, o["c1"], o["s1"])
        self.linear("qkv", o["c1"], o["s1"], o["qkv"], self.d, stream)
        kv.launch_paged_rope_append(o["qkv"], m, self.pool, 0, self.dslots, self.dpos, self.dc, self.ds,
                                    128, self.nq, stream=stream)
        kv.launch_paged_attention(o["qkv"], self.qkv_dim, self.pool, 0, self.dt, 8, self.dlens, m, 128,
                                  o["attn"], self.d, self.nq, self.ws, stream=stream)
        kv.launch_quantize_rows(o["attn"], self.d, m, self.d, o["c2"], self.d, o["s2"], stream=stream)
        self.linear("o", o["c2"], o["s2"], o["o"], self.d, stream)
        self.norm(o["o"], 1, stream, o["c3"], o["s3"])
        self.linear("gate_up", o["c3"], o["s3"], o["gu"], self.d, stream)
        kv.launch_silu_mul_quantize(o["gu"], o["gu"].ptr + 2 * self.ffn, 2 * self.ffn, m, self.ffn,
                                    o["c4"], self.ffn, o["s4"], stream=stream)
        self.linear("down", o["c4"], o["s4"], o["down"], self.ffn, stream)
        self.norm(o["down"], 2, stream, normed=o["final"])

    def bits(self):
        got = {k: b.download(np.uint8) for k, b in self.out.items()}
        got["res"], got["pool"] = self.dres.download(np.uint8), self.pool_mem.download(np.uint8)
        return got


@pytest.mark.parametrize("m", [1, 5, 37, 80])
def test_layer(gpu, m):
    """Each operator of the layer on what the one before it wrote, against 64 bits; the
    attention between them has its own tests."""
    say(f"int8 layer of {m} tokens")
    t = Layer(m, 11 + m)
    t.reset()
    t.run()
    d, ffn, o = t.d, t.ffn, t.out
    f16 = lambda k, n: o[k].download(np.float16, (m, n))
    codes = lambda k, n: (o["c" + k].download(np.int8, (m, n)), o["s" + k].download(np.float32, (m,)))

    def product(name, key, y, k):
        c, s = codes(key, k)
        w, ws = t.w[name]
        _, p, want = gemm_parts(c, s, w, ws)
        got = f16(y, len(ws)).astype(np.float64)
        assert np.all(np.abs(got - want) <= gemm_bound(p, want, np.float16)), name

    s, v = rmsnorm(t.x, t.res, t.norms[0], t.eps)
    assert_codes(*codes("1", d), v, norm_delta(d), "norm 1")
    # qkv is rotated in place by the append: check its V part, which stays, and the pool's rows
    c, sc = codes("1", d)
    _, p, want = gemm_parts(c, sc, *t.w["qkv"])
    got = f16("qkv", t.qkv_dim).astype(np.float64)
    vp = slice(d + t.kvd, None)
    assert np.all(np.abs(got - want)[:, vp] <= gemm_bound(p, want, np.float16)[:, vp])
    pool = t.pool_mem.download(np.float16, t.pool0.shape)
    assert np.array_equal(pool[1][t.slots].view(np.uint16), f16("qkv", t.qkv_dim)[:, vp].view(np.uint16))
    assert np.isfinite(f16("attn", d)).all()
    assert_codes(*codes("2", d), f16("attn", d).astype(np.float64), 0.0, "attention's output")
    product("o", "2", "o", d)
    r1 = t.x.astype(np.float32) + t.res
    s, v = rmsnorm(f16("o", d), r1, t.norms[1], t.eps)
    assert_codes(*codes("3", d), v, norm_delta(d), "norm 2")
    product("gate_up", "3", "gu", d)
    gu = f16("gu", 2 * ffn)
    assert_codes(*codes("4", ffn), silu_mul(gu[:, :ffn], gu[:, ffn:]), silu_delta(gu[:, :ffn]), "mlp")
    product("down", "4", "down", ffn)
    r2 = f16("o", d).astype(np.float32) + r1
    r3 = f16("down", d).astype(np.float32) + r2
    assert np.array_equal(t.dres.download(np.float32, (m, d)), r3)
    _, v = rmsnorm(f16("down", d), r2, t.norms[2], t.eps)
    err = np.abs(f16("final", d).astype(np.float64) - v)
    assert np.all(err <= 1.01 * norm_delta(d) * np.abs(v) + 0.5 * fp16_ulp(v))


@pytest.mark.parametrize("m", [1, 37])
def test_layer_graph_replays(gpu, m):
    """The layer captured and replayed, eager work and other inputs between the replays."""
    say(f"int8 layer of {m} tokens under graph replay")
    t = Layer(m, 50 + m)
    stream = dev.Stream()
    t.reset()
    graph = dev.Graph.capture(stream, lambda: t.run(stream))
    for i in range(4):
        t.x = np.random.default_rng(i).standard_normal((m, t.d)).astype(np.float16)
        t.dx.upload(t.x)
        t.reset()
        t.run()
        dev.synchronize()
        eager = t.bits()
        t.reset()
        graph.launch(stream)
        stream.sync()
        replay = t.bits()
        for key in eager:
            assert np.array_equal(eager[key], replay[key]), (i, key)
    graph.destroy()
    stream.destroy()


def test_two_streams_at_once(gpu):
    """No call keeps state of its own: launches on two streams may overlap."""
    say("products and quantisers on two streams")
    cases = [product_case(40, 3000, 1024, 1), product_case(300, 500, 4096, 2)]
    want = [product_gpu(*c) for c in cases]
    streams = [dev.Stream(), dev.Stream()]
    bufs = [[up(a) for a in c] for c in cases]
    outs = [dev.DeviceBuffer(2 * w.size) for w in want]
    for _ in range(6):
        for s, c, b, y in zip(streams, cases, bufs, outs):
            (m, k), n = c[0].shape, c[2].shape[0]
            kv.launch_w8a8_gemm(b[0], k, b[1], m, b[2], k, b[3], y, n, n, k, bias=b[4], stream=s)
    for s in streams:
        s.sync()
    for y, w in zip(outs, want):
        assert y.download(np.uint16).tobytes() == w.tobytes()
    for s in streams:
        s.destroy()
