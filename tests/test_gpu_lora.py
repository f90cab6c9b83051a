"""Low-rank adapters beside a shared projection on the GPU (af_lora_add) against the same operator
in 64 bits, within a bound that counts each rounding (rows_ref), and in whole numbers, bit for
bit."""
import numpy as np
import pytest

import atomflow_amd
from atomflow_amd import AF_FP16, AF_FP32
from atomflow_amd import device as dev
from atomflow_amd import kv
from rows_ref import Rows, assert_lora, lora

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


def up(a):
    return dev.DeviceBuffer.from_array(a)


class Case:
    """One projection's adapters and a batch of tokens; `whole`: small whole numbers, so that every
    sum is exact in fp32 and in the two fp16 halves of v."""

    def __init__(self, m, k, ends, rmax, count, seed, whole=False, y_dtype=np.float16, none=0.2, ranks=True):
        r = np.random.default_rng(seed)
        self.m, self.k, self.ends, self.rmax, self.count = m, k, list(ends), rmax, count
        n = self.n = ends[-1]
        if whole:
            self.x = r.integers(-3, 4, (m, k)).astype(np.float16)
            self.a = (r.integers(-2, 3, (count, len(ends), rmax, k)) * (r.random((count, len(ends), rmax, k)) < 0.3)
                      ).astype(np.float16)
            self.b = r.integers(-2, 3, (count, n, rmax)).astype(np.float16)
            self.y = r.integers(-50, 51, (m, n)).astype(y_dtype)
            self.scales = r.choice([0.5, 1.0, 2.0, -1.0], count).astype(np.float32)
        else:
            self.x = (r.standard_normal((m, k)) * np.where(r.random(k) < 0.01, 12, 1)).astype(np.float16)
            self.a = (r.standard_normal((count, len(ends), rmax, k)) / np.sqrt(k)).astype(np.float16)
            self.b = (0.1 * r.standard_normal((count, n, rmax))).astype(np.float16)
            self.y = r.standard_normal((m, n)).astype(y_dtype)
            self.scales = (0.5 + r.random(count)).astype(np.float32)
        self.ranks = np.full(count, rmax, np.int32)
        if ranks:
            self.ranks[:] = r.integers(0, rmax + 1, count)
            self.ranks[0] = rmax
        self.ids = np.where(r.random(m) < none, -1, r.integers(0, count, m)).astype(np.int32)
        # what lies behind an adapter's rank is not read as a number
        for i in range(count):
            self.a[i, :, self.ranks[i]:] = np.nan
            self.b[i, :, self.ranks[i]:] = np.inf

    def want(self):
        return lora(self.x, self.ids, self.a, self.b, self.ranks, self.scales, self.ends, self.y)

    def device(self, x_pad=0, y_pad=0, y_off=0):
        self.dx = Rows(up, np.float16, self.m, self.k, self.k + x_pad, 0, self.x)
        self.dy = Rows(up, self.y.dtype, self.m, self.n, self.n + y_pad, y_off, self.y)
        self.do = Rows(up, self.y.dtype, self.m, self.n, self.n + 2 * y_pad, y_off)
        self.da, self.db, self.dr, self.ds, self.di = (
            up(t) for t in (self.a, self.b, self.ranks, self.scales, self.ids))
        self.lora = kv.make_lora(self.da, self.db, self.count, self.rmax, self.k, self.ends, ranks=self.dr,
                                 scales=self.ds)
        self.ws = dev.DeviceBuffer(kv.lora_workspace_size(self.lora, self.m))
        self.ws.fill_u32(0x7fc00000)  # (NaN)
        return self

    def call(self, out=None, stream=None, ids=None, m=None):
        out = out or self.do
        kv.launch_lora_add(self.dx.ptr, self.dx.stride, self.m if m is None else m, ids or self.di, self.lora,
                           self.dy.ptr, self.dy.stride, out.ptr, out.stride, self.ws, self.ws.nbytes,
                           y_dtype=AF_FP16 if self.y.dtype == np.float16 else AF_FP32, stream=stream)

    def check(self):
        out, bound = self.want()
        got = self.do.get()
        assert_lora(got, out, bound)
        none = (self.ids < 0) | (self.ids >= self.count)
        none[~none] = self.ranks[self.ids[~none]] == 0
        assert got[none].tobytes() == self.y[none].tobytes(), "tokens without an adapter keep y"


SHAPES = [  # m, k, slice ends, max_rank, adapters
    (1, 4096, [512], 16, 3), (1, 8, [1], 8, 1), (2, 40, [5, 9], 8, 2), (16, 512, [64, 128, 131], 24, 5),
    (17, 520, [300], 32, 40), (33, 2048, [100, 133, 166], 16, 7), (45, 1536, [700, 1400], 64, 24),
    (64, 4104, [257], 128, 64), (100, 256, [63, 64, 65, 66], 40, 9), (257, 640, [320, 500], 32, 6),
    (300, 1000, [1025], 64, 300), (513, 136, [40, 80], 128, 2), (700, 2048, [2100], 16, 12),
    (1030, 328, [1024, 1030], 8, 70)]


@pytest.mark.parametrize("m,k,ends,rmax,count", SHAPES)
@pytest.mark.parametrize("y_dtype,pad,off", [(np.float16, 0, 0), (np.float32, 5, 3), (np.float16, 3, 1)])
def test_lora(gpu, m, k, ends, rmax, count, y_dtype, pad, off):
    say(f"lora m={m} k={k} ends={ends} rank={rmax} adapters={count} {np.dtype(y_dtype)} pad {pad} offset {off}")
    c = Case(m, k, ends, rmax, count, m + k, y_dtype=y_dtype).device(8 * pad, pad, off)
    c.call()
    c.check()
    before = c.do.get().tobytes()
    c.call(out=c.dy)  # in place
    assert c.dy.get().tobytes() == before


@pytest.mark.parametrize("m,k,ends,rmax,count", SHAPES)
def test_lora_whole_numbers(gpu, m, k, ends, rmax, count):
    say(f"lora in whole numbers m={m} k={k} ends={ends} rank={rmax} adapters={count}")
    c = Case(m, k, ends, rmax, count, m * 3 + k, whole=True, y_dtype=np.float32).device()
    c.call()
    out, _ = c.want()
    assert np.abs(out).max() < 2 ** 22
    assert np.array_equal(c.do.get().astype(np.float64), out)


@pytest.mark.parametrize("mix", ["one", "chunks", "step", "all"])
@pytest.mark.parametrize("m", [64, 500, 1300])
def test_lora_mixes(gpu, m, mix):
    """One adapter for all, prompt chunks, decoded tokens before chunks, a new adapter each token."""
    say(f"lora mix {mix} m={m}")
    c = Case(m, 264, [130, 200], 16, 90, m, none=0.0)
    at = np.arange(m)
    c.ids[:] = {"one": at * 0 + 5, "chunks": at // 97, "step": np.where(at < 40, (at * 37) % 90, 3 + at // 300),
                "all": at % 90}[mix]
    c.device().call()
    c.check()


def test_lora_row_does_not_depend_on_the_launch(gpu):
    """A token's bits are the same alone, in a decode batch and in a large step."""
    say("lora, a row's bits in every launch")
    for k, ends, rmax in ((4096, [300, 420], 32), (1304, [129], 64), (14336, [64], 16), (600, [100], 128)):
        c = Case(1000, k, ends, rmax, 6, k).device()
        c.call()
        all_rows = c.do.get()
        for at, m in ((0, 1), (5, 16), (100, 45), (999, 1), (300, 257), (64, 700)):
            part = Case(m, k, ends, rmax, 6, k)
            for name in ("a", "b", "ranks", "scales"):
                setattr(part, name, getattr(c, name))
            part.x, part.y, part.ids = (t[at:at + m].copy() for t in (c.x, c.y, c.ids))
            part.device().call()
            assert part.do.get().tobytes() == all_rows[at:at + m].tobytes(), (k, at, m)


def test_lora_ids_outside(gpu):
    say("lora, ids outside the adapters")
    c = Case(70, 128, [90], 16, 4, 3)
    c.ids[::3] = [4, 5, -2, 2 ** 31 - 1, -2 ** 31, 100] * 4
    c.device().call()
    c.check()


def test_lora_without_ranks_and_scales(gpu):
    say("lora, max_rank and scale 1 for all")
    c = Case(20, 128, [90], 16, 4, 3, ranks=False)
    c.scales[:] = 1
    c.device()
    c.lora = kv.make_lora(c.da, c.db, 4, 16, 128, [90])
    c.call()
    c.check()


def test_lora_ranks_outside(gpu):
    """Ranks are clamped to [0, max_rank]."""
    say("lora, ranks outside")
    c = Case(40, 128, [90], 16, 4, 3, ranks=False)
    c.device()
    bad = up(np.array([99, -3, 16, 2 ** 31 - 1], np.int32))
    c.ranks[1] = 0
    c.lora = kv.make_lora(c.da, c.db, 4, 16, 128, [90], ranks=bad, scales=c.ds)
    c.call()
    c.check()


def test_lora_not_finite(gpu):
    """A NaN in a token's x, in an adapter or in y stays with the token, or with the tokens of that
    adapter; large and tiny values lose nothing to fp16's range."""
    say("lora, NaN and extremes")
    c = Case(40, 256, [70], 16, 3, 8, none=0.0, ranks=False, y_dtype=np.float32)
    c.x[3, 7] = np.nan
    c.x[10] = (c.x[10].astype(np.float32) * 3000).astype(np.float16)
    c.x[11] = 6e-8 * np.sign(c.x[11].astype(np.float32))
    c.y[20, 5] = np.nan
    c.a[2, 0, 3, 9] = np.nan
    c.ids[10:12], c.ids[3], c.ids[20] = 0, 1, 0
    c.device().call()
    got = c.do.get()
    bad = np.zeros(got.shape, bool)
    bad[3], bad[c.ids == 2], bad[20, 5] = True, True, True
    assert np.array_equal(np.isnan(got), bad)
    c.x[3], c.x[c.ids == 2], c.y[20, 5], c.a[2, 0, 3, 9] = 0, 0, 0, 0
    out, bound = c.want()
    assert_lora(got[~bad], out[~bad], bound[~bad])


def test_lora_captured(gpu):
    """A captured launch reads ids, ranks and scales as they are at each replay."""
    say("lora, captured, ids change between replays")
    st = dev.Stream()
    c = Case(50, 512, [200, 300], 16, 8, 4).device()
    c.call(stream=st)
    st.sync()
    g = dev.Graph.capture(st, lambda: c.call(stream=st))
    r = np.random.default_rng(1)
    for i in range(4):
        c.ids = r.integers(-1, 8, 50).astype(np.int32) if i else np.full(50, -1, np.int32)
        c.di.upload(c.ids, st)
        c.do.buf.fill_u32(0x5b5b5b5b, st)
        c.ws.fill_u32(0x7fc00000, st)
        g.launch(st)
        st.sync()
        c.check()
        eager = c.do.get().tobytes()
        c.call(stream=st)
        st.sync()
        assert c.do.get().tobytes() == eager
    g.destroy()
    st.destroy()


def test_lora_fewer_tokens_than_the_workspace(gpu):
    say("lora, a workspace of more tokens")
    c = Case(300, 512, [200], 16, 8, 4).device()
    c.call()
    whole = c.do.get()
    part = c.do.get()
    c.do.buf.fill_u32(0x5b5b5b5b)
    c.call(m=7)
    part = c.do.buf.download(np.float16, (len(c.do.before),))
    assert part[:7 * 200].tobytes() == whole[:7].tobytes()
    assert np.all(part[7 * 200:].view(np.uint8) == 0x5b)


def test_lora_far_rows(gpu):
    """Rows whose byte offsets pass 32 bits: in x, y and an adapter's b."""
    say("lora, far rows")
    m, k, n, r = 20, 64, 96, 8
    stride = 1 << 28  # elements: 4.5 GiB apart at the ninth row
    x = dev.DeviceBuffer((m - 1) * stride * 2 + k * 2)
    y = dev.DeviceBuffer((m - 1) * stride * 2 + n * 2)
    c = Case(m, k, [n], r, 2, 6)
    for i in range(m):
        x.upload(c.x[i], offset=i * stride * 2)
        y.upload(c.y[i], offset=i * stride * 2)
    c.device()
    kv.launch_lora_add(x, stride, m, c.di, c.lora, y, stride, y, stride, c.ws, c.ws.nbytes)
    got = np.stack([y.download(np.float16, (n,), offset=i * stride * 2) for i in range(m)])
    out, bound = c.want()
    assert_lora(got, out, bound)


def test_lora_workspace_too_small(gpu):
    c = Case(4, 64, [8], 8, 1, 1).device()
    with pytest.raises(atomflow_amd.AfError) as e:
        kv.launch_lora_add(c.dx.ptr, 64, 4, c.di, c.lora, c.dy.ptr, 8, c.do.ptr, 8, c.ws,
                           kv.lora_workspace_size(c.lora, 4) - 1)
    assert e.value.status == atomflow_amd.AF_ERR_WORKSPACE


LARGE = [  # launches whose tiles fill the device: m, k, slice ends, max_rank, adapters
    (12300, 72, [130], 8, 5), (12289, 520, [33], 24, 3), (12290, 1288, [20, 41], 24, 6),
    (3100, 1304, [60, 120, 180, 215], 128, 3), (8300, 64, [2050, 4111], 16, 4), (4100, 64, [8200], 64, 3),
    (2100, 64, [16400], 128, 5), (2000, 4104, [40], 16, 12), (1500, 2056, [70, 100], 40, 5),
    (900, 6152, [9, 18, 30], 64, 3)]


@pytest.mark.parametrize("m,k,ends,rmax,count", LARGE)
@pytest.mark.parametrize("y_dtype,pad,off", [(np.float16, 3, 1), (np.float32, 0, 0)])
def test_lora_large(gpu, m, k, ends, rmax, count, y_dtype, pad, off):
    """Prompt chunks, runs of one token of each adapter, and tokens without one; in place too, and a
    few of the rows alone, bit for bit."""
    say(f"lora large m={m} k={k} ends={ends} rank={rmax} adapters={count} {np.dtype(y_dtype)}")
    c = Case(m, k, ends, rmax, count, m + k, y_dtype=y_dtype)
    at = np.arange(m)
    c.ids[:] = np.where(at < 70, at % (count + 1) - 1, (at // 700) % (count + 1) - 1)
    c.device(8 * pad, pad, off).call()
    c.check()
    got = c.do.get()
    c.call(out=c.dy)
    assert c.dy.get().tobytes() == got.tobytes()
    some = np.concatenate([np.arange(60, 75), np.arange(m - 20, m)])
    part = Case(len(some), k, ends, rmax, count, m + k, y_dtype=y_dtype)
    for name in ("a", "b", "ranks", "scales"):
        setattr(part, name, getattr(c, name))
    part.x, part.y, part.ids = (t[some].copy() for t in (c.x, c.y, c.ids))
    part.device().call()
    assert part.do.get().tobytes() == got[some].tobytes()


@pytest.mark.parametrize("m,k,ends,rmax,count", [(2000, 4104, [40], 16, 12), (4100, 1032, [8200], 64, 3)])
def test_lora_large_captured(gpu, m, k, ends, rmax, count):
    """Prompt-sized launches replayed with other adapters, against eager launches of the same ids."""
    say(f"lora large, captured m={m} k={k}")
    st = dev.Stream()
    c = Case(m, k, ends, rmax, count, 3).device()
    c.call(stream=st)
    st.sync()
    g = dev.Graph.capture(st, lambda: c.call(stream=st))
    r = np.random.default_rng(2)
    for _ in range(3):
        c.di.upload(np.repeat(r.integers(-1, count, m // 50 + 1), 50)[:m].astype(np.int32), st)
        c.do.buf.fill_u32(0x5b5b5b5b, st)
        c.ws.fill_u32(0x7fc00000, st)
        g.launch(st)
        st.sync()
        got = c.do.get().tobytes()
        c.call(stream=st)
        st.sync()
        assert c.do.get().tobytes() == got
    g.destroy()
    st.destroy()


def test_lora_two_streams(gpu):
    """Two projections' launches at once, each with its own workspace."""
    say("lora, two streams")
    cases = [Case(300, 2048, [700], 32, 9, 1).device(), Case(45, 4096, [512, 900], 16, 20, 2).device()]
    want = []
    for c in cases:
        c.call()
        want.append(c.do.get().tobytes())
    streams = [dev.Stream(), dev.Stream()]
    for _ in range(5):
        for c, st in zip(cases, streams):
            c.do.buf.fill_u32(0x5b5b5b5b, st)
        for _ in range(4):
            for c, st in zip(cases, streams):
                c.call(stream=st)
        for st in streams:
            st.sync()
        assert [c.do.get().tobytes() for c in cases] == want
    for st in streams:
        st.destroy()
