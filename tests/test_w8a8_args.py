"""Refusals of the int8 projection path, all before any device call: the pointers are
never dereferenced."""
import os
import subprocess

import numpy as np
import pytest

import atomflow_amd
import w8a8_ref
from atomflow_amd import weights
from atomflow_amd import (AF_ERR_INVALID_ARG, AF_ERR_UNSUPPORTED, AF_FP16, AF_FP32, AF_KV_FP8_E4M3, AF_OK,
                          kv)

FAKE = 0x10000


def call(name, defaults, **changes):
    args = dict(defaults)
    assert set(changes) <= set(args)
    args.update(changes)
    return getattr(atomflow_amd.lib(), name)(*args.values())


GEMM = dict(x=FAKE, x_stride=64, xs=FAKE, m=4, w=FAKE, w_stride=64, ws=FAKE, bias=None, y=FAKE,
            y_stride=32, y_dtype=AF_FP16, n=32, k=64, stream=None)
QUANT = dict(x=FAKE, x_stride=64, m=4, n=64, codes=FAKE, codes_stride=64, scales=FAKE, stream=None)
SILU = dict(gate=FAKE, up=FAKE, stride=64, m=4, n=64, codes=FAKE, codes_stride=64, scales=FAKE,
            stream=None)
NORM = dict(x=FAKE, x_stride=64, residual=FAKE, residual_out=FAKE, residual_stride=64,
            residual_dtype=AF_FP16, weight=FAKE, eps=1e-5, m=4, n=64, codes=FAKE, codes_stride=64,
            scales=FAKE, normed=FAKE, normed_stride=64, stream=None)
BAD, NOT = AF_ERR_INVALID_ARG, AF_ERR_UNSUPPORTED


@pytest.mark.parametrize("changes,status", [
    (dict(x=None), BAD), (dict(xs=None), BAD), (dict(w=None), BAD), (dict(ws=None), BAD),
    (dict(y=None), BAD), (dict(m=-1), BAD), (dict(n=0), BAD), (dict(k=0), BAD),
    (dict(k=-16), BAD), (dict(k=40), NOT), (dict(k=131072, x_stride=131072, w_stride=131072), NOT),
    (dict(x_stride=48), BAD), (dict(w_stride=48), BAD), (dict(x_stride=72), BAD),
    (dict(w_stride=72), BAD), (dict(y_stride=31), BAD), (dict(x_stride=1 << 23), NOT),
    (dict(w_stride=1 << 23), NOT), (dict(x=FAKE + 8), BAD), (dict(w=FAKE + 1), BAD),
    (dict(xs=FAKE + 2), BAD), (dict(ws=FAKE + 2), BAD), (dict(bias=FAKE + 2), BAD),
    (dict(y=FAKE + 1), BAD), (dict(y=FAKE + 2, y_dtype=AF_FP32), BAD), (dict(y_dtype=2), NOT),
    (dict(y_dtype=AF_KV_FP8_E4M3), NOT), (dict(m=(1 << 25) + 1), NOT),
    (dict(n=(1 << 25) + 1, y_stride=1 << 27), NOT),
    (dict(m=1 << 20, n=1 << 17, y_stride=1 << 17), NOT), (dict(m=0), AF_OK)])
def test_w8a8_gemm_refusals(changes, status):
    assert call("af_w8a8_gemm", GEMM, **changes) == status


COMMON = [(dict(m=-1), BAD), (dict(n=0), BAD), (dict(scales=None), BAD), (dict(codes_stride=63), BAD),
          (dict(scales=FAKE + 2), BAD), (dict(m=0), AF_OK)]


@pytest.mark.parametrize("changes,status", COMMON + [
    (dict(x=None), BAD), (dict(x=FAKE + 1), BAD), (dict(x_stride=63), BAD), (dict(codes=None), BAD),
    (dict(n=(1 << 30) + 1, x_stride=1 << 31, codes_stride=1 << 31), NOT)])
def test_quantize_rows_refusals(changes, status):
    assert call("af_quantize_rows", QUANT, **changes) == status


@pytest.mark.parametrize("changes,status", COMMON + [
    (dict(gate=None), BAD), (dict(up=None), BAD), (dict(gate=FAKE + 1), BAD), (dict(up=FAKE + 1), BAD),
    (dict(stride=63), BAD), (dict(codes=None), BAD),
    (dict(n=(1 << 30) + 1, stride=1 << 31, codes_stride=1 << 31), NOT)])
def test_silu_mul_quantize_refusals(changes, status):
    assert call("af_silu_mul_quantize", SILU, **changes) == status


@pytest.mark.parametrize("changes,status", COMMON + [
    (dict(x=None), BAD), (dict(x=FAKE + 1), BAD), (dict(x_stride=63), BAD), (dict(weight=None), BAD),
    (dict(weight=FAKE + 2), BAD), (dict(eps=0.0), BAD), (dict(eps=-1e-6), BAD),
    (dict(eps=float("nan")), BAD), (dict(eps=float("inf")), BAD), (dict(residual=None), BAD),
    (dict(residual_out=None), BAD), (dict(residual_stride=63), BAD), (dict(residual_dtype=2), NOT),
    (dict(residual=FAKE + 1), BAD), (dict(residual=FAKE + 2, residual_dtype=AF_FP32), BAD),
    (dict(residual_out=FAKE + 2, residual_dtype=AF_FP32), BAD), (dict(normed_stride=63), BAD),
    (dict(normed=FAKE + 1), BAD), (dict(codes=None, normed=None), BAD),
    (dict(codes=None, scales=None, m=0), AF_OK), (dict(normed=None, normed_stride=0, m=0), AF_OK),
    (dict(residual=None, residual_out=None, residual_stride=0, m=0), AF_OK)])
def test_rmsnorm_quantize_refusals(changes, status):
    assert call("af_rmsnorm_quantize", NORM, **changes) == status


def test_python_mirror_raises():
    with pytest.raises(atomflow_amd.AfError) as e:
        kv.launch_w8a8_gemm(FAKE, 40, FAKE, 1, FAKE, 40, FAKE, FAKE, 8, 8, 40)
    assert e.value.status == NOT
    with pytest.raises(atomflow_amd.AfError) as e:
        kv.launch_rmsnorm_quantize(FAKE, 8, FAKE, 1e-5, 1, 8)
    assert e.value.status == BAD
    with pytest.raises(atomflow_amd.AfError):
        kv.launch_quantize_rows(FAKE, 4, 1, 8, FAKE, 8, FAKE)
    with pytest.raises(atomflow_amd.AfError):
        kv.launch_silu_mul_quantize(FAKE, None, 8, 1, 8, FAKE, 8, FAKE)


def test_cpp_launchers_refuse(tmp_path):
    """The C++ wrappers check their Views and throw with the status text; nothing reaches a device."""
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include <cstdio>
#include <functional>
#include <stdexcept>
#include <string>
#include "ops/kernel.h"
static int bad = 0;
static void throws(const char* what, const char* text, const std::function<void()>& f) {
    try { f(); } catch (const std::runtime_error& e) {
        if (std::string(e.what()).find(text) == std::string::npos) { std::printf("%s: %s\n", what, e.what()); ++bad; }
        return;
    }
    std::printf("%s did not throw\n", what);
    ++bad;
}
int main() {
    char* fake = reinterpret_cast<char*>(0x10000);
    auto h = reinterpret_cast<__half*>(fake);
    auto c = reinterpret_cast<int8_t*>(fake);
    auto f = reinterpret_cast<float*>(fake);
    View y = create_contiguous_view(fake, DataType::FP16, {4, 32});
    View res = create_contiguous_view(fake, DataType::FP32, {4, 64});
    View w = create_contiguous_view(fake, DataType::FP32, {64});
    throws("gemm k", "unsupported", [&] { launch_w8a8_gemm(c, 48, f, c, 48, f, nullptr, y, 40, nullptr); });
    throws("gemm x", "invalid", [&] { launch_w8a8_gemm(nullptr, 64, f, c, 64, f, nullptr, y, 64, nullptr); });
    View y3 = create_contiguous_view(fake, DataType::FP16, {2, 2, 32});
    throws("gemm dims", "output", [&] { launch_w8a8_gemm(c, 64, f, c, 64, f, nullptr, y3, 64, nullptr); });
    View y8 = create_contiguous_view(fake, DataType::FP8_E4M3, {4, 32});
    throws("gemm type", "unsupported", [&] { launch_w8a8_gemm(c, 64, f, c, 64, f, nullptr, y8, 64, nullptr); });
    throws("norm eps", "invalid", [&] { launch_rmsnorm_quantize(h, 64, res, w, 0.0f, c, 64, f, nullptr); });
    View wh = create_contiguous_view(fake, DataType::FP16, {64});
    View ws = create_contiguous_view(fake, DataType::FP32, {63});
    throws("norm length", "weight", [&] { launch_rmsnorm_quantize(h, 64, res, ws, 1e-5f, c, 64, f, nullptr); });
    View far = create_contiguous_view(fake, DataType::FP16, {int64_t(1) << 32, 32});
    throws("gemm rows", "output", [&] { launch_w8a8_gemm(c, 64, f, c, 64, f, nullptr, far, 64, nullptr); });
    View tr = y;
    tr.strides[1] = 2;
    throws("gemm columns", "output", [&] { launch_w8a8_gemm(c, 64, f, c, 64, f, nullptr, tr, 64, nullptr); });
    throws("norm weight", "weight", [&] { launch_rmsnorm_quantize(h, 64, res, wh, 1e-5f, c, 64, f, nullptr); });
    View rb = create_contiguous_view(fake, DataType::BF16, {4, 64});
    throws("norm residual", "unsupported", [&] { launch_rmsnorm_quantize(h, 64, rb, w, 1e-5f, c, 64, f, nullptr); });
    throws("quantize", "invalid", [&] { launch_quantize_rows(h, 63, 4, 64, c, 64, f, nullptr); });
    throws("silu", "invalid", [&] { launch_silu_mul_quantize(h, nullptr, 64, 4, 64, c, 64, f, nullptr); });
    if (!bad) std::puts("ok");
    return bad;
}
''')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.dirname(atomflow_amd.LIB_PATH)
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    os.path.join(root, "include"), str(src), "-L", lib, "-latomflow_kv",
                    "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{lib}:/opt/rocm/lib", "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.stdout, r.stderr)


@pytest.mark.parametrize("n,k", [(5, 64), (3, 100), (1, 1), (40, 4096)])
def test_quantize_int8(n, k):
    r = np.random.default_rng(n + k)
    w = (r.standard_normal((n, k)) * r.uniform(1e-3, 3.0, (n, 1))).astype(np.float32)
    w[n // 2] = 0.0
    codes, scales = weights.quantize_int8(w)
    assert codes.dtype == np.int8 and codes.shape == (n, -(-k // 16) * 16) and scales.dtype == np.float32
    assert np.all(codes[:, k:] == 0)
    w8a8_ref.assert_codes(codes[:, :k], scales, w.astype(np.float64), 0.0)


def test_quantize_int8_halves():
    """Odd multiples of a / 254 lie halfway between two codes: to the even one, whatever a is."""
    r = np.random.default_rng(5)
    unit = r.integers(1, 1 << 15, (300, 1)) * np.exp2(r.integers(-40, 20, (300, 1)))
    odd = 2 * r.integers(-127, 127, (300, 64)) + 1
    w = (odd * unit).astype(np.float32)  # exact
    w[:, 7] = 254 * unit[:, 0]
    codes, scales = weights.quantize_int8(w)
    want = np.rint(odd / 2.0)
    want[:, 7] = 127
    assert np.array_equal(codes, want)
    assert np.array_equal(scales, (2 * unit[:, 0]).astype(np.float32))


def test_quantize_int8_refuses():
    for bad in (np.zeros(4), np.full((2, 3), np.nan), np.array([[1.0, np.inf]])):
        with pytest.raises(ValueError):
            weights.quantize_int8(bad)


def test_cpp_norm_refuses_a_null_residual(tmp_path):
    """The C++ norm adds into its residual: a View without memory is refused (the C ABI takes a null
    residual as the norm of x alone), unless it has no rows."""
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include <cstdio>
#include <stdexcept>
#include "ops/kernel.h"
static const char* text(View res) {
    static char said[256];
    char* fake = reinterpret_cast<char*>(0x10000);
    View w = create_contiguous_view(fake, DataType::FP32, {64});
    std::snprintf(said, sizeof said, "nothing");
    try {
        launch_rmsnorm_quantize(reinterpret_cast<__half*>(fake), 64, res, w, 1e-5f,
                                reinterpret_cast<int8_t*>(fake), 64, reinterpret_cast<float*>(fake), nullptr);
    } catch (const std::runtime_error& e) {
        std::snprintf(said, sizeof said, "%s", e.what());
    }
    return said;
}
int main() {
    std::puts(text(create_contiguous_view(nullptr, DataType::FP32, {4, 64})));
    std::puts(text(create_contiguous_view(nullptr, DataType::FP16, {4, 64})));
    std::puts(text(create_contiguous_view(nullptr, DataType::FP16, {0, 64})));
}
''')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.dirname(atomflow_amd.LIB_PATH)
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    os.path.join(root, "include"), str(src), "-L", lib, "-latomflow_kv",
                    "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{lib}:/opt/rocm/lib", "-o", str(exe)],
                   check=True)
    # (no device is shown to the program: a call that passes the checks ends in the runtime's error)
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1")
    r = subprocess.run([str(exe)], capture_output=True, text=True, env=env)
    said = r.stdout.split("\n")
    assert r.returncode == 0 and all("null residual" in s for s in said[:2]) and said[2] == "nothing", r


def test_product_shapes_reach_every_form():
    """The shapes that the GPU tests of the product run, by its rule on a device of 256 CUs (what a
    host without a device assumes): every form that sizes drawn at random reach is among them, streamed
    and not, and none of these launches passes 2^32 threads."""
    import test_gpu_w8a8 as shapes

    for form, cases in shapes.STREAMED.items():
        for q in cases:
            assert kv.w8a8_gemm_form(*q) == (*form, True), q
    lists = shapes.SHAPES + shapes.FORMS + shapes.WIDE + shapes.UNSTREAMED
    covered = {kv.w8a8_gemm_form(*q) for q in lists + sum(shapes.STREAMED.values(), [])}
    tiles = {f[:4] for f in covered if f[0] > 1 and f[:2] != (256, 256)}
    assert tiles == set(shapes.STREAMED)
    r = np.random.default_rng(1)
    for top_m, top_n in ((3, 18), (6, 14), (8, 18), (13, 15), (25, 25)):
        m = np.exp2(r.uniform(0, top_m, 20000)).astype(int)
        n = np.exp2(r.uniform(0, top_n, 20000)).astype(int)
        k = 16 * np.exp2(r.uniform(0, 12.9, 20000)).astype(int)
        for q in zip(m.tolist(), n.tolist(), k.tolist()):
            if q[0] * q[1] > 1 << 36:
                continue
            form = kv.w8a8_gemm_form(*q)
            assert form in covered, (q, form)
            assert form[0] == 1 or -(-q[0] // form[0]) * -(-q[1] // form[1]) * 512 < 1 << 32, (q, form)


def test_product_form_refusals():
    form = np.zeros(5, np.int32)
    f = atomflow_amd.lib().af_w8a8_gemm_form
    for bad in ((0, 8, 16), (-1, 8, 16), (4, 0, 16), (4, 8, 0)):
        assert f(*bad, form.ctypes.data) == BAD
    assert f(4, 8, 16, None) == BAD
    for no in ((4, 8, 40), (4, 8, 131072), ((1 << 25) + 1, 8, 16), (4, (1 << 25) + 1, 16),
               (1 << 20, 1 << 17, 16)):
        assert f(*no, form.ctypes.data) == NOT
    assert not form.any()
    assert kv.w8a8_gemm_form(1, 64, 4096) == (1, 1, 1, 0, True)
    assert kv.w8a8_gemm_form(1, 64, 4112) == (1, 2, 1, 0, True)
