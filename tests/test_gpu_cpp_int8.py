"""The int8 projection path driven from a C++ host (tests/cpp/int8_step, built with the
library): the MLP half of a layer through include/ops/kernel.h, each step's output checked in
64 bits on what the step before it wrote."""
import os
import subprocess

import numpy as np
import pytest

from w8a8_ref import assert_codes, gemm_bound, gemm_parts, norm_delta, rmsnorm, silu_delta, silu_mul

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "int8_step")
M, D, F = 21, 272, 400


def test_cpp_host_mlp(gpu, tmp_path):
    print("[case] C++ host: int8 MLP", flush=True)
    assert os.path.exists(EXE), "tests/cpp/int8_step is built by the library's Makefile"
    r = subprocess.run([EXE, str(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.returncode, r.stdout, r.stderr)
    load = lambda name, dtype, *shape: np.fromfile(tmp_path / f"{name}.bin", dtype).reshape(shape)
    f32, f16, i8 = np.float32, np.float16, np.int8
    x = load("x", f16, M, D + 8)[:, :D]
    res = load("res", f32, M, D)
    assert np.array_equal(load("res_out", f32, M, D), x.astype(f32) + res)
    _, v = rmsnorm(x, res, load("norm", f32, D), 1e-5)
    c1, s1 = load("c1", i8, M, D), load("s1", f32, M)
    assert_codes(c1, s1, v, norm_delta(D))
    _, p, y = gemm_parts(c1, s1, load("w_gate_up", i8, 2 * F, D), load("s_gate_up", f32, 2 * F),
                         load("bias", f32, 2 * F))
    gu = load("gate_up", f16, M, 2 * F)
    assert np.all(np.abs(gu.astype(np.float64) - y) <= gemm_bound(p, y, f16))
    c2, s2 = load("c2", i8, M, F), load("s2", f32, M)
    assert_codes(c2, s2, silu_mul(gu[:, :F], gu[:, F:]), silu_delta(gu[:, :F]))
    _, p, y = gemm_parts(c2, s2, load("w_down", i8, D, F), load("s_down", f32, D))
    down = load("down", f32, M, D)
    assert np.all(np.abs(down.astype(np.float64) - y) <= gemm_bound(p, y, f32))
    assert_codes(load("c3", i8, M, 2 * F), load("s3", f32, M), gu.astype(np.float64), 0.0)
