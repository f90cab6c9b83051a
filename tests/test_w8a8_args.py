"""Refusals of the int8 projection path, all before any device call: the pointers are
never dereferenced."""
import pytest

import atomflow_amd
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
    (dict(y_dtype=AF_KV_FP8_E4M3), NOT), (dict(m=(1 << 26) + 1), NOT),
    (dict(n=(1 << 26) + 1, y_stride=1 << 27), NOT),
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
