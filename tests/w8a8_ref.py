"""The int8 projection path in 64 bits, for the tests of its GPU operators."""
import numpy as np

from inputs import fp16_ulp

EPS24 = 2.0 ** -24  # half a step of fp32, relative


def gemm_parts(x, xs, w, ws, bias=None):
    """(exact integer sums, their scaled values, y) of the int8 product in 64 bits."""
    acc = x.astype(np.float64) @ w.astype(np.float64).T  # whole numbers below 2^53: exact
    p = acc * xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None, :]
    y = p if bias is None else p + bias.astype(np.float64)[None, :]
    return acc, p, y


def gemm_bound(p, y, out):
    """Sum to fp32, two products (half a step of fp32 each), the bias's addition, and the
    result's rounding; second-order terms within 1 %."""
    b = 1.01 * EPS24 * (3 * np.abs(p) + np.abs(y))
    if out == np.float16:
        b = b + 0.5 * fp16_ulp(y)
    return b + 2.0 ** -149


def codes_of(v):
    """Unrounded codes v * 127 / a, scales and the rows' largest magnitudes, 64 bits."""
    a = np.abs(v).max(axis=1, keepdims=True)
    zero = a < 2.0 ** -100
    scale = np.where(zero, 1.0, a / 127.0)
    return np.where(zero, 0.0, v / scale), scale[:, 0], a[:, 0]


def assert_codes(codes, scales, v, delta, what=""):
    """codes and scales of rows v (64 bits) whose fp32 values are off by at most `delta`
    (relative, per row): 127 / a and a / 127 add half a step each."""
    want, scale, _ = codes_of(v)
    delta = np.broadcast_to(np.asarray(delta, np.float64), scale.shape)
    assert np.all(np.abs(scales - scale) <= 1.01 * (delta + EPS24) * scale), what
    err = np.abs(codes.astype(np.float64) - want)
    assert np.all(err <= 0.5 + 1.01 * 127 * (2 * delta + EPS24)[:, None]), (what, err.max())
    assert np.all(np.abs(codes.astype(np.int32)) <= 127), what
    zero = np.abs(v).max(axis=1) == 0
    assert np.all(codes[zero] == 0) and np.all(scales[zero] == 1.0), what


def silu_mul(gate, up):
    g, u = gate.astype(np.float64), up.astype(np.float64)
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def silu_delta(gate):
    """Relative error of silu(g) * u in fp32, per row: the exponent g * log2 e (its constant's
    and its product's rounding) moves e^-g by |g| 2^-23, which counts where g < 0; e^x and the
    reciprocal are within a step (2^-23) each, the sum and two products within half of one."""
    worst = np.maximum(0.0, -gate.astype(np.float64)).max(axis=1)
    return (np.minimum(worst, 90.0) + 4.0) * 2.0 ** -23


def rmsnorm(x, residual, weight, eps):
    """(s, v) in 64 bits: the residual's sum and its norm."""
    s = x.astype(np.float64)
    if residual is not None:
        s = s + residual.astype(np.float64)
    with np.errstate(invalid="ignore"):
        v = s / np.sqrt((s * s).mean(axis=1, keepdims=True) + eps) * weight.astype(np.float64)
    return s, v


def norm_delta(n):
    """Relative error of v in fp32: the sum of squares adds at most max(32, n / 1024) terms in
    one thread, then 6 + 16 partial sums (all terms positive; halved by the root); s, the
    mean, eps, the root, its reciprocal and two products each within half a step. Generously
    without the halving."""
    return (max(32, -(-n // 1024)) + 22 + 10) * EPS24
