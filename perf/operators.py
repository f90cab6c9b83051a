"""Performance cases of the 8-bit integer projection path: the operators around an int8 linear layer.

* ``norm``   RMSNorm with the residual's addition: the new residual stream, and the normed rows as int8
             codes with one scale per row (``out``: "codes"), as fp16 ("normed"), or as both;
* ``quant``  rows to int8 codes with one scale per row, of plain fp16 rows (attention's output, before the
             output projection) or, ``gated``, of silu(gate) * up (the MLP's, before the down projection);
* ``gemm``   the int8 matrix product with one scale per token and one per output channel.

Codes are returned as the values they stand for, in the activations' type (fp16), next to their scales.
"""
import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # One decoded token, model width 4096: pure latency.
        {"name": "norm_token", "kind": "norm", "m": 1, "n": 4096, "res": "fp16", "out": "codes"},
        # A ragged decode batch over an fp32 residual stream, the normed rows kept for an fp16 consumer too.
        {"name": "norm_b45", "kind": "norm", "m": 45, "n": 5120, "res": "fp32", "out": "both"},
        # The rows of a large prefill step: the stream from HBM and back.
        {"name": "norm_prompt", "kind": "norm", "m": 8192, "n": 8192, "res": "fp16", "out": "codes"},
        # Attention's output of a decode batch, before the output projection.
        {"name": "quant_b32", "kind": "quant", "m": 32, "n": 4096, "gated": False},
        # The MLP activation of one token: one long row.
        {"name": "silu_token", "kind": "quant", "m": 1, "n": 14336, "gated": True},
        # The MLP activation of a large prefill step.
        {"name": "silu_prompt", "kind": "quant", "m": 8192, "n": 14336, "gated": True},
        # One token's QKV projection (32 query and 8 KV heads of 128): the weights' stream.
        {"name": "gemm_token", "kind": "gemm", "m": 1, "n": 6144, "k": 4096, "out": "fp16", "bias": False},
        # The gate and up projections of a ragged decode batch, in one product.
        {"name": "gemm_b45", "kind": "gemm", "m": 45, "n": 28672, "k": 4096, "out": "fp16", "bias": False},
        # The logits of a decode batch over a 128256-entry vocabulary, fp32 out.
        {"name": "gemm_logits", "kind": "gemm", "m": 32, "n": 128256, "k": 4096, "out": "fp32", "bias": False},
        # A prefill chunk's down projection, one token past a tile: long k, few tiles, with a bias.
        {"name": "gemm_513", "kind": "gemm", "m": 513, "n": 4096, "k": 14336, "out": "fp16", "bias": True},
        # A serving step's tokens (decode rows and chunks together, ragged) through a small model's MLP.
        {"name": "gemm_2011", "kind": "gemm", "m": 2011, "n": 8192, "k": 2048, "out": "fp16", "bias": False},
        # The gate and up projections of a large prefill step: the largest product.
        {"name": "gemm_prompt", "kind": "gemm", "m": 8192, "n": 28672, "k": 4096, "out": "fp16", "bias": False},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "quant", "gemm", "gemm"])
    if kind == "gemm":
        m, n, k = _log(rng, 1, 8192), _log(rng, 128, 28672), 16 * _log(rng, 16, 896)
        m = min(m, 8192 * 28672 * 4096 // (n * k))
        return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(["fp16", "fp16", "fp32"]),
                "bias": rng.random() < 0.3}
    if kind == "norm":
        return {"kind": kind, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 8192),
                "res": rng.choice(["fp16", "fp16", "fp32"]),
                "out": rng.choice(["codes", "codes", "both", "normed"])}
    return {"kind": kind, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 14336),
            "gated": rng.random() < 0.6}


# ---- inputs -----------------------------------------------------------------------------------


class State:
    pass


def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + salt)


def _rows(m, n, gen):
    """fp16 activations: N(0, 1) with a few channels ten times as large, as hidden states have."""
    channel = 1.0 + 9.0 * (torch.rand(n, device="cuda", generator=gen) < 0.005)
    return (torch.randn(m, n, device="cuda", generator=gen) * channel).half()


def _codes(m, n, gen):
    """int8 codes of normally distributed rows whose largest magnitude takes 127."""
    return torch.randn(m, n, device="cuda", generator=gen).mul_(34.0).round_().clamp_(-127, 127).to(
        torch.int8)


def _scales(n, size, gen):
    return size * (0.75 + 0.5 * torch.rand(n, device="cuda", generator=gen))


def _code_buffers(s, m, n):
    """Codes in rows of whole 16 bytes, as the product reads them, their scales and values."""
    s.code_stride = -(-n // 16) * 16
    s.codes = torch.zeros(m, s.code_stride, device="cuda", dtype=torch.int8)
    s.scales = torch.zeros(m, 1, device="cuda")
    s.values = torch.zeros(m, n, device="cuda", dtype=torch.float16)


def prepare(case, seed):
    s = State()
    s.case = case
    m, n, gen = case["m"], case["n"], _generator(seed, 1)
    if case["kind"] == "norm":
        s.x = _rows(m, n, gen)
        s.residual = _rows(m, n, gen).mul_(3.0)
        if case["res"] == "fp32":
            s.residual = s.residual.float().add_(1e-4 * torch.randn(m, n, device="cuda", generator=gen))
        s.weight = 1.0 + 0.2 * torch.randn(n, device="cuda", generator=gen)
        s.residual_out = torch.zeros_like(s.residual)
        s.normed = torch.zeros(m, n, device="cuda", dtype=torch.float16)
        _code_buffers(s, m, n)
    elif case["kind"] == "quant":
        # gated: one buffer of rows [gate | up], as a fused gate and up product writes them
        s.x = _rows(m, 2 * n if case["gated"] else n, gen)
        _code_buffers(s, m, n)
    else:
        k = case["k"]
        s.x, s.x_scales = _codes(m, k, gen), _scales(m, 4.0 / 127, gen)
        s.w, s.w_scales = _codes(n, k, gen), _scales(n, 4.0 / 127 / math.sqrt(k), gen)
        s.bias = 0.1 * torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
        s.y = torch.zeros(m, n, device="cuda",
                          dtype=torch.float32 if case["out"] == "fp32" else torch.float16)
    return s


# ---- passes -----------------------------------------------------------------------------------


def run(s):
    case = s.case
    if own:
        return {"norm": _own_norm, "quant": _own_quant, "gemm": _own_gemm}[case["kind"]](s, case)
    return {"norm": _plain_norm, "quant": _plain_quant, "gemm": _plain_gemm}[case["kind"]](s, case)


def _quantized(v):
    """The values that int8 codes with one scale per row stand for, and the scales."""
    a = v.abs().amax(dim=1, keepdim=True)
    zero = a == 0
    scale = torch.where(zero, 1.0, a / 127.0)
    codes = torch.round(v * torch.where(zero, 0.0, 127.0 / a))
    return (codes * scale).half(), scale


def _plain_norm(s, case):
    h = s.x.float() + s.residual.float()
    out = {"residual": h.to(s.residual.dtype)}
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * s.weight
    if case["out"] != "normed":
        out["values"], out["scales"] = _quantized(y)
    if case["out"] != "codes":
        out["normed"] = y.half()
    return out


def _plain_quant(s, case):
    v = s.x.float()
    if case["gated"]:
        gate, up = v[:, :case["n"]], v[:, case["n"]:]
        v = gate / (1.0 + torch.exp(-gate)) * up
    values, scales = _quantized(v)
    return {"values": values, "scales": scales}


def _plain_gemm(s, case):
    y = (s.x.float() @ s.w.float().t()) * s.x_scales[:, None] * s.w_scales
    if s.bias is not None:
        y = y + s.bias
    return y.to(s.y.dtype)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _values(s, n):
    torch.mul(s.codes[:, :n], s.scales, out=s.values)
    return {"values": s.values, "scales": s.scales}


def _own_norm(s, case):
    from atomflow_amd import AF_FP16, AF_FP32, kv

    m, n = case["m"], case["n"]
    codes, normed = case["out"] != "normed", case["out"] != "codes"
    kv.launch_rmsnorm_quantize(
        s.x.data_ptr(), n, s.weight.data_ptr(), EPS, m, n,
        codes=s.codes.data_ptr() if codes else None, codes_stride=s.code_stride,
        scales=s.scales.data_ptr() if codes else None,
        residual=s.residual.data_ptr(), residual_out=s.residual_out.data_ptr(), residual_stride=n,
        residual_dtype=AF_FP32 if case["res"] == "fp32" else AF_FP16,
        normed=s.normed.data_ptr() if normed else None, normed_stride=n, stream=_stream())
    out = {"residual": s.residual_out}
    if codes:
        out.update(_values(s, n))
    if normed:
        out["normed"] = s.normed
    return out


def _own_quant(s, case):
    from atomflow_amd import kv

    m, n = case["m"], case["n"]
    if case["gated"]:
        gate = s.x.data_ptr()
        kv.launch_silu_mul_quantize(gate, gate + 2 * n, 2 * n, m, n, s.codes.data_ptr(), s.code_stride,
                                    s.scales.data_ptr(), stream=_stream())
    else:
        kv.launch_quantize_rows(s.x.data_ptr(), n, m, n, s.codes.data_ptr(), s.code_stride,
                                s.scales.data_ptr(), stream=_stream())
    return _values(s, n)


def _own_gemm(s, case):
    from atomflow_amd import AF_FP16, AF_FP32, kv

    m, n, k = case["m"], case["n"], case["k"]
    kv.launch_w8a8_gemm(s.x.data_ptr(), k, s.x_scales.data_ptr(), m, s.w.data_ptr(), k,
                        s.w_scales.data_ptr(), s.y.data_ptr(), n, n, k,
                        bias=None if s.bias is None else s.bias.data_ptr(),
                        y_dtype=AF_FP32 if case["out"] == "fp32" else AF_FP16, stream=_stream())
    return s.y


# ---- what a pass cannot do without, and its result from the definition --------------------------


def work(case):
    m, n = case["m"], case["n"]
    if case["kind"] == "gemm":
        k = case["k"]
        size = 4 if case["out"] == "fp32" else 2
        return {"bytes": m * k + n * k + size * m * n + 4 * (m + n) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if case["kind"] == "norm":
        res = 4 if case["res"] == "fp32" else 2
        per = 2 + 2 * res + (case["out"] != "normed") + 2 * (case["out"] != "codes")
        return {"bytes": per * m * n + 4 * n + (4 * m if case["out"] != "normed" else 0),
                "flops": 8 * m * n}
    return {"bytes": (5 if case["gated"] else 3) * m * n + 4 * m, "flops": (8 if case["gated"] else 4) * m * n}


def exact(case, seed):
    s = prepare(case, seed)
    m, n = case["m"], case["n"]
    if case["kind"] == "gemm":
        # sums of 1024 products of codes are whole numbers below 2^24: each fp32 block product is exact
        acc = torch.zeros(m, n, device="cuda", dtype=torch.float64)
        for at in range(0, case["k"], 1024):
            acc += torch.mm(s.x[:, at:at + 1024].float(), s.w[:, at:at + 1024].float().t().contiguous())
        acc *= s.x_scales.double().unsqueeze(1)
        acc *= s.w_scales.double().unsqueeze(0)
        return acc if s.bias is None else acc + s.bias.double()

    def codes(v):
        top = torch.amax(torch.abs(v), 1).unsqueeze(1)
        step = top / 127
        step[top == 0] = 1
        return torch.round(v / step) * step, step

    v = s.x.to(torch.float64)
    if case["kind"] == "quant":
        if case["gated"]:
            v = v[:, :n] * torch.sigmoid(v[:, :n]) * v[:, n:]
        values, scales = codes(v)
        return {"values": values, "scales": scales}
    v = v + s.residual.to(torch.float64)
    y = v / torch.sqrt(torch.sum(v ** 2, 1).unsqueeze(1) / n + EPS) * s.weight.to(torch.float64)
    out = {"residual": v, "normed": y}
    out["values"], out["scales"] = codes(y)
    drop = {"codes": ("normed",), "normed": ("values", "scales"), "both": ()}[case["out"]]
    return {key: value for key, value in out.items() if key not in drop}
