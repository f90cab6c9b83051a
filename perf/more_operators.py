"""Performance cases of what happens to a token's rows beside the shared projections and on the way into the cache:

* ``lora``     low-rank adapters of many requests, added to a projection that they share;
* ``table``    the cos/sin table of rotary positions scaled for long contexts;
* ``rope``     rotary positions in any layout, over rows of Q and K, or with K and V appended to a paged cache;
* ``compact``  rows dropped out of cached sequences: what stays moves up, its keys turned to the new positions.

FP8 caches are returned as the values that their codes stand for, without the heads' scales.
"""
import math

import torch

own = False

BLOCK = 16  # rows of a cache page


def listed():
    return [
        # One decoded token's QKV projection, one adapter out of sixteen loaded: pure latency.
        {"name": "lora_token", "kind": "lora", "m": 1, "k": 4096, "n": 6144, "slices": "qkv", "rank": 16,
         "adapters": 16, "mix": "scattered"},
        # A ragged decode batch through the fused gate and up projection, some requests without an adapter.
        {"name": "lora_b45", "kind": "lora", "m": 45, "k": 4096, "n": 28672, "slices": "pair", "rank": 32,
         "adapters": 24, "mix": "scattered"},
        # A serving step through the down projection: decoded tokens and prompt chunks of several tenants.
        {"name": "lora_step", "kind": "lora", "m": 2011, "k": 14336, "n": 4096, "slices": "one", "rank": 16,
         "adapters": 12, "mix": "step"},
        # The gate and up projections of a large prefill step with few tenants: the largest product.
        {"name": "lora_prompt", "kind": "lora", "m": 8192, "k": 4096, "n": 28672, "slices": "pair", "rank": 64,
         "adapters": 8, "mix": "chunks"},
        # The table of a context stretched 16 times, whole: built when an engine starts.
        {"name": "table_128k", "kind": "table", "rows": 131072, "first": 0, "rot": 128, "scaling": "yarn"},
        # The next rows of a table that grows with its longest sequence, far out; half of the head turns.
        {"name": "table_grow", "kind": "table", "rows": 4096, "first": 1000000, "rot": 64, "scaling": "bands"},
        # One decoded token: interleaved pairs, half of the head, into an fp16 cache: pure latency.
        {"name": "rope_token", "kind": "rope", "m": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "layout": "interleaved", "cache": "fp16"},
        # The rows of a large prefill step into an FP8 cache.
        {"name": "rope_prompt_fp8", "kind": "rope", "m": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "layout": "half", "cache": "fp8"},
        # Packed sequences of several lengths, Q and K alone, heads of 80 of which 32 elements turn.
        {"name": "rope_pack", "kind": "rope", "m": 4001, "q_heads": 32, "kv_heads": 32, "dim": 80, "rot": 32,
         "layout": "interleaved", "cache": "none"},
        # A long conversation cut to its first rows and its latest ones, in place, all layers.
        {"name": "compact_window", "kind": "compact", "seqs": 1, "length": 8192, "layers": 28, "kv_heads": 8,
         "dim": 128, "rot": 128, "layout": "half", "cache": "fp16", "keep": "window"},
        # A batch of forked sequences that keep a scattered half of their rows, FP8.
        {"name": "compact_batch_fp8", "kind": "compact", "seqs": 13, "length": 3000, "layers": 4, "kv_heads": 8,
         "dim": 128, "rot": 128, "layout": "half", "cache": "fp8", "keep": "scattered"},
        # One short sequence of a small model that drops some of its rows.
        {"name": "compact_short", "kind": "compact", "seqs": 1, "length": 300, "layers": 16, "kv_heads": 4,
         "dim": 64, "rot": 32, "layout": "interleaved", "cache": "fp16", "keep": "scattered"},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["lora", "lora", "table", "rope", "rope", "compact"])
    if kind == "lora":
        m, n, k = _log(rng, 1, 8192), 8 * _log(rng, 32, 3584), 8 * _log(rng, 32, 1792)
        m = min(m, 8192 * 30720 // (n + k // 2))
        mix = "scattered" if m <= 256 else rng.choice(["step", "chunks"])
        return {"kind": kind, "m": m, "k": k, "n": n, "slices": rng.choice(["one", "pair", "qkv"]),
                "rank": rng.choice([8, 16, 16, 24, 32, 64]), "adapters": _log(rng, 1, 32 if m <= 256 else 12),
                "mix": mix}
    if kind == "table":
        return {"kind": kind, "rows": _log(rng, 256, 131072), "first": rng.choice([0, 0, _log(rng, 1000, 1000000)]),
                "rot": 2 * _log(rng, 16, 64), "scaling": rng.choice(["linear", "ntk", "bands", "yarn"])}
    dim = rng.choice([64, 80, 96, 128, 128])
    case = {"kind": kind, "kv_heads": rng.choice([2, 4, 8]), "dim": dim,
            "rot": rng.choice([dim, dim, dim // 2, 16 * rng.randint(1, dim // 16)]),
            "layout": rng.choice(["half", "interleaved"])}
    if kind == "rope":
        case.update(m=_log(rng, 1, 8192), q_heads=case["kv_heads"] * rng.choice([1, 3, 4]),
                    cache=rng.choice(["none", "fp16", "fp8"]))
    else:
        case.update(cache=rng.choice(["fp16", "fp8"]), seqs=_log(rng, 1, 16), layers=rng.randint(2, 8),
                    keep=rng.choice(["window", "scattered"]))
        case["length"] = _log(rng, 200, 16000 // case["seqs"])
    return case


# ---- inputs -----------------------------------------------------------------------------------


class State:
    pass


def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + salt)


def _rows(m, n, gen):
    """fp16 activations: N(0, 1) with a few channels ten times as large, as hidden states have."""
    channel = 1.0 + 9.0 * (torch.rand(n, device="cuda", generator=gen) < 0.005)
    return (torch.randn(m, n, device="cuda", generator=gen) * channel).half()


def _ints(lo, hi, n, gen):
    return torch.randint(lo, hi, (n,), device="cuda", generator=gen)


def _slice_ends(case):
    """Columns of a fused product: QKV (two thirds, a sixth, a sixth), gate and up, or one projection."""
    n = case["n"]
    return {"one": [n], "pair": [n // 2, n], "qkv": [2 * n // 3, 2 * n // 3 + n // 6, n]}[case["slices"]]


def _ids(case, gen):
    """Adapters of the step's tokens, -1 for none: one for each decoded token, one for each prompt chunk."""
    m, count = case["m"], case["adapters"]
    chunks = {"scattered": m, "step": 72, "chunks": 9}[case["mix"]]
    of_chunk = torch.where(torch.rand(chunks, device="cuda", generator=gen) < 0.15, -1, _ints(0, count, chunks, gen))
    of_chunk[0] = of_chunk[0].clamp(min=0)
    if case["mix"] == "scattered":
        return of_chunk.int()
    singles = 64 if case["mix"] == "step" else 0
    at = torch.arange(m, device="cuda")
    cuts = singles + torch.sort(_ints(1, max(2, m - singles), chunks - singles - 1, gen)).values
    return of_chunk[torch.where(at < singles, at, singles + torch.searchsorted(cuts, at, right=True))].int()


def _prepare_lora(s, case, gen):
    m, k, n, rank, count = (case[x] for x in ("m", "k", "n", "rank", "adapters"))
    s.ends = _slice_ends(case)
    s.x, s.y = _rows(m, k, gen), torch.randn(m, n, device="cuda", generator=gen).half()
    s.a = (torch.randn(count, len(s.ends), rank, k, device="cuda", generator=gen) / math.sqrt(k)).half()
    s.b = (0.05 * torch.randn(count, n, rank, device="cuda", generator=gen)).half()
    s.ids = _ids(case, gen)
    s.ranks = torch.where(torch.rand(count, device="cuda", generator=gen) < 0.5, rank,
                          _ints(1, rank + 1, count, gen)).int()
    s.scales = 0.5 + 1.5 * torch.rand(count, device="cuda", generator=gen)
    s.out = torch.empty_like(s.y)
    if own:
        from atomflow_amd import kv

        s.lora = kv.make_lora(s.a.data_ptr(), s.b.data_ptr(), count, rank, k, s.ends, ranks=s.ranks.data_ptr(),
                              scales=s.scales.data_ptr())
        s.ws_bytes = kv.lora_workspace_size(s.lora, m)
        s.ws = torch.empty(max(s.ws_bytes, 16), device="cuda", dtype=torch.uint8)


def _prepare_table(s, case, gen):
    s.factor = 4.0 + 12.0 * float(torch.rand(1, device="cuda", generator=gen))
    s.base = 500000.0
    s.cos = torch.empty(case["rows"], case["rot"] // 2, device="cuda")
    s.sin = torch.empty_like(s.cos)


def _angles(rows, rot):
    """A plain table's angles, in 64 bits."""
    freq = 500000.0 ** (torch.arange(rot // 2, device="cuda", dtype=torch.float64) * (-2.0 / rot))
    return torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq


def _tables(s, rows, rot):
    angle = _angles(rows, rot)
    s.cos, s.sin, s.max_pos = torch.cos(angle).float(), torch.sin(angle).float(), rows


def _prepare_rope(s, case, gen):
    m, dim, heads = case["m"], case["dim"], case["q_heads"] + 2 * case["kv_heads"]
    _tables(s, 16384, case["rot"])
    s.x = torch.randn(m, heads * dim, device="cuda", generator=gen).half()  # rows [Q | K | V]
    start = torch.where(torch.rand(m, device="cuda", generator=gen) < 0.004, _ints(0, 4096, m, gen), 0)
    s.positions = ((torch.arange(m, device="cuda") + torch.cumsum(start, 0)) % 16384).int()
    s.q_out = torch.zeros(m, case["q_heads"] * dim, device="cuda", dtype=torch.float16)
    if case["cache"] == "none":
        s.k_out = torch.zeros(m, case["kv_heads"] * dim, device="cuda", dtype=torch.float16)
        return
    blocks = -(-m // BLOCK) + 5
    s.slots = torch.randperm(blocks * BLOCK, device="cuda", generator=gen)[:m].contiguous()
    s.pool, s.scales = _pool(case, 2, blocks, gen)
    if own:
        s.desc = _descriptor(s, case, 2, blocks)


def _pool(case, layers, blocks, gen):
    """[layer, K and V, row, head, element] with values in place, and an FP8 cache's scales."""
    shape = (layers, 2, blocks * BLOCK, case["kv_heads"], case["dim"])
    x = torch.randn(shape, device="cuda", generator=gen, dtype=torch.float16)
    if case["cache"] == "fp16":
        return x, None
    scales = 0.01 + 0.02 * torch.rand(layers, 2, case["kv_heads"], device="cuda", generator=gen)
    return (x * 40.0).to(torch.float8_e4m3fn), scales


def _descriptor(s, case, layers, blocks):
    from atomflow_amd import AF_KV_FP16, AF_KV_FP8_E4M3, kv

    return kv.make_pool(s.pool.data_ptr(), AF_KV_FP16 if case["cache"] == "fp16" else AF_KV_FP8_E4M3, BLOCK,
                        layers, case["kv_heads"], case["dim"], blocks,
                        scales=None if s.scales is None else s.scales.data_ptr())


def _prepare_compact(s, case, gen):
    seqs, top = case["seqs"], case["length"]
    lengths = _ints(3 * top // 4, top + 1, seqs, gen)
    lengths[0] = top
    _tables(s, top, case["rot"])
    pages = -(-top // BLOCK)
    at = torch.arange(top, device="cuda").expand(seqs, top)
    if case["keep"] == "window":
        # the first four rows stay, the latest eighth moves up behind them: in place
        keep = (at >= lengths[:, None] - lengths[:, None] // 8) & (at < lengths[:, None])
        s.first = torch.full((seqs,), 4, device="cuda", dtype=torch.int32)
        tables = torch.randperm(seqs * pages, device="cuda", generator=gen).int().reshape(seqs, pages)
        s.src_tables, s.dst_tables, blocks = tables, tables, seqs * pages
    else:
        # a scattered half, into pages of its own: the old ones belong to the sequence that this one forked
        keep = (torch.rand(seqs, top, device="cuda", generator=gen) < 0.5) & (at < lengths[:, None])
        s.first = torch.zeros(seqs, device="cuda", dtype=torch.int32)
        tables = torch.randperm(2 * seqs * pages, device="cuda", generator=gen).int().reshape(2, seqs, pages)
        s.src_tables, s.dst_tables, blocks = tables[0].contiguous(), tables[1].contiguous(), 2 * seqs * pages
    s.rows = torch.nonzero(keep)  # (sequence, row) of what moves, in order
    s.kept = s.rows[:, 1].int().contiguous()
    count = keep.sum(1)
    s.start = torch.zeros(seqs + 1, device="cuda", dtype=torch.int32)
    s.start[1:] = torch.cumsum(count, 0)
    s.most = int(count.max())
    s.pool, s.scales = _pool(case, case["layers"], blocks, gen)
    if own:
        s.desc = _descriptor(s, case, case["layers"], blocks)


def prepare(case, seed):
    s = State()
    s.case = case
    {"lora": _prepare_lora, "table": _prepare_table, "rope": _prepare_rope,
     "compact": _prepare_compact}[case["kind"]](s, case, _generator(seed, 1))
    return s


# ---- passes -----------------------------------------------------------------------------------


def run(s):
    kind = s.case["kind"]
    if own:
        return {"lora": _own_lora, "table": _own_table, "rope": _own_rope, "compact": _own_compact}[kind](s, s.case)
    return {"lora": _plain_lora, "table": _plain_table, "rope": _plain_rope,
            "compact": _plain_compact}[kind](s, s.case)


def _column_slice(s, n):
    """The slice that each of the product's columns belongs to."""
    ends = torch.tensor(s.ends, device="cuda")
    return torch.searchsorted(ends, torch.arange(n, device="cuda"), right=True)


def _plain_lora(s, case):
    count, slices, rank, k = s.a.shape
    m, n = case["m"], case["n"]
    # every adapter's down projection of every token, then the token's own adapter's ranks
    v = (s.x.float() @ s.a.float().reshape(-1, k).t()).reshape(m, count, slices, rank)
    own_rank = torch.arange(rank, device="cuda") < s.ranks[:, None]
    mine = (s.ids[:, None] == torch.arange(count, device="cuda"))[:, :, None, None] & own_rank[:, None, :]
    v = torch.where(mine, v * s.scales[:, None, None], 0.0)
    # the up projection, whose columns read their own slice's ranks
    in_slice = _column_slice(s, n)[:, None] == torch.arange(slices, device="cuda")
    b = torch.where(in_slice[None, :, :, None], s.b.float()[:, :, None, :], 0.0)
    b = b.permute(0, 2, 3, 1).reshape(-1, n)
    return (s.y.float() + v.reshape(m, -1) @ b).half()


def _frequencies(case, base, factor):
    """Angle of a pair per position, and the factor on cos and sin, in 64 bits."""
    rot, context = case["rot"], 8192.0
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    if case["scaling"] == "ntk":
        base = base * factor ** (rot / (rot - 2.0))
    freq = base ** (i * (-2.0 / rot))
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "bands":
        low, high = 1.0, 4.0
        smooth = ((context * freq / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return freq * (smooth + (1.0 - smooth) / factor), 1.0
    if case["scaling"] == "yarn":
        pair = [rot * math.log(context / (turns * 2.0 * math.pi)) / (2.0 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return freq * (1.0 - ramp + ramp / factor), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _plain_table(s, case):
    freq, mult = _frequencies(case, s.base, s.factor)
    angle = (case["first"] + torch.arange(case["rows"], device="cuda", dtype=torch.float64))[:, None] * freq
    return {"cos": (torch.cos(angle) * mult).float(), "sin": (torch.sin(angle) * mult).float()}


def _turn(x, cos, sin, rot, layout):
    """Rotary positions of x [..., heads, dim] by cos and sin [..., 1, rot / 2], in 32 bits."""
    part, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)
    a, b = part[..., 0::2], part[..., 1::2]
    return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)


def _fp8(v):
    return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _plain_rope(s, case):
    m, dim, q, kv_heads = case["m"], case["dim"], case["q_heads"], case["kv_heads"]
    x = s.x.float().reshape(m, -1, dim)
    at = s.positions.long()
    turned = _turn(x[:, :q + kv_heads], s.cos[at][:, None], s.sin[at][:, None], case["rot"], case["layout"])
    out = {"q": turned[:, :q].reshape(m, -1).half()}
    k, v = turned[:, q:], x[:, q + kv_heads:]
    if case["cache"] == "none":
        out["k"] = k.reshape(m, -1).half()
        return out
    cache = s.pool[1]  # the layer's K and V
    if case["cache"] == "fp16":
        cache[0][s.slots], cache[1][s.slots] = k.half(), v.half()
    else:
        codes, scales = cache.view(torch.uint8), s.scales[1][:, :, None]
        codes[0][s.slots] = _fp8(k / scales[0]).view(torch.uint8)
        codes[1][s.slots] = _fp8(v / scales[1]).view(torch.uint8)
    out["cache"] = cache
    return out


def _places(s):
    """Physical rows that rows move from and to, and how far each moves."""
    seq, row = s.rows[:, 0], s.rows[:, 1]
    to = torch.arange(len(row), device="cuda") - s.start[seq].long() + s.first[seq].long()
    src = s.src_tables[seq, row // BLOCK].long() * BLOCK + row % BLOCK
    dst = s.dst_tables[seq, to // BLOCK].long() * BLOCK + to % BLOCK
    return src, dst, row - to


def _plain_compact(s, case):
    src, dst, moved = _places(s)
    pool = s.pool if case["cache"] == "fp16" else s.pool.view(torch.uint8)
    rows = pool[:, :, src]
    k = (rows[:, 0] if case["cache"] == "fp16" else rows[:, 0].view(torch.float8_e4m3fn)).float()
    k = _turn(k, s.cos[moved][:, None], -s.sin[moved][:, None], case["rot"], case["layout"])
    pool[:, 0, dst] = k.half() if case["cache"] == "fp16" else _fp8(k).view(torch.uint8)
    pool[:, 1, dst] = rows[:, 1]
    return s.pool


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_lora(s, case):
    from atomflow_amd import kv

    m, n = case["m"], case["n"]
    kv.launch_lora_add(s.x.data_ptr(), case["k"], m, s.ids.data_ptr(), s.lora, s.y.data_ptr(), n,
                       s.out.data_ptr(), n, s.ws.data_ptr(), s.ws_bytes, stream=_stream())
    return s.out


def _own_table(s, case):
    from atomflow_amd import kv

    freq, mult = kv.rope_frequencies(case["rot"], s.base, scaling=case["scaling"], factor=s.factor,
                                     original_max_pos=8192, low_freq_factor=1.0, high_freq_factor=4.0,
                                     beta_fast=32.0, beta_slow=1.0)
    kv.build_rope_table_scaled(s.cos.data_ptr(), s.sin.data_ptr(), case["first"], case["rows"], case["rot"], freq,
                               mult, stream=_stream())
    return {"cos": s.cos, "sin": s.sin}


def _layout(case):
    from atomflow_amd import AF_ROPE_HALF, AF_ROPE_INTERLEAVED

    return AF_ROPE_HALF if case["layout"] == "half" else AF_ROPE_INTERLEAVED


def _own_rope(s, case):
    from atomflow_amd import kv

    m, dim, q, kv_heads = case["m"], case["dim"], case["q_heads"], case["kv_heads"]
    stride, x = (q + 2 * kv_heads) * dim, s.x.data_ptr()
    if case["cache"] == "none":
        kv.launch_rope_rows(x, stride, s.q_out.data_ptr(), q * dim, q, x + 2 * q * dim, stride, s.k_out.data_ptr(),
                            kv_heads * dim, kv_heads, m, dim, case["rot"], _layout(case), s.cos.data_ptr(),
                            s.sin.data_ptr(), s.max_pos, positions=s.positions.data_ptr(), stream=_stream())
        return {"q": s.q_out, "k": s.k_out}
    kv.launch_paged_rope_append_rows(x, stride, m, s.q_out.data_ptr(), q * dim, q, s.desc, 1, s.slots.data_ptr(),
                                     s.positions.data_ptr(), case["rot"], _layout(case), s.cos.data_ptr(),
                                     s.sin.data_ptr(), s.max_pos, stream=_stream())
    return {"q": s.q_out, "cache": s.pool[1]}


def _own_compact(s, case):
    from atomflow_amd import kv

    kv.kv_compact(s.desc, s.src_tables.data_ptr(), s.dst_tables.data_ptr(), s.src_tables.shape[1], case["seqs"],
                  s.kept.data_ptr(), s.start.data_ptr(), s.first.data_ptr(), s.most, case["rot"], _layout(case),
                  s.cos.data_ptr(), s.sin.data_ptr(), s.max_pos, stream=_stream())
    return s.pool


# ---- what a pass cannot do without, and its result from the definition --------------------------


def work(case):
    if case["kind"] == "lora":
        m, k, n, rank = case["m"], case["k"], case["n"], case["rank"]
        down = len(_slice_ends(case)) * rank
        used = min(case["adapters"], m)
        return {"bytes": 2 * m * k + 4 * m * n + 4 * m + 2 * used * (down * k + rank * n),
                "flops": 2 * m * (down * k + rank * n)}
    if case["kind"] == "table":
        return {"bytes": 4 * case["rows"] * case["rot"], "flops": 40 * case["rows"] * case["rot"] // 2}
    kv_dim = case["kv_heads"] * case["dim"]
    if case["kind"] == "rope":
        m, q_dim, table = case["m"], case["q_heads"] * case["dim"], 4 * min(case["m"], 16384) * case["rot"]
        size = {"none": 2, "fp16": 2, "fp8": 1}[case["cache"]]
        values = 1 if case["cache"] == "none" else 2  # K alone, or K and V
        return {"bytes": m * (4 * q_dim + values * (2 + size) * kv_dim + 12) + table,
                "flops": 3 * m * (case["q_heads"] + case["kv_heads"]) * case["rot"]}
    # sequences of 7/8 of the length on average, of which an eighth or a half moves
    rows = case["seqs"] * case["length"] * 7 // 8 // (8 if case["keep"] == "window" else 2)
    return {"bytes": rows * case["layers"] * 4 * kv_dim * (2 if case["cache"] == "fp16" else 1),
            "flops": 3 * rows * case["layers"] * case["kv_heads"] * case["rot"]}


def _exact_lora(s, case):
    m, n, slices = case["m"], case["n"], len(s.ends)
    if m * n > 1 << 26:
        # the tokens of one adapter at a time would do; all at once take too much memory
        tokens = torch.split(torch.arange(m, device="cuda"), 1024)
    else:
        tokens = [torch.arange(m, device="cuda")]
    out = s.y.to(torch.float64)
    begin = [0] + s.ends[:-1]
    for some in tokens:
        for adapter in torch.unique(s.ids[some]).tolist():
            if adapter < 0:
                continue
            t = some[s.ids[some] == adapter]
            r = int(s.ranks[adapter])
            x = s.x[t].to(torch.float64)
            for j in range(slices):
                down = torch.mm(x, s.a[adapter, j, :r].to(torch.float64).t().contiguous())
                up = s.b[adapter, begin[j]:s.ends[j], :r].to(torch.float64).t().contiguous()
                out[t, begin[j]:s.ends[j]] += s.scales[adapter].double() * torch.mm(down, up)
    return out


def _exact_table(s, case):
    rot, context, factor = case["rot"], 8192, s.factor
    base = s.base * factor ** (rot / (rot - 2)) if case["scaling"] == "ntk" else s.base
    freqs, mult = [], 1.0
    edge = lambda turns: rot * math.log(context / (2 * math.pi * turns)) / 2 / math.log(base)  # noqa: E731
    low, high = max(0, math.floor(edge(32))), min(rot - 1, math.ceil(edge(1)))
    for i in range(rot // 2):
        f = math.exp(-2 * i / rot * math.log(base))
        if case["scaling"] == "linear":
            f /= factor
        elif case["scaling"] == "bands":
            wave = 2 * math.pi / f
            if wave > context / 1.0:
                f /= factor
            elif wave >= context / 4.0:
                part = (context / wave - 1.0) / 3.0
                f = (1 - part) * f / factor + part * f
        elif case["scaling"] == "yarn":
            part = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            f = f / factor * part + f * (1 - part)
            mult = 0.1 * math.log(factor) + 1.0
        freqs.append(f)
    position = torch.arange(case["first"], case["first"] + case["rows"], device="cuda").double()
    turned = torch.polar(torch.full_like(position, mult)[:, None].expand(-1, len(freqs)).contiguous(),
                         torch.outer(position, torch.tensor(freqs, device="cuda", dtype=torch.float64)))
    return {"cos": turned.real.contiguous(), "sin": turned.imag.contiguous()}


def _exact_turn(x, cos, sin, rot, layout):
    """x in 64 bits as complex numbers, times cos + i sin."""
    out = x.clone()
    if layout == "half":
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous())
    else:
        z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous())
    z = z * torch.complex(cos.double(), sin.double())
    if layout == "half":
        out[..., :rot // 2], out[..., rot // 2:rot] = z.real, z.imag
    else:
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    return out


def _nearest_fp8(v):
    """The E4M3 value nearest to each of v, in 64 bits: 3 bits behind the leading one, steps of 2^-9 at least."""
    v = torch.clamp(v, -448, 448)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -20))), min=-6) - 3)
    return torch.round(v / step) * step


def _exact_rope(s, case):
    m, dim, q, kv_heads, fp8 = case["m"], case["dim"], case["q_heads"], case["kv_heads"], case["cache"] == "fp8"
    x = s.x.double().reshape(m, -1, dim)
    p = s.positions.long()
    y = _exact_turn(x[:, :q + kv_heads], s.cos[p].unsqueeze(1), s.sin[p].unsqueeze(1), case["rot"], case["layout"])
    out = {"q": y[:, :q].reshape(m, -1)}
    if case["cache"] == "none":
        out["k"] = y[:, q:].reshape(m, -1)
        return out
    cache = s.pool[1].float().double()
    for which, value in enumerate((y[:, q:], x[:, q + kv_heads:])):
        if fp8:
            value = _nearest_fp8(value / s.scales[1, which].double()[:, None])
        cache[which].index_copy_(0, s.slots, value)
    out["cache"] = cache
    return out


def _exact_compact(s, case):
    src, dst, moved = _places(s)
    out = torch.empty(s.pool.shape, device="cuda", dtype=torch.float64)
    for layer in range(case["layers"]):
        old = s.pool[layer].float().double()
        k = _exact_turn(old[0][src], s.cos[moved].unsqueeze(1), -s.sin[moved].unsqueeze(1), case["rot"],
                        case["layout"])
        out[layer] = old
        out[layer, 0].index_copy_(0, dst, _nearest_fp8(k) if case["cache"] == "fp8" else k)
        out[layer, 1].index_copy_(0, dst, old[1][src])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"lora": _exact_lora, "table": _exact_table, "rope": _exact_rope,
            "compact": _exact_compact}[case["kind"]](s, case)
