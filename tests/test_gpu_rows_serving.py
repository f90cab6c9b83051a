"""A token's way from the projection into the cache and out of it: projection, adapters, rotary positions of a
stretched table, append, attention, and compaction in between, enqueued one after the other as an engine would;
each stage against 64 bits on what the stage before left. And a decode step captured and replayed."""
import numpy as np
import pytest

from atomflow_amd import AF_KV_FP16, AF_KV_FP8_E4M3, AF_ROPE_INTERLEAVED
from atomflow_amd import device as dev
from atomflow_amd import kv
from inputs import ATOL_FP8, ATOL_F16, RTOL_F16, RTOL_FP8, assert_attn_close, gemv_case
from rows_ref import EPS24, assert_compact, assert_fp8, assert_lora, e4m3_decode, lora, turn, turn_bound

pytestmark = pytest.mark.gpu
NQ, NK, HD, ROT, K, BS, LAYERS, BLOCKS, MAX_POS = 4, 2, 128, 64, 256, 16, 2, 40, 256
N = (NQ + 2 * NK) * HD
ENDS = [NQ * HD, (NQ + NK) * HD, N]
RANK, ADAPTERS = 16, 3


def say(msg):
    print(f"[case] {msg}", flush=True)


def up(a):
    return dev.DeviceBuffer.from_array(np.ascontiguousarray(a))


class Engine:
    def __init__(self, fp8, seed):
        r = self.r = np.random.default_rng(seed)
        self.fp8 = fp8
        self.w, _, self.ws = gemv_case(N, K, seed)
        self.a = (r.standard_normal((ADAPTERS, 3, RANK, K)) / 16).astype(np.float16)
        self.b = (0.1 * r.standard_normal((ADAPTERS, N, RANK))).astype(np.float16)
        self.ranks = np.array([16, 5, 0], np.int32)
        self.lscales = np.array([1.5, 0.5, 1.0], np.float32)
        freq, self.mult = kv.rope_frequencies(ROT, 10000.0, "yarn", 4.0, 64)
        self.cos, self.sin = (dev.DeviceBuffer(MAX_POS * ROT // 2 * 4) for _ in range(2))
        kv.build_rope_table_scaled(self.cos, self.sin, 0, MAX_POS, ROT, freq, self.mult)
        self.c, self.s = (t.download(np.float32, (MAX_POS, ROT // 2)) for t in (self.cos, self.sin))
        shape = (LAYERS, 2, BLOCKS * BS, NK, HD)
        self.pool = dev.DeviceBuffer(int(np.prod(shape)) * (1 if fp8 else 2))
        self.pool.fill_u32(0)
        self.shape, self.dtype = shape, np.uint8 if fp8 else np.float16
        self.scales = (0.02 + 0.02 * r.random((LAYERS, 2, NK))).astype(np.float32)
        self.bufs = [up(t) for t in (self.w, self.ws, self.a, self.b, self.ranks, self.lscales, self.scales)]
        dw, dws, da, db, dr, dl, dsc = self.bufs
        self.desc = kv.make_pool(self.pool.ptr, AF_KV_FP8_E4M3 if fp8 else AF_KV_FP16, BS, LAYERS, NK, HD, BLOCKS,
                                 scales=dsc.ptr if fp8 else None)
        self.lora = kv.make_lora(da, db, ADAPTERS, RANK, K, ENDS, ranks=dr, scales=dl)
        self.lws = dev.DeviceBuffer(kv.lora_workspace_size(self.lora, 256))

    def get(self):
        return self.pool.download(self.dtype, self.shape)

    def enqueue(self, layer, m, x, ids, slots, pos, y, z, q, stream=None):
        kv.launch_w8a16_gemm_batched(x, K, m, self.bufs[0], self.bufs[1], y, N, N, K, stream=stream)
        kv.launch_lora_add(x, K, m, ids, self.lora, y, N, z, N, self.lws, self.lws.nbytes, stream=stream)
        kv.launch_paged_rope_append_rows(z, N, m, q, NQ * HD, NQ, self.desc, layer, slots, pos, ROT,
                                         AF_ROPE_INTERLEAVED, self.cos, self.sin, MAX_POS, stream=stream)

    def step(self, layer, ids, slots, pos):
        """One layer's projections and append of m tokens, checked; returns Q on the device."""
        m = len(ids)
        x = self.r.standard_normal((m, K)).astype(np.float16)
        y, z, q = (dev.DeviceBuffer(m * n * 2) for n in (N, N, NQ * HD))
        before = self.get()
        d = [up(t) for t in (x, np.asarray(ids, np.int32), np.asarray(slots, np.int64), np.asarray(pos, np.int32))]
        self.enqueue(layer, m, *d, y, z, q)
        yh, zh, qh = (t.download(np.float16, (m, n)) for t, n in ((y, N), (z, N), (q, NQ * HD)))
        assert_lora(zh, *lora(x, ids, self.a, self.b, self.ranks, self.lscales, ENDS, yh))
        heads = zh.reshape(m, -1, HD)
        t, mag = turn(heads[:, :NQ + NK], self.c[pos], self.s[pos], ROT, AF_ROPE_INTERLEAVED)
        assert np.all(np.abs(qh.reshape(m, NQ, HD) - t[:, :NQ]) <= turn_bound(t, mag)[:, :NQ])
        after = self.get()
        k, v = after[layer, 0][slots], after[layer, 1][slots]
        kx, vx = t[:, NQ:], heads[:, NQ + NK:].astype(np.float64)
        if self.fp8:
            ks, vs = (self.scales[layer, i].astype(np.float64)[:, None] for i in (0, 1))
            assert_fp8(k, kx / ks, 1.01 * EPS24 * (mag[:, NQ:] + 2 * np.abs(kx)) / ks)
            assert_fp8(v, vx / vs, 1.01 * EPS24 * np.abs(vx) / vs)
        else:
            assert np.all(np.abs(k - kx) <= turn_bound(kx, mag[:, NQ:])) and np.array_equal(v, vx)
        want = before.copy()
        want[layer, 0][slots], want[layer, 1][slots] = k, v
        assert after.tobytes() == want.tobytes()
        return q

    def attend(self, layer, q, tables, lens):
        batch = len(lens)
        out = dev.DeviceBuffer(batch * NQ * HD * 2)
        ws = kv.AttentionWorkspace(batch, NQ, NK, HD, 0)
        kv.launch_paged_attention(q, NQ * HD, self.desc, layer, up(tables), tables.shape[1], up(lens), batch,
                                  int(lens.max()), out, NQ * HD, NQ, ws)
        got = out.download(np.float16, (batch, NQ, HD))
        qh = q.download(np.float16, (batch, NQ, HD)).astype(np.float64)
        pool = self.get()[layer]
        rows = e4m3_decode(pool) * self.scales[layer][:, None, :, None] if self.fp8 else pool.astype(np.float64)
        for i in range(batch):
            at = np.arange(lens[i])
            k, v = rows[:, tables[i][at // BS].astype(np.int64) * BS + at % BS]
            for h in range(NQ):
                s = k[:, h // (NQ // NK)] @ qh[i, h] / np.sqrt(HD)
                p = np.exp(s - s.max())
                want = p / p.sum() @ v[:, h // (NQ // NK)]
                assert_attn_close(got[i, h], want, ATOL_FP8 if self.fp8 else ATOL_F16,
                                  RTOL_FP8 if self.fp8 else RTOL_F16, f"sequence {i} head {h}")


@pytest.mark.parametrize("fp8", [False, True])
def test_prompt_compaction_decode(gpu, fp8):
    say(f"prompt, fork, compaction, decode; fp8={fp8}")
    e = Engine(fp8, 77)
    bm = kv.BlockManager(BLOCKS, BS, LAYERS, NK, HD, AF_KV_FP8_E4M3 if fp8 else AF_KV_FP16)
    a, c = bm.seq_create(), bm.seq_create()
    lengths = {a: 60, c: 23}
    for s, n in lengths.items():
        bm.seq_extend(s, n)
    slots = np.array([bm.seq_slot(s, i) for s, n in lengths.items() for i in range(n)], np.int64)
    pos = np.concatenate([np.arange(n) for n in lengths.values()]).astype(np.int32)
    ids = np.where(pos < 0, 0, np.repeat([0, 1], list(lengths.values()))).astype(np.int32)
    for layer in range(LAYERS):
        e.step(layer, ids, slots, pos)
    # a fork keeps a third of the prompt, and the short sequence drops its first rows, in one launch
    b = bm.seq_fork(a)
    keeps = [np.concatenate([np.arange(4), np.arange(44, 60)]), np.arange(5, 23)]
    plan = bm.plan_compact([b, c], keeps)
    before = e.get()
    d = [up(plan[k]) for k in ("src_tables", "dst_tables", "keep", "start", "first")]
    kv.kv_compact(e.desc, d[0], d[1], plan["src_tables"].shape[1], 2, d[2], d[3], d[4], plan["max_rows"], ROT,
                  AF_ROPE_INTERLEAVED, e.cos, e.sin, MAX_POS, e.mult)
    moves = [(plan["src_tables"][i], plan["dst_tables"][i], plan["first"][i],
              plan["keep"][plan["start"][i]:plan["start"][i + 1]]) for i in range(2)]
    assert_compact(e.get(), before, moves, BS, ROT, AF_ROPE_INTERLEAVED, e.c, e.s, np.float64(np.float32(e.mult)))
    # the next tokens of all three, each behind its own rows
    seqs = [a, b, c]
    slots, pos, copies = bm.plan_decode(seqs)
    assert list(pos) == [60, 20, 18]
    if len(copies):
        kv.kv_copy_blocks(e.desc, up(copies), up(np.array([len(copies)], np.int32)), len(copies))
    tables, lens = bm.export_tables(seqs, 8)
    for layer in range(LAYERS):
        q = e.step(layer, [2, 0, -1], slots, pos)
        e.attend(layer, q, tables, lens)
    bm.close()


def test_decode_step_captured(gpu):
    """Projection, adapters and append as a graph, replayed with other tokens, adapters and slots, with
    eager launches of another batch between the replays."""
    say("decode step, captured")
    e = Engine(False, 5)
    st = dev.Stream()
    m = 19
    x, ids, slots, pos = (dev.DeviceBuffer(m * n) for n in (2 * K, 4, 8, 4))
    y, z, q, y2, z2, q2 = (dev.DeviceBuffer(m * n * 2) for n in 2 * (N, N, NQ * HD))
    r = e.r

    def fill():
        x.upload(r.standard_normal((m, K)).astype(np.float16), st)
        ids.upload(r.integers(-1, ADAPTERS, m).astype(np.int32), st)
        slots.upload(r.permutation(BLOCKS * BS)[:m].astype(np.int64), st)
        pos.upload(r.integers(0, MAX_POS, m).astype(np.int32), st)

    fill()
    e.enqueue(0, m, x, ids, slots, pos, y, z, q, stream=st)
    st.sync()
    g = dev.Graph.capture(st, lambda: e.enqueue(0, m, x, ids, slots, pos, y, z, q, stream=st))
    for _ in range(4):
        fill()
        e.pool.fill_u32(0, st)
        g.launch(st)
        st.sync()
        got = [t.download(np.uint16) for t in (z, q, e.pool)]
        e.pool.fill_u32(0, st)
        e.enqueue(0, m, x, ids, slots, pos, y2, z2, q2, stream=st)
        st.sync()
        for a, b in zip(got, (z2, q2, e.pool)):
            assert np.array_equal(a, b.download(np.uint16))
    g.destroy()
    st.destroy()
