// kv_compact.hip — rows dropped out of cached sequences, what stays moved up, for gfx950.
//
// Rows move in place: row i is overwritten with row keep[i] >= i of the same sequence, which may
// itself be overwritten later. Columns do not mix (a head's pairs aside), so a workgroup takes
// some heads of one layer's K or V and walks down the sequence's rows, a chunk at a time: it
// loads the chunk's rows, meets at a barrier, and stores them. Two facts keep it right:
//   * keep is strictly increasing, so a later chunk's sources lie behind this chunk's
//     destinations: its loads may be issued before this chunk's stores, and are;
//   * stores of a chunk follow a barrier that every wave reaches with its loads in registers, so
//     no source within the chunk (or before it) is overwritten unread.
// No workspace, no copy to spare blocks, no order between workgroups.
#include <algorithm>

#include "af_common.h"
#include "af_device.h"
#include "af_kv_pool.h"
#include "af_rope.h"

namespace af {
namespace {

constexpr int kMaxChunkRows = 256;

struct CompactArgs {
    uint8_t* base;
    int64_t slab;          // bytes of a layer's K (or V)
    int64_t row_bytes;
    int64_t total_blocks;
    int bs_log2;
    int n_kv_heads, head_dim;
    const int32_t* src_tables;
    const int32_t* dst_tables;
    int max_blocks;
    const int32_t* keep;
    const int32_t* start;
    const int32_t* first;
    int max_rows;
    int rot;               // 0: no turn
    const float* cos_t;
    const float* sin_t;
    int max_pos;
    float inv_factor;
    int32_t* status;
    int chunks;            // of a head: 2 W elements each
    int rows;              // rows of a chunk of the walk
    int groups;            // of heads
};

// A run of W elements, as it lies in memory.
template <int BYTES>
struct RunOf;
template <>
struct RunOf<8> {
    typedef uint2 type;
};
template <>
struct RunOf<2> {
    typedef uint16_t type;
};
template <>
struct RunOf<1> {
    typedef uint8_t type;
};

struct Meta {
    int64_t src, dst;  // physical rows; src < 0: nothing moves
    int moved;
};

template <int LAYOUT, bool FP8, int W, int HU>
__global__ __launch_bounds__(1024) void kv_compact_kernel(const CompactArgs p) {
    constexpr int kBytes = FP8 ? 1 : 2;
    typedef typename RunOf<W * kBytes>::type Run;
    __shared__ Meta meta[3][kMaxChunkRows];
    const int seq = blockIdx.y;
    const int group = int(blockIdx.x) % p.groups;
    const int which = int(blockIdx.x) / p.groups;  // 2 layer + {K, V}
    const bool is_k = (which & 1) == 0;
    const int chunk = int(threadIdx.x) % p.chunks;
    const int lane_row = int(threadIdx.x) / p.chunks;
    const bool here = lane_row < p.rows;

    const int begin = p.start[seq];
    const int n = min(p.start[seq + 1] - begin, p.max_rows);
    if (n <= 0) return;
    const int first = p.first[seq];
    const int steps = (n + p.rows - 1) / p.rows;
    const int64_t capacity = int64_t(p.max_blocks) << p.bs_log2;
    const int in_block = (1 << p.bs_log2) - 1;

    auto plan = [&](int step) {
        for (int t = threadIdx.x; t < p.rows; t += blockDim.x) {
            Meta r{-1, 0, 0};
            const int i = step * p.rows + t;
            if (i < n) {
                const int from = p.keep[begin + i];
                const int64_t to = int64_t(first) + i;
                const int64_t moved = from - to;
                bool ok = to >= 0 && moved >= 0 && from < capacity &&
                          (p.rot == 0 || moved < p.max_pos);
                if (ok) {
                    const int64_t sb = p.src_tables[size_t(seq) * p.max_blocks + (from >> p.bs_log2)];
                    const int64_t db = p.dst_tables[size_t(seq) * p.max_blocks + (to >> p.bs_log2)];
                    ok = sb >= 0 && sb < p.total_blocks && db >= 0 && db < p.total_blocks;
                    const int64_t src = (sb << p.bs_log2) | (from & in_block);
                    const int64_t dst = (db << p.bs_log2) | (to & in_block);
                    if (ok && src != dst) r = Meta{src, dst, int(moved)};
                }
                if (!ok && p.status && blockIdx.x == 0) *p.status = AF_ERR_OUT_OF_RANGE;
            }
            meta[step % 3][t] = r;
        }
    };

    const bool turns = is_k && p.rot > 0;
    const bool rotated = turns && chunk < p.rot / (2 * W);
    const int e0 = LAYOUT == AF_ROPE_HALF && rotated ? chunk * W : chunk * 2 * W;
    const int e1 = LAYOUT == AF_ROPE_HALF && rotated ? p.rot / 2 + chunk * W : e0 + W;
    const int head0 = group * HU;
    uint8_t* slab = p.base + size_t(which) * p.slab;

    struct Held {
        Run a[HU], b[HU];
        float c[W], s[W];
        int64_t dst;
        bool live, turn;
    };
    auto load = [&](int step, Held& h) {
        h.live = h.turn = false;
        if (!here || step >= steps) return;
        const Meta r = meta[step % 3][lane_row];
        h.live = r.src >= 0;
        if (!h.live) return;
        h.dst = r.dst;
        const uint8_t* row = slab + r.src * p.row_bytes;
#pragma unroll
        for (int i = 0; i < HU; ++i) {
            if (head0 + i >= p.n_kv_heads) break;
            const uint8_t* head = row + size_t(head0 + i) * p.head_dim * kBytes;
            h.a[i] = *reinterpret_cast<const Run*>(head + e0 * kBytes);
            h.b[i] = *reinterpret_cast<const Run*>(head + e1 * kBytes);
        }
        h.turn = rotated && r.moved != 0;
        if (h.turn) {
            const size_t at = size_t(r.moved) * (p.rot / 2) + chunk * W;
            load_floats<W>(p.cos_t + at, h.c);
            load_floats<W>(p.sin_t + at, h.s);
        }
    };
    auto store = [&](Held& h) {
        if (!h.live) return;
        uint8_t* row = slab + h.dst * p.row_bytes;
        float c[W], s[W];
        if (h.turn) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                c[i] = h.c[i] * p.inv_factor;
                s[i] = -h.s[i] * p.inv_factor;
            }
        }
#pragma unroll
        for (int i = 0; i < HU; ++i) {
            if (head0 + i >= p.n_kv_heads) break;
            uint8_t* head = row + size_t(head0 + i) * p.head_dim * kBytes;
            if (!h.turn) {
                *reinterpret_cast<Run*>(head + e0 * kBytes) = h.a[i];
                *reinterpret_cast<Run*>(head + e1 * kBytes) = h.b[i];
            } else if constexpr (FP8) {
                float x[W], y[W];
                load_fp8<W>(reinterpret_cast<const uint8_t*>(&h.a[i]), x);
                load_fp8<W>(reinterpret_cast<const uint8_t*>(&h.b[i]), y);
                rotate_floats<LAYOUT, W>(x, y, c, s);
                store_fp8<W>(head + e0, x);
                store_fp8<W>(head + e1, y);
            } else {
                uint16_t x[W], y[W];
                load_halves<W>(reinterpret_cast<const uint16_t*>(&h.a[i]), x);
                load_halves<W>(reinterpret_cast<const uint16_t*>(&h.b[i]), y);
                rotate_halves<LAYOUT, W>(x, y, c, s);
                store_halves<W>(reinterpret_cast<uint16_t*>(head) + e0, x);
                store_halves<W>(reinterpret_cast<uint16_t*>(head) + e1, y);
            }
        }
    };

    plan(0);
    plan(1);
    __syncthreads();
    Held now, next;
    load(0, now);
    for (int step = 0; step < steps; ++step) {
        plan(step + 2);      // (its slot was last read before the barrier of the step before)
        wait_vmcnt<0>();     // this wave's rows of the step are in registers
        __syncthreads();
        load(step + 1, next);
        store(now);
        now = next;
    }
}

template <int LAYOUT, bool FP8, int W>
int launch_compact(CompactArgs& p, int n_seqs, int n_layers, hipStream_t s) {
    constexpr int HU = 2;
    p.chunks = p.head_dim / (2 * W);
    p.groups = ceil_div(p.n_kv_heads, HU);
    const int64_t blocks = int64_t(p.groups) * 2 * n_layers;
    if (blocks > INT32_MAX || p.chunks > 1024) return AF_ERR_UNSUPPORTED;
    const int threads = p.chunks > 256 || (blocks * n_seqs < 1024 && p.max_rows > 256 / p.chunks)
                            ? 1024 : 256;
    p.rows = std::min(kMaxChunkRows, threads / p.chunks);
    hipLaunchKernelGGL((kv_compact_kernel<LAYOUT, FP8, W, HU>), dim3(unsigned(blocks), n_seqs),
                       dim3(threads), 0, s, p);
    AF_TRY_LAUNCH();
    return AF_OK;
}

template <int LAYOUT>
int launch_compact(CompactArgs& p, bool fp8, int n_seqs, int n_layers, hipStream_t s) {
    const int w = fp8 ? 8 : 4;  // 8-byte runs
    const bool wide = p.head_dim % (2 * w) == 0 && p.rot % (2 * w) == 0;
    if (fp8)
        return wide ? launch_compact<LAYOUT, true, 8>(p, n_seqs, n_layers, s)
                    : launch_compact<LAYOUT, true, 1>(p, n_seqs, n_layers, s);
    return wide ? launch_compact<LAYOUT, false, 4>(p, n_seqs, n_layers, s)
                : launch_compact<LAYOUT, false, 1>(p, n_seqs, n_layers, s);
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" int af_kv_compact(const af_kv_pool* pool, const int32_t* d_src_tables,
                             const int32_t* d_dst_tables, int max_blocks, int n_seqs,
                             const int32_t* d_keep, const int32_t* d_start, const int32_t* d_first,
                             int max_rows, int rot_dim, int layout, const float* cos_table,
                             const float* sin_table, int max_pos, float table_factor,
                             int32_t* d_status, af_stream_t stream) {
    if (int st = check_pool(pool)) return st;
    auto on = [](const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; };
    if (n_seqs < 0 || max_blocks <= 0 || max_rows < 0 || rot_dim < 0 || rot_dim % 2 ||
        rot_dim > pool->head_dim || pool->head_dim % 2)
        return AF_ERR_INVALID_ARG;
    if (layout != AF_ROPE_HALF && layout != AF_ROPE_INTERLEAVED) return AF_ERR_UNSUPPORTED;
    if (rot_dim > 0 && (!cos_table || !sin_table || !on(cos_table, 16) || !on(sin_table, 16) ||
                        max_pos <= 0 || !(table_factor > 0.0f) || !(1.0f / table_factor > 0.0f)))
        return AF_ERR_INVALID_ARG;
    if (n_seqs > 65535) return AF_ERR_UNSUPPORTED;
    if (n_seqs == 0 || max_rows == 0) return AF_OK;
    if (!d_src_tables || !d_dst_tables || !d_keep || !d_start || !d_first ||
        !on(d_src_tables, 4) || !on(d_dst_tables, 4) || !on(d_keep, 4) || !on(d_start, 4) ||
        !on(d_first, 4) || !on(d_status, 4))
        return AF_ERR_INVALID_ARG;
    CompactArgs p{};
    p.base = static_cast<uint8_t*>(pool->base);
    p.slab = int64_t(pool_slab_bytes(*pool));
    p.row_bytes = int64_t(pool_row_bytes(*pool));
    p.total_blocks = pool->total_blocks;
    p.bs_log2 = __builtin_ctz(unsigned(pool->block_size));
    p.n_kv_heads = pool->n_kv_heads;
    p.head_dim = pool->head_dim;
    p.src_tables = d_src_tables;
    p.dst_tables = d_dst_tables;
    p.max_blocks = max_blocks;
    p.keep = d_keep;
    p.start = d_start;
    p.first = d_first;
    p.max_rows = max_rows;
    p.rot = rot_dim;
    p.cos_t = cos_table;
    p.sin_t = sin_table;
    p.max_pos = max_pos;
    p.inv_factor = rot_dim > 0 ? 1.0f / table_factor : 1.0f;
    p.status = d_status;
    const bool fp8 = pool->dtype == AF_KV_FP8_E4M3;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return layout == AF_ROPE_HALF
               ? launch_compact<AF_ROPE_HALF>(p, fp8, n_seqs, pool->n_layers, s)
               : launch_compact<AF_ROPE_INTERLEAVED>(p, fp8, n_seqs, pool->n_layers, s);
}
