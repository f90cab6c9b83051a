// kv_compact.hip — rows dropped out of cached sequences, what stays moved up, for gfx950.
//
// Rows move in place: row i is overwritten with row keep[i] >= i of the same sequence, which may
// itself be overwritten later. Two ways through, and the device says which, sequence by sequence:
//
// Apart. What is written is read by nobody: either the first source lies behind the last destination
// (a window's latest rows move up behind the first ones), or every block written is a new one (the old ones
// are shared). Any order will do: workgroups take rows, threads a chunk of some heads.
//
// In order. Columns do not mix (a head's pairs aside), so a workgroup takes some heads of one
// layer's K or V and walks down the sequence's rows, a step at a time: it loads the step's rows,
// meets at a barrier, and stores them. Two facts keep it right:
//   * keep is strictly increasing, so a later step's sources lie behind this step's
//     destinations: its loads may be issued before this step's stores, and are;
//   * stores of a step follow a barrier that every wave reaches with its loads in registers, so
//     no source within the step (or before it) is overwritten unread.
// No workspace, no copy to spare blocks, no order between workgroups.
//
// Bound by memory: one sequence of 8192 rows cut to 1028, 28 layers, fp16, in 52 us (206 MB read and
// written, 3.9 TB/s); 13 sequences of 3000 cut to half, 4 layers, FP8, into new blocks 77 us (3.7
// TB/s), in place 87. Runs of 8 instead of 16 bytes, 8 heads to a thread instead of 4, and 2 or 4
// rows measured the same within 10 %.
#include <algorithm>

#include "af_common.h"
#include "af_device.h"
#include "af_kv_pool.h"
#include "af_rope.h"

namespace af {
namespace {

constexpr int kThreads = 512;        // at most
constexpr int kHeadsOfThread = 4;  // apart: heads of a thread at a time, which share their cos and sin
constexpr int kHeadsInOrder = 2;   // in order: heads of a workgroup
constexpr int kMaxStepRows = kThreads;
constexpr int kManyParts = 4096;   // apart: workgroups

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
    int rows;              // in order: rows of a step
    int groups;            // in order: of heads
    int lanes, apart_rows; // apart: threads of a row's heads, rows at a time
    int parts, part_rows;  // apart: workgroups of a sequence's rows, rows of each
};

// A run of W elements, as it lies in memory.
template <int BYTES>
struct RunOf;
template <>
struct RunOf<16> {
    typedef uint4 type;
};
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

// Element offsets of a chunk's two runs.
struct Runs {
    int a, b;
};

template <int LAYOUT, bool FP8, int W>
struct Mover {
    static constexpr int kBytes = FP8 ? 1 : 2;
    typedef typename RunOf<W * kBytes>::type Run;

    // Where row i of the sequence's moves comes from and goes to.
    static __device__ __forceinline__ Meta plan(const CompactArgs& p, int seq, int begin, int first, int i,
                                                bool report) {
        const int64_t capacity = int64_t(p.max_blocks) << p.bs_log2;
        const int in_block = (1 << p.bs_log2) - 1;
        Meta r{-1, 0, 0};
        const int from = p.keep[begin + i];
        const int64_t to = int64_t(first) + i;
        const int64_t moved = from - to;
        bool ok = to >= 0 && moved >= 0 && from < capacity && (p.rot == 0 || moved < p.max_pos);
        if (ok) {
            const int64_t sb = p.src_tables[size_t(seq) * p.max_blocks + (from >> p.bs_log2)];
            const int64_t db = p.dst_tables[size_t(seq) * p.max_blocks + (to >> p.bs_log2)];
            ok = sb >= 0 && sb < p.total_blocks && db >= 0 && db < p.total_blocks;
            const int64_t src = (sb << p.bs_log2) | (from & in_block);
            const int64_t dst = (db << p.bs_log2) | (to & in_block);
            if (ok && src != dst) r = Meta{src, dst, int(moved)};
        }
        if (!ok && p.status && report) *p.status = AF_ERR_OUT_OF_RANGE;
        return r;
    }
    static __device__ __forceinline__ Runs runs(const CompactArgs& p, int chunk, bool turns, bool rotated) {
        if (!turns) return {chunk * W, p.head_dim / 2 + chunk * W};
        const int a = LAYOUT == AF_ROPE_HALF && rotated ? chunk * W : chunk * 2 * W;
        return {a, LAYOUT == AF_ROPE_HALF && rotated ? p.rot / 2 + chunk * W : a + W};
    }
    static __device__ __forceinline__ void load_turn(const CompactArgs& p, int moved, int chunk, float (&c)[W],
                                                     float (&s)[W]) {
        const size_t at = size_t(moved) * (p.rot / 2) + chunk * W;
        load_floats<W>(p.cos_t + at, c);
        load_floats<W>(p.sin_t + at, s);
    }
    static __device__ __forceinline__ void store(uint8_t* head, Runs e, const Run& a, const Run& b, bool turn,
                                                 const float (&c)[W], const float (&s)[W]) {
        if (!turn) {
            *reinterpret_cast<Run*>(head + e.a * kBytes) = a;
            *reinterpret_cast<Run*>(head + e.b * kBytes) = b;
        } else if constexpr (FP8) {
            float x[W], y[W];
            load_fp8<W>(reinterpret_cast<const uint8_t*>(&a), x);
            load_fp8<W>(reinterpret_cast<const uint8_t*>(&b), y);
            rotate_floats<LAYOUT, W>(x, y, c, s);
            store_fp8<W>(head + e.a, x);
            store_fp8<W>(head + e.b, y);
        } else {
            uint16_t x[W], y[W];
            load_halves<W>(reinterpret_cast<const uint16_t*>(&a), x);
            load_halves<W>(reinterpret_cast<const uint16_t*>(&b), y);
            rotate_halves<LAYOUT, W>(x, y, c, s);
            store_halves<W>(reinterpret_cast<uint16_t*>(head) + e.a, x);
            store_halves<W>(reinterpret_cast<uint16_t*>(head) + e.b, y);
        }
    }
    static __device__ __forceinline__ void turn_back(const CompactArgs& p, float (&c)[W], float (&s)[W]) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            c[i] = c[i] * p.inv_factor;
            s[i] = -s[i] * p.inv_factor;
        }
    }
};

template <int LAYOUT, bool FP8, int W>
__global__ __launch_bounds__(kThreads) void kv_compact_kernel(const CompactArgs p) {
    typedef Mover<LAYOUT, FP8, W> M;
    typedef typename M::Run Run;
    constexpr int kBytes = M::kBytes;
    constexpr int HU = kHeadsOfThread, HO = kHeadsInOrder;
    __shared__ Meta meta[3][kMaxStepRows];
    const int seq = blockIdx.y;
    const int which = blockIdx.x;  // 2 layer + {K, V}
    const bool is_k = (which & 1) == 0;
    const int begin = p.start[seq];
    const int n = min(p.start[seq + 1] - begin, p.max_rows);
    if (n <= 0) return;
    const int first = p.first[seq];
    const int chunk = int(threadIdx.x) % p.chunks;
    const bool rotated = is_k && chunk < p.rot / (2 * W);
    const Runs e = M::runs(p, chunk, is_k && p.rot > 0, rotated);
    uint8_t* slab = p.base + size_t(which) * p.slab;

    bool apart = p.keep[begin] >= int64_t(first) + n;
    if (!apart) {
        bool same = false;
        const int64_t last = min((int64_t(first) + n - 1) >> p.bs_log2, int64_t(p.max_blocks) - 1);
        for (int64_t b = (int64_t(max(first, 0)) >> p.bs_log2) + threadIdx.x; b <= last; b += blockDim.x) {
            const size_t at = size_t(seq) * p.max_blocks + b;
            same |= p.src_tables[at] == p.dst_tables[at];
        }
        apart = !__syncthreads_or(same);
    }
    if (apart) {
        if (int(blockIdx.z) >= p.parts) return;
        const int lane = int(threadIdx.x) / p.chunks % p.lanes;  // heads lane, lane + lanes, ...
        const int row0 = int(threadIdx.x) / (p.chunks * p.lanes);
        Meta* plans = &meta[0][0];
#pragma unroll 1
        for (int64_t rows0 = int64_t(blockIdx.z) * p.part_rows; rows0 < n; rows0 += int64_t(p.parts) * p.part_rows) {
            // the rows, planned at once
            const int mine = min(p.part_rows, int(n - rows0));
            for (int t = threadIdx.x; t < mine; t += blockDim.x)
                plans[t] = M::plan(p, seq, begin, first, int(rows0) + t, which == 0);
            __syncthreads();
#pragma unroll 1
            for (int i = row0; i < mine && row0 < p.apart_rows; i += p.apart_rows) {
                const Meta r = plans[i];
                if (r.src < 0) continue;
                const uint8_t* from = slab + r.src * p.row_bytes;
                uint8_t* to = slab + r.dst * p.row_bytes;
                const bool turn = rotated && r.moved != 0;
                float c[W], s[W];
                if (turn) M::load_turn(p, r.moved, chunk, c, s);
                for (int h0 = lane; h0 < p.n_kv_heads; h0 += HU * p.lanes) {
                    Run a[HU], b[HU];
#pragma unroll
                    for (int j = 0; j < HU; ++j) {
                        const int h = h0 + j * p.lanes;
                        if (h >= p.n_kv_heads) break;
                        const uint8_t* head = from + size_t(h) * p.head_dim * kBytes;
                        a[j] = *reinterpret_cast<const Run*>(head + e.a * kBytes);
                        b[j] = *reinterpret_cast<const Run*>(head + e.b * kBytes);
                    }
                    if (turn && h0 == lane) M::turn_back(p, c, s);
#pragma unroll
                    for (int j = 0; j < HU; ++j) {
                        const int h = h0 + j * p.lanes;
                        if (h >= p.n_kv_heads) break;
                        M::store(to + size_t(h) * p.head_dim * kBytes, e, a[j], b[j], turn, c, s);
                    }
                }
            }
            __syncthreads();
        }
        return;
    }

    if (int(blockIdx.z) >= p.groups) return;
    const int head0 = int(blockIdx.z) * HO;
    const int lane_row = int(threadIdx.x) / p.chunks;
    const bool here = lane_row < p.rows;
    const int steps = (n - 1) / p.rows + 1;
    auto plan = [&](int step) {
        const int t = threadIdx.x;
        const int64_t i = int64_t(step) * p.rows + t;  // (steps past the last one are planned too)
        if (t < p.rows)
            meta[step % 3][t] = i < n ? M::plan(p, seq, begin, first, int(i), which == 0 && blockIdx.z == 0)
                                      : Meta{-1, 0, 0};
    };
    struct Held {
        Run a[HO], b[HO];
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
        for (int i = 0; i < HO; ++i) {
            if (head0 + i >= p.n_kv_heads) break;
            const uint8_t* head = row + size_t(head0 + i) * p.head_dim * kBytes;
            h.a[i] = *reinterpret_cast<const Run*>(head + e.a * kBytes);
            h.b[i] = *reinterpret_cast<const Run*>(head + e.b * kBytes);
        }
        h.turn = rotated && r.moved != 0;
        if (h.turn) M::load_turn(p, r.moved, chunk, h.c, h.s);
    };
    auto store = [&](Held& h) {
        if (!h.live) return;
        uint8_t* row = slab + h.dst * p.row_bytes;
        if (h.turn) M::turn_back(p, h.c, h.s);
#pragma unroll
        for (int i = 0; i < HO; ++i) {
            if (head0 + i >= p.n_kv_heads) break;
            M::store(row + size_t(head0 + i) * p.head_dim * kBytes, e, h.a[i], h.b[i], h.turn, h.c, h.s);
        }
    };
    plan(0);
    plan(1);
    __syncthreads();
    Held now, next;
    load(0, now);
#pragma unroll 1
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
    p.chunks = p.head_dim / (2 * W);
    if (p.chunks > kThreads || n_layers > INT32_MAX / 2) return AF_ERR_UNSUPPORTED;
    p.groups = ceil_div(p.n_kv_heads, kHeadsInOrder);
    const int64_t others = int64_t(2) * n_layers * n_seqs;
    // Long sequences, in order, where workgroups are few: longer steps (one sequence of 2000 rows,
    // 28 layers, half of them kept in place: 43 us, with 256 threads 59). Else 256 threads: 13
    // sequences of 3000 rows, 4 layers, FP8, into new blocks: 76 us, with 512 threads 82.
    const int threads = p.chunks > 256 || (others * p.groups < 400 && p.max_rows > 512) ? 512 : 256;
    p.rows = threads / p.chunks;
    p.lanes = std::min(ceil_div(p.n_kv_heads, kHeadsOfThread), threads / p.chunks);
    p.apart_rows = std::max(1, threads / (p.chunks * p.lanes));
    // apart: one row to a thread, two where there are many workgroups anyway
    p.part_rows = p.apart_rows;
    p.parts = ceil_div(p.max_rows, p.part_rows);
    if (others * p.parts > kManyParts) {
        p.part_rows *= 2;
        p.parts = ceil_div(p.max_rows, p.part_rows);
    }
    p.parts = std::min(p.parts, kManyParts);
    const int z = std::max(p.groups, p.parts);
    if (z > 65535) return AF_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((kv_compact_kernel<LAYOUT, FP8, W>), dim3(2 * n_layers, n_seqs, z), dim3(threads), 0, s, p);
    AF_TRY_LAUNCH();
    return AF_OK;
}

template <int LAYOUT, bool FP8>
int launch_compact(CompactArgs& p, int n_seqs, int n_layers, hipStream_t s) {
    // 16-byte, 8-byte or single runs
    constexpr int w = FP8 ? 16 : 8;
    auto fits = [&](int w) { return p.head_dim % (2 * w) == 0 && p.rot % (2 * w) == 0; };
    if (fits(w)) return launch_compact<LAYOUT, FP8, w>(p, n_seqs, n_layers, s);
    if (fits(w / 2)) return launch_compact<LAYOUT, FP8, w / 2>(p, n_seqs, n_layers, s);
    return launch_compact<LAYOUT, FP8, 1>(p, n_seqs, n_layers, s);
}

template <int LAYOUT>
int launch_compact(CompactArgs& p, bool fp8, int n_seqs, int n_layers, hipStream_t s) {
    return fp8 ? launch_compact<LAYOUT, true>(p, n_seqs, n_layers, s)
               : launch_compact<LAYOUT, false>(p, n_seqs, n_layers, s);
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
