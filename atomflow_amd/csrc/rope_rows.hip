// rope_rows.hip — rotary positions in other forms for gfx950: the table of scaled angles, and
// rows turned in either pair layout, over part of the head, in place, out of place, or on their
// way into a paged cache.
#include <algorithm>
#include <cmath>

#include "af_common.h"
#include "af_device.h"
#include "af_kv_pool.h"
#include "af_rope.h"

namespace af {
namespace {

constexpr double kTwoPi = 6.283185307179586476925286766559;
constexpr int kMaxPairs = 128;  // rot_dim up to 256
constexpr int kMaxHeadDim = 512;
constexpr int kTableBlocks = 2048;  // 8 to a compute unit

// ---- the table -------------------------------------------------------------------------------
struct TableArgs {
    float* cos_t;
    float* sin_t;
    int64_t first;
    int n_rows, pairs;
    double factor;
    double turns[kMaxPairs];  // full turns per position
};

// cos and sin of t full turns, in 64 bits: t less the nearest quarter is within an eighth, an
// angle within pi/4, where Taylor's series up to x^12 (x^13 / 13! < 7e-12) is exact to fp32.
__device__ __forceinline__ void turned(double t, double& c, double& s) {
    const double r = t - __builtin_rint(t);  // within half a turn, exact
    const double q = __builtin_rint(4.0 * r);
    const double x = __builtin_fma(-0.25, q, r) * kTwoPi;
    const double z = x * x;
    double a = 1.0 / 39916800.0;
    a = __builtin_fma(-a, z, 1.0 / 362880.0);
    a = __builtin_fma(-a, z, 1.0 / 5040.0);
    a = __builtin_fma(-a, z, 1.0 / 120.0);
    a = __builtin_fma(-a, z, 1.0 / 6.0);
    const double sn = __builtin_fma(-a * z, x, x);
    double b = 1.0 / 479001600.0;
    b = __builtin_fma(-b, z, 1.0 / 3628800.0);
    b = __builtin_fma(-b, z, 1.0 / 40320.0);
    b = __builtin_fma(-b, z, 1.0 / 720.0);
    b = __builtin_fma(-b, z, 1.0 / 24.0);
    b = __builtin_fma(-b, z, 0.5);
    const double cs = __builtin_fma(-b, z, 1.0);
    const int quarter = int(q) & 3;
    const bool swap = quarter & 1;
    c = swap ? sn : cs;
    s = swap ? cs : sn;
    if (quarter == 1 || quarter == 2) c = -c;
    if (quarter >= 2) s = -s;
}

// V neighbouring pairs per thread, of every `step`-th row: their turns stay in registers, and the
// loop has no division (with one, and the turns in LDS, 40 us). About 30 64-bit operations a pair
// hide behind its 8 bytes: bound by the writes, 131072 rows of 64 pairs in 15.0 us, 4.5 TB/s.
template <int V>
__global__ __launch_bounds__(256) void rope_table_kernel(const TableArgs p) {
    const int chunks = p.pairs / V, rows = 256 / chunks;
    const int i0 = int(threadIdx.x) % chunks * V, lane_row = int(threadIdx.x) / chunks;
    if (lane_row >= rows) return;
    // (the arguments as memory: an index into a by-value argument that differs by lane would go
    // through private memory)
    typedef const __attribute__((address_space(4))) TableArgs* Args;
    const Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    double turns[V];
#pragma unroll
    for (int i = 0; i < V; ++i) turns[i] = args->turns[i0 + i];
    const int64_t step = int64_t(gridDim.x) * rows;
    for (int64_t row = int64_t(blockIdx.x) * rows + lane_row; row < p.n_rows; row += step) {
        const double pos = double(p.first + row);
        float c[V], s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            double cd, sd;
            turned(pos * turns[i], cd, sd);
            c[i] = float(cd * p.factor);
            s[i] = float(sd * p.factor);
        }
        const size_t at = size_t(row) * p.pairs + i0;
        if constexpr (V == 4) {
            *reinterpret_cast<float4*>(p.cos_t + at) = make_float4(c[0], c[1], c[2], c[3]);
            *reinterpret_cast<float4*>(p.sin_t + at) = make_float4(s[0], s[1], s[2], s[3]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) p.cos_t[at + i] = c[i], p.sin_t[at + i] = s[i];
        }
    }
}

// ---- rows ------------------------------------------------------------------------------------
enum { kNoCache, kFp16, kFp8 };

struct RowsArgs {
    const uint16_t* q;
    const uint16_t* k;  // K heads; kFp16, kFp8: V's heads follow them
    uint16_t* q_out;
    uint16_t* k_out;    // kNoCache
    int64_t q_stride, k_stride, q_out_stride, k_out_stride;
    int m, q_heads, k_heads;
    int head_dim, rot;
    float direction;    // 1, or -1 to turn back
    const float* cos_t;
    const float* sin_t;
    int max_pos;
    const int32_t* positions;
    int p0;
    const int64_t* slots;
    int64_t max_rows;
    uint8_t* k_dst;     // the layer's slabs
    uint8_t* v_dst;
    const float* k_scales;
    const float* v_scales;
    int32_t* status;
    int chunks;         // of a head, 2 W elements each
    int lanes;          // heads that a row's threads take at a time, per workgroup
    int rows;           // rows of a workgroup
};

// Threads: row, head, chunk of 2 W elements (W pairs where they turn), the chunk fastest. A thread
// keeps its row and chunk, so its cos and sin, and walks over heads: the table costs 512 bytes a
// row instead of a head. Bound by memory: 8192 rows of 48 heads of 128 into an FP8 cache in 42.8
// us, 4.4 TB/s read and written (a plain copy reaches 4.9); one row 2.7 us, the launch.
template <int LAYOUT, int CACHE, int W>
__global__ __launch_bounds__(256) void rope_rows_kernel(const RowsArgs a) {
    const int chunk = int(threadIdx.x) % a.chunks;
    const int rest = int(threadIdx.x) / a.chunks;
    const int row = int(blockIdx.x) * a.rows + rest / a.lanes;
    if (rest / a.lanes >= a.rows || row >= a.m) return;
    const int first = int(blockIdx.y) * a.lanes + rest % a.lanes;
    const int step = a.lanes * int(gridDim.y);

    const int pos = a.positions ? a.positions[row] : a.p0 + row;
    const bool turn = pos >= 0 && pos < a.max_pos;
    bool bad = !turn;
    int64_t slot = -1;
    if constexpr (CACHE != kNoCache) {
        slot = a.slots[row];
        const bool in = slot >= 0 && slot < a.max_rows;
        if (slot != -1 && !in) bad = true;
        if (!in || !turn) slot = -1;
    }
    if (bad && a.status && first == 0 && chunk == 0) *a.status = AF_ERR_OUT_OF_RANGE;

    const bool rotated = chunk < a.rot / (2 * W);  // else past the part that turns
    // the chunk's two runs of W elements
    const int e0 = LAYOUT == AF_ROPE_HALF && rotated ? chunk * W
                                                     : chunk * 2 * W;
    const int e1 = LAYOUT == AF_ROPE_HALF && rotated ? a.rot / 2 + chunk * W : e0 + W;
    float c[W], s[W];
#pragma unroll
    for (int i = 0; i < W; ++i) c[i] = 1.0f, s[i] = 0.0f;
    if (rotated && turn) {
        const size_t at = size_t(pos) * (a.rot / 2) + chunk * W;
        load_floats<W>(a.cos_t + at, c);
        load_floats<W>(a.sin_t + at, s);
#pragma unroll
        for (int i = 0; i < W; ++i) s[i] *= a.direction;
    }

    const int heads = a.q_heads + a.k_heads * (CACHE == kNoCache ? 1 : 2);
    for (int h = first; h < heads; h += step) {
        const bool is_q = h < a.q_heads;
        const int kh = h - a.q_heads;
        if (!is_q && CACHE != kNoCache && slot < 0) break;  // (K and V follow Q)
        const uint16_t* src = is_q ? a.q + size_t(row) * a.q_stride + size_t(h) * a.head_dim
                                   : a.k + size_t(row) * a.k_stride + size_t(kh) * a.head_dim;
        const bool is_v = CACHE != kNoCache && kh >= a.k_heads;
        const bool change = rotated && turn && !is_v;
        if (CACHE == kNoCache || is_q) {
            uint16_t* dst = is_q ? a.q_out + size_t(row) * a.q_out_stride + size_t(h) * a.head_dim
                                 : a.k_out + size_t(row) * a.k_out_stride + size_t(kh) * a.head_dim;
            if (!change && src == dst) continue;
            uint16_t u[W], v[W];
            load_halves<W>(src + e0, u);
            load_halves<W>(src + e1, v);
            if (change) rotate_halves<LAYOUT, W>(u, v, c, s);
            store_halves<W>(dst + e0, u);
            store_halves<W>(dst + e1, v);
            continue;
        }
        // (V's chunks lie one after the other, whatever the layout)
        const int f0 = is_v ? chunk * 2 * W : e0, f1 = is_v ? f0 + W : e1;
        uint16_t u[W], v[W];
        load_halves<W>(src + f0, u);
        load_halves<W>(src + f1, v);
        const int ch = is_v ? kh - a.k_heads : kh;
        const size_t to = size_t(slot) * a.k_heads * a.head_dim + size_t(ch) * a.head_dim;
        uint8_t* slab = is_v ? a.v_dst : a.k_dst;
        if constexpr (CACHE == kFp16) {
            if (change) rotate_halves<LAYOUT, W>(u, v, c, s);
            store_halves<W>(reinterpret_cast<uint16_t*>(slab) + to + f0, u);
            store_halves<W>(reinterpret_cast<uint16_t*>(slab) + to + f1, v);
        } else {
            float x[W], y[W];
#pragma unroll
            for (int i = 0; i < W; ++i) x[i] = h2f(u[i]), y[i] = h2f(v[i]);
            if (change) rotate_floats<LAYOUT, W>(x, y, c, s);
            const float scale = (is_v ? a.v_scales : a.k_scales)[ch];
#pragma unroll
            for (int i = 0; i < W; ++i) x[i] /= scale, y[i] /= scale;
            store_fp8<W>(slab + to + f0, x);
            store_fp8<W>(slab + to + f1, y);
        }
    }
}

// ---- launch ----------------------------------------------------------------------------------
bool on(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Pairs per chunk that sizes and alignments allow: 16-, 8- or 2-byte accesses.
int pairs_per_chunk(const RowsArgs& a) {
    auto fits = [&](int w) {
        const size_t bytes = size_t(2 * w);
        return a.head_dim % (2 * w) == 0 && a.rot % (2 * w) == 0 && a.q_stride % w == 0 &&
               a.k_stride % w == 0 && a.q_out_stride % w == 0 && a.k_out_stride % w == 0 &&
               on(a.q, bytes) && on(a.k, bytes) && on(a.q_out, bytes) && on(a.k_out, bytes);
    };
    return fits(8) ? 8 : fits(4) ? 4 : 1;
}

template <int LAYOUT, int CACHE>
int launch_rows(RowsArgs& a, hipStream_t s) {
    const int w = pairs_per_chunk(a);
    a.chunks = a.head_dim / (2 * w);
    const int heads = a.q_heads + a.k_heads * (CACHE == kNoCache ? 1 : 2);
    const int fit = std::max(1, 256 / a.chunks);
    // few rows: a thread for every chunk; many: a thread walks over some heads with its cos and sin
    const int64_t all = int64_t(a.m) * heads * a.chunks;
    const int walk = int(std::min<int64_t>(6, std::max<int64_t>(1, all / (256 * 2048))));
    a.lanes = std::min(fit, ceil_div(heads, walk));
    a.rows = std::max(1, fit / a.lanes);
    const dim3 grid(ceil_div(a.m, a.rows), ceil_div(heads, a.lanes * walk));
    switch (w) {
        case 8:
            hipLaunchKernelGGL((rope_rows_kernel<LAYOUT, CACHE, 8>), grid, dim3(256), 0, s, a);
            break;
        case 4:
            hipLaunchKernelGGL((rope_rows_kernel<LAYOUT, CACHE, 4>), grid, dim3(256), 0, s, a);
            break;
        default:
            hipLaunchKernelGGL((rope_rows_kernel<LAYOUT, CACHE, 1>), grid, dim3(256), 0, s, a);
    }
    AF_TRY_LAUNCH();
    return AF_OK;
}

template <int CACHE>
int launch_rows(RowsArgs& a, int layout, hipStream_t s) {
    return layout == AF_ROPE_HALF ? launch_rows<AF_ROPE_HALF, CACHE>(a, s)
                                  : launch_rows<AF_ROPE_INTERLEAVED, CACHE>(a, s);
}

// The checks that both entry points share.
int check_form(int head_dim, int rot_dim, int layout, const float* cos_t, const float* sin_t,
               int max_pos) {
    if (head_dim <= 0 || rot_dim <= 0 || rot_dim % 2 || rot_dim > head_dim || max_pos <= 0 ||
        !cos_t || !sin_t || !on(cos_t, 16) || !on(sin_t, 16))
        return AF_ERR_INVALID_ARG;
    if (layout != AF_ROPE_HALF && layout != AF_ROPE_INTERLEAVED) return AF_ERR_UNSUPPORTED;
    if (head_dim % 2 || head_dim > kMaxHeadDim) return AF_ERR_UNSUPPORTED;
    return AF_OK;
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" int af_rope_frequencies(const af_rope_scaling* sc, int rot_dim, double* h_freq,
                                   double* h_factor) {
    if (!sc || !h_freq || !h_factor || rot_dim <= 0 || rot_dim % 2) return AF_ERR_INVALID_ARG;
    if (rot_dim > 2 * kMaxPairs || sc->kind < AF_ROPE_SCALE_NONE || sc->kind > AF_ROPE_SCALE_YARN)
        return AF_ERR_UNSUPPORTED;
    auto positive = [](double v) { return v > 0.0 && std::isfinite(v); };
    if (!positive(sc->base) || !(sc->attention_factor == 0.0 || positive(sc->attention_factor)))
        return AF_ERR_INVALID_ARG;
    if (sc->kind != AF_ROPE_SCALE_NONE && !positive(sc->factor)) return AF_ERR_INVALID_ARG;
    const double context = sc->original_max_pos;
    double base = sc->base, factor = 1.0, lo = 0.0, hi = 0.0;
    if (sc->kind == AF_ROPE_SCALE_NTK && rot_dim > 2)
        base *= std::pow(sc->factor, double(rot_dim) / double(rot_dim - 2));
    if (sc->kind == AF_ROPE_SCALE_BANDS &&
        (sc->original_max_pos <= 0 || !positive(sc->low_freq_factor) ||
         !positive(sc->high_freq_factor) || sc->low_freq_factor >= sc->high_freq_factor))
        return AF_ERR_INVALID_ARG;
    if (sc->kind == AF_ROPE_SCALE_YARN) {
        if (sc->original_max_pos <= 0 || !positive(sc->beta_fast) || !positive(sc->beta_slow) ||
            !(base > 1.0))
            return AF_ERR_INVALID_ARG;
        auto pair_of = [&](double turns) {
            return rot_dim * std::log(context / (turns * kTwoPi)) / (2.0 * std::log(base));
        };
        lo = std::max(std::floor(pair_of(sc->beta_fast)), 0.0);
        hi = std::min(std::ceil(pair_of(sc->beta_slow)), double(rot_dim - 1));
        factor = 0.1 * std::log(std::max(sc->factor, 1.0)) + 1.0;
    }
    for (int i = 0; i < rot_dim / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / rot_dim);
        double r = f;
        if (sc->kind == AF_ROPE_SCALE_LINEAR) {
            r = f / sc->factor;
        } else if (sc->kind == AF_ROPE_SCALE_BANDS) {
            const double t = (context * f / kTwoPi - sc->low_freq_factor) /
                             (sc->high_freq_factor - sc->low_freq_factor);
            const double u = std::min(std::max(t, 0.0), 1.0);
            r = (1.0 - u) * f / sc->factor + u * f;
        } else if (sc->kind == AF_ROPE_SCALE_YARN) {
            const double t = std::min(std::max((i - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
            r = (1.0 - t) * f + t * f / sc->factor;
        }
        h_freq[i] = r;
    }
    *h_factor = sc->attention_factor != 0.0 ? sc->attention_factor : factor;
    return AF_OK;
}

extern "C" int af_rope_table_scaled(float* d_cos, float* d_sin, int64_t first_pos, int n_rows,
                                    int rot_dim, const double* h_freq, double factor,
                                    af_stream_t stream) {
    if (!h_freq || first_pos < 0 || n_rows < 0 || rot_dim <= 0 || rot_dim % 2 ||
        !std::isfinite(factor))
        return AF_ERR_INVALID_ARG;
    if (rot_dim > 2 * kMaxPairs || first_pos > INT32_MAX) return AF_ERR_UNSUPPORTED;
    TableArgs a{};
    a.cos_t = d_cos;
    a.sin_t = d_sin;
    a.first = first_pos;
    a.n_rows = n_rows;
    a.pairs = rot_dim / 2;
    a.factor = factor;
    for (int i = 0; i < a.pairs; ++i) {
        if (!std::isfinite(h_freq[i])) return AF_ERR_INVALID_ARG;
        a.turns[i] = h_freq[i] / kTwoPi;
    }
    if (n_rows == 0) return AF_OK;
    if (!d_cos || !d_sin || !on(d_cos, 16) || !on(d_sin, 16)) return AF_ERR_INVALID_ARG;
    const int v = a.pairs % 4 == 0 ? 4 : 1;
    const int grid = std::min(ceil_div(n_rows, 256 / (a.pairs / v)), kTableBlocks);
    if (v == 4)
        hipLaunchKernelGGL(rope_table_kernel<4>, dim3(grid), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
    else
        hipLaunchKernelGGL(rope_table_kernel<1>, dim3(grid), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
    AF_TRY_LAUNCH();
    return AF_OK;
}

extern "C" int af_rope_rows(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride,
                            int n_q_heads, const void* k, int64_t k_stride, void* k_out,
                            int64_t k_out_stride, int n_k_heads, int m, int head_dim, int rot_dim,
                            int layout, int inverse, const float* cos_table, const float* sin_table,
                            int max_pos, const int32_t* d_positions, int p0, int32_t* d_status,
                            af_stream_t stream) {
    if (int st = check_form(head_dim, rot_dim, layout, cos_table, sin_table, max_pos)) return st;
    if (!k || !n_k_heads) {
        if (n_k_heads < 0) return AF_ERR_INVALID_ARG;
        k = nullptr, k_out = nullptr, n_k_heads = 0, k_stride = k_out_stride = 0;
    }
    if (m < 0 || n_q_heads <= 0 || n_k_heads < 0 || (inverse != 0 && inverse != 1) ||
        q_stride < int64_t(n_q_heads) * head_dim || q_out_stride < int64_t(n_q_heads) * head_dim ||
        k_stride < int64_t(n_k_heads) * head_dim || k_out_stride < int64_t(n_k_heads) * head_dim)
        return AF_ERR_INVALID_ARG;
    if (n_q_heads > 65535 || n_k_heads > 65535) return AF_ERR_UNSUPPORTED;
    if (!d_positions && (p0 < 0 || int64_t(p0) + m > max_pos)) return AF_ERR_OUT_OF_RANGE;
    if (m == 0) return AF_OK;
    if (!q || !q_out || (n_k_heads && !k_out) || !on(q, 2) || !on(q_out, 2) || !on(k, 2) ||
        !on(k_out, 2) || !on(d_positions, 4) || !on(d_status, 4))
        return AF_ERR_INVALID_ARG;
    if ((q == q_out && q_stride != q_out_stride) || (k && k == k_out && k_stride != k_out_stride))
        return AF_ERR_INVALID_ARG;
    RowsArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.q_out = static_cast<uint16_t*>(q_out);
    a.k_out = static_cast<uint16_t*>(k_out);
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.q_out_stride = q_out_stride;
    a.k_out_stride = k_out_stride;
    a.m = m;
    a.q_heads = n_q_heads;
    a.k_heads = n_k_heads;
    a.head_dim = head_dim;
    a.rot = rot_dim;
    a.direction = inverse ? -1.0f : 1.0f;
    a.cos_t = cos_table;
    a.sin_t = sin_table;
    a.max_pos = max_pos;
    a.positions = d_positions;
    a.p0 = p0;
    a.status = d_status;
    return launch_rows<kNoCache>(a, layout, static_cast<hipStream_t>(stream));
}

extern "C" int af_paged_rope_append_rows(const void* qkv, int64_t qkv_stride, int m, void* q_out,
                                         int64_t q_out_stride, int n_q_heads,
                                         const af_kv_pool* pool, int layer, const int64_t* d_slots,
                                         const int32_t* d_positions, int rot_dim, int layout,
                                         const float* cos_table, const float* sin_table,
                                         int max_pos, int32_t* d_status, af_stream_t stream) {
    if (int st = check_pool(pool)) return st;
    const bool fp8 = pool->dtype == AF_KV_FP8_E4M3;
    const int hd = pool->head_dim, kvh = pool->n_kv_heads;
    if (int st = check_form(hd, rot_dim, layout, cos_table, sin_table, max_pos)) return st;
    if (m < 0 || n_q_heads <= 0 || layer < 0 || layer >= pool->n_layers || (fp8 && !pool->scales) ||
        qkv_stride < (int64_t(n_q_heads) + 2 * kvh) * hd ||
        q_out_stride < int64_t(n_q_heads) * hd)
        return AF_ERR_INVALID_ARG;
    if (n_q_heads > 65535 || kvh > 65535) return AF_ERR_UNSUPPORTED;
    if (m == 0) return AF_OK;
    if (!qkv || !q_out || !d_slots || !d_positions || !on(qkv, 2) || !on(q_out, 2) ||
        !on(d_slots, 8) || !on(d_positions, 4) || !on(d_status, 4) ||
        (qkv == q_out && qkv_stride != q_out_stride))
        return AF_ERR_INVALID_ARG;
    const PoolLayer at(*pool, layer);
    RowsArgs a{};
    a.q = static_cast<const uint16_t*>(qkv);
    a.k = a.q + size_t(n_q_heads) * hd;
    a.q_out = static_cast<uint16_t*>(q_out);
    a.q_stride = a.k_stride = qkv_stride;
    a.q_out_stride = q_out_stride;
    a.m = m;
    a.q_heads = n_q_heads;
    a.k_heads = kvh;
    a.head_dim = hd;
    a.rot = rot_dim;
    a.direction = 1.0f;
    a.cos_t = cos_table;
    a.sin_t = sin_table;
    a.max_pos = max_pos;
    a.positions = d_positions;
    a.slots = d_slots;
    a.max_rows = int64_t(pool->total_blocks) * pool->block_size;
    a.k_dst = at.k;
    a.v_dst = at.v;
    a.k_scales = at.k_scales;
    a.v_scales = at.v_scales;
    a.status = d_status;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return fp8 ? launch_rows<kFp8>(a, layout, s) : launch_rows<kFp16>(a, layout, s);
}
