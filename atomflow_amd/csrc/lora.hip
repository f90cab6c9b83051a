// lora.hip — low-rank adapters of many requests beside a shared projection, for gfx950.
//
//   y_out[i, j] = y[i, j] + scale[a] * sum_r B[a, j, r] * v[i, s(j), r],   a = ids[i]
//   v[i, s, r]  = sum_k A[a, s, r, k] x[i, k],                             r < rank[a]
//
// Two launches. `down` computes v: tiles of 16 or 64 tokens, K cut into at most eight parts whose
// sums it leaves in the workspace. `up` adds the parts, and its tiles' products to y. Both run on
// the matrix cores (16x16x32, fp16 operands, fp32 sums), with the adapter's rows as the first
// operand and the tokens as the second, so a token's sums depend on no other token.
//
// Tokens come in any order. A tile's workgroups (grid z) each take one of the adapters that its
// tokens name, every J-th from z on, compute the whole tile with that adapter's weights and write
// the rows that are its own: a prompt's tile has one adapter, a decode batch's tile of 16 has up
// to 16, side by side. No plan, no sort, no host data: ids, ranks and scales may change between
// the replays of a graph.
//
// Sums: K's parts and the order in which they are added are fixed by k alone, and every form adds
// a token's products in the same order, so a token's row has the same bits whatever the launch.
#include <algorithm>

#include "af_common.h"
#include "af_device.h"

namespace af {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// y's rows start at any element
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMaxSlices = AF_LORA_MAX_SLICES;
constexpr int kMaxRank = 128;
constexpr int kParts = 8;     // parts of K, at most
constexpr int kPartMin = 512; // k of a part, at least

struct LoraArgs {
    const uint16_t* x;
    int64_t x_stride;
    int m;
    const int32_t* ids;
    const uint16_t* a;      // [n_adapters][n_slices * rmax][k]
    const uint16_t* b;      // [n_adapters][n][rmax]
    const int32_t* ranks;
    const float* scales;
    int n_adapters, rmax, rows, k, n;  // rows = n_slices * rmax
    const void* y;
    int64_t y_stride;
    void* y_out;
    int64_t y_out_stride;
    float* v;               // [parts][m][rows]
    int parts, part_k;
    int n_slices;
    int slice_begin[kMaxSlices + 1];
    int slice_block[kMaxSlices + 1];  // `up`: first column block of each slice
    int cols;                         // `up`: columns of a workgroup
};

__device__ __forceinline__ f16x8 load_f16x8(const uint16_t* p) {
    return __builtin_bit_cast(f16x8, *reinterpret_cast<const u32x4*>(p));
}

// The adapters that a tile's tokens name, in order of first appearance. Lane t holds token t's.
struct Adapters {
    uint64_t todo;
    int id;
    __device__ __forceinline__ Adapters(int id, bool valid) : todo(__ballot(valid)), id(id) {}
    // Skips `skip` adapters; false when there is none behind them. mask: the tokens of `adapter`.
    __device__ __forceinline__ bool next(int skip, int& adapter, uint64_t& mask) {
        while (todo) {
            const int lead = __builtin_ctzll(todo);
            adapter = __builtin_amdgcn_readlane(id, lead);
            mask = __ballot(id == adapter) & todo;
            todo &= ~mask;
            if (skip-- == 0) return true;
        }
        return false;
    }
};

// ---- down: v ------------------------------------------------------------------------------
// MT 16-token tiles by NT 16-row tiles of A. The four waves take a quarter of the part's k each,
// operands straight from memory into registers (no barrier in the loop); their sums meet in LDS.
template <int MT, int NT>
__global__ __launch_bounds__(256) void lora_down_kernel(const LoraArgs p) {
    __shared__ f32x4 sums[4][MT * NT][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int t0 = blockIdx.x * (16 * MT);
    const int part = blockIdx.y % p.parts;
    const int row0 = (blockIdx.y / p.parts) * (16 * NT);
    int id = -1;
    if (lane < 16 * MT && t0 + lane < p.m) id = p.ids[t0 + lane];
    Adapters todo(id, id >= 0 && id < p.n_adapters);

    const int sub = 8 * (lane >> 4);
    const uint16_t* xp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = min(t0 + 16 * i + (lane & 15), p.m - 1);
        xp[i] = p.x + size_t(row) * p.x_stride + sub;
    }
    const int kw = p.part_k / 4;
    const int k0 = part * p.part_k + wave * kw;
    const int k1 = min(k0 + kw, p.k);

    int adapter;
    uint64_t mask;
    for (int skip = blockIdx.z; todo.next(skip, adapter, mask); skip = int(gridDim.z) - 1) {
        const int rank = p.ranks ? min(max(p.ranks[adapter], 0), p.rmax) : p.rmax;
        const uint16_t* ap[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int r = row0 + 16 * i + (lane & 15);
            const bool ok = r < p.rows && r % p.rmax < rank;
            // (a row past the rank touches its own sums alone, and those are not used)
            ap[i] = p.a + (size_t(adapter) * p.rows + (ok ? r : row0)) * p.k + sub;
        }
        f32x4 acc[MT][NT] = {};
        int k = k0;
        for (; k + 32 <= k1; k += 32) {
            f16x8 xf[MT], af[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) xf[i] = load_f16x8(xp[i] + k);
#pragma unroll
            for (int i = 0; i < NT; ++i) af[i] = load_f16x8(ap[i] + k);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[j], xf[i], acc[i][j], 0, 0, 0);
        }
        if (k < k1) {  // k is a multiple of 8: whole pieces of 8, or none
            const bool in = k + sub < k1;
            f16x8 xf[MT], af[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) xf[i] = in ? load_f16x8(xp[i] + k) : f16x8{};
#pragma unroll
            for (int i = 0; i < NT; ++i) af[i] = in ? load_f16x8(ap[i] + k) : f16x8{};
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[j], xf[i], acc[i][j], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) sums[wave][i * NT + j][lane] = acc[i][j];
        __syncthreads();
        // lane: token lane & 15 of the tile, rows 4 * (lane >> 4) ...
        for (int t = wave; t < MT * NT; t += 4) {
            const int token = 16 * (t / NT) + (lane & 15);
            const int r = row0 + 16 * (t % NT) + 4 * (lane >> 4);
            if (((mask >> token) & 1) && r < p.rows) {
                f32x4 s = (sums[0][t][lane] + sums[1][t][lane]) + (sums[2][t][lane] + sums[3][t][lane]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if ((r + e) % p.rmax >= rank) s[e] = 0.0f;
                *reinterpret_cast<f32x4*>(p.v + (size_t(part) * p.m + t0 + token) * p.rows + r) = s;
            }
        }
        __syncthreads();
    }
}

// ---- up: y_out = y + scale * B v ------------------------------------------------------------
// v in two fp16 halves, v = 2^e (hi + lo): 22 bits, so that fp16 matrix instructions lose nothing
// that fp32 sums would keep (one fp16 half alone would be off by half a step of fp16, as much as
// y's own rounding). e follows the token's largest v, so that neither half leaves fp16's range.
__device__ __forceinline__ int scale_exponent(float top) {
    const int e = int((__builtin_bit_cast(uint32_t, top) >> 23) & 255) - 127;
    return e == 128 ? 0 : max(e, -100) - 12;  // largest v to [2^12, 2^13); not finite: as it is
}

__device__ __forceinline__ float pow2f(int e) { return __builtin_ldexpf(1.0f, e); }

template <typename Y>
__device__ __forceinline__ void load_y16(const Y* p, int n, float (&v)[16]);
template <>
__device__ __forceinline__ void load_y16(const uint16_t* p, int n, float (&v)[16]) {
    if (n >= 16) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4_a2 w = *reinterpret_cast<const u32x4_a2*>(p + 8 * h);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[8 * h + i] = h2f(uint16_t(w[i >> 1] >> (16 * (i & 1))));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < n ? h2f(p[i]) : 0.0f;
    }
}
template <>
__device__ __forceinline__ void load_y16(const float* p, int n, float (&v)[16]) {
    if (n >= 16) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const f32x4_a4 w = *reinterpret_cast<const f32x4_a4*>(p + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * h + i] = w[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
}
__device__ __forceinline__ void store_y16(uint16_t* p, int n, const float (&v)[16]) {
    if (n >= 16) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4_a2 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = uint32_t(f2h(v[8 * h + 2 * i])) | (uint32_t(f2h(v[8 * h + 2 * i + 1])) << 16);
            *reinterpret_cast<u32x4_a2*>(p + 8 * h) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n) p[i] = f2h(v[i]);
    }
}
__device__ __forceinline__ void store_y16(float* p, int n, const float (&v)[16]) {
    if (n >= 16) {
#pragma unroll
        for (int h = 0; h < 4; ++h)
            *reinterpret_cast<f32x4_a4*>(p + 4 * h) =
                f32x4_a4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n) p[i] = v[i];
    }
}

// 16 * MT tokens by p.cols columns of one slice; rank up to 32 * KS. A wave takes 64 columns at a
// time: four first operands whose rows are the columns 16 g + 4 t + i (g, i the result's lane
// group and element, t the operand), so that a lane ends up with 16 columns in a row of one token.
template <int MT, int KS, typename Y>
__global__ __launch_bounds__(256) void lora_up_kernel(const LoraArgs p) {
    constexpr int kTokens = 16 * MT, kLd = 32 * KS + 8;
    __shared__ __attribute__((aligned(16))) uint16_t hi[kTokens * kLd];
    __shared__ __attribute__((aligned(16))) uint16_t lo[kTokens * kLd];
    __shared__ float back[kTokens];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int t0 = blockIdx.y * kTokens;
    int s = 0;
    while (s + 1 < p.n_slices && int(blockIdx.x) >= p.slice_block[s + 1]) ++s;
    const int col0 = p.slice_begin[s] + (int(blockIdx.x) - p.slice_block[s]) * p.cols;
    const int col1 = min(col0 + p.cols, p.slice_begin[s + 1]);

    const bool copy = p.y != p.y_out;  // tokens without an adapter are copied
    int id = -1;
    const bool token_in = lane < kTokens && t0 + lane < p.m;
    if (token_in) id = p.ids[t0 + lane];
    if (id < 0 || id >= p.n_adapters) id = -1;
    Adapters todo(id, token_in && (copy || id >= 0));

    int adapter;
    uint64_t mask;
    for (int skip = blockIdx.z; todo.next(skip, adapter, mask); skip = int(gridDim.z) - 1) {
        int rank = 0;
        if (adapter >= 0) rank = p.ranks ? min(max(p.ranks[adapter], 0), p.rmax) : p.rmax;
        if (rank == 0) {  // y as it is, bit for bit
            if (copy) {
                const int cols = col1 - col0;
                for (int t = 0; t < kTokens; ++t) {
                    if (!((mask >> t) & 1)) continue;
                    const Y* src = static_cast<const Y*>(p.y) + size_t(t0 + t) * p.y_stride + col0;
                    Y* dst = static_cast<Y*>(p.y_out) + size_t(t0 + t) * p.y_out_stride + col0;
                    for (int c = threadIdx.x; c < cols; c += 256) dst[c] = src[c];
                }
            }
            continue;
        }
        {  // the parts' sums, times the scale, in two halves
            constexpr int kPer = 256 / kTokens;      // threads of a token
            constexpr int kEach = 32 * KS / kPer;    // ranks of a thread
            const int t = threadIdx.x / kPer, r0 = (threadIdx.x % kPer) * kEach;
            const float scale = p.scales ? p.scales[adapter] : 1.0f;
            const bool mine = (mask >> t) & 1;
            float v[kEach];
#pragma unroll
            for (int i = 0; i < kEach; ++i) v[i] = 0.0f;
            if (mine) {
                const float* src = p.v + size_t(t0 + t) * p.rows + s * p.rmax + r0;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    if (r0 + i < rank) {
                        float sum = src[i];
                        for (int q = 1; q < p.parts; ++q) sum += src[size_t(q) * p.m * p.rows + i];
                        v[i] = sum * scale;
                    }
                }
            }
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
#pragma unroll
            for (int o = 1; o < kPer; o *= 2) top = max(top, uint32_t(__shfl_xor(int(top), o)));
            const int e = scale_exponent(__builtin_bit_cast(float, top));
            const float down = pow2f(-e);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const float w = v[i] * down;
                const uint16_t h = f2h(w);
                hi[t * kLd + r0 + i] = h;
                lo[t * kLd + r0 + i] = (h & 0x7c00u) == 0x7c00u ? uint16_t(0) : f2h(w - h2f(h));
            }
            if (threadIdx.x % kPer == 0) back[t] = pow2f(e);
        }
        __syncthreads();
        // which of a lane's 8 ranks there are: what lies behind an adapter's rank is not used
        u32x4 keep[KS];
#pragma unroll
        for (int q = 0; q < KS; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 32 * q + 8 * (lane >> 4) + 2 * i;
                keep[q][i] = (r < rank ? 0xffffu : 0u) | (r + 1 < rank ? 0xffff0000u : 0u);
            }
        for (int c = col0 + 64 * wave; c < col1; c += 256) {
            f16x8 bf[4][KS];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int col = c + 16 * ((lane & 15) >> 2) + 4 * t + (lane & 3);
                const uint16_t* bp =
                    p.b + (size_t(adapter) * p.n + min(col, col1 - 1)) * p.rmax + 8 * (lane >> 4);
#pragma unroll
                for (int q = 0; q < KS; ++q) {
                    u32x4 w = {0, 0, 0, 0};
                    if (32 * q + 8 * (lane >> 4) < rank)
                        w = *reinterpret_cast<const u32x4*>(bp + 32 * q) & keep[q];
                    bf[t][q] = __builtin_bit_cast(f16x8, w);
                }
            }
            const int col = c + 16 * (lane >> 4);
            const int left = col1 - col;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (((mask >> (16 * i)) & 0xffffu) == 0) continue;
                const int t = 16 * i + (lane & 15);
                const bool mine = ((mask >> t) & 1) && left > 0;
                float y[16];
                if (mine)
                    load_y16(static_cast<const Y*>(p.y) + size_t(t0 + t) * p.y_stride + col, left, y);
                f32x4 acc[4] = {};
#pragma unroll
                for (int q = 0; q < KS; ++q) {
                    const f16x8 h = load_f16x8(hi + t * kLd + 32 * q + 8 * (lane >> 4));
                    const f16x8 l = load_f16x8(lo + t * kLd + 32 * q + 8 * (lane >> 4));
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[u][q], l, acc[u], 0, 0, 0);
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[u][q], h, acc[u], 0, 0, 0);
                    }
                }
                if (mine) {
                    const float up = back[t];
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[e] += up * acc[e >> 2][e & 3];
                    store_y16(static_cast<Y*>(p.y_out) + size_t(t0 + t) * p.y_out_stride + col, left, y);
                }
            }
        }
        __syncthreads();
    }
}

// ---- launch ---------------------------------------------------------------------------------
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int parts_of(int k) { return std::min(kParts, ceil_div(k, kPartMin)); }

int lora_check(const af_lora* l) {
    if (!l || l->n_adapters <= 0 || l->max_rank <= 0 || l->n_slices <= 0 || l->k <= 0 || l->n <= 0)
        return AF_ERR_INVALID_ARG;
    if (l->max_rank % 8 || l->max_rank > kMaxRank || l->n_slices > kMaxSlices || l->k % 8 ||
        l->k > (1 << 24) || l->n > (1 << 24) || l->n_adapters > (1 << 20))
        return AF_ERR_UNSUPPORTED;
    int begin = 0;
    for (int s = 0; s < l->n_slices; ++s) {
        if (l->slice_end[s] <= begin) return AF_ERR_INVALID_ARG;
        begin = l->slice_end[s];
    }
    return begin == l->n ? AF_OK : AF_ERR_INVALID_ARG;
}

template <int MT>
void launch_down(const LoraArgs& p, dim3 grid, int nt, hipStream_t s) {
    switch (nt) {
        case 1: hipLaunchKernelGGL((lora_down_kernel<MT, 1>), grid, dim3(256), 0, s, p); break;
        case 2: hipLaunchKernelGGL((lora_down_kernel<MT, 2>), grid, dim3(256), 0, s, p); break;
        case 3: hipLaunchKernelGGL((lora_down_kernel<MT, 3>), grid, dim3(256), 0, s, p); break;
        default: hipLaunchKernelGGL((lora_down_kernel<MT, 4>), grid, dim3(256), 0, s, p); break;
    }
}

template <int MT, typename Y>
void launch_up(const LoraArgs& p, dim3 grid, hipStream_t s) {
    if (p.rmax <= 32)
        hipLaunchKernelGGL((lora_up_kernel<MT, 1, Y>), grid, dim3(256), 0, s, p);
    else if (p.rmax <= 64)
        hipLaunchKernelGGL((lora_up_kernel<MT, 2, Y>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((lora_up_kernel<MT, 4, Y>), grid, dim3(256), 0, s, p);
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" size_t af_lora_workspace_size(const af_lora* lora, int m) {
    if (lora_check(lora) || m < 0) return 0;
    return align_up(size_t(parts_of(lora->k)) * size_t(m > 0 ? m : 1) * lora->n_slices *
                        lora->max_rank * sizeof(float),
                    256);
}

extern "C" int af_lora_add(const void* x, int64_t x_stride, int m, const int32_t* d_ids,
                           const af_lora* lora, const void* y, int64_t y_stride, void* y_out,
                           int64_t y_out_stride, int y_dtype, void* workspace,
                           size_t workspace_bytes, af_stream_t stream) {
    if (int st = lora_check(lora)) return st;
    if (y_dtype != AF_FP16 && y_dtype != AF_FP32) return AF_ERR_UNSUPPORTED;
    const size_t esz = y_dtype == AF_FP16 ? 2 : 4;
    if (!lora->a || !lora->b || m < 0 || x_stride < lora->k || x_stride % 8 ||
        y_stride < lora->n || y_out_stride < lora->n)
        return AF_ERR_INVALID_ARG;
    if (!aligned16(lora->a) || !aligned16(lora->b) || !aligned_to(lora->ranks, 4) ||
        !aligned_to(lora->scales, 4))
        return AF_ERR_INVALID_ARG;
    if (m == 0) return AF_OK;
    if (!x || !d_ids || !y || !y_out || !aligned16(x) || !aligned_to(d_ids, 4) ||
        !aligned_to(y, esz) || !aligned_to(y_out, esz))
        return AF_ERR_INVALID_ARG;
    if (y == y_out && y_stride != y_out_stride) return AF_ERR_INVALID_ARG;
    if (m > (1 << 20)) return AF_ERR_UNSUPPORTED;
    if (!workspace || !aligned16(workspace) || workspace_bytes < af_lora_workspace_size(lora, m))
        return AF_ERR_WORKSPACE;

    LoraArgs p{};
    p.x = static_cast<const uint16_t*>(x);
    p.x_stride = x_stride;
    p.m = m;
    p.ids = d_ids;
    p.a = static_cast<const uint16_t*>(lora->a);
    p.b = static_cast<const uint16_t*>(lora->b);
    p.ranks = lora->ranks;
    p.scales = lora->scales;
    p.n_adapters = lora->n_adapters;
    p.rmax = lora->max_rank;
    p.rows = lora->n_slices * lora->max_rank;
    p.k = lora->k;
    p.n = lora->n;
    p.y = y;
    p.y_stride = y_stride;
    p.y_out = y_out;
    p.y_out_stride = y_out_stride;
    p.v = static_cast<float*>(workspace);
    p.parts = parts_of(p.k);
    p.part_k = int(align_up(size_t(ceil_div(p.k, p.parts)), 128));
    p.n_slices = lora->n_slices;

    const int mt = m > 256 ? 4 : 1;
    const int tiles = ceil_div(m, 16 * mt);
    const int side = std::min(mt == 4 ? 4 : 16, p.n_adapters);
    hipStream_t s = static_cast<hipStream_t>(stream);

    const int row_tiles = ceil_div(p.rows, 16);
    const int nt = std::min(4, row_tiles);
    const dim3 down(tiles, p.parts * ceil_div(row_tiles, nt), side);
    if (mt == 4)
        launch_down<4>(p, down, nt, s);
    else
        launch_down<1>(p, down, nt, s);
    AF_TRY_LAUNCH();

    p.cols = mt == 4 ? 1024 : 256;
    int blocks = 0;
    for (int i = 0; i < p.n_slices; ++i) {
        p.slice_begin[i + 1] = lora->slice_end[i];
        p.slice_block[i] = blocks;
        blocks += ceil_div(lora->slice_end[i] - p.slice_begin[i], p.cols);
    }
    p.slice_block[p.n_slices] = blocks;
    const dim3 up(blocks, tiles, std::min(mt == 4 ? 4 : 16, p.n_adapters + (y != y_out)));
    if (up.y > 65535) return AF_ERR_UNSUPPORTED;
    if (y_dtype == AF_FP16) {
        if (mt == 4)
            launch_up<4, uint16_t>(p, up, s);
        else
            launch_up<1, uint16_t>(p, up, s);
    } else {
        if (mt == 4)
            launch_up<4, float>(p, up, s);
        else
            launch_up<1, float>(p, up, s);
    }
    AF_TRY_LAUNCH();
    return AF_OK;
}
