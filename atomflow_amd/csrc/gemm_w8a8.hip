// gemm_w8a8.hip — the int8 x int8 projection on the gfx950 matrix cores:
//
//   y[i, j] = (sum_k x[i, k] * W[j, k]) * sx[i] * sw[j] (+ bias[j])
//
// One scale per token and one per output channel factor out of the sum, so the matrix
// cores add whole products of codes in 32 bits. These sums are exact (|sum| <= 2^14 k <
// 2^31 for k <= 131056): every order, split and tile gives the same bits, and a token's
// row does not depend on the launch it is in. The sum becomes fp32 (its one rounding
// before the result's, 2^-25 relative at most) and takes the scales and the bias there.
//
// Two kernels: few tokens (w8a8_few_kernel), bound by the weights' stream, and tiles
// (w8a8_tiled_kernel), bound by the matrix cores.
#include "af_common.h"
#include "af_device.h"

namespace af {
namespace {

typedef int int4v_t __attribute__((ext_vector_type(4)));
typedef int int16v_t __attribute__((ext_vector_type(16)));

struct W8A8Args {
    const int8_t* x;      // rows x_stride bytes apart
    int64_t x_stride;
    const float* xs;
    const int8_t* w;      // rows w_stride bytes apart
    int64_t w_stride;
    const float* ws;
    const float* bias;    // optional
    void* y;              // fp16 or fp32 rows, y_stride elements apart
    int64_t y_stride;
    int y32;
    int m, n, k;
};

// What tail chunks past k load in place of codes.
__device__ const uint4 kZeroChunk = {0, 0, 0, 0};

// One form of the last steps, so that every kernel gives the same bits.
__device__ __forceinline__ float finish(int sum, float sx, float sw, float bias) {
    return fmaf(float(sum) * sx, sw, bias);
}

__device__ __forceinline__ void put(const W8A8Args& a, int t, int j, float v) {
    const size_t at = size_t(t) * a.y_stride + j;
    if (a.y32) static_cast<float*>(a.y)[at] = v;
    else static_cast<uint16_t*>(a.y)[at] = f2h(v);
}

// ---- few tokens ---------------------------------------------------------------
// D = W X^T on v_mfma_i32_16x16x64_i8: A = 16 weight rows, B = 16 tokens (rows past n or
// m repeat the last; their products are not stored). Lane (row r, group g) holds bytes
// [16 g, 16 g + 16) of its row's 64, for both operands. A workgroup is 8 waves over 16 NT
// weight rows and up to 16 TT tokens; wave p takes the 64-byte steps p, p + 8, .. of K, so
// that the workgroup reads 512 contiguous bytes of each row at a time and each weight byte
// is read by one lane of the launch. The waves' sums meet in LDS.
constexpr int kFewWaves = 8;

template <int TT, int NT>
__global__ __launch_bounds__(64 * kFewWaves) void w8a8_few_kernel(const W8A8Args a) {
    __shared__ __align__(16) int s_red[kFewWaves * TT * NT * 256];
    const int lane = threadIdx.x & 63, p = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT);
    const int8_t* wp[NT];
    const int8_t* xp[TT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
        wp[i] = a.w + size_t(min(n0 + 16 * i + r, a.n - 1)) * a.w_stride;
#pragma unroll
    for (int i = 0; i < TT; ++i) xp[i] = a.x + size_t(min(16 * i + r, a.m - 1)) * a.x_stride;
    int4v_t acc[TT][NT];
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = int4v_t{0, 0, 0, 0};

    auto load = [](const int8_t* q) { return *reinterpret_cast<const int4v_t*>(q); };
    const int full = a.k / 64;
    constexpr int U = 4;
    int s = p;
    for (; s + kFewWaves * (U - 1) < full; s += kFewWaves * U) {
        int4v_t wf[U][NT], xf[U][TT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = 64 * (s + kFewWaves * u) + 16 * g;
#pragma unroll
            for (int j = 0; j < NT; ++j) wf[u][j] = load(wp[j] + at);
#pragma unroll
            for (int i = 0; i < TT; ++i) xf[u][i] = load(xp[i] + at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][j], xf[u][i], acc[i][j],
                                                                      0, 0, 0);
    }
    for (; 64 * s < a.k; s += kFewWaves) {  // the last may be part of a step
        const bool in = 64 * s + 16 * g < a.k;
        const int at = in ? 64 * s + 16 * g : 0;
        int4v_t wf[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) wf[j] = load(wp[j] + at);
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            int4v_t xf = load(xp[i] + at);
            if (!in) xf = int4v_t{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf, acc[i][j], 0, 0, 0);
        }
    }
    int4v_t* red = reinterpret_cast<int4v_t*>(s_red);
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) red[((p * TT + i) * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // Register q of lane (r, g) is weight row 4 g + q, token r.
    for (int e = threadIdx.x; e < TT * NT * 256; e += 64 * kFewWaves) {
        const int row = e % (16 * NT), t = e / (16 * NT);
        const int at = (((t >> 4) * NT + (row >> 4)) * 64 + 16 * ((row & 15) >> 2) + (t & 15)) * 4 +
                       (row & 3);
        int sum = 0;
#pragma unroll
        for (int q = 0; q < kFewWaves; ++q) sum += s_red[q * TT * NT * 256 + at];
        const int j = n0 + row;
        if (t < a.m && j < a.n) {
            put(a, t, j, finish(sum, a.xs[t], a.ws[j], a.bias ? a.bias[j] : 0.0f));
        }
    }
}

// ---- tiles ----------------------------------------------------------------------
// A workgroup of WR x WC waves makes a BM x BN tile of y in steps of 128 bytes of k. A
// stage of LDS holds the step's BM + BN rows of 128 bytes, fetched without registers (16
// bytes per lane, a wave-instruction 8 rows); 16-byte chunk c of row r sits at chunk
// c ^ (r % 8), so the 8 lanes of a 128-byte LDS access of an operand read (8 rows, one
// chunk) cover all banks. ST stages: while one is multiplied, ST - 1 load. Rows past m or n
// load the last row (not stored); chunks past k load zeros.
constexpr int kStep = 128;

template <int BM, int BN, int WR, int WC, int ST>
__global__ __launch_bounds__(64 * WR * WC) void w8a8_tiled_kernel(const W8A8Args a) {
    constexpr int NW = WR * WC;
    constexpr int MT = BM / WR / 32, NT = BN / WC / 32;  // 32x32 tiles of a wave
    constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW;    // DMA instructions of a wave per step
    constexpr int kStage = (BM + BN) * kStep;
    constexpr int D = ST - 1;                            // steps in flight ahead
    static_assert(XI * 8 * NW == BM && WI * 8 * NW == BN, "uneven DMA");
    static_assert(MT >= 1 && NT >= 1 && ST >= 2, "tile too small for its waves");
    __shared__ __align__(16) char s_lds[ST * kStage];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, hi = lane >> 5;

    // Workgroup ids go round-robin over the 8 XCDs: those of one XCD take a contiguous
    // range of tiles, in bands of 8 token tiles (a band's x and a few weight tiles stay in
    // the XCD's L2).
    const int mb = (a.m + BM - 1) / BM, nb = (a.n + BN - 1) / BN;
    const int tiles = mb * nb;
    const int xcd = int(blockIdx.x) & 7, per = tiles >> 3, rest = tiles & 7;
    const int tile = xcd * per + min(xcd, rest) + (int(blockIdx.x) >> 3);
    const int band = tile / (8 * nb), in_band = tile - band * 8 * nb;
    const int wide = min(8, mb - 8 * band);
    const int t0 = (8 * band + in_band % wide) * BM, n0 = in_band / wide * BN;

    const int chunk = (lane & 7) ^ (lane >> 3);
    const char* xb = reinterpret_cast<const char*>(a.x) + size_t(t0) * a.x_stride;
    const char* wb = reinterpret_cast<const char*>(a.w) + size_t(n0) * a.w_stride;
    uint32_t xoff[XI], woff[WI];
#pragma unroll
    for (int i = 0; i < XI; ++i)
        xoff[i] = uint32_t(min(8 * (wave * XI + i) + (lane >> 3), a.m - 1 - t0)) *
                      uint32_t(a.x_stride) + 16u * chunk;
#pragma unroll
    for (int i = 0; i < WI; ++i)
        woff[i] = uint32_t(min(8 * (wave * WI + i) + (lane >> 3), a.n - 1 - n0)) *
                      uint32_t(a.w_stride) + 16u * chunk;
    const uint32_t lds0 = lds_address(s_lds);
    const int steps = (a.k + kStep - 1) / kStep;
    auto issue = [&](int step, int buf) {
        const uint32_t dst = lds0 + buf * kStage;
        const char* xs = xb + size_t(step) * kStep;
        const char* ws = wb + size_t(step) * kStep;
        if ((step + 1) * kStep <= a.k) {
#pragma unroll
            for (int i = 0; i < XI; ++i) lds_dma16(xs, xoff[i], dst + 1024 * (wave * XI + i));
#pragma unroll
            for (int i = 0; i < WI; ++i)
                lds_dma16(ws, woff[i], dst + BM * kStep + 1024 * (wave * WI + i));
        } else {
            const bool in = step * kStep + 16 * chunk < a.k;
            const char* zero = reinterpret_cast<const char*>(&kZeroChunk);
#pragma unroll
            for (int i = 0; i < XI; ++i)
                lds_dma16(in ? xs + xoff[i] : zero, dst + 1024 * (wave * XI + i));
#pragma unroll
            for (int i = 0; i < WI; ++i)
                lds_dma16(in ? ws + woff[i] : zero, dst + BM * kStep + 1024 * (wave * WI + i));
        }
    };
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (i < steps) issue(i, i);

    // Operand reads: x row wm + 32 mt + col, weight row wn + 32 nt + col, chunk 2 q + hi.
    const int wm = (wave / WC) * (BM / WR), wn = (wave % WC) * (BN / WC);
    uint32_t at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
        at[q] = uint32_t(col) * kStep + 16u * uint32_t((2 * q + hi) ^ (col & 7));
    int16v_t acc[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[mt][nt][r] = 0;

    int buf = 0;
    for (int st = 0; st < steps; ++st) {
        // The step's loads have arrived (later ones may be in flight); the barrier covers
        // the other waves' and frees the stage read a step ago, which the next loads take.
        if (st + D - 1 < steps) wait_vmcnt<(D - 1) * (XI + WI)>();
        else wait_vmcnt<0>();
        __syncthreads();
        if (st + D < steps) issue(st + D, buf == 0 ? D : buf - 1);
        const char* sx = s_lds + buf * kStage + wm * kStep;
        const char* sw = s_lds + buf * kStage + (BM + wn) * kStep;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            int4v_t xf[MT], wf[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                wf[nt] = *reinterpret_cast<const int4v_t*>(sw + at[q] + nt * 32 * kStep);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                xf[mt] = *reinterpret_cast<const int4v_t*>(sx + at[q] + mt * 32 * kStep);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    acc[mt][nt] =
                        __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[mt], wf[nt], acc[mt][nt], 0, 0, 0);
        }
        buf = buf == D ? 0 : buf + 1;
    }

    // Register r of (mt, nt) is token 32 mt + 8 (r / 4) + 4 hi + r % 4 of the wave's piece,
    // column 32 nt + col.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int j = n0 + wn + 32 * nt + col;
        const bool has = j < a.n;
        const float sj = has ? a.ws[j] : 0.0f;
        const float bj = has && a.bias ? a.bias[j] : 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = t0 + wm + 32 * mt + 8 * (r >> 2) + 4 * hi + (r & 3);
                if (has && t < a.m) put(a, t, j, finish(acc[mt][nt][r], a.xs[t], sj, bj));
            }
    }
}

template <int TT, int NT>
void launch_few(const W8A8Args& a, hipStream_t s) {
    hipLaunchKernelGGL((w8a8_few_kernel<TT, NT>), dim3((a.n + 16 * NT - 1) / (16 * NT)),
                       dim3(64 * kFewWaves), 0, s, a);
}

template <int BM, int BN, int WR, int WC, int ST>
void launch_tiled(const W8A8Args& a, hipStream_t s) {
    const int tiles = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
    hipLaunchKernelGGL((w8a8_tiled_kernel<BM, BN, WR, WC, ST>), dim3(tiles), dim3(64 * WR * WC), 0,
                       s, a);
}

void launch_w8a8(const W8A8Args& a, hipStream_t s) {
    if (a.m <= 16) launch_few<1, 1>(a, s);
    else if (a.m <= 32) launch_few<2, 1>(a, s);
    else if (a.m <= 64) launch_few<4, 1>(a, s);
    else launch_tiled<128, 128, 2, 2, 2>(a, s);
}

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace
}  // namespace af

using namespace af;

extern "C" int af_w8a8_gemm(const int8_t* x, int64_t x_stride, const float* x_scales, int m,
                            const int8_t* weight, int64_t w_stride, const float* w_scales,
                            const float* bias, void* y, int64_t y_stride, int y_dtype, int n, int k,
                            af_stream_t stream) {
    if (!x || !x_scales || !weight || !w_scales || !y || m < 0 || n <= 0 || k <= 0)
        return AF_ERR_INVALID_ARG;
    if (y_dtype != AF_FP16 && y_dtype != AF_FP32) return AF_ERR_UNSUPPORTED;
    if (k % 16 || k > 131056) return AF_ERR_UNSUPPORTED;  // 2^14 k < 2^31
    if (x_stride < k || w_stride < k || x_stride % 16 || w_stride % 16 || y_stride < n)
        return AF_ERR_INVALID_ARG;
    // 32-bit lane offsets within a tile's rows
    if (x_stride >= int64_t(1) << 23 || w_stride >= int64_t(1) << 23) return AF_ERR_UNSUPPORTED;
    if (!aligned(x, 16) || !aligned(weight, 16) || !aligned(x_scales, 4) || !aligned(w_scales, 4) ||
        !aligned(bias, 4) || !aligned(y, y_dtype == AF_FP32 ? 4 : 2))
        return AF_ERR_INVALID_ARG;
    // a launch has fewer than 2^32 threads
    if (m > 1 << 26 || n > 1 << 26 || int64_t(m) * n > int64_t(1) << 36) return AF_ERR_UNSUPPORTED;
    if (m == 0) return AF_OK;
    W8A8Args a{};
    a.x = x;
    a.x_stride = x_stride;
    a.xs = x_scales;
    a.w = weight;
    a.w_stride = w_stride;
    a.ws = w_scales;
    a.bias = bias;
    a.y = y;
    a.y_stride = y_stride;
    a.y32 = y_dtype == AF_FP32;
    a.m = m;
    a.n = n;
    a.k = k;
    launch_w8a8(a, static_cast<hipStream_t>(stream));
    AF_TRY_LAUNCH();
    return AF_OK;
}
