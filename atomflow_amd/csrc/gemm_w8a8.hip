// gemm_w8a8.hip — the int8 x int8 projection on the gfx950 matrix cores:
//
//   y[i, j] = (sum_k x[i, k] * W[j, k]) * sx[i] * sw[j] (+ bias[j])
//
// One scale per token and one per output channel factor out of the sum, so the matrix
// cores add whole products of codes in 32 bits. These sums are exact (|sum| <= 2^14 k <
// 2^31 for k <= 131056): every order, split and tile gives the same bits, and a token's
// row does not depend on the launch it is in. The sum becomes fp32 and takes the scales and
// the bias there: its conversion and its product with sx round by 2^-24 at most each, before
// the rounding of the multiply-add with sw and the bias and the one to the result's type.
//
// Three kernels: one token (w8a8_row_kernel) and the tiles of few tokens (w8a8_tiled_kernel)
// are bound by the weights' stream, large launches (w8a8_wide_kernel) by the card's power;
// launches in between reach no ceiling. pick_form chooses by measured cost.
#include <algorithm>

#include "af_common.h"
#include "af_device.h"

namespace af {
namespace {

typedef int int4v_t __attribute__((ext_vector_type(4)));
typedef int int16v_t __attribute__((ext_vector_type(16)));
typedef float float2v_t __attribute__((ext_vector_type(2)));
typedef float float4v_t __attribute__((ext_vector_type(4)));
typedef f16 half2v_t __attribute__((ext_vector_type(2)));
// y's rows may start at any element (global memory takes any alignment).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

struct W8A8Args {
    const int8_t* x;      // rows x_stride bytes apart
    int64_t x_stride;
    const float* xs;
    const int8_t* w;      // rows w_stride bytes apart
    int64_t w_stride;
    const float* ws;
    const float* bias;    // optional
    void* y;              // fp16 (Y = uint16_t) or fp32 (float) rows, y_stride elements apart
    int64_t y_stride;
    int m, n, k;
    int stream_w;         // each weight row is read by one workgroup: see launch_tiled
};

// What tail chunks past k load in place of codes.
__device__ const uint4 kZeroChunk = {0, 0, 0, 0};

// One form of the last steps, so that every kernel gives the same bits.
__device__ __forceinline__ float finish(int sum, float sx, float sw, float bias) {
    return fmaf(float(sum) * sx, sw, bias);
}

// Two fp16 values, the first in the low half (v_cvt_pk_f16_f32, round to nearest even).
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v_t{lo, hi}), half2v_t));
}

// ---- one token ------------------------------------------------------------------
// A wave owns R weight rows (rows past n repeat the last; not stored) and reads them in
// contiguous 1 KB chunks, 16 bytes per lane, non-temporally (each weight byte is read once
// by the launch); a chunk of the token's codes is loaded once for the R rows. All loads of a
// pass of U chunks go out before any is used. v_dot4_i32_i8 adds four products a lane, and
// the lanes' sums meet by cross-lane adds. Bound by HBM: 28672 x 4096 in 18.7 us (6.3 TB/s, the
// launch in it), 128256 x 4096 in 76 (6.9; a 16 x 16 x 64 matrix-core product fed with 64-byte
// pieces of 16 rows took 25.6 and 123). Two tokens are no faster here than on the tiles.
constexpr int kRowWaves = 4;

__device__ __forceinline__ int wave_sum_i32(int v) {
#define AF_DPP_ADD(ctrl) v += __builtin_amdgcn_update_dpp(0, v, ctrl, 0xf, 0xf, true)
    AF_DPP_ADD(0xB1);
    AF_DPP_ADD(0x4E);
    AF_DPP_ADD(0x141);
    AF_DPP_ADD(0x128);
#undef AF_DPP_ADD
    uint32_t a = uint32_t(v), b = a;
    swap16(a, b);
    a = b = a + b;
    swap32(a, b);
    return int(a + b);
}

template <typename Y, int R, int U>
__global__ __launch_bounds__(64 * kRowWaves) void w8a8_row_kernel(const W8A8Args a) {
    const int lane = threadIdx.x & 63;
    const int row0 = (int(blockIdx.x) * kRowWaves + int(threadIdx.x >> 6)) * R;
    if (row0 >= a.n) return;
    const int8_t* wp[R];
#pragma unroll
    for (int r = 0; r < R; ++r) wp[r] = a.w + size_t(min(row0 + r, a.n - 1)) * a.w_stride;
    int acc[R] = {};
    for (int base = 0; base < a.k; base += 1024 * U) {
        int4v_t wv[U][R], xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = base + 1024 * u + 16 * lane;
            const bool in = k0 < a.k;
            const int at = in ? k0 : 0;
#pragma unroll
            for (int r = 0; r < R; ++r)
                wv[u][r] = __builtin_nontemporal_load(reinterpret_cast<const int4v_t*>(wp[r] + at));
            xv[u] = *reinterpret_cast<const int4v_t*>(a.x + at);
            if (!in) xv[u] = int4v_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[r] = __builtin_amdgcn_sdot4(wv[u][r][e], xv[u][e], acc[r], false);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int sum = wave_sum_i32(acc[r]);
        const int j = row0 + r;
        if (lane != 0 || j >= a.n) continue;
        const float v = finish(sum, a.xs[0], a.ws[j], a.bias ? a.bias[j] : 0.0f);
        if constexpr (sizeof(Y) == 4) static_cast<float*>(a.y)[j] = v;
        else static_cast<uint16_t*>(a.y)[j] = f2h(v);
    }
}

// ---- tiles ----------------------------------------------------------------------
// A workgroup of WR x WC waves for each of KS parts of K makes a BM x BN tile of y (tokens x
// weight rows) in steps of 128 bytes of k per part; D = W X^T, so that a lane's registers run
// along y's rows. A stage of LDS holds a step's BM + BN rows of 128 bytes (per part), fetched
// without registers (16 bytes per lane, 8 rows per wave-instruction); ST stages. Rows past m
// or n load the last row (not stored); chunks past k load zeros. The parts' sums meet in LDS.
//
// Operands are read one sub-step ahead of the products, over the step's end: when a step's
// last operands are in registers and the next stage has arrived, one barrier both publishes
// that stage and frees the one just read, whose place the step ST ahead takes; the next
// stage's first operands are read under the last products of this one. A part of one wave
// needs no barrier: it loads what it reads.
//
// Between a few dozen and a few hundred tokens it reaches no ceiling, and what holds it is not
// established. 513 x 4096 x 14336 runs in 60 us (weights from HBM): the matrix cores are busy a
// quarter of the time, HBM moves 1.2 TB/s, and each of the 215 workgroups loads 53 GB/s, where
// loads of 8 rows of 128 bytes an instruction reach 98 per CU from L2 (1 KB pieces 145). All
// workgroups ask for the same k of rows a fixed stride apart at a time; where one row of tiles
// reads the weights that alone cost a third (the turned start, below). Stages twice as many or
// as long, operands a whole step ahead, waves of 64 x 64 and 64 x 96 (which read a third less
// from LDS), and a wave that touches the weights' lines early gave nothing or cost time.
constexpr int kStep = 128;

// lds_dma16 of a wave-uniform base and lane offsets, non-temporal.
__device__ __forceinline__ void lds_dma16_nt(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds),
                 "v"(off), "s"(base)
                 : "memory");
}

// S x S products of one instruction. Lane l holds row l % S of either operand, chunk l / S of
// a sub-step's kChunks; its registers are kGroups groups of four rows of D (weight rows),
// group g from 8 g + 4 (l / S), in column l % S (a token).
template <int S>
struct Mfma;
template <>
struct Mfma<32> {
    typedef int16v_t Acc;
    [[maybe_unused]] static constexpr int kChunks = 2, kGroups = 4;
    static __device__ __forceinline__ Acc mul(int4v_t w, int4v_t x, Acc c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(w, x, c, 0, 0, 0);
    }
};
template <>
struct Mfma<16> {
    typedef int4v_t Acc;
    [[maybe_unused]] static constexpr int kChunks = 4, kGroups = 1;
    static __device__ __forceinline__ Acc mul(int4v_t w, int4v_t x, Acc c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
    }
};

// 16-byte chunk c of row r sits at chunk c ^ (r / 2 % 8): the 16 lanes of a 256-byte LDS
// access of an operand read (16 rows, one chunk) cover all 64 banks. (With the pattern
// repeating after 8 rows, half of the LDS's cycles were conflicts.)
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
    return uint32_t(chunk ^ ((row >> 1) & 7));
}

template <int kY, int S, int BM, int BN, int WR, int WC, int KS, int ST>
struct TileLds {
    static constexpr int kPart = (BM + BN) * kStep;     // a part of K's rows in a stage
    static constexpr int kStage = KS * kPart;
    static constexpr int kRows = S * WR;            // tokens of an output pass
    static constexpr int kOut = kRows * (kY * BN + 16);
    static constexpr int kLoop = ST * kStage;
    static constexpr int kSums = (KS - 1) * BM * BN * 4;
    static constexpr int kMost = kOut > kLoop ? kOut : kLoop;
    static constexpr int kScales = kSums > kMost ? kSums : kMost;  // xs, ws, bias
    static constexpr int kLds = kScales + 4 * (BM + 2 * BN);
};

// Stores the rows of one output pass from LDS.
template <typename Y, int S, int BN, int ROWS, int WROWS, int THREADS>
__device__ __forceinline__ void store_pass(const W8A8Args& a, const char* s_out, int t0, int n0,
                                           int mt) {
    constexpr int E = 16 / sizeof(Y), kChunks = BN / E, kStride = BN * sizeof(Y) + 16;
    for (int c = threadIdx.x; c < ROWS * kChunks; c += THREADS) {
        const int r = c / kChunks, q = c % kChunks;
        const int t = t0 + r / S * WROWS + S * mt + r % S, j = n0 + E * q;
        if (t >= a.m || j >= a.n) continue;
        const Y* from = reinterpret_cast<const Y*>(s_out + r * kStride + 16 * q);
        Y* dst = static_cast<Y*>(a.y) + size_t(t) * a.y_stride + j;
        if (j + E <= a.n) {
            const uint4 v = *reinterpret_cast<const uint4*>(from);
            *reinterpret_cast<u32x4_any*>(dst) = u32x4_any{v.x, v.y, v.z, v.w};
        } else {
#pragma unroll 1
            for (int e = 0; j + e < a.n; ++e) dst[e] = from[e];
        }
    }
}

template <typename Y, int S, int BM, int BN, int WR, int WC, int KS, int ST, int WGS>
__global__ __launch_bounds__(64 * WR * WC * KS, (WGS * WR * WC * KS + 3) / 4) void
w8a8_tiled_kernel(const W8A8Args a) {
    using L = TileLds<sizeof(Y), S, BM, BN, WR, WC, KS, ST>;
    constexpr int NW = WR * WC, THREADS = 64 * NW * KS;
    constexpr int MT = BM / WR / S, NT = BN / WC / S;  // S x S tiles of a wave
    constexpr int C = Mfma<S>::kChunks, G = Mfma<S>::kGroups;
    constexpr int kRowLanes = kStep / 16, kDmaRows = 64 / kRowLanes;  // a DMA instruction's rows
    constexpr int XI = BM / kDmaRows / NW, WI = BN / kDmaRows / NW;
    constexpr int Q = kStep / 16 / C;  // sub-steps
    static_assert(XI * kDmaRows * NW == BM && WI * kDmaRows * NW == BN, "uneven DMA");
    static_assert(MT >= 1 && NT >= 1 && ST >= 2, "tile too small for its waves");
    static_assert(Q % 2 == 0, "the next step's first operands take the slot that its last leave");
    __shared__ __align__(16) char s_lds[L::kLds];

    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = KS > 1 ? wid / NW : 0, wave = KS > 1 ? wid % NW : wid;
    const int col = lane % S, hi = lane / S;

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

    // The chunk that the lane's place in DMA instruction `block` (kDmaRows rows) holds.
    const int drow = lane / kRowLanes;
    auto chunk = [&](int block) {
        return int(swizzled(kDmaRows * block + drow, lane % kRowLanes));
    };
    const char* xb = reinterpret_cast<const char*>(a.x) + size_t(t0) * a.x_stride;
    const char* wb = reinterpret_cast<const char*>(a.w) + size_t(n0) * a.w_stride;
    uint32_t xoff[XI], woff[WI];
#pragma unroll
    for (int i = 0; i < XI; ++i)
        xoff[i] = uint32_t(min(kDmaRows * (wave * XI + i) + drow, a.m - 1 - t0)) *
                      uint32_t(a.x_stride) + 16u * chunk(wave * XI + i);
#pragma unroll
    for (int i = 0; i < WI; ++i)
        woff[i] = uint32_t(min(kDmaRows * (wave * WI + i) + drow, a.n - 1 - n0)) *
                      uint32_t(a.w_stride) + 16u * chunk(wave * WI + i);
    const uint32_t lds0 = lds_address(s_lds) + ks * L::kPart;
    const int steps = (a.k + KS * kStep - 1) / (KS * kStep);
    // Workgroups that stream weights of their own begin at different steps: side by side at one
    // k they would ask the same few memory channels for rows a power of two apart, and miss x
    // together (45 x 28672 x 4096: 27.9 to 21.6 us, 32 x 128256 x 4096 118 to 79; without the
    // non-temporal loads too, 31 and 127). The others share each step's operands in L2: turned,
    // launches of two to four token tiles took 9 % less to 24 % more time, of five and more up
    // to a third more (513 x 4096 x 14336 on 128 x 64 tiles: 82 and 92).
    const uint32_t spread = uint32_t(n0 / BN) * 2654435769u;  // (2^32 over the golden ratio)
    const int turn = a.stream_w ? int(__umulhi(spread, uint32_t(steps))) : 0;
    auto issue = [&](int step, int buf) __attribute__((always_inline)) {
        const uint32_t dst = lds0 + buf * L::kStage;
        const int turned = step + turn;
        const int k0 = ((turned >= steps ? turned - steps : turned) * KS + ks) * kStep;
        const char* xs = xb + k0;
        const char* ws = wb + k0;
        if (k0 + kStep <= a.k) {
#pragma unroll
            for (int i = 0; i < XI; ++i) lds_dma16(xs, xoff[i], dst + 1024 * (wave * XI + i));
            if (a.stream_w) {
#pragma unroll
                for (int i = 0; i < WI; ++i)
                    lds_dma16_nt(ws, woff[i], dst + BM * kStep + 1024 * (wave * WI + i));
            } else {
#pragma unroll
                for (int i = 0; i < WI; ++i)
                    lds_dma16(ws, woff[i], dst + BM * kStep + 1024 * (wave * WI + i));
            }
        } else {
            auto in = [&](int block) { return k0 + 16 * chunk(block) < a.k; };
            const char* zero = reinterpret_cast<const char*>(&kZeroChunk);
#pragma unroll
            for (int i = 0; i < XI; ++i)
                lds_dma16(in(wave * XI + i) ? xs + xoff[i] : zero, dst + 1024 * (wave * XI + i));
#pragma unroll
            for (int i = 0; i < WI; ++i)
                lds_dma16(in(wave * WI + i) ? ws + woff[i] : zero,
                          dst + BM * kStep + 1024 * (wave * WI + i));
        }
    };
#pragma unroll
    for (int i = 0; i < ST; ++i)
        if (i < steps) issue(i, i);

    // Operand reads: x row wm + S mt + col, weight row wn + S nt + col, chunk C q + hi.
    const int wm = (wave / WC) * (BM / WR), wn = (wave % WC) * (BN / WC);
    uint32_t at[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q)
        at[q] = uint32_t(col) * kStep + 16u * swizzled(col, C * q + hi);
    typename Mfma<S>::Acc acc[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 4 * G; ++r) acc[mt][nt][r] = 0;
    int4v_t xf[2][MT], wf[2][NT];
    auto read = [&](int slot, int buf, int q) __attribute__((always_inline)) {
        const char* sx = s_lds + buf * L::kStage + ks * L::kPart + wm * kStep + at[q];
        const char* sw = sx + (BM + wn - wm) * kStep;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            wf[slot][nt] = *reinterpret_cast<const int4v_t*>(sw + nt * S * kStep);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
            xf[slot][mt] = *reinterpret_cast<const int4v_t*>(sx + mt * S * kStep);
        // (left to itself the compiler moves each read down to its use)
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                acc[mt][nt] = Mfma<S>::mul(wf[slot][nt], xf[slot][mt], acc[mt][nt]);
        __builtin_amdgcn_sched_barrier(0);
    };

    // The tile's scales and bias, staged for the output. Loaded once no stage is left to load,
    // so that they arrive under the last steps.
    constexpr int kOwn = (BM + 2 * BN + THREADS - 1) / THREADS;
    float own[kOwn];
    auto load_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int e = threadIdx.x + i * THREADS;
            const int t = t0 + e, j = n0 + (e - BM) % BN;
            const float* from = e < BM ? a.xs + t : (e < BM + BN ? a.ws + j : a.bias + j);
            const bool has = e < BM ? t < a.m
                                    : e < BM + 2 * BN && j < a.n && (e < BM + BN || a.bias);
            own[i] = 0.0f;
            if (has) own[i] = *from;
        }
    };
    // The waves of a part share its stages. One wave alone waits for its own reads only.
    auto meet = [&]() __attribute__((always_inline)) {
        if constexpr (NW > 1) {
            __syncthreads();
        } else {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
            asm volatile("" ::: "memory");
        }
    };
    if (steps >= ST) wait_vmcnt<(ST - 1) * (XI + WI)>();
    else wait_vmcnt<0>();
    meet();
    read(0, 0, 0);
    int buf = 0;
    if (steps <= ST) load_scales();
    for (int st = 0; st + 1 < steps; ++st) {
        if (st + ST == steps && st > 0) load_scales();
#pragma unroll
        for (int q = 0; q + 1 < Q; ++q) {
            read((q + 1) & 1, buf, q + 1);
            multiply(q & 1);
        }
        if (st + ST <= steps) wait_vmcnt<(ST - 2) * (XI + WI)>();
        else wait_vmcnt<0>();
        meet();
        const int next = buf == ST - 1 ? 0 : buf + 1;
        read(0, next, 0);
        if (st + ST < steps) issue(st + ST, buf);
        buf = next;
        multiply((Q - 1) & 1);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        if (q + 1 < Q) read((q + 1) & 1, buf, q + 1);
        multiply(q & 1);
    }

    float* s_xs = reinterpret_cast<float*>(s_lds + L::kScales);
    float *s_ws = s_xs + BM, *s_bias = s_ws + BN;
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
        if (int(threadIdx.x) + i * THREADS < BM + 2 * BN) s_xs[threadIdx.x + i * THREADS] = own[i];

    // The parts' sums, to the first part's waves.
    if constexpr (KS > 1) {
        int4v_t* sums = reinterpret_cast<int4v_t*>(s_lds) + wave * MT * NT * G * 64 + lane;
        constexpr int kSlot = NW * MT * NT * G * 64;
        __syncthreads();
        if (ks > 0)
#pragma unroll
            for (int i = 0; i < MT * NT * G; ++i) {
                const auto& c = acc[i / G / NT][i / G % NT];
                const int r = 4 * (i % G);
                sums[(ks - 1) * kSlot + i * 64] = int4v_t{c[r], c[r + 1], c[r + 2], c[r + 3]};
            }
        __syncthreads();
        if (ks == 0)
#pragma unroll
            for (int p = 0; p < KS - 1; ++p)
#pragma unroll
                for (int i = 0; i < MT * NT * G; ++i) {
                    const int4v_t v = sums[p * kSlot + i * 64];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i / G / NT][i / G % NT][4 * (i % G) + e] += v[e];
                }
    }

    // Register 4 g + e of (mt, nt) is column S nt + 8 g + 4 hi + e, token S mt + col of the
    // wave's piece. y's rows go through LDS, S tokens of each wave row at a time.
    const int orow = (wave / WC) * S + col;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        __syncthreads();  // the loop's, or the last pass's, reads of LDS are done
        if (KS == 1 || ks == 0) {
            const float sx = s_xs[wm + S * mt + col];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int c = wn + S * nt + 8 * g + 4 * hi;
                    const float4 sw = *reinterpret_cast<const float4*>(s_ws + c);
                    const float4 b = *reinterpret_cast<const float4*>(s_bias + c);
                    const float v0 = finish(acc[mt][nt][4 * g], sx, sw.x, b.x);
                    const float v1 = finish(acc[mt][nt][4 * g + 1], sx, sw.y, b.y);
                    const float v2 = finish(acc[mt][nt][4 * g + 2], sx, sw.z, b.z);
                    const float v3 = finish(acc[mt][nt][4 * g + 3], sx, sw.w, b.w);
                    char* to = s_lds + orow * (sizeof(Y) * BN + 16) + sizeof(Y) * c;
                    if constexpr (sizeof(Y) == 4)
                        *reinterpret_cast<float4*>(to) = make_float4(v0, v1, v2, v3);
                    else
                        *reinterpret_cast<uint2*>(to) =
                            make_uint2(half_pair(v0, v1), half_pair(v2, v3));
                }
        }
        __syncthreads();
        store_pass<Y, S, BN, S * WR, BM / WR, THREADS>(a, s_lds, t0, n0, mt);
    }
}

// ---- 256 x 256 tiles --------------------------------------------------------------
// Large launches: a workgroup of eight waves (128 x 64 of y each, two per SIMD) per CU, which
// walks its tiles. What bounds it is the card's power: the matrix cores are busy 71 % of the
// cycles at 1.5 GHz (a form that kept them busy half of the cycles ran at 1.9 GHz), so the
// rest is kept off them: 32x32x32 products, 128-byte rows from L2, no LDS conflict.
//
// LDS is a ring of five 32 KB slots: load L of the sequence x0, w0, x1, w1, .. (the step's 256
// token rows, its 256 weight rows) takes slot L % 5. One barrier per step, before its last
// sub-step: by then the step's operands are in registers, so the two slots it read are free
// for w of the next step but one and x of the one after, a few 1 KB loads between two products
// each; x then has a step and a half to arrive, w one and a quarter. The sequence runs on
// across tiles: the next tile's first loads are issued before this tile's output, which goes
// through the two slots that its last step leaves. 8192 x 28672 x 4096 takes 786 us (a library
// product of the same integers 908; this kernel's first form 811, where one workgroup per
// tile with stages of whole steps took 872).
template <typename Y, int MT, int NT>
__device__ __forceinline__ void store_wide(const W8A8Args& a, int t0, int n0, int lane, char* s,
                                           const int16v_t (&acc)[MT][NT]) {
    // Register 4 g + e of (mt, nt) is column 32 nt + 8 g + 4 hi + e, token 32 mt + col. Rows
    // go through the wave's own part of LDS (s: 32 rows of PB bytes, then scales), 32 tokens
    // at a time, and leave as PB contiguous bytes. No other wave takes part and LDS serves a
    // wave's accesses in order, so nothing waits but the compiler (the empty asm). 16-byte
    // chunk c of row r sits at c ^ (r % CH).
    constexpr int PB = NT * 64, CH = PB / 16, RI = 1024 / PB;  // rows of a wave's 1 KB access
    constexpr int E = 16 / sizeof(Y);
    const int col = lane & 31, hi = lane >> 5;
    const int rr = lane / CH, rc = lane % CH;
    float* s_ws = reinterpret_cast<float*>(s + 32 * PB);
    float *s_b = s_ws + 32 * NT, *s_xs = s_b + 32 * NT;
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) {
        const int c = 64 * i + lane, j = n0 + c;
        s_ws[c] = j < a.n ? a.ws[j] : 0.0f;
        s_b[c] = a.bias && j < a.n ? a.bias[j] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < MT / 2; ++i) {
        const int t = t0 + 64 * i + lane;
        s_xs[64 * i + lane] = t < a.m ? a.xs[t] : 0.0f;
    }
    asm volatile("" ::: "memory");
    float4v_t sw[NT][4], sb[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            sw[nt][g] = *reinterpret_cast<const float4v_t*>(s_ws + 32 * nt + 8 * g + 4 * hi);
            sb[nt][g] = *reinterpret_cast<const float4v_t*>(s_b + 32 * nt + 8 * g + 4 * hi);
        }
    const bool inside = t0 + 32 * MT <= a.m && n0 + 32 * NT <= a.n;
    auto rows_out = [&](int mt, int first) __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        Y* y = static_cast<Y*>(a.y) + size_t(t0 + 32 * mt) * a.y_stride + n0 + first;
        if (inside) {
            Y* dst = y + rr * a.y_stride + E * rc;
#pragma unroll
            for (int i = 0; i < 32 / RI; ++i) {
                const int r = i * RI + rr;
                const uint4 v = *reinterpret_cast<const uint4*>(s + r * PB + 16 * (rc ^ (r % CH)));
                *reinterpret_cast<u32x4_any*>(dst + size_t(i * RI) * a.y_stride) =
                    u32x4_any{v.x, v.y, v.z, v.w};
            }
        } else {
#pragma unroll 1
            for (int r = rr; r < 32 && t0 + 32 * mt + r < a.m; r += RI) {
                const int left = a.n - (n0 + first + E * rc);
                const Y* from = reinterpret_cast<const Y*>(s + r * PB + 16 * (rc ^ (r % CH)));
#pragma unroll 1
                for (int e = 0; e < E && e < left; ++e) y[r * a.y_stride + E * rc + e] = from[e];
            }
        }
        asm volatile("" ::: "memory");
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float sx = s_xs[32 * mt + col];
        __builtin_amdgcn_sched_barrier(0);
        constexpr int P = sizeof(Y) / 2;  // passes: 32 rows of PB bytes hold NT / P column tiles
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int nt = p * NT / P; nt < (p + 1) * NT / P; ++nt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = finish(acc[mt][nt][4 * g + e], sx, sw[nt][g][e], sb[nt][g][e]);
                    const int c = 4 * P * (nt - p * NT / P) + P * g;  // chunks of the column tile
                    if constexpr (sizeof(Y) == 4)
                        *reinterpret_cast<float4*>(s + col * PB + 16 * ((c + hi) ^ (col % CH))) =
                            make_float4(v[0], v[1], v[2], v[3]);
                    else
                        *reinterpret_cast<uint2*>(s + col * PB + 16 * (c ^ (col % CH)) + 8 * hi) =
                            make_uint2(half_pair(v[0], v[1]), half_pair(v[2], v[3]));
                }
            rows_out(mt, p * NT * 32 / P);
        }
    }
}

constexpr int kWide = 256;

template <typename Y>
__global__ __launch_bounds__(512, 2) void w8a8_wide_kernel(const W8A8Args a) {
    constexpr int WC = 4, kSlot = kWide * kStep, kSlots = 5;
    constexpr int MT = 4, NT = 2, MF = MT * NT, FR = MT + NT;  // a wave's 32x32 tiles, operands
    constexpr int DI = 4;                                      // a wave's loads of a slot
    __shared__ __align__(16) char s_lds[kSlots * kSlot];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, hi = lane >> 5;
    // The XCDs' ranges of tiles and the bands of w8a8_tiled_kernel.
    const int mb = (a.m + kWide - 1) / kWide, nb = (a.n + kWide - 1) / kWide;
    const int tiles = mb * nb;
    const int xcd = int(blockIdx.x) & 7, per = tiles >> 3, rest = tiles & 7;
    const int first = xcd * per + min(xcd, rest), end = first + per + (xcd < rest ? 1 : 0);
    const int stride = (int(gridDim.x) + 7 - xcd) >> 3;  // workgroups of this XCD
    int tile = first + (int(blockIdx.x) >> 3);
    if (tile >= end) return;

    const int steps = (a.k + kStep - 1) / kStep;
    const int part = a.k % kStep / 16;  // chunks of a last, partial step
    // Instruction i of a slot fetches rows 8 (wave DI + i) .. + 7; the chunk of the lane's place
    // for even and odd i.
    const int drow = lane >> 3;
    const uint32_t ch0 = swizzled(drow, lane & 7), ch1 = ch0 ^ 4;
    const char *xb, *wb;
    uint32_t xoff[DI], woff[DI];
    int t0, n0;
    auto aim = [&](int tl) __attribute__((always_inline)) {
        const int band = tl / (8 * nb), in_band = tl - band * 8 * nb;
        const int wide = min(8, mb - 8 * band);
        t0 = (8 * band + in_band % wide) * kWide;
        n0 = in_band / wide * kWide;
        xb = reinterpret_cast<const char*>(a.x) + size_t(t0) * a.x_stride;
        wb = reinterpret_cast<const char*>(a.w) + size_t(n0) * a.w_stride;
#pragma unroll
        for (int i = 0; i < DI; ++i) {
            const int r = 8 * (wave * DI + i) + drow;
            const uint32_t c = 16u * (i & 1 ? ch1 : ch0);
            xoff[i] = uint32_t(min(r, a.m - 1 - t0)) * uint32_t(a.x_stride) + c;
            woff[i] = uint32_t(min(r, a.n - 1 - n0)) * uint32_t(a.w_stride) + c;
        }
    };
    const uint32_t lds0 = lds_address(s_lds) + 1024 * wave * DI;
    // Past a partial step's chunks a lane loads its row's first one (x is zeroed where it is used).
    const uint32_t back0 = part && ch0 >= uint32_t(part) ? 16 * ch0 : 0;
    const uint32_t back1 = part && ch1 >= uint32_t(part) ? 16 * ch1 : 0;
    auto dma = [&](const char* base, const uint32_t (&off)[DI], int step, int slot, int i)
        __attribute__((always_inline)) {
        lds_dma16(base + size_t(step) * kStep, off[i], lds0 + slot * kSlot + 1024 * i);
    };
    auto load = [&](const char* base, const uint32_t (&off)[DI], int step, int slot)
        __attribute__((always_inline)) {
        if (step >= steps) return;
        const bool cut = part && step + 1 == steps;
#pragma unroll
        for (int i = 0; i < DI; ++i)
            lds_dma16(base + size_t(step) * kStep, cut ? off[i] - (i & 1 ? back1 : back0) : off[i],
                      lds0 + slot * kSlot + 1024 * i);
    };
    auto up = [](int slot, int by) { return slot + by >= kSlots ? slot + by - kSlots : slot + by; };

    const int wm = wave / WC * 128, wn = wave % WC * (kWide / WC);
    uint32_t at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) at[q] = uint32_t(col) * kStep + 16u * swizzled(col, 2 * q + hi);
    int16v_t acc[MT][NT];
    int4v_t xf[2][MT], wf[2][NT];
    // operand f of sub-step q: the weight rows', then the tokens'
    auto read1 = [&](int p, int xs, int ws, int q, int f) __attribute__((always_inline)) {
        if (f < NT)
            wf[p][f] = *reinterpret_cast<const int4v_t*>(s_lds + ws * kSlot + wn * kStep + at[q] +
                                                         f * 32 * kStep);
        else
            xf[p][f - NT] = *reinterpret_cast<const int4v_t*>(
                s_lds + xs * kSlot + wm * kStep + at[q] + (f - NT) * 32 * kStep);
    };
    auto mfma = [&](int p, int i) __attribute__((always_inline)) {
        acc[i / NT][i % NT] = Mfma<32>::mul(wf[p][i % NT], xf[p][i / NT], acc[i / NT][i % NT]);
    };
    auto fence = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };

    int xs = 0;  // slot of the current step's x; its w, the next x, w and the x after that follow
    aim(tile);
    load(xb, xoff, 0, 0);
    load(wb, woff, 0, 1);
    load(xb, xoff, 1, 2);
    wait_vmcnt<0>();
    while (true) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[mt][nt][r] = 0;
        __syncthreads();  // step 0 has arrived; the last tile's output is out of LDS
#pragma unroll
        for (int f = 0; f < FR; ++f) read1(0, xs, up(xs, 1), 0, f);
        load(wb, woff, 1, up(xs, 3));
        load(xb, xoff, 2, up(xs, 4));
        fence();
        int st = 0;
        const int whole = a.k / kStep;
        for (; st + 3 < whole; ++st) {  // the loads that these steps issue are of whole steps
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int i = 0; i < MF; ++i) {
                    mfma(q & 1, i);
                    if (i < FR) read1((q + 1) & 1, xs, up(xs, 1), q + 1, i);
                    if (q == 0 && i >= MF - DI && st > 0)
                        dma(xb, xoff, st + 2, up(xs, 4), i - (MF - DI));
                    fence();
                }
            wait_vmcnt<DI>();  // the next step has arrived (x of the one after may not have)
            __syncthreads();
            fence();
            const int x1 = up(xs, 2), w1 = up(xs, 3);
#pragma unroll
            for (int i = 0; i < MF; ++i) {
                mfma(1, i);
                if (i < FR) read1(0, x1, w1, 0, i);
                if (i >= MF - DI) dma(wb, woff, st + 2, xs, i - (MF - DI));
                fence();
            }
            xs = x1;
        }
        for (; st < steps; ++st) {
            const bool cut = part && st + 1 == steps;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q == 0 && st > 0) load(xb, xoff, st + 2, up(xs, 4));
                if (q == 3) {
                    wait_vmcnt<0>();
                    __syncthreads();
                    if (st + 1 < steps) {
                        load(wb, woff, st + 2, xs);
#pragma unroll
                        for (int f = 0; f < FR; ++f) read1(0, up(xs, 2), up(xs, 3), 0, f);
                    }
                } else {
#pragma unroll
                    for (int f = 0; f < FR; ++f) read1((q + 1) & 1, xs, up(xs, 1), q + 1, f);
                }
                if (cut && 2 * q + hi >= part)
#pragma unroll
                    for (int f = 0; f < MT; ++f) xf[q & 1][f] = int4v_t{0, 0, 0, 0};
                fence();
#pragma unroll
                for (int i = 0; i < MF; ++i) mfma(q & 1, i);
                fence();
            }
            if (st + 1 < steps) xs = up(xs, 2);
        }
        // Every wave has read its last operands (the last step's barrier): all slots are free.
        const int c0 = t0 + wm, c1 = n0 + wn, out = xs;
        tile += stride;
        const bool more = tile < end;
        if (more) {
            aim(tile);
            load(xb, xoff, 0, up(xs, 2));
            load(wb, woff, 0, up(xs, 3));
            load(xb, xoff, 1, up(xs, 4));
            // (waited for here, before the output's stores, which count as later loads do)
            wait_vmcnt<0>();
        }
        char* mine = s_lds + (wave < WC ? out : up(out, 1)) * kSlot + wave % WC * (kSlot / WC);
        store_wide<Y, MT, NT>(a, c0, c1, lane, mine, acc);
        if (!more) return;
        xs = up(xs, 2);
    }
}

template <typename Y, int R, int U>
void launch_row(const W8A8Args& a, hipStream_t s) {
    const int per = kRowWaves * R;
    hipLaunchKernelGGL((w8a8_row_kernel<Y, R, U>), dim3((a.n + per - 1) / per), dim3(64 * kRowWaves),
                       0, s, a);
}

// Weights that one row of tiles (mb) reads are streamed, as the FP8 GEMV streams its own: those
// under 12 MB may stay in the caches from one launch to the next.
bool streams_weights(int mb, int n, int k) { return mb == 1 && int64_t(n) * k > 12 << 20; }

template <typename Y, int S, int BM, int BN, int WR, int WC, int KS, int ST, int WGS>
void launch_tiled(const W8A8Args& a, hipStream_t s) {
    const int mb = (a.m + BM - 1) / BM, tiles = mb * ((a.n + BN - 1) / BN);
    W8A8Args b = a;
    b.stream_w = streams_weights(mb, a.n, a.k);
    hipLaunchKernelGGL((w8a8_tiled_kernel<Y, S, BM, BN, WR, WC, KS, ST, WGS>), dim3(tiles),
                       dim3(64 * WR * WC * KS), 0, s, b);
}

template <typename Y>
void launch_wide(const W8A8Args& a, hipStream_t s) {
    const int tiles = ((a.m + kWide - 1) / kWide) * ((a.n + kWide - 1) / kWide);
    const int wgs = std::min(tiles, device_compute_units());
    hipLaunchKernelGGL(w8a8_wide_kernel<Y>, dim3(wgs), dim3(512), 0, s, a);
}

// The forms (token rows, weight rows, parts of K, workgroups per CU), and what a launch of
// each was measured to cost on MI355X (21 (n, k) shapes from 8192 x 64 to 151936 x 2048, 2
// to 4096 tokens, weights read from HBM): a round of workgroups, `wgs` of them per CU while
// tiles last, takes `round` plus per step (128 k of each part) `step`, for each workgroup of
// the busiest CUs `share` and of the average CU `spread` (us); a launch `fixed` besides, and
// `stream` per MB of weights. Small tiles with several parts of K at a time fill the device
// when tokens or rows are few, large ones read the least and keep the matrix cores busiest.
// The rule's form takes 1.4 % more than the best measured one on average, 23 % at most, of the
// launches that the costs were fitted to.
struct TileCost {
    int bm, bn, ks, wgs;
    float fixed, round, step, share, spread, stream;
};
enum {
    k16x16k8, k16x32k4, k32x32k4, k32x64k2, k64x32k4, k64x64x2, k64x64k2,
    k128x64k2, k128x96, k128x128, k192x128, k256x256, k192x256, k64x128,
    k128x128x2, k32x256,
    kForms
};
constexpr TileCost kTileCost[kForms] = {
    {16, 16, 8, 1, 1.5253f, 1.1634f, 0.2820f, 0.0f, 0.2026f, 0.0435f},
    {16, 32, 4, 2, 1.6584f, 1.0537f, 0.0427f, 0.2422f, 0.0421f, 0.0677f},
    {32, 32, 4, 1, 1.4628f, 1.5650f, 0.3373f, 0.0f, 0.1539f, 0.0428f},
    {32, 64, 2, 2, 1.5800f, 1.3526f, 0.1062f, 0.2143f, 0.0824f, 0.0599f},
    {64, 32, 4, 1, 1.1681f, 2.0336f, 0.5269f, 0.0f, 0.1022f, 0.0762f},
    {64, 64, 1, 2, 1.1423f, 2.1340f, 0.0735f, 0.1634f, 0.0245f, 0.0575f},
    {64, 64, 2, 1, 1.1364f, 2.1727f, 0.4097f, 0.0f, 0.0791f, 0.0573f},
    {128, 64, 2, 1, 1.5647f, 2.7491f, 0.5400f, 0.0f, 0.2365f, 0.0436f},
    {128, 96, 1, 1, 1.4953f, 3.6545f, 0.3755f, 0.0f, 0.1381f, 0.0299f},
    {128, 128, 1, 1, 1.0881f, 3.0483f, 0.4148f, 0.0f, 0.1950f, 0.0440f},
    {192, 128, 1, 1, 1.5970f, 3.7784f, 0.4931f, 0.0f, 0.3379f, 0.0246f},
    {256, 256, 1, 1, 1.2085f, 6.8190f, 0.9115f, 0.0f, 0.6966f, 0.0614f},
    {192, 256, 1, 1, 2.0918f, 5.7229f, 0.8791f, 0.0f, 0.5041f, 0.0339f},
    {64, 128, 1, 2, 1.4440f, 2.5838f, 0.0989f, 0.2060f, 0.0959f, 0.0652f},
    {128, 128, 1, 2, 0.8969f, 4.2947f, 0.4938f, 0.0303f, 0.2533f, 0.0530f},
    {32, 256, 1, 2, 1.3309f, 2.1394f, 0.4646f, 0.1685f, 0.1281f, 0.0776f}
};

int pick_form(unsigned m, unsigned n, unsigned k) {
    // (called for every launch: constant tile sizes, 32-bit arithmetic; tiles are below 2^29)
    const unsigned cus = unsigned(device_compute_units());
    const float weights = float(n) * float(k) * 1e-6f;  // MB
    int best = 0;
    float best_cost = 0.0f;
#pragma clang loop unroll(full)
    for (int i = 0; i < kForms; ++i) {
        constexpr auto up = [](unsigned x, int by) { return (x + by - 1) / unsigned(by); };
        const TileCost& c = kTileCost[i];
        const unsigned tiles = up(m, c.bm) * up(n, c.bn);
        const unsigned per_cu = (tiles + cus - 1) / cus;  // of the busiest CUs
        const float steps = float(up(k, 128 * c.ks));
        const float all = float(tiles) / float(cus);
        const float cost = c.fixed + float(up(per_cu, c.wgs)) * (c.round + steps * c.step) +
                           steps * (float(per_cu) * c.share + all * c.spread) + weights * c.stream;
        if (i == 0 || cost < best_cost) {
            best = i;
            best_cost = cost;
        }
    }
    return best;
}

// One token: rows of one pass (four 1 KB chunks) each to a wave; longer ones in pairs. (us,
// one row / two per wave: 6144 x 4096 5.8 / 5.9, 28672 x 4096 18.2 / 18.6, 4096 x 14336
// 11.2 / 10.8; the best tiles 6.7, 20.9 and 11.5.)
bool row_pairs(int k) { return k > 4096; }

template <typename Y>
void launch_w8a8(const W8A8Args& a, hipStream_t s) {
    if (a.m == 1)
        return row_pairs(a.k) ? launch_row<Y, 2, 4>(a, s) : launch_row<Y, 1, 4>(a, s);
    switch (pick_form(a.m, a.n, a.k)) {
        case k16x16k8: return launch_tiled<Y, 16, 16, 16, 1, 1, 8, 4, 1>(a, s);
        case k16x32k4: return launch_tiled<Y, 16, 16, 32, 1, 1, 4, 3, 2>(a, s);
        case k32x32k4: return launch_tiled<Y, 32, 32, 32, 1, 1, 4, 4, 1>(a, s);
        case k32x64k2: return launch_tiled<Y, 32, 32, 64, 1, 2, 2, 3, 2>(a, s);
        case k64x32k4: return launch_tiled<Y, 32, 64, 32, 2, 1, 4, 3, 1>(a, s);
        case k64x64x2: return launch_tiled<Y, 32, 64, 64, 2, 2, 1, 4, 2>(a, s);
        case k64x64k2: return launch_tiled<Y, 32, 64, 64, 2, 2, 2, 4, 1>(a, s);
        case k128x64k2: return launch_tiled<Y, 32, 128, 64, 2, 2, 2, 3, 1>(a, s);
        case k128x96: return launch_tiled<Y, 32, 128, 96, 4, 1, 1, 4, 1>(a, s);
        case k128x128: return launch_tiled<Y, 32, 128, 128, 4, 2, 1, 3, 1>(a, s);
        case k192x128: return launch_tiled<Y, 32, 192, 128, 2, 4, 1, 3, 1>(a, s);
        case k256x256: return launch_wide<Y>(a, s);
        case k192x256: return launch_tiled<Y, 32, 192, 256, 2, 4, 1, 2, 1>(a, s);
        case k64x128: return launch_tiled<Y, 32, 64, 128, 2, 2, 1, 3, 2>(a, s);
        case k128x128x2: return launch_tiled<Y, 32, 128, 128, 2, 2, 1, 2, 2>(a, s);
        case k32x256: return launch_tiled<Y, 32, 32, 256, 1, 4, 1, 2, 2>(a, s);
    }
}

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Sums below 2^31 (2^14 k), and a launch of fewer than 2^32 threads.
bool supported_sizes(int m, int n, int k) {
    return k % 16 == 0 && k <= 131056 && m <= 1 << 25 && n <= 1 << 25 &&
           int64_t(m) * n <= int64_t(1) << 36;
}

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
    if (!supported_sizes(m, n, k)) return AF_ERR_UNSUPPORTED;
    if (x_stride < k || w_stride < k || x_stride % 16 || w_stride % 16 || y_stride < n)
        return AF_ERR_INVALID_ARG;
    // 32-bit lane offsets within a tile's rows
    if (x_stride >= int64_t(1) << 23 || w_stride >= int64_t(1) << 23) return AF_ERR_UNSUPPORTED;
    if (!aligned(x, 16) || !aligned(weight, 16) || !aligned(x_scales, 4) || !aligned(w_scales, 4) ||
        !aligned(bias, 4) || !aligned(y, y_dtype == AF_FP32 ? 4 : 2))
        return AF_ERR_INVALID_ARG;
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
    a.m = m;
    a.n = n;
    a.k = k;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (y_dtype == AF_FP32) launch_w8a8<float>(a, s);
    else launch_w8a8<uint16_t>(a, s);
    AF_TRY_LAUNCH();
    return AF_OK;
}

extern "C" int af_w8a8_gemm_form(int m, int n, int k, int32_t* form) {
    if (!form || m <= 0 || n <= 0 || k <= 0) return AF_ERR_INVALID_ARG;
    if (!supported_sizes(m, n, k)) return AF_ERR_UNSUPPORTED;
    if (m == 1) {
        const int32_t row[5] = {1, row_pairs(k) ? 2 : 1, 1, 0, 1};
        std::copy(row, row + 5, form);
        return AF_OK;
    }
    const int i = pick_form(m, n, k);
    const TileCost& c = kTileCost[i];
    const bool streams = i != k256x256 && streams_weights((m + c.bm - 1) / c.bm, n, k);
    const int32_t tile[5] = {c.bm, c.bn, c.ks, c.wgs, streams};
    std::copy(tile, tile + 5, form);
    return AF_OK;
}
