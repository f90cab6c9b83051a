// quantize_rows.hip — rows of int8 codes with one fp32 scale each, the activations of
// the int8 product (gemm_w8a8.hip), and what produces them in the same pass:
//
//   v = x                                        (attention's output)
//   v = silu(gate) * up,  silu(g) = g / (1 + e^-g)    (the MLP's activation)
//   v = s * rsqrt(mean(s^2) + eps) * w,  s = x + residual   (RMSNorm, residual added)
//
//   a = max |v| over the row;  scale = a / 127 (1 for a zero row);  code = rne(v * 127 / a)
//
// Memory-bound: every input element is read once and every output written once.
// A row is held in fp32 registers by the threads that own it, 8 consecutive elements
// (one 16-byte load of fp16) per thread and chunk, so the norm's sum, the row's
// maximum and the codes need one pass; two reductions (a wave's by DPP, the waves' of
// a row through LDS) stand between the loads and the stores. Sums, the norm and the
// products stay in fp32 until the one rounding to a code (or to fp16). The maximum is
// taken over the magnitudes' bits, where NaN > infinity > every finite value: a row
// that holds one gets scale NaN and codes 0, so what is computed from it is NaN.
#include "af_common.h"
#include "af_device.h"

namespace af {
namespace {

// Rows may start at any element: the 16- and 8-byte accesses are declared with the
// element's own alignment (global memory takes any).
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));

enum { kPlain, kSiluMul, kNorm, kNormAdd16, kNormAdd32 };

struct RowArgs {
    const uint16_t* x;     // kSiluMul: gate
    const uint16_t* up;
    int64_t x_stride;
    const void* res_in;    // fp16 or fp32, rows res_stride elements apart
    void* res_out;
    int64_t res_stride;
    const float* weight;
    float eps;
    int row0, m, n;        // the launch's rows [row0, row0 + m)
    int8_t* codes;         // optional with kNorm*
    int64_t codes_stride;
    float* scales;
    uint16_t* normed;      // kNorm*, optional
    int64_t normed_stride;
};

// Elements [e, e + 8) of a row of n; past the end 0.
__device__ __forceinline__ void load8(const uint16_t* p, int e, int n, float (&v)[8]) {
    if (e + 8 <= n) {
        const u32x4_a2 w = *reinterpret_cast<const u32x4_a2*>(p + e);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = h2f(uint16_t(w[i >> 1] >> (16 * (i & 1))));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e + i < n ? h2f(p[e + i]) : 0.0f;
    }
}
__device__ __forceinline__ void load8(const float* p, int e, int n, float (&v)[8]) {
    if (e + 8 <= n) {
        const f32x4_a4 a = *reinterpret_cast<const f32x4_a4*>(p + e);
        const f32x4_a4 b = *reinterpret_cast<const f32x4_a4*>(p + e + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e + i < n ? p[e + i] : 0.0f;
    }
}
__device__ __forceinline__ void store8(uint16_t* p, int e, int n, const float (&v)[8]) {
    if (e + 8 <= n) {
        u32x4_a2 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = uint32_t(f2h(v[2 * i])) | (uint32_t(f2h(v[2 * i + 1])) << 16);
        *reinterpret_cast<u32x4_a2*>(p + e) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < n) p[e + i] = f2h(v[i]);
    }
}
__device__ __forceinline__ void store8(float* p, int e, int n, const float (&v)[8]) {
    if (e + 8 <= n) {
        *reinterpret_cast<f32x4_a4*>(p + e) = f32x4_a4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_a4*>(p + e + 4) = f32x4_a4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < n) p[e + i] = v[i];
    }
}

// Codes of v: adding 1.5 * 2^23 to a quotient rounds it to a whole number, to nearest even (the
// sum's last place is 1), and leaves that in the low byte.
//
// Computed values (v is rounded itself): the quotient is v * inv, within 2^-23 of v * 127 / a,
// rounded by itself, so that a program that computes the formula in fp32 gets the same codes.
// Plain rows (EXACT): v and a are fp16, and quotients that lie halfway between two codes are
// common (v = a / 2 is 63.5), so the rounding of inv would choose between them. With the rest
// of 127 / a in inv_lo the quotient is the exact one to nearest: a half stays a half, and what
// is none is at least 16 times that rounding away from one (v has 11 bits, a too). It costs
// 1 to 3 % (8192 rows of 8192 36.5 -> 37.2 us).
template <bool EXACT>
__device__ __forceinline__ void store_codes(int8_t* p, int e, int n, const float (&v)[8],
                                            float inv, float inv_lo) {
#pragma clang fp contract(off)
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = EXACT ? __builtin_fmaf(v[i], inv, v[i] * inv_lo) : v[i] * inv;
        b[i] = __builtin_bit_cast(uint32_t, q + 12582912.0f);
    }
    if (e + 8 <= n) {
        u32x2_a1 w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000c0cu);
            w[i] = lo | hi;
        }
        *reinterpret_cast<u32x2_a1*>(p + e) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < n) p[e + i] = int8_t(b[i]);
    }
}

__device__ __forceinline__ uint32_t magnitude(float v) {
    return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
}

// Non-negative floats and NaN bits order as unsigned integers.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](uint32_t o) { v = o > v ? o : v; };
#define AF_DPP_MAX(ctrl) \
    step(uint32_t(__builtin_amdgcn_update_dpp(0, int(v), ctrl, 0xf, 0xf, true)))
    AF_DPP_MAX(0xB1);
    AF_DPP_MAX(0x4E);
    AF_DPP_MAX(0x141);
    AF_DPP_MAX(0x128);
#undef AF_DPP_MAX
    uint32_t a = v, b = v;
    swap16(a, b);
    a = b = a > b ? a : b;
    swap32(a, b);
    return a > b ? a : b;
}

// One value per wave of the row (or one for each of P chunks) to all of the row's threads,
// combined in the order of chunks and waves.
template <int WAVES, int P, typename V, typename F>
__device__ __forceinline__ V across_waves(const V (&v)[P], V* s, F op) {
    if constexpr (WAVES == 1) {
        static_assert(P == 1, "one value");
        return v[0];
    } else {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int p = 0; p < P; ++p) s[p * WAVES + (threadIdx.x >> 6)] = v[p];
        __syncthreads();
        V r = s[0];
#pragma unroll
        for (int i = 1; i < P * WAVES; ++i) r = op(r, s[i]);
        return r;
    }
}

// A chunk of v before the norm's factor: x, silu(gate) * up, or x + residual.
template <int MODE>
__device__ __forceinline__ void load_chunk(const RowArgs& a, size_t row, int e, float (&v)[8]) {
    load8(a.x + row * a.x_stride, e, a.n, v);
    float o[8];
    if constexpr (MODE == kSiluMul) {
        load8(a.up + row * a.x_stride, e, a.n, o);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ex = fast_exp2(v[i] * -1.4426950408889634f);
            v[i] = v[i] * __builtin_amdgcn_rcpf(1.0f + ex) * o[i];
        }
    } else if constexpr (MODE == kNormAdd16) {
        load8(static_cast<const uint16_t*>(a.res_in) + row * a.res_stride, e, a.n, o);
    } else if constexpr (MODE == kNormAdd32) {
        load8(static_cast<const float*>(a.res_in) + row * a.res_stride, e, a.n, o);
    }
    if constexpr (MODE >= kNormAdd16)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += o[i];
}

template <int MODE>
__device__ __forceinline__ void store_residual(const RowArgs& a, size_t row, int e,
                                               const float (&v)[8]) {
    if constexpr (MODE == kNormAdd16)
        store8(static_cast<uint16_t*>(a.res_out) + row * a.res_stride, e, a.n, v);
    else if constexpr (MODE == kNormAdd32)
        store8(static_cast<float*>(a.res_out) + row * a.res_stride, e, a.n, v);
}

// rsqrt(mean + eps) of a row's sum of squares; NaN where the sum is not finite.
__device__ __forceinline__ float norm_factor(float sum, const RowArgs& a) {
    const float r = 1.0f / sqrtf(sum / float(a.n) + a.eps);
    return magnitude(sum) < 0x7f800000u ? r : __builtin_nanf("");
}

// Rows whose largest magnitude is below 2^-100 count as zero rows: 127 / a stays finite.
struct Scale {
    float inv, scale;
    bool bad;
    float inv_lo;  // of 127 / a, what inv's rounding leaves
};
__device__ __forceinline__ Scale row_scale(uint32_t bits) {
    const float top = __builtin_bit_cast(float, bits);
    const bool zero = bits < 0x0d800000u;
    Scale r;
    r.bad = bits >= 0x7f800000u;
    r.inv = zero ? 0.0f : 127.0f / top;
    r.inv_lo = zero ? 0.0f : __builtin_fmaf(-r.inv, top, 127.0f) / top;
    r.scale = r.bad ? __builtin_nanf("") : (zero ? 1.0f : top / 127.0f);
    return r;
}

// T threads per row (a wave's, or the whole workgroup), CH chunks of 8 elements per
// thread in registers: n <= 8 * T * CH.
template <int MODE, int T, int CH>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rows_kernel(const RowArgs a) {
    constexpr int WAVES = T / 64, ROWS = T < 256 ? 256 / T : 1;
    // Rows that few of them give 1024 threads and many 512 with two chunks each are summed in
    // the first's order by both, so that a row's bits do not depend on how many there are.
    constexpr int SUMS = T == 512 ? CH : 1;
    __shared__ float s_sum[SUMS * WAVES];
    __shared__ uint32_t s_max[WAVES];
    const int t = threadIdx.x % T;
    const int row_i = int(blockIdx.x) * ROWS + int(threadIdx.x) / T;
    if (ROWS > 1 && row_i >= a.m) return;  // whole waves; such a kernel has no barrier
    const size_t row = size_t(a.row0) + row_i;
    float v[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) load_chunk<MODE>(a, row, 8 * (t + c * T), v[c]);
    if constexpr (MODE >= kNorm) {
        float sums[SUMS] = {};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                sums[c % SUMS] = fmaf(v[c][i], v[c][i], sums[c % SUMS]);
        float w[CH][8];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            load8(a.weight, 8 * (t + c * T), a.n, w[c]);
            store_residual<MODE>(a, row, 8 * (t + c * T), v[c]);
        }
#pragma unroll
        for (int i = 0; i < SUMS; ++i) sums[i] = wave_sum(sums[i]);
        const float f = norm_factor(
            across_waves<WAVES>(sums, s_sum, [](float p, float q) { return p + q; }), a);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = v[c][i] * f * w[c][i];
            if (a.normed) store8(a.normed + row * a.normed_stride, 8 * (t + c * T), a.n, v[c]);
        }
        if (!a.codes) return;
    }
    uint32_t top[1] = {0};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) top[0] = max(top[0], magnitude(v[c][i]));
    top[0] = wave_max_u32(top[0]);
    const Scale sc = row_scale(across_waves<WAVES>(
        top, s_max, [](uint32_t p, uint32_t q) { return p > q ? p : q; }));
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if (sc.bad)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0.0f;
        store_codes<MODE == kPlain>(a.codes + row * a.codes_stride, 8 * (t + c * T), a.n, v[c],
                                    sc.bad ? 0.0f : sc.inv, sc.bad ? 0.0f : sc.inv_lo);
    }
    if (t == 0) a.scales[row] = sc.scale;
}

// Rows longer than the registers of a workgroup: the same steps, the row's chunks read
// again (from cache) for each. The residual is written by the last pass, so that it may
// be the one that is read.
template <int MODE>
__global__ __launch_bounds__(1024) void long_rows_kernel(const RowArgs a) {
    __shared__ float s_sum[16];
    __shared__ uint32_t s_max[16];
    const size_t row = size_t(a.row0) + blockIdx.x;
    float f = 1.0f;
    float v[8], w[8];
    if constexpr (MODE >= kNorm) {
        float sum[1] = {0.0f};
        for (int e = 8 * threadIdx.x; e < a.n; e += 8 * 1024) {
            load_chunk<MODE>(a, row, e, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[0] = fmaf(v[i], v[i], sum[0]);
        }
        sum[0] = wave_sum(sum[0]);
        f = norm_factor(across_waves<16>(sum, s_sum, [](float p, float q) { return p + q; }), a);
    }
    auto scaled = [&](int e, bool raw) {
        load_chunk<MODE>(a, row, e, v);
        if constexpr (MODE >= kNorm) {
            if (raw) store_residual<MODE>(a, row, e, v);
            load8(a.weight, e, a.n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * f * w[i];
        }
    };
    Scale sc{0.0f, 1.0f, false, 0.0f};
    if (a.codes) {
        uint32_t top[1] = {0};
        for (int e = 8 * threadIdx.x; e < a.n; e += 8 * 1024) {
            scaled(e, false);
#pragma unroll
            for (int i = 0; i < 8; ++i) top[0] = max(top[0], magnitude(v[i]));
        }
        top[0] = wave_max_u32(top[0]);
        sc = row_scale(across_waves<16>(top, s_max,
                                        [](uint32_t p, uint32_t q) { return p > q ? p : q; }));
        if (threadIdx.x == 0) a.scales[row] = sc.scale;
    }
    for (int e = 8 * threadIdx.x; e < a.n; e += 8 * 1024) {
        scaled(e, true);
        if (MODE >= kNorm && a.normed) store8(a.normed + row * a.normed_stride, e, a.n, v);
        if (a.codes) {
            if (sc.bad)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
            store_codes<MODE == kPlain>(a.codes + row * a.codes_stride, e, a.n, v,
                                        sc.bad ? 0.0f : sc.inv, sc.bad ? 0.0f : sc.inv_lo);
        }
    }
}

template <int MODE, int T, int CH>
void launch_rows(const RowArgs& a, hipStream_t s) {
    constexpr int ROWS = T < 256 ? 256 / T : 1;
    const unsigned blocks = unsigned((int64_t(a.m) + ROWS - 1) / ROWS);
    hipLaunchKernelGGL((rows_kernel<MODE, T, CH>), dim3(blocks), dim3(T < 256 ? 256 : T), 0, s, a);
}

// Threads per row and chunks per thread by the row's length, measured for 1 to 8192 rows on
// MI355X (us, plain / gated / norm with an fp16 residual). A thread's one chunk is best while
// a workgroup can hold the row so: 45 rows of 4096 on 512 threads 2.2 / 2.6 / 3.0, on 256 with
// two chunks each 2.4 / 2.9 / 3.6; 8192 rows 21.4 / 31.7 / 44.2 and 21.0 / 35.6 / 48.4. Short
// rows take a wave each, which needs no barrier: 8192 rows of 1024 8.2 / 13.1 / 15.1, on 256
// threads 9.9 / 13.5 / 17.5. Above 4096, 1024 threads suit few rows (45 of 5120: 2.4 / 3.0 /
// 3.7, on 512 threads 2.6 / 3.5 / 4.2), and many only where the row fills them (8192 of 8192:
// 40.9 / 61.7 / 85.0 and 37.2 / 62.1 / 88.1; of 5120: 34.0 / 47.8 / 66.1 and 26.8 / 43.4 / 59.4).
// 85.0 us are 5.5 TB/s, what a large copy reaches on this card (5.15) and more.
template <int MODE>
void launch_slice(const RowArgs& a, hipStream_t s) {
    const bool few = a.m < 2 * device_compute_units();
    if (a.n <= 512) launch_rows<MODE, 64, 1>(a, s);
    else if (a.n <= 1024) launch_rows<MODE, 64, 2>(a, s);
    else if (a.n <= 2048) launch_rows<MODE, 256, 1>(a, s);
    else if (a.n <= 4096) launch_rows<MODE, 512, 1>(a, s);
    else if (a.n <= 8192 && (few || (MODE != kPlain && a.n > 7168)))
        launch_rows<MODE, 1024, 1>(a, s);
    else if (a.n <= 8192) launch_rows<MODE, 512, 2>(a, s);
    else if (a.n <= 16384) launch_rows<MODE, 1024, 2>(a, s);
    else if (a.n <= 32768) launch_rows<MODE, 1024, 4>(a, s);
    else hipLaunchKernelGGL((long_rows_kernel<MODE>), dim3(unsigned(a.m)), dim3(1024), 0, s, a);
}

// A launch has fewer than 2^32 threads: more rows than kSlice take several.
constexpr int kSlice = 1 << 21;

template <int MODE>
int launch_mode(const RowArgs& a, hipStream_t s) {
    RowArgs b = a;
    for (int64_t row = 0; row < a.m; row += kSlice) {
        b.row0 = int(row);
        b.m = int(a.m - row < kSlice ? a.m - row : kSlice);
        launch_slice<MODE>(b, s);
        AF_TRY_LAUNCH();
    }
    return AF_OK;
}

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_rows(const void* x, int64_t x_stride, int m, int n) {
    if (!x || m < 0 || n <= 0 || x_stride < n || !aligned(x, 2)) return AF_ERR_INVALID_ARG;
    if (n > 1 << 30) return AF_ERR_UNSUPPORTED;  // 32-bit element indices, one step past the end
    return AF_OK;
}
int check_codes(const int8_t* codes, int64_t codes_stride, const float* scales, int n) {
    if (!codes || !scales || codes_stride < n || !aligned(scales, 4)) return AF_ERR_INVALID_ARG;
    return AF_OK;
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" int af_quantize_rows(const void* x, int64_t x_stride, int m, int n, int8_t* codes,
                                int64_t codes_stride, float* scales, af_stream_t stream) {
    if (int st = check_rows(x, x_stride, m, n)) return st;
    if (int st = check_codes(codes, codes_stride, scales, n)) return st;
    if (m == 0) return AF_OK;
    RowArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.m = m;
    a.n = n;
    a.codes = codes;
    a.codes_stride = codes_stride;
    a.scales = scales;
    return launch_mode<kPlain>(a, static_cast<hipStream_t>(stream));
}

extern "C" int af_silu_mul_quantize(const void* gate, const void* up, int64_t stride, int m, int n,
                                    int8_t* codes, int64_t codes_stride, float* scales,
                                    af_stream_t stream) {
    if (int st = check_rows(gate, stride, m, n)) return st;
    if (int st = check_rows(up, stride, m, n)) return st;
    if (int st = check_codes(codes, codes_stride, scales, n)) return st;
    if (m == 0) return AF_OK;
    RowArgs a{};
    a.x = static_cast<const uint16_t*>(gate);
    a.up = static_cast<const uint16_t*>(up);
    a.x_stride = stride;
    a.m = m;
    a.n = n;
    a.codes = codes;
    a.codes_stride = codes_stride;
    a.scales = scales;
    return launch_mode<kSiluMul>(a, static_cast<hipStream_t>(stream));
}

extern "C" int af_rmsnorm_quantize(const void* x, int64_t x_stride, const void* residual,
                                   void* residual_out, int64_t residual_stride, int residual_dtype,
                                   const float* weight, float eps, int m, int n, int8_t* codes,
                                   int64_t codes_stride, float* scales, void* normed,
                                   int64_t normed_stride, af_stream_t stream) {
    if (int st = check_rows(x, x_stride, m, n)) return st;
    if (!weight || !aligned(weight, 4) || !(eps > 0.0f) || !(eps < __builtin_inff()))
        return AF_ERR_INVALID_ARG;
    if (!codes && !normed) return AF_ERR_INVALID_ARG;
    if (codes)
        if (int st = check_codes(codes, codes_stride, scales, n)) return st;
    if (normed && (normed_stride < n || !aligned(normed, 2))) return AF_ERR_INVALID_ARG;
    if (!residual != !residual_out) return AF_ERR_INVALID_ARG;
    if (residual) {
        if (residual_dtype != AF_FP16 && residual_dtype != AF_FP32) return AF_ERR_UNSUPPORTED;
        const size_t to = residual_dtype == AF_FP32 ? 4 : 2;
        if (residual_stride < n || !aligned(residual, to) || !aligned(residual_out, to))
            return AF_ERR_INVALID_ARG;
    }
    if (m == 0) return AF_OK;
    RowArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.res_in = residual;
    a.res_out = residual_out;
    a.res_stride = residual_stride;
    a.weight = weight;
    a.eps = eps;
    a.m = m;
    a.n = n;
    a.codes = codes;
    a.codes_stride = codes_stride;
    a.scales = scales;
    a.normed = static_cast<uint16_t*>(normed);
    a.normed_stride = normed_stride;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!residual) return launch_mode<kNorm>(a, s);
    if (residual_dtype == AF_FP32) return launch_mode<kNormAdd32>(a, s);
    return launch_mode<kNormAdd16>(a, s);
}
