// af_rope.h — device helpers of the rotary operators: runs of W elements, and W turned pairs.
#pragma once

#include "af_device.h"
#include "af_kv.h"

namespace af {

template <int W>
__device__ __forceinline__ void load_halves(const uint16_t* p, uint16_t (&v)[W]) {
    if constexpr (W == 8) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = uint16_t(u[i >> 1] >> (16 * (i & 1)));
    } else if constexpr (W == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        v[0] = uint16_t(w.x), v[1] = uint16_t(w.x >> 16);
        v[2] = uint16_t(w.y), v[3] = uint16_t(w.y >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = p[i];
    }
}
template <int W>
__device__ __forceinline__ void store_halves(uint16_t* p, const uint16_t (&v)[W]) {
    auto pair = [&](int i) { return uint32_t(v[i]) | (uint32_t(v[i + 1]) << 16); };
    if constexpr (W == 8)
        *reinterpret_cast<uint4*>(p) = make_uint4(pair(0), pair(2), pair(4), pair(6));
    else if constexpr (W == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(pair(0), pair(2));
    else
#pragma unroll
        for (int i = 0; i < W; ++i) p[i] = v[i];
}
template <int W>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[W]) {
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const float4 w = *reinterpret_cast<const float4*>(p + i);
            v[i] = w.x, v[i + 1] = w.y, v[i + 2] = w.z, v[i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = p[i];
    }
}

// Four fp32 values to E4M3, to nearest even and clamped to +-448 (v_cvt_pk_fp8_f32); a NaN stays
// one (the clamp alone would make it a bound).
__device__ __forceinline__ float clamp_fp8(float v) {
    return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f);
}
template <int W>
__device__ __forceinline__ void store_fp8(uint8_t* p, const float (&v)[W]) {
    if constexpr (W % 4 == 0) {
        uint32_t w[W / 4];
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            int x = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_fp8(v[4 * i]), clamp_fp8(v[4 * i + 1]), 0,
                                                    false);
            x = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_fp8(v[4 * i + 2]), clamp_fp8(v[4 * i + 3]), x,
                                                true);
            w[i] = uint32_t(x);
        }
        if constexpr (W == 16)
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (W == 8)
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            p[i] = uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(clamp_fp8(v[i]), 0.0f, 0, false));
    }
}
template <int W>
__device__ __forceinline__ void load_fp8(const uint8_t* p, float (&v)[W]) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
    if constexpr (W % 4 == 0) {
        uint32_t w[W / 4];
        if constexpr (W == 16) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else if constexpr (W == 8) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            w[0] = u.x, w[1] = u.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), false);
            const float2_t b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), true);
            v[4 * i] = a[0], v[4 * i + 1] = a[1], v[4 * i + 2] = b[0], v[4 * i + 3] = b[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = __builtin_amdgcn_cvt_f32_fp8(int(p[i]), 0);
    }
}

// One turned pair in fp32: separately rounded products and sums, as rope_rotate's.
__device__ __forceinline__ void turn_pair(float& x, float& y, float c, float s) {
#pragma clang fp contract(off)
    const float xc = x * c, ys = y * s, xs = x * s, yc = y * c;
    x = xc - ys;
    y = xs + yc;
}
// The pairs of a chunk's two runs u and v of W elements: (u[i], v[i]) in halves of the head, or
// neighbours in the 2 W elements u, v.
template <int LAYOUT, int W>
__device__ __forceinline__ void rotate_floats(float (&u)[W], float (&v)[W], const float (&c)[W],
                                              const float (&s)[W]) {
    if constexpr (LAYOUT == AF_ROPE_HALF || W == 1) {
#pragma unroll
        for (int i = 0; i < W; ++i) turn_pair(u[i], v[i], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            turn_pair(u[2 * i], u[2 * i + 1], c[i], s[i]);
            turn_pair(v[2 * i], v[2 * i + 1], c[W / 2 + i], s[W / 2 + i]);
        }
    }
}
template <int LAYOUT, int W>
__device__ __forceinline__ void rotate_halves(uint16_t (&u)[W], uint16_t (&v)[W],
                                              const float (&c)[W], const float (&s)[W]) {
    float x[W], y[W];
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = h2f(u[i]), y[i] = h2f(v[i]);
    rotate_floats<LAYOUT, W>(x, y, c, s);
#pragma unroll
    for (int i = 0; i < W; ++i) u[i] = f2h(x[i]), v[i] = f2h(y[i]);
}

}  // namespace af
