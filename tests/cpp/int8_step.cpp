// int8_step.cpp — a C++ host that runs the MLP half of a layer on the int8 projection path
// through include/ops/kernel.h: the residual's addition and norm, the gate and up product
// (with a bias), silu(gate) * up, the down product in fp32, and the quantiser of plain rows.
// Inputs come from a fixed xorshift stream; inputs and outputs are written to
// <out_dir>/*.bin so tests/test_gpu_cpp_int8.py can check them in 64 bits.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <stdexcept>
#include <string>
#include <vector>

#include "ops/kernel.h"

namespace {

constexpr int M = 21, D = 272, F = 400;
constexpr int XS = D + 8;  // row stride of x

#define HIP_OK(x)                                                                        \
    do {                                                                                 \
        hipError_t e_ = (x);                                                             \
        if (e_ != hipSuccess)                                                            \
            throw std::runtime_error(std::string(#x) + ": " + hipGetErrorString(e_));   \
    } while (0)

struct Rng {
    uint64_t s;
    uint64_t next() {
        s ^= s >> 12;
        s ^= s << 25;
        s ^= s >> 27;
        return s * 0x2545F4914F6CDD1Dull;
    }
    float uniform() { return float(int64_t(next() >> 11) - (int64_t(1) << 52)) * 0x1p-51f; }  // [-2, 2)
};

std::string out_dir;

void save(const char* name, const void* p, size_t bytes) {
    const std::string path = out_dir + "/" + name + ".bin";
    FILE* f = std::fopen(path.c_str(), "wb");
    if (!f || std::fwrite(p, 1, bytes, f) != bytes) throw std::runtime_error("write " + path);
    std::fclose(f);
}

// A host array written to a file and copied to the device.
template <typename T>
T* input(const char* name, const std::vector<T>& h) {
    save(name, h.data(), h.size() * sizeof(T));
    T* d = nullptr;
    HIP_OK(hipMalloc(&d, h.size() * sizeof(T)));
    HIP_OK(hipMemcpy(d, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice));
    return d;
}

template <typename T>
T* room(size_t n) {
    T* d = nullptr;
    HIP_OK(hipMalloc(&d, n * sizeof(T)));
    return d;
}

template <typename T>
void output(const char* name, const T* d, size_t n) {
    std::vector<T> h(n);
    HIP_OK(hipMemcpy(h.data(), d, n * sizeof(T), hipMemcpyDeviceToHost));
    save(name, h.data(), n * sizeof(T));
}

void run(hipStream_t s) {
    Rng r{0x9E3779B97F4A7C15ull};
    auto floats = [&](size_t n, float size, float mid) {
        std::vector<float> v(n);
        for (auto& x : v) x = mid + size * r.uniform();
        return v;
    };
    auto codes = [&](size_t n) {
        std::vector<int8_t> v(n);
        for (auto& x : v) x = int8_t(int(r.next() >> 40) % 255 - 127);
        return v;
    };
    std::vector<uint16_t> x(size_t(M) * XS);
    for (auto& v : x) v = __half_as_ushort(__float2half_rn(r.uniform()));
    __half* d_x = reinterpret_cast<__half*>(input("x", x));
    float* d_res = input("res", floats(size_t(M) * D, 1.5f, 0.0f));
    float* d_norm = input("norm", floats(D, 0.1f, 1.0f));
    int8_t* d_wgu = input("w_gate_up", codes(size_t(2 * F) * D));
    float* d_sgu = input("s_gate_up", floats(2 * F, 1e-4f, 6e-4f));
    float* d_bias = input("bias", floats(2 * F, 0.2f, 0.0f));
    int8_t* d_wd = input("w_down", codes(size_t(D) * F));
    float* d_sd = input("s_down", floats(D, 1e-4f, 6e-4f));

    int8_t *c1 = room<int8_t>(size_t(M) * D), *c2 = room<int8_t>(size_t(M) * F);
    int8_t* c3 = room<int8_t>(size_t(M) * 2 * F);
    float *s1 = room<float>(M), *s2 = room<float>(M), *s3 = room<float>(M);
    uint16_t* gu = room<uint16_t>(size_t(M) * 2 * F);
    float* down = room<float>(size_t(M) * D);

    View res = create_contiguous_view(d_res, DataType::FP32, {M, D});
    View norm = create_contiguous_view(d_norm, DataType::FP32, {D});
    View v_gu = create_contiguous_view(gu, DataType::FP16, {M, 2 * F});
    View v_down = create_contiguous_view(down, DataType::FP32, {M, D});
    __half* h_gu = reinterpret_cast<__half*>(gu);
    launch_rmsnorm_quantize(d_x, XS, res, norm, 1e-5f, c1, D, s1, s);
    launch_w8a8_gemm(c1, D, s1, d_wgu, D, d_sgu, d_bias, v_gu, D, s);
    launch_silu_mul_quantize(h_gu, h_gu + F, 2 * F, M, F, c2, F, s2, s);
    launch_w8a8_gemm(c2, F, s2, d_wd, F, d_sd, nullptr, v_down, F, s);
    launch_quantize_rows(h_gu, 2 * F, M, 2 * F, c3, 2 * F, s3, s);
    HIP_OK(hipStreamSynchronize(s));
    output("res_out", d_res, size_t(M) * D);
    output("c1", c1, size_t(M) * D);
    output("s1", s1, M);
    output("gate_up", gu, size_t(M) * 2 * F);
    output("c2", c2, size_t(M) * F);
    output("s2", s2, M);
    output("down", down, size_t(M) * D);
    output("c3", c3, size_t(M) * 2 * F);
    output("s3", s3, M);
}

}  // namespace

int main(int argc, char** argv) {
    if (argc != 2) {
        std::fprintf(stderr, "usage: %s OUT_DIR\n", argv[0]);
        return 2;
    }
    out_dir = argv[1];
    try {
        HIP_OK(hipSetDevice(0));
        hipStream_t s = nullptr;
        HIP_OK(hipStreamCreate(&s));
        run(s);
        HIP_OK(hipStreamDestroy(s));
    } catch (const std::exception& e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
    std::puts("ok");
    return 0;
}
