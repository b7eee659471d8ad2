// Compiled and run by tests/test_host_experts.py: the C++ binding converts the weights of all experts, a rank-3 tensor, in one call.
// Without an argument only its guards run; with `gpu` it is compared with a call for each expert.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include <cuda_runtime_api.h>

#include "../beantensor_b200/host/MatMulOps.h"

using namespace BeanTensor::Tensors::detail;

static btm_tensor_view view(void *data, int dtype, std::vector<uint64_t> shape)
{
    btm_tensor_view v;
    std::memset(&v, 0, sizeof(v));
    v.data = data;
    v.dtype = dtype;
    v.device = 1;
    v.ndim = (int)shape.size();
    uint64_t stride = 1;
    for (int i = v.ndim - 1; i >= 0; --i) {
        v.shape[i] = shape[i];
        v.strides[i] = stride;
        stride *= shape[i];
    }
    return v;
}

static int guards()
{
    int passed = 0;
    void *p = reinterpret_cast<void *>(0x1000);
    auto x = view(p, BTM_F16, {3, 40, 64}), q = view(p, BTM_U8, {3, 40, 32}), s = view(p, BTM_U8, {3 * 512}), off = view(p, BTM_I32, {4});
    auto refused = [&](const char *text, auto &&f) {
        try { f(); } catch (const std::invalid_argument &e) { passed += std::strstr(e.what(), text) != nullptr; }
    };
    // all guards passed: the C ABI then refuses a type that it does not know, without a device
    auto accepted = [&](auto &&f) { try { f(); } catch (const BeanTensor::ErrorHandling::NotImplemented &) { ++passed; } catch (...) {} };
    accepted([&] { auto c = x; c.dtype = BTM_I16; quantize_mxfp4_gpu(c, q, s); });
    accepted([&] { auto c = x; c.dtype = BTM_I16; dequant_mxfp4_gpu(q, s, c); });
    refused("offsets go with", [&] { quantize_mxfp4_gpu(x, q, s, &off); });
    refused("offsets go with", [&] { dequant_mxfp4_gpu(q, s, x, &off); });
    refused("too few scale", [&] { auto c = view(p, BTM_U8, {3 * 512 - 1}); quantize_mxfp4_gpu(x, q, c); });
    refused("shape mismatch", [&] { auto c = view(p, BTM_U8, {3, 41, 32}); quantize_mxfp4_gpu(x, c, s); });
    refused("shape mismatch", [&] { auto c = view(p, BTM_U8, {2, 40, 32}); dequant_mxfp4_gpu(c, s, x); });
    refused("wrong rank", [&] { auto c = view(p, BTM_U8, {120, 32}); quantize_mxfp4_gpu(x, c, s); });
    refused("contiguous", [&] { auto c = x; c.strides[0] = 41 * 64; quantize_mxfp4_gpu(c, q, s); });
    refused("contiguous", [&] { auto c = x; c.strides[1] = 72; c.strides[0] = 40 * 72; dequant_mxfp4_gpu(q, s, c); });
    refused("32 bits", [&] { auto c = view(p, BTM_F16, {1ull << 20, 1ull << 20, 64}); auto d = view(p, BTM_U8, {1ull << 20, 1ull << 20, 32}); quantize_mxfp4_gpu(c, d, s); });
    auto y = view(p, BTM_F16, {40, 64}), yq = view(p, BTM_U8, {40, 32});
    refused("offsets must be", [&] { auto c = view(p, BTM_I32, {0}); quantize_mxfp4_gpu(y, yq, s, &c); });
    refused("offsets must be", [&] { auto c = view(p, BTM_I32, {2, 2}); quantize_mxfp4_gpu(y, yq, s, &c); });
    return passed;
}

struct Device {
    void *p = nullptr;
    Device(size_t bytes, const void *src = nullptr)
    {
        if (cudaMalloc(&p, bytes) != cudaSuccess) std::exit(3);
        if (src) cudaMemcpy(p, src, bytes, cudaMemcpyHostToDevice);
        else cudaMemset(p, 0x5A, bytes);
    }
    ~Device() { cudaFree(p); }
    std::vector<uint8_t> read(size_t n) const
    {
        std::vector<uint8_t> h(n);
        cudaMemcpy(h.data(), p, n, cudaMemcpyDeviceToHost);
        return h;
    }
};

static int experts()
{
    const size_t G = 3, N = 200, K = 160, one = btm_mxfp4_scale_bytes(1, N, K);
    std::vector<float> w(G * N * K);
    unsigned s = 1;
    for (auto &x : w) {
        s = s * 1664525u + 1013904223u;
        x = (float)((int)(s >> 20) - 2048) / 64.0f;
    }
    Device dw(w.size() * 4, w.data()), q(G * N * K / 2), sc(G * one), back(w.size() * 4), q1(G * N * K / 2), sc1(G * one), back1(w.size() * 4);
    auto vw = view(dw.p, BTM_F32, {G, N, K}), vq = view(q.p, BTM_U8, {G, N, K / 2}), vs = view(sc.p, BTM_U8, {G * one}), vb = view(back.p, BTM_F32, {G, N, K});
    quantize_mxfp4_gpu(vw, vq, vs);
    dequant_mxfp4_gpu(vq, vs, vb);
    for (size_t g = 0; g < G; ++g) {
        auto x = view(static_cast<float *>(dw.p) + g * N * K, BTM_F32, {N, K}), y = view(static_cast<char *>(q1.p) + g * N * K / 2, BTM_U8, {N, K / 2});
        auto z = view(static_cast<char *>(sc1.p) + g * one, BTM_U8, {one}), o = view(static_cast<float *>(back1.p) + g * N * K, BTM_F32, {N, K});
        quantize_mxfp4_gpu(x, y, z);
        dequant_mxfp4_gpu(y, z, o);
    }
    if (btm_check_device_status(0, nullptr) != BTM_OK) return -100;
    return (q.read(G * N * K / 2) == q1.read(G * N * K / 2)) + (sc.read(G * one) == sc1.read(G * one)) + (back.read(w.size() * 4) == back1.read(w.size() * 4));
}

int main(int argc, char **argv)
{
    int passed = guards();
    if (argc > 1 && !std::strcmp(argv[1], "gpu")) passed += experts();
    std::printf("passed=%d\n", passed);
    return 0;
}
