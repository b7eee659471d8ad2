// Compiled and run by tests/test_host_grouped.py: the C++ binding of the grouped and microscaled operators. Without an argument
// only its guards and the status mapping run; with `gpu` real products of small whole numbers, exact in every format.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include <cuda_runtime_api.h>

#include "../beantensor_b200/host/MatMulOps.h"

using namespace BeanTensor::Tensors::detail;

static btm_tensor_view view(void *data, int dtype, int device, std::vector<uint64_t> shape)
{
    btm_tensor_view v;
    std::memset(&v, 0, sizeof(v));
    v.data = data;
    v.dtype = dtype;
    v.device = device;
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
    auto a = view(p, BTM_F16, 1, {8, 32}), b = view(p, BTM_F16, 1, {2, 32, 16}), off = view(p, BTM_I32, 1, {3}), o = view(p, BTM_F16, 1, {8, 16});
    auto refused = [&](auto &&f) { try { f(); } catch (const std::invalid_argument &) { ++passed; } };
    refused([&] { auto c = a; c.device = 0; grouped_matmul_gpu(c, b, off, o); });
    refused([&] { auto c = view(p, BTM_I32, 1, {2}); grouped_matmul_gpu(a, b, c, o); });
    refused([&] { auto c = view(p, BTM_I64, 1, {3}); grouped_matmul_gpu(a, b, c, o); });
    refused([&] { auto c = view(p, BTM_F16, 1, {8, 17}); grouped_matmul_gpu(a, b, off, c); });
    refused([&] { auto c = b; c.strides[1] = 3; c.strides[2] = 2; grouped_matmul_gpu(a, c, off, o); });
    refused([&] { auto c = view(p, BTM_F16, 1, {1ull << 32, 32}); auto d = view(p, BTM_F16, 1, {1ull << 32, 16}); grouped_matmul_gpu(c, b, off, d); });
    refused([&] { auto c = view(p, BTM_F16, 1, {2, 16, 32}); grouped_matmul_wgrad_gpu(a, o, off, c); });
    try { // the C ABI's own refusal
        auto x = view(p, BTM_F32, 1, {8, 32}), y = view(p, BTM_F32, 1, {2, 32, 16}), z = view(p, BTM_F32, 1, {8, 16});
        grouped_matmul_gpu(x, y, off, z);
    } catch (const BeanTensor::ErrorHandling::NotImplemented &) { ++passed; }
    auto q = view(p, BTM_U8, 1, {8, 16}), s = view(p, BTM_U8, 1, {512}), w = view(p, BTM_U8, 1, {2, 16, 16});
    refused([&] { auto c = view(p, BTM_U8, 1, {511}); quantize_mxfp4_gpu(a, q, c); });
    refused([&] { auto c = view(p, BTM_U8, 1, {8, 17}); quantize_mxfp4_gpu(a, c, s); });
    refused([&] { auto c = view(p, BTM_I8, 1, {8, 16}); quantize_mxfp4_gpu(a, c, s); });
    refused([&] { auto c = view(p, BTM_F16, 1, {8, 48}); auto d = view(p, BTM_U8, 1, {8, 24}); quantize_mxfp4_gpu(c, d, s); });
    refused([&] { auto c = view(p, BTM_U8, 1, {16, 24}); matmul_mxfp4_gpu(q, s, c, s, o); });
    refused([&] { auto c = view(p, BTM_U8, 1, {512}); grouped_matmul_mxfp4_gpu(q, c, w, c, off, o); });
    return passed;
}

// small whole numbers as fp16 bits and back
static uint16_t f16(int n)
{
    if (n == 0) return 0;
    const uint16_t sign = n < 0 ? 0x8000 : 0;
    unsigned m = (unsigned)std::abs(n);
    int e = 31 - __builtin_clz(m);
    return (uint16_t)(sign | ((e + 15) << 10) | ((m << (10 - e)) & 0x3FF));
}

struct Device {
    void *p = nullptr;
    Device(size_t bytes, const void *src = nullptr)
    {
        if (cudaMalloc(&p, bytes) != cudaSuccess) std::exit(3);
        if (src) cudaMemcpy(p, src, bytes, cudaMemcpyHostToDevice);
        else cudaMemset(p, 0, bytes);
    }
    ~Device() { cudaFree(p); }
    std::vector<uint16_t> read(size_t n) const
    {
        std::vector<uint16_t> h(n);
        cudaMemcpy(h.data(), p, n * 2, cudaMemcpyDeviceToHost);
        return h;
    }
};

static int products()
{
    int passed = 0;
    const int rows = 50, K = 64, N = 40, G = 3;
    const int32_t offs[G + 1] = {2, 20, 20, 47};
    static const int grid[8] = {0, 1, 2, 3, 4, 6, -1, -6}; // values that the 4-bit format holds beside a largest one of 6
    std::vector<int> a(rows * K), b(G * K * N), d(rows * N);
    unsigned s = 1;
    auto next = [&] { s = s * 1664525u + 1013904223u; return s >> 24; };
    for (auto &x : a) x = grid[next() % 8];
    for (auto &x : b) x = grid[next() % 8];
    for (auto &x : d) x = (int)(next() % 5) - 2;
    for (int r = 0; r < rows; ++r) for (int k = 0; k < K; k += 32) a[r * K + k] = 6; // fixes the scale of every block to 1
    for (int g = 0; g < G; ++g) for (int n = 0; n < N; ++n) for (int k = 0; k < K; k += 32) b[(g * K + k) * N + n] = 6;
    std::vector<uint16_t> ab(a.size()), bb(b.size()), bt(b.size()), db(d.size());
    for (size_t i = 0; i < a.size(); ++i) ab[i] = f16(a[i]);
    for (size_t i = 0; i < b.size(); ++i) bb[i] = f16(b[i]);
    for (size_t i = 0; i < d.size(); ++i) db[i] = f16(d[i]);
    for (int g = 0; g < G; ++g) for (int k = 0; k < K; ++k) for (int n = 0; n < N; ++n) bt[(g * N + n) * K + k] = bb[(g * K + k) * N + n];
    Device da(ab.size() * 2, ab.data()), dw(bb.size() * 2, bb.data()), dt(bt.size() * 2, bt.data()), dd(db.size() * 2, db.data());
    Device doff(sizeof(offs), offs), out(rows * N * 2), grad(G * K * N * 2), back(rows * K * 2), o4(rows * N * 2);
    auto va = view(da.p, BTM_F16, 1, {rows, K}), vb = view(dw.p, BTM_F16, 1, {G, K, N}), vd = view(dd.p, BTM_F16, 1, {rows, N});
    auto voff = view(doff.p, BTM_I32, 1, {G + 1}), vo = view(out.p, BTM_F16, 1, {rows, N}), vg = view(grad.p, BTM_F16, 1, {G, K, N});
    auto vback = view(back.p, BTM_F16, 1, {rows, K}), vo4 = view(o4.p, BTM_F16, 1, {rows, N});
    auto vbt = vb; // b transposed: [G, N, K] in the place of [G, K, N]
    vbt.shape[1] = N; vbt.shape[2] = K; vbt.strides[1] = 1; vbt.strides[2] = N;

    grouped_matmul_gpu(va, vb, voff, vo);
    grouped_matmul_wgrad_gpu(va, vd, voff, vg);
    grouped_matmul_gpu(vd, vbt, voff, vback);
    // 4 bits: activations by groups, the experts' weights one after the other
    Device q(rows * K / 2), qs(btm_mxfp4_scale_bytes(G, rows, K)), w((size_t)G * N * K / 2), ws(G * btm_mxfp4_scale_bytes(1, N, K)), values(rows * K * 2), dense(N * 2);
    auto vq = view(q.p, BTM_U8, 1, {rows, K / 2}), vqs = view(qs.p, BTM_U8, 1, {btm_mxfp4_scale_bytes(G, rows, K)});
    quantize_mxfp4_gpu(va, vq, vqs, &voff);
    auto vv = view(values.p, BTM_F16, 1, {rows, K});
    dequant_mxfp4_gpu(vq, vqs, vv, &voff);
    for (int g = 0; g < G; ++g) {
        auto x = view(static_cast<char *>(dt.p) + (size_t)g * N * K * 2, BTM_F16, 1, {N, K});
        auto y = view(static_cast<char *>(w.p) + (size_t)g * N * K / 2, BTM_U8, 1, {N, K / 2});
        auto z = view(static_cast<char *>(ws.p) + g * btm_mxfp4_scale_bytes(1, N, K), BTM_U8, 1, {btm_mxfp4_scale_bytes(1, N, K)});
        quantize_mxfp4_gpu(x, y, z);
    }
    auto vw = view(w.p, BTM_U8, 1, {G, N, K / 2}), vws = view(ws.p, BTM_U8, 1, {G * btm_mxfp4_scale_bytes(1, N, K)});
    grouped_matmul_mxfp4_gpu(vq, vqs, vw, vws, voff, vo4);
    // one row of the first group through the plain product
    auto row = view(static_cast<char *>(da.p) + (size_t)offs[0] * K * 2, BTM_F16, 1, {1, K});
    Device rq(K / 2), rs(512);
    auto vrq = view(rq.p, BTM_U8, 1, {1, K / 2}), vrs = view(rs.p, BTM_U8, 1, {512});
    quantize_mxfp4_gpu(row, vrq, vrs);
    auto w0 = view(w.p, BTM_U8, 1, {N, K / 2}), ws0 = view(ws.p, BTM_U8, 1, {btm_mxfp4_scale_bytes(1, N, K)}), vdense = view(dense.p, BTM_F16, 1, {1, N});
    matmul_mxfp4_gpu(vrq, vrs, w0, ws0, vdense);
    if (btm_check_device_status(0, nullptr) != BTM_OK) return -1;

    auto ho = out.read(rows * N), hg = grad.read(G * K * N), hb = back.read(rows * K), h4 = o4.read(rows * N), hv = values.read(rows * K), hd = dense.read(N);
    bool product = true, gradient = true, activation = true, four = true, same = true, plain = true;
    for (int r = 0; r < rows; ++r) {
        int g = -1;
        for (int i = 0; i < G; ++i) if (r >= offs[i] && r < offs[i + 1]) g = i;
        for (int n = 0; n < N; ++n) {
            int sum = 0;
            for (int k = 0; k < K && g >= 0; ++k) sum += a[r * K + k] * b[(g * K + k) * N + n];
            product &= ho[r * N + n] == f16(sum);
            four &= h4[r * N + n] == f16(sum);
            if (r == offs[0]) plain &= hd[n] == f16(sum);
        }
        for (int k = 0; k < K; ++k) {
            int sum = 0;
            for (int n = 0; n < N && g >= 0; ++n) sum += d[r * N + n] * b[(g * K + k) * N + n];
            activation &= hb[r * K + k] == f16(sum);
            same &= hv[r * K + k] == (g >= 0 ? ab[r * K + k] : 0);
        }
    }
    for (int g = 0; g < G; ++g)
        for (int k = 0; k < K; ++k)
            for (int n = 0; n < N; ++n) {
                int sum = 0;
                for (int r = offs[g]; r < offs[g + 1]; ++r) sum += a[r * K + k] * d[r * N + n];
                gradient &= hg[(g * K + k) * N + n] == f16(sum);
            }
    passed += product + gradient + activation + four + same + plain;
    if (passed != 6) std::printf("product %d gradient %d activation %d four %d same %d plain %d\n", product, gradient, activation, four, same, plain);
    return passed;
}

int main(int argc, char **argv)
{
    int passed = guards();
    if (argc > 1 && !std::strcmp(argv[1], "gpu")) passed += products();
    std::printf("passed=%d\n", passed);
    return 0;
}
