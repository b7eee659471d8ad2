// C++23 binding of libbtm.so in the style of the reference's GPU operator boundary
// (namespace BeanTensor::Tensors::detail, Tensor/TensorOps.h:15-65): free functions that guard
// the device, enqueue the work and leave the result in a pre-allocated tensor, raising the
// reference's exception types (Errors/Logic.h:13-59) on failure.
//
// The functions take btm_tensor_view, a POD mirror of the Tensor fields the path reads
// (Tensor/Tensor.h:173-201). Inside the reference tree a maintainer fills it from a Tensor in a
// friend function and defines BT_HAVE_REFERENCE_ERRORS so that the
// exception types come from Errors/Logic.h instead of the stand-ins below.
#pragma once
#include <cstdint>
#include <new>
#include <stdexcept>
#include <string>

#include "../../include/btm.h"

#if defined(BT_HAVE_REFERENCE_ERRORS)
#include "Errors/Logic.h"
#else
namespace BeanTensor::ErrorHandling {
class NotImplemented : public std::logic_error {
public:
    NotImplemented() : std::logic_error("Function not yet implemented") {}
};
class OutOfMemory : public std::bad_alloc {
public:
    OutOfMemory() = default;
};
} // namespace BeanTensor::ErrorHandling
#endif

namespace BeanTensor::Tensors::detail {

// Status -> exception, the inverse of what a C ABI has to do to the reference's throw sites.
inline void btm_raise(int status)
{
    if (status == BTM_OK) return;
    const std::string msg = btm_last_error_string();
    switch (status) {
    case BTM_ERR_INVALID: throw std::invalid_argument(msg);                       // Tensor/TensorOps.cu:241,269
    case BTM_ERR_UNSUPPORTED: throw BeanTensor::ErrorHandling::NotImplemented();  // Errors/Logic.h:13-17
    case BTM_ERR_OOM: throw BeanTensor::ErrorHandling::OutOfMemory();             // Errors/Logic.h:22-25
    default: throw std::runtime_error(msg);                                       // "CUDA Error: ..." Errors/Logic.h:50-59
    }
}

inline void btm_require_gpu_rowmajor(const btm_tensor_view &t, int ndim, const char *name)
{
    if (t.device != 1) throw std::invalid_argument(std::string(name) + ": Tensor is not on the GPU"); // guard of TensorOps.cu:89-93
    if (t.ndim != ndim) throw std::invalid_argument(std::string(name) + ": wrong rank");
    if (t.shape[ndim - 1] > 1 && t.strides[ndim - 1] != 1)
        throw std::invalid_argument(std::string(name) + ": last dimension must be contiguous (row-major, Tensor.cpp:157-162)");
}

inline const void *btm_base(const btm_tensor_view &t)
{
    return static_cast<const char *>(t.data) + t.offset * btm_dtype_size(t.dtype);
}

// out[M,N] = act(a[M,K] . b[K,N] + bias[N]). Float16/BFloat16 (fp32 accumulate) or Float32 (3xTF32).
// `bias` may be null (none); `relu` applies max(x, 0) after the bias. The product, the reference's broadcast Add
// (Ops/Elementwise/Add/Add.h:28) and its Relu stub (Ops/Elementwise/Relu/Relu.h) in one kernel: out is written once.
inline void matmul_bias_act_gpu(const btm_tensor_view &a, const btm_tensor_view &b, const btm_tensor_view *bias, bool relu,
                                btm_tensor_view &out, void *stream = nullptr)
{
    btm_require_gpu_rowmajor(a, 2, "matmul_gpu(a)");
    btm_require_gpu_rowmajor(b, 2, "matmul_gpu(b)");
    btm_require_gpu_rowmajor(out, 2, "matmul_gpu(out)");
    if (a.dtype != b.dtype || a.dtype != out.dtype) throw std::invalid_argument("matmul_gpu: dtypes differ");
    if (a.gpu_id != b.gpu_id || a.gpu_id != out.gpu_id) throw std::invalid_argument("matmul_gpu: tensors live on different GPUs");
    if (a.shape[1] != b.shape[0] || out.shape[0] != a.shape[0] || out.shape[1] != b.shape[1])
        throw std::invalid_argument("matmul_gpu: shape mismatch");
    if (bias) {
        btm_require_gpu_rowmajor(*bias, 1, "matmul_gpu(bias)");
        if (bias->dtype != out.dtype || bias->gpu_id != out.gpu_id || bias->shape[0] != out.shape[1])
            throw std::invalid_argument("matmul_gpu: bias must be a [N] tensor of the output's dtype on the output's GPU");
    }
    const int M = (int)a.shape[0], K = (int)a.shape[1], N = (int)b.shape[1];
    const int64_t lda = M > 1 ? (int64_t)a.strides[0] : (K > 0 ? K : 1);
    const int64_t ldb = K > 1 ? (int64_t)b.strides[0] : (N > 0 ? N : 1);
    const int64_t ldc = M > 1 ? (int64_t)out.strides[0] : (N > 0 ? N : 1);
    btm_raise(btm_gemm_bias_act(a.gpu_id, stream, a.dtype, M, N, K, btm_base(a), lda, btm_base(b), ldb, bias ? btm_base(*bias) : nullptr,
                                relu ? BTM_ACT_RELU : BTM_ACT_NONE, const_cast<void *>(btm_base(out)), ldc));
}

// Operands may be any 2-D view (Tensor::strides, Tensor/Tensor.h:173-195): row-major, transposed or strided.
inline void btm_require_gpu_2d(const btm_tensor_view &t, const char *name)
{
    if (t.device != 1) throw std::invalid_argument(std::string(name) + ": Tensor is not on the GPU"); // guard of TensorOps.cu:89-93
    if (t.ndim != 2) throw std::invalid_argument(std::string(name) + ": wrong rank");
}

// out[M,N] = a[M,K] . b[K,N]. Float16/BFloat16 (fp32 accumulate) or Float32 (3xTF32). a and b may be transposed or
// strided views (no copy is made); out is row-major.
inline void matmul_gpu(const btm_tensor_view &a, const btm_tensor_view &b, btm_tensor_view &out, void *stream = nullptr)
{
    btm_require_gpu_2d(a, "matmul_gpu(a)");
    btm_require_gpu_2d(b, "matmul_gpu(b)");
    btm_require_gpu_rowmajor(out, 2, "matmul_gpu(out)");
    if (a.dtype != b.dtype || a.dtype != out.dtype) throw std::invalid_argument("matmul_gpu: dtypes differ");
    if (a.gpu_id != b.gpu_id || a.gpu_id != out.gpu_id) throw std::invalid_argument("matmul_gpu: tensors live on different GPUs");
    if (a.shape[1] != b.shape[0] || out.shape[0] != a.shape[0] || out.shape[1] != b.shape[1])
        throw std::invalid_argument("matmul_gpu: shape mismatch");
    const int M = (int)a.shape[0], K = (int)a.shape[1], N = (int)b.shape[1];
    const int64_t ldc = M > 1 ? (int64_t)out.strides[0] : (N > 0 ? N : 1);
    btm_raise(btm_gemm_strided(a.gpu_id, stream, a.dtype, M, N, K, btm_base(a), (int64_t)a.strides[0], (int64_t)a.strides[1], btm_base(b),
                               (int64_t)b.strides[0], (int64_t)b.strides[1], const_cast<void *>(btm_base(out)), ldc));
}

// out[b] = a[b] . b[b]; dense row-major matrices with a batch stride.
inline void bmm_gpu(const btm_tensor_view &a, const btm_tensor_view &b, btm_tensor_view &out, void *stream = nullptr)
{
    btm_require_gpu_rowmajor(a, 3, "bmm_gpu(a)");
    btm_require_gpu_rowmajor(b, 3, "bmm_gpu(b)");
    btm_require_gpu_rowmajor(out, 3, "bmm_gpu(out)");
    if (a.dtype != b.dtype || a.dtype != out.dtype) throw std::invalid_argument("bmm_gpu: dtypes differ");
    if (a.shape[0] != b.shape[0] || a.shape[0] != out.shape[0] || a.shape[2] != b.shape[1] || out.shape[1] != a.shape[1] ||
        out.shape[2] != b.shape[2])
        throw std::invalid_argument("bmm_gpu: shape mismatch");
    const int B = (int)a.shape[0], M = (int)a.shape[1], K = (int)a.shape[2], N = (int)b.shape[2];
    if ((M > 1 && a.strides[1] != (uint64_t)K) || (K > 1 && b.strides[1] != (uint64_t)N) || (M > 1 && out.strides[1] != (uint64_t)N))
        throw std::invalid_argument("bmm_gpu: each matrix must be dense row-major");
    btm_raise(btm_bmm(a.gpu_id, stream, a.dtype, B, M, N, K, btm_base(a), (int64_t)a.strides[0], btm_base(b), (int64_t)b.strides[0],
                      const_cast<void *>(btm_base(out)), (int64_t)out.strides[0]));
}

// out[M,N] (Float16) = act[M,K] (Float16) . dequant(w_packed[N,K/2], scales[N,K/group])^T
inline void matmul_int4_gpu(const btm_tensor_view &act, const btm_tensor_view &w_packed, const btm_tensor_view &scales,
                            btm_tensor_view &out, uint32_t group = 128, void *stream = nullptr)
{
    btm_require_gpu_rowmajor(act, 2, "matmul_int4_gpu(act)");
    btm_require_gpu_rowmajor(w_packed, 2, "matmul_int4_gpu(w)");
    btm_require_gpu_rowmajor(scales, 2, "matmul_int4_gpu(scales)");
    btm_require_gpu_rowmajor(out, 2, "matmul_int4_gpu(out)");
    if (act.dtype != BTM_F16 || scales.dtype != BTM_F16 || out.dtype != BTM_F16 || w_packed.dtype != BTM_INT4X2)
        throw std::invalid_argument("matmul_int4_gpu: expected Float16 activations/scales/output and packed int4 weights");
    const int M = (int)act.shape[0], K = (int)act.shape[1], N = (int)w_packed.shape[0];
    if (group == 0 || w_packed.shape[1] * 2 != (uint64_t)K || scales.shape[0] != (uint64_t)N || scales.shape[1] * group != (uint64_t)K ||
        out.shape[0] != (uint64_t)M || out.shape[1] != (uint64_t)N)
        throw std::invalid_argument("matmul_int4_gpu: shape mismatch");
    btm_raise(btm_int4_matmul(act.gpu_id, stream, M, N, K, (int)group, btm_base(act), btm_base(w_packed), btm_base(scales),
                              const_cast<void *>(btm_base(out))));
}

// A dimension as the C ABI takes it.
inline int btm_dim(uint64_t n)
{
    if (n > 0x7FFFFFFFull) throw std::invalid_argument("dimension does not fit 32 bits");
    return static_cast<int>(n);
}

// Row offsets of the groups: a rank-1 Int32 tensor of groups + 1 entries on the operands' GPU.
inline const int32_t *btm_group_offsets(const btm_tensor_view &offsets, uint64_t groups, int32_t gpu_id, const char *name)
{
    btm_require_gpu_rowmajor(offsets, 1, name);
    if (offsets.dtype != BTM_I32 || offsets.shape[0] != groups + 1 || offsets.gpu_id != gpu_id)
        throw std::invalid_argument(std::string(name) + ": offsets must be an Int32 tensor of groups + 1 entries on the operands' GPU");
    return static_cast<const int32_t *>(btm_base(offsets));
}

inline int64_t btm_pitch(const btm_tensor_view &t) // leading dimension of the last two dimensions; a single row has none of its own
{
    const uint64_t rows = t.shape[t.ndim - 2], cols = t.shape[t.ndim - 1];
    return rows > 1 ? (int64_t)t.strides[t.ndim - 2] : (int64_t)(cols > 0 ? cols : 1);
}

// out[r,:] = a[r,:] . b[g] for the rows r of group g (offsets[g] <= r < offsets[g+1]); a [rows,K], b [groups,K,N], out [rows,N],
// Float16/BFloat16. Each matrix of b may be transposed (b [groups,K,N] with unit stride along K): with the output gradient as
// a this is the gradient of the activations. Rows outside the groups keep what out held.
inline void grouped_matmul_gpu(const btm_tensor_view &a, const btm_tensor_view &b, const btm_tensor_view &offsets, btm_tensor_view &out,
                               void *stream = nullptr)
{
    btm_require_gpu_rowmajor(a, 2, "grouped_matmul_gpu(a)");
    btm_require_gpu_rowmajor(out, 2, "grouped_matmul_gpu(out)");
    if (b.device != 1) throw std::invalid_argument("grouped_matmul_gpu(b): Tensor is not on the GPU");
    if (b.ndim != 3) throw std::invalid_argument("grouped_matmul_gpu(b): wrong rank");
    if (a.dtype != b.dtype || a.dtype != out.dtype) throw std::invalid_argument("grouped_matmul_gpu: dtypes differ");
    if (a.gpu_id != b.gpu_id || a.gpu_id != out.gpu_id) throw std::invalid_argument("grouped_matmul_gpu: tensors live on different GPUs");
    if (a.shape[1] != b.shape[1] || out.shape[0] != a.shape[0] || out.shape[1] != b.shape[2])
        throw std::invalid_argument("grouped_matmul_gpu: shape mismatch");
    const int32_t *offs = btm_group_offsets(offsets, b.shape[0], a.gpu_id, "grouped_matmul_gpu(offsets)");
    const uint64_t K = b.shape[1], N = b.shape[2];
    const bool trans = N > 1 && b.strides[2] != 1;
    if (trans && K > 1 && b.strides[1] != 1) throw std::invalid_argument("grouped_matmul_gpu(b): each matrix must be row-major or transposed row-major");
    const int64_t ldb = trans ? (int64_t)b.strides[2] : (K > 1 ? (int64_t)b.strides[1] : (int64_t)(N > 0 ? N : 1));
    const int64_t sb = b.shape[0] > 1 ? (int64_t)b.strides[0] : ldb * (int64_t)(trans ? N : K);
    btm_raise(btm_gemm_grouped(a.gpu_id, stream, a.dtype, btm_dim(b.shape[0]), btm_dim(a.shape[0]), btm_dim(N), btm_dim(K), offs, btm_base(a), btm_pitch(a), btm_base(b),
                               sb, ldb, trans ? 1 : 0, const_cast<void *>(btm_base(out)), btm_pitch(out)));
}

// The weight gradient of the above: out[g] = a[rows of g]^T . dout[rows of g]; a [rows,K], dout [rows,N], out [groups,K,N].
inline void grouped_matmul_wgrad_gpu(const btm_tensor_view &a, const btm_tensor_view &dout, const btm_tensor_view &offsets, btm_tensor_view &out,
                                     void *stream = nullptr)
{
    btm_require_gpu_rowmajor(a, 2, "grouped_matmul_wgrad_gpu(a)");
    btm_require_gpu_rowmajor(dout, 2, "grouped_matmul_wgrad_gpu(dout)");
    btm_require_gpu_rowmajor(out, 3, "grouped_matmul_wgrad_gpu(out)");
    if (a.dtype != dout.dtype || a.dtype != out.dtype) throw std::invalid_argument("grouped_matmul_wgrad_gpu: dtypes differ");
    if (a.gpu_id != dout.gpu_id || a.gpu_id != out.gpu_id) throw std::invalid_argument("grouped_matmul_wgrad_gpu: tensors live on different GPUs");
    if (a.shape[0] != dout.shape[0] || out.shape[1] != a.shape[1] || out.shape[2] != dout.shape[1])
        throw std::invalid_argument("grouped_matmul_wgrad_gpu: shape mismatch");
    const int32_t *offs = btm_group_offsets(offsets, out.shape[0], a.gpu_id, "grouped_matmul_wgrad_gpu(offsets)");
    const int64_t ldc = btm_pitch(out);
    const int64_t sc = out.shape[0] > 1 ? (int64_t)out.strides[0] : ldc * (int64_t)out.shape[1];
    btm_raise(btm_gemm_grouped_wgrad(a.gpu_id, stream, a.dtype, btm_dim(out.shape[0]), btm_dim(a.shape[0]), btm_dim(out.shape[1]), btm_dim(out.shape[2]), offs, btm_base(a),
                                     btm_pitch(a), btm_base(dout), btm_pitch(dout), const_cast<void *>(btm_base(out)), sc, ldc));
}

// A microscaled operand: packed [.., K/2] UInt8, dense, and its scale blocks, a rank-1 UInt8 tensor of at least `bytes`.
inline void btm_require_mxfp4(const btm_tensor_view &packed, const btm_tensor_view &scales, int ndim, uint64_t bytes, const char *name)
{
    btm_require_gpu_rowmajor(packed, ndim, name);
    btm_require_gpu_rowmajor(scales, 1, name);
    if (packed.dtype != BTM_U8 || scales.dtype != BTM_U8) throw std::invalid_argument(std::string(name) + ": packed values and scales are UInt8");
    if (scales.shape[0] < bytes) throw std::invalid_argument(std::string(name) + ": too few scale bytes");
    uint64_t stride = 1;
    for (int i = ndim - 1; i >= 0; --i) {
        if (packed.shape[i] > 1 && packed.strides[i] != stride) throw std::invalid_argument(std::string(name) + ": packed values must be contiguous");
        stride *= packed.shape[i];
    }
    if (packed.gpu_id != scales.gpu_id) throw std::invalid_argument(std::string(name) + ": tensors live on different GPUs");
}

// The plain side t of a conversion to or from microscaled values beside its packed side: [rows,K], one group or ragged ones by
// offsets, or the matrices of all experts [groups,N,K], which are dense and have no offsets.
struct btm_mxfp4_rows {
    int groups, rows, K;
    int64_t ld;
    const int32_t *offsets;
};
inline btm_mxfp4_rows btm_require_mxfp4_conversion(const btm_tensor_view &t, const btm_tensor_view &packed, const btm_tensor_view &scales,
                                                   const btm_tensor_view *offsets, const std::string &name)
{
    const int nd = t.ndim == 3 ? 3 : 2;
    btm_require_gpu_rowmajor(t, nd, name.c_str());
    if (offsets && nd == 3) throw std::invalid_argument(name + ": offsets go with rank-2 tensors; the groups of a rank-3 one are its first dimension");
    if (offsets && (offsets->ndim != 1 || offsets->shape[0] == 0)) throw std::invalid_argument(name + ": offsets must be an Int32 tensor of groups + 1 entries");
    btm_mxfp4_rows r;
    r.K = btm_dim(t.shape[nd - 1]);
    uint64_t bytes;
    if (nd == 3) {
        r.groups = btm_dim(t.shape[0]);
        const int N = btm_dim(t.shape[1]);
        r.rows = btm_dim((uint64_t)r.groups * (uint64_t)N);
        r.ld = r.K;
        if ((N > 1 && t.strides[1] != (uint64_t)r.K) || (r.groups > 1 && t.strides[0] != (uint64_t)N * (uint64_t)r.K))
            throw std::invalid_argument(name + ": a rank-3 tensor must be contiguous");
        bytes = (uint64_t)r.groups * btm_mxfp4_scale_bytes(1, N, r.K);
    } else {
        r.groups = offsets ? btm_dim(offsets->shape[0]) - 1 : 1;
        r.rows = btm_dim(t.shape[0]);
        r.ld = btm_pitch(t);
        bytes = btm_mxfp4_scale_bytes(r.groups, r.rows, r.K);
    }
    btm_require_mxfp4(packed, scales, nd, bytes, (name + "(packed)").c_str());
    bool fits = packed.gpu_id == t.gpu_id && packed.shape[nd - 1] * 2 == t.shape[nd - 1];
    for (int i = 0; i < nd - 1; ++i) fits = fits && packed.shape[i] == t.shape[i];
    if (!fits) throw std::invalid_argument(name + ": shape mismatch");
    r.offsets = offsets ? btm_group_offsets(*offsets, (uint64_t)r.groups, t.gpu_id, (name + "(offsets)").c_str()) : nullptr;
    return r;
}

// x [rows,K] (Float32/Float16/BFloat16) -> packed [rows,K/2] and scales; with offsets the scales are laid out for those groups.
// x [groups,N,K] -> packed [groups,N,K/2] and the scales of one group after the other: the weights of all experts in one call.
inline void quantize_mxfp4_gpu(const btm_tensor_view &x, btm_tensor_view &packed, btm_tensor_view &scales, const btm_tensor_view *offsets = nullptr,
                               void *stream = nullptr)
{
    const btm_mxfp4_rows r = btm_require_mxfp4_conversion(x, packed, scales, offsets, "quantize_mxfp4_gpu");
    btm_raise(btm_mxfp4_quantize(x.gpu_id, stream, x.dtype, r.groups, r.rows, r.K, r.offsets, btm_base(x), r.ld, const_cast<void *>(btm_base(packed)),
                                 const_cast<void *>(btm_base(scales))));
}

// The inverse: out = the values that packed and scales stand for, rounded once to out's dtype; shapes as above.
inline void dequant_mxfp4_gpu(const btm_tensor_view &packed, const btm_tensor_view &scales, btm_tensor_view &out, const btm_tensor_view *offsets = nullptr,
                              void *stream = nullptr)
{
    const btm_mxfp4_rows r = btm_require_mxfp4_conversion(out, packed, scales, offsets, "dequant_mxfp4_gpu");
    btm_raise(btm_mxfp4_dequant(out.gpu_id, stream, out.dtype, r.groups, r.rows, r.K, r.offsets, btm_base(packed), btm_base(scales),
                                const_cast<void *>(btm_base(out)), r.ld));
}

// out[M,N] (Float16/BFloat16) = act[M,K] . w[N,K]^T of microscaled operands.
inline void matmul_mxfp4_gpu(const btm_tensor_view &act, const btm_tensor_view &act_scales, const btm_tensor_view &w, const btm_tensor_view &w_scales,
                             btm_tensor_view &out, void *stream = nullptr)
{
    btm_require_gpu_rowmajor(act, 2, "matmul_mxfp4_gpu(act)");
    btm_require_gpu_rowmajor(w, 2, "matmul_mxfp4_gpu(w)");
    btm_require_gpu_rowmajor(out, 2, "matmul_mxfp4_gpu(out)");
    const int M = btm_dim(act.shape[0]), N = btm_dim(w.shape[0]), K = btm_dim(act.shape[1] * 2);
    btm_require_mxfp4(act, act_scales, 2, btm_mxfp4_scale_bytes(1, M, K), "matmul_mxfp4_gpu(act)");
    btm_require_mxfp4(w, w_scales, 2, btm_mxfp4_scale_bytes(1, N, K), "matmul_mxfp4_gpu(w)");
    if (w.shape[1] != act.shape[1] || out.shape[0] != act.shape[0] || out.shape[1] != w.shape[0])
        throw std::invalid_argument("matmul_mxfp4_gpu: shape mismatch");
    if (act.gpu_id != w.gpu_id || act.gpu_id != out.gpu_id) throw std::invalid_argument("matmul_mxfp4_gpu: tensors live on different GPUs");
    btm_raise(btm_mxfp4_matmul(act.gpu_id, stream, out.dtype, M, N, K, btm_base(act), btm_base(act_scales), btm_base(w), btm_base(w_scales),
                               const_cast<void *>(btm_base(out)), btm_pitch(out)));
}

// out[r,:] = act[r,:] . w[g]^T for the rows r of group g; act [rows,K/2] quantised with these offsets, w [groups,N,K/2].
inline void grouped_matmul_mxfp4_gpu(const btm_tensor_view &act, const btm_tensor_view &act_scales, const btm_tensor_view &w,
                                     const btm_tensor_view &w_scales, const btm_tensor_view &offsets, btm_tensor_view &out, void *stream = nullptr)
{
    btm_require_gpu_rowmajor(act, 2, "grouped_matmul_mxfp4_gpu(act)");
    btm_require_gpu_rowmajor(w, 3, "grouped_matmul_mxfp4_gpu(w)");
    btm_require_gpu_rowmajor(out, 2, "grouped_matmul_mxfp4_gpu(out)");
    const int groups = btm_dim(w.shape[0]), rows = btm_dim(act.shape[0]), N = btm_dim(w.shape[1]), K = btm_dim(act.shape[1] * 2);
    btm_require_mxfp4(act, act_scales, 2, btm_mxfp4_scale_bytes(groups, rows, K), "grouped_matmul_mxfp4_gpu(act)");
    btm_require_mxfp4(w, w_scales, 3, (uint64_t)groups * btm_mxfp4_scale_bytes(1, N, K), "grouped_matmul_mxfp4_gpu(w)");
    if (w.shape[2] != act.shape[1] || out.shape[0] != act.shape[0] || out.shape[1] != w.shape[1])
        throw std::invalid_argument("grouped_matmul_mxfp4_gpu: shape mismatch");
    if (act.gpu_id != w.gpu_id || act.gpu_id != out.gpu_id) throw std::invalid_argument("grouped_matmul_mxfp4_gpu: tensors live on different GPUs");
    const int32_t *offs = btm_group_offsets(offsets, (uint64_t)groups, act.gpu_id, "grouped_matmul_mxfp4_gpu(offsets)");
    btm_raise(btm_mxfp4_matmul_grouped(act.gpu_id, stream, out.dtype, groups, rows, N, K, offs, btm_base(act), btm_base(act_scales), btm_base(w),
                                       btm_base(w_scales), const_cast<void *>(btm_base(out)), btm_pitch(out)));
}

} // namespace BeanTensor::Tensors::detail
