"""Host-side mirror of the reference's GPU operator boundary for the matmul path.

The reference declares its GPU operators as free functions `detail::*_gpu(Tensor&, ...)`
(Tensor/TensorOps.h:15-65) that check the device, then enqueue work and leave the result in a
pre-allocated tensor. The functions here have the names and argument meaning a
`matmul_gpu` / `bmm_gpu` / `matmul_int4_gpu` family added beside them would have; torch
tensors stand in for BeanTensor's Tensor (torch is used for device memory and streams only —
every product is computed by libbtm.so).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .errors import GPUTaskOnCPUBuild, raise_for_status

_DT = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}


# A call into the library makes its device current on the calling thread; the functions here put back the one that was. With one
# GPU there is nothing to put back, and looking it up takes 0.2 us of a call's 6.5: the first call counts them.
_ONE_GPU = _counted = False
_set_device = torch._C._cuda_setDevice


def _current_device() -> int:
    global _ONE_GPU, _counted
    if not _counted:
        _counted, _ONE_GPU = True, torch.cuda.device_count() == 1
    return torch._C._cuda_getDevice()


def _LIB():
    return _lib._lib or _lib.lib()


def _require_gpu(*tensors: torch.Tensor) -> int:
    if not torch.cuda.is_available():
        raise GPUTaskOnCPUBuild("GPU task cannot be run on CPU build")  # TensorOps.hpp:5-30
    dev = None
    for t in tensors:
        if t.device.type != "cuda":
            raise ValueError("Tensor is not on the GPU")  # guard of Tensor/TensorOps.cu:89-93
        if dev is None:
            dev = t.device.index
        elif t.device.index != dev:
            raise ValueError("Tensors live on different GPUs")
    return int(dev)


def _stream(dev: int | None = None) -> int:
    """The calling thread's current CUDA stream of `dev` as a raw handle (what the C ABI takes as void*)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if dev is None else dev)


def _rowmajor(t: torch.Tensor, name: str) -> None:
    if t.stride(-1) != 1 and t.size(-1) > 1:
        raise ValueError(f"{name} must be row-major (last stride 1)")  # Tensor/Tensor.cpp:157-162


def init(device: int = 0) -> None:
    raise_for_status(_lib.lib().btm_init(device))


def check_device_status(device: int = 0) -> None:
    cur = device if _ONE_GPU else _current_device()
    rc = _lib.lib().btm_check_device_status(device, _stream(device))
    if cur != device:
        _set_device(cur)
    raise_for_status(rc)


def matmul_gpu(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor, bias: torch.Tensor | None = None,
               relu: bool = False) -> None:
    """out[M,N] = a[M,K] . b[K,N]; fp16/bf16 (fp32 accumulate) or fp32 (3xTF32).

    With `bias` ([N], dtype of out) and/or `relu` the epilogue is fused: out = relu(a.b + bias), rounded once.
    """
    dev = _require_gpu(a, b, out)
    if bias is not None:
        if not bias.is_cuda or bias.device != out.device:
            raise ValueError("matmul_gpu: bias is not on the output's GPU")
        if bias.dim() != 1 or bias.shape[0] != out.shape[-1] or bias.dtype != out.dtype or not bias.is_contiguous():
            raise ValueError("matmul_gpu: bias must be a contiguous [N] tensor of the output's dtype")
    if a.dim() != 2 or b.dim() != 2 or out.dim() != 2:
        raise ValueError("matmul_gpu takes 2-D tensors")
    if a.dtype != b.dtype or a.dtype != out.dtype:
        raise ValueError("matmul_gpu: dtypes differ")
    if a.dtype not in _DT:
        from .errors import NotImplementedOp
        raise NotImplementedOp(f"matmul_gpu: dtype {a.dtype} is not supported")
    M, K = a.shape
    K2, N = b.shape
    if K != K2 or out.shape != (M, N):
        raise ValueError(f"matmul_gpu: shape mismatch {tuple(a.shape)} x {tuple(b.shape)} -> {tuple(out.shape)}")
    _rowmajor(out, "out")
    ldc = out.stride(0) if M > 1 else max(N, 1)
    a_row = a.stride(1) == 1 or K <= 1
    b_row = b.stride(1) == 1 or N <= 1
    if not (a_row and b_row):
        # Transposed or strided views (Tensor::strides, Tensor/Tensor.h:173-195) go through without a copy.
        if bias is not None or relu:
            raise ValueError("matmul_gpu: the fused epilogue takes row-major operands")
        cur = dev if _ONE_GPU else _current_device()
        rc = _LIB().btm_gemm_strided(dev, _stream(dev), _DT[a.dtype], M, N, K, a.data_ptr(), a.stride(0), a.stride(1),
                                     b.data_ptr(), b.stride(0), b.stride(1), out.data_ptr(), ldc)
        if cur != dev:
            _set_device(cur)
        raise_for_status(rc)
        return
    lda = a.stride(0) if M > 1 else max(K, 1)
    ldb = b.stride(0) if K > 1 else max(N, 1)
    cur = dev if _ONE_GPU else _current_device()
    if bias is None and not relu:
        rc = _lib.lib().btm_gemm(dev, _stream(dev), _DT[a.dtype], M, N, K, a.data_ptr(), lda, b.data_ptr(), ldb,
                                 out.data_ptr(), ldc)
    else:
        rc = _lib.lib().btm_gemm_bias_act(dev, _stream(dev), _DT[a.dtype], M, N, K, a.data_ptr(), lda, b.data_ptr(), ldb,
                                          bias.data_ptr() if bias is not None else None, 1 if relu else 0,
                                          out.data_ptr(), ldc)
    if cur != dev:
        _set_device(cur)
    raise_for_status(rc)


def bmm_gpu(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor) -> None:
    """out[b] = a[b] . b[b] for dense row-major 3-D tensors (fp16/bf16)."""
    dev = _require_gpu(a, b, out)
    if a.dim() != 3 or b.dim() != 3 or out.dim() != 3:
        raise ValueError("bmm_gpu takes 3-D tensors")
    if a.dtype != b.dtype or a.dtype != out.dtype:
        raise ValueError("bmm_gpu: dtypes differ")
    if a.dtype not in (torch.float16, torch.bfloat16):
        from .errors import NotImplementedOp
        raise NotImplementedOp(f"bmm_gpu: dtype {a.dtype} is not supported")
    B, M, K = a.shape
    B2, K2, N = b.shape
    if B != B2 or K != K2 or out.shape != (B, M, N):
        raise ValueError("bmm_gpu: shape mismatch")
    for t in (a, b, out):
        if not t[0].is_contiguous() if B > 0 else False:
            raise ValueError("bmm_gpu: each matrix must be dense row-major")
    sa = a.stride(0) if B > 1 else M * K
    sb = b.stride(0) if B > 1 else K * N
    sc = out.stride(0) if B > 1 else M * N
    cur = dev if _ONE_GPU else _current_device()
    rc = _lib.lib().btm_bmm(dev, _stream(dev), _DT[a.dtype], B, M, N, K, a.data_ptr(), sa, b.data_ptr(), sb,
                            out.data_ptr(), sc)
    if cur != dev:
        _set_device(cur)
    raise_for_status(rc)


def matmul_int4_gpu(act: torch.Tensor, w_packed: torch.Tensor, scales: torch.Tensor, out: torch.Tensor,
                    group: int = 128) -> None:
    """out[M,N] (fp16) = act[M,K] (fp16) . dequant(w_packed[N,K/2], scales[N,K/group])^T."""
    # One pass over the operands: this call sits in front of a kernel of a few microseconds (a decoder calls it once
    # per layer and token), so the guards are written to cost little. Same checks as the other operators.
    dev = out.device.index
    f16 = torch.float16
    if not (act.is_cuda and w_packed.is_cuda and scales.is_cuda and out.is_cuda):
        _require_gpu(act, w_packed, scales, out)  # raises with the operator boundary's messages
    if act.device != out.device or w_packed.device != out.device or scales.device != out.device:
        raise ValueError("Tensors live on different GPUs")
    if act.dtype != f16 or scales.dtype != f16 or out.dtype != f16:
        raise ValueError("matmul_int4_gpu: activations, scales and output are Float16")
    if w_packed.dtype != torch.uint8:
        raise ValueError("matmul_int4_gpu: packed weights are bytes (two nibbles each)")
    M, K = act.shape
    N = w_packed.shape[0]
    if w_packed.shape != (N, K // 2) or scales.shape != (N, K // group if group else 0) or out.shape != (M, N):
        raise ValueError("matmul_int4_gpu: shape mismatch")
    if not (act.is_contiguous() and w_packed.is_contiguous() and scales.is_contiguous() and out.is_contiguous()):
        raise ValueError("matmul_int4_gpu: tensors must be contiguous")
    cur = dev if _ONE_GPU else _current_device()
    rc = _LIB().btm_int4_matmul(dev, torch._C._cuda_getCurrentRawStream(dev), M, N, K, group, act.data_ptr(), w_packed.data_ptr(),
                                scales.data_ptr(), out.data_ptr())
    if cur != dev:
        _set_device(cur)
    if rc:
        raise_for_status(rc)


def dequant_int4_gpu(w_packed: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, group: int = 128) -> None:
    dev = _require_gpu(w_packed, scales, out)
    N, K2 = w_packed.shape
    K = K2 * 2
    if out.shape != (N, K) or out.dtype != torch.float16 or scales.dtype != torch.float16:
        raise ValueError("dequant_int4_gpu: shape or dtype mismatch")
    cur = dev if _ONE_GPU else _current_device()
    rc = _lib.lib().btm_int4_dequant(dev, _stream(dev), N, K, group, w_packed.data_ptr(), scales.data_ptr(), out.data_ptr())
    if cur != dev:
        _set_device(cur)
    raise_for_status(rc)


def unpack_int4_gpu(w_packed: torch.Tensor, out: torch.Tensor) -> None:
    dev = _require_gpu(w_packed, out)
    N, K2 = w_packed.shape
    if out.shape != (N, K2 * 2) or out.dtype != torch.int8:
        raise ValueError("unpack_int4_gpu: shape or dtype mismatch")
    cur = dev if _ONE_GPU else _current_device()
    rc = _lib.lib().btm_int4_unpack(dev, _stream(dev), N, K2 * 2, w_packed.data_ptr(), out.data_ptr())
    if cur != dev:
        _set_device(cur)
    raise_for_status(rc)


def quantize_int4_gpu(w: torch.Tensor, w_packed: torch.Tensor, scales: torch.Tensor, group: int = 128) -> None:
    """fp16 weights [N,K] -> packed nibbles [N,K/2] + fp16 scales [N,K/group] (max-abs / 7 per group)."""
    dev = _require_gpu(w, w_packed, scales)
    N, K = w.shape
    if w.dtype != torch.float16 or scales.dtype != torch.float16 or w_packed.dtype != torch.uint8:
        raise ValueError("quantize_int4_gpu: Float16 weights and scales, byte output")
    if group <= 0 or K % group or w_packed.shape != (N, K // 2) or scales.shape != (N, K // group):
        raise ValueError("quantize_int4_gpu: shape mismatch")
    for t in (w, w_packed, scales):
        if not t.is_contiguous():
            raise ValueError("quantize_int4_gpu: tensors must be contiguous")
    cur = dev if _ONE_GPU else _current_device()
    rc = _lib.lib().btm_int4_quantize(dev, _stream(dev), N, K, group, w.data_ptr(), w_packed.data_ptr(), scales.data_ptr())
    if cur != dev:
        _set_device(cur)
    raise_for_status(rc)


# The grouped and microscaled operators sit in front of kernels of a few microseconds: their guards look at each tensor once
# and cost little; whatever fails goes through the slower functions that find out why and raise.
_U8, _I32 = torch.uint8, torch.int32
_DT16 = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_raw_stream = torch._C._cuda_getCurrentRawStream


def _same_gpu(*tensors: torch.Tensor) -> None:
    """Raises with the operator boundary's messages; called when the tensors are not all on one GPU."""
    _require_gpu(*tensors)
    raise ValueError("Tensors live on different GPUs")


def _not_supported(what: str, dtype) -> None:
    from .errors import NotImplementedOp
    raise NotImplementedOp(f"{what}: dtype {dtype} is not supported")


def _bad_offsets(what: str) -> None:
    raise ValueError(f"{what}: offsets must be a contiguous Int32 tensor of groups + 1 entries")


def _too_large(what: str) -> None:
    from .errors import NotImplementedOp
    raise NotImplementedOp(f"{what}: dimensions must fit 32 bits")


def _row_pitch(t: torch.Tensor, rows: int, cols: int, name: str) -> int:
    """Leading dimension of a row-major matrix, the last two dimensions of t; a single row has none of its own."""
    st = t.stride()
    if cols > 1 and st[-1] != 1:
        raise ValueError(f"{name} must be row-major (last stride 1)")  # Tensor/Tensor.cpp:157-162
    return st[-2] if rows > 1 else (cols or 1)


def grouped_matmul_gpu(a: torch.Tensor, b: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor) -> None:
    """out[r] = a[r] . b[g] for the rows r of group g: offsets[g] <= r < offsets[g+1] (Int32, on the GPU).

    a [rows,K], b [groups,K,N], out [rows,N], fp16/bf16 with fp32 accumulation. b may be a transposed view: with
    b.transpose(1, 2) and the output gradient as `a` this is the gradient of the activations. Rows outside the groups
    keep what `out` held.
    """
    dev = out.get_device()
    if dev < 0 or a.get_device() != dev or b.get_device() != dev or offsets.get_device() != dev:
        _same_gpu(a, b, offsets, out)
    sa, sb = a.shape, b.shape
    if len(sa) != 2 or len(sb) != 3 or out.dim() != 2:
        raise ValueError("grouped_matmul_gpu takes a 2-D, b 3-D and out 2-D")
    dtype = a.dtype
    if b.dtype != dtype or out.dtype != dtype:
        raise ValueError("grouped_matmul_gpu: dtypes differ")
    dt = _DT16.get(dtype)
    if dt is None:
        _not_supported("grouped_matmul_gpu", dtype)
    rows, K = sa
    G, K2, N = sb
    if K != K2 or out.shape != (rows, N):
        raise ValueError(f"grouped_matmul_gpu: shape mismatch {tuple(sa)} x {tuple(sb)} -> {tuple(out.shape)}")
    if offsets.dtype != _I32 or offsets.shape != (G + 1,) or not offsets.is_contiguous():
        _bad_offsets("grouped_matmul_gpu")
    if (rows | N | K | G) >> 31:
        _too_large("grouped_matmul_gpu")
    lda, ldc = _row_pitch(a, rows, K, "a"), _row_pitch(out, rows, N, "out")
    bg, bk, bn = b.stride()
    trans = bn != 1 and N > 1
    if not trans:
        ldb, outer = (bk if K > 1 else N or 1), K
    elif bk == 1 or K <= 1:
        ldb, outer = (bn if N > 1 else K or 1), N
    else:
        raise ValueError("grouped_matmul_gpu: each matrix of b must be row-major or transposed row-major")
    cur = dev if _ONE_GPU else _current_device()
    rc = _LIB().btm_gemm_grouped(dev, _raw_stream(dev), dt, G, rows, N, K, offsets.data_ptr(), a.data_ptr(), lda, b.data_ptr(),
                                 bg if G > 1 else outer * ldb, ldb, 1 if trans else 0, out.data_ptr(), ldc)
    if cur != dev:
        _set_device(cur)
    if rc:
        raise_for_status(rc)


def grouped_matmul_wgrad_gpu(a: torch.Tensor, dout: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor) -> None:
    """The weight gradient of grouped_matmul_gpu: out[g] = a[rows of g]^T . dout[rows of g], zero for an empty group.

    a [rows,K], dout [rows,N], out [groups,K,N], fp16/bf16 with fp32 accumulation."""
    dev = out.get_device()
    if dev < 0 or a.get_device() != dev or dout.get_device() != dev or offsets.get_device() != dev:
        _same_gpu(a, dout, offsets, out)
    sa, sd = a.shape, dout.shape
    if len(sa) != 2 or len(sd) != 2 or out.dim() != 3:
        raise ValueError("grouped_matmul_wgrad_gpu takes a 2-D, dout 2-D and out 3-D")
    dtype = a.dtype
    if dout.dtype != dtype or out.dtype != dtype:
        raise ValueError("grouped_matmul_wgrad_gpu: dtypes differ")
    dt = _DT16.get(dtype)
    if dt is None:
        _not_supported("grouped_matmul_wgrad_gpu", dtype)
    rows, K = sa
    rows2, N = sd
    G, Ko, No = out.shape
    if rows != rows2 or Ko != K or No != N:
        raise ValueError(f"grouped_matmul_wgrad_gpu: shape mismatch {tuple(sa)} x {tuple(sd)} -> {tuple(out.shape)}")
    if offsets.dtype != _I32 or offsets.shape != (G + 1,) or not offsets.is_contiguous():
        _bad_offsets("grouped_matmul_wgrad_gpu")
    if (rows | N | K | G) >> 31:
        _too_large("grouped_matmul_wgrad_gpu")
    lda, ldd, ldc = _row_pitch(a, rows, K, "a"), _row_pitch(dout, rows, N, "dout"), _row_pitch(out, K, N, "out")
    cur = dev if _ONE_GPU else _current_device()
    rc = _LIB().btm_gemm_grouped_wgrad(dev, _raw_stream(dev), dt, G, rows, K, N, offsets.data_ptr(), a.data_ptr(), lda, dout.data_ptr(), ldd,
                                       out.data_ptr(), out.stride(0) if G > 1 else K * ldc, ldc)
    if cur != dev:
        _set_device(cur)
    if rc:
        raise_for_status(rc)


def mxfp4_scale_bytes(rows: int, K: int, groups: int = 1) -> int:
    """Bytes that hold the scales of `rows` microscaled rows of K values in `groups` groups, however the rows are divided
    (btm_mxfp4_scale_bytes)."""
    if rows <= 0 or K <= 0 or groups <= 0:
        return 0
    return (rows + 127 * (groups if groups < rows else rows)) // 128 * ((K + 127) // 128) * 512


def _bad_mxfp4(packed: torch.Tensor, scales: torch.Tensor, K: int, what: str, fits: bool = True) -> None:
    """Raises: why packed values and scales do not fit the operator."""
    if packed.dtype != _U8 or scales.dtype != _U8:
        raise ValueError(f"{what}: packed values and scales are bytes")
    if K % 32:
        raise ValueError(f"{what}: K={K} must be a multiple of 32")
    if not fits:
        raise ValueError(f"{what}: shape mismatch")
    raise ValueError(f"{what}: packed values and scales must be contiguous")


def _mxfp4_convert(fn, x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor | None, what: str, quantize: bool) -> None:
    """quantize_mxfp4_gpu and dequant_mxfp4_gpu; x is the plain side."""
    dev = x.get_device()
    if dev < 0 or packed.get_device() != dev or scales.get_device() != dev or (offsets is not None and offsets.get_device() != dev):
        _same_gpu(*((x, packed, scales) if offsets is None else (x, packed, scales, offsets)))
    dt = _DT.get(x.dtype)
    if dt is None:
        _not_supported(what, x.dtype)
    shape = x.shape
    if len(shape) == 2:
        rows, K = shape
        ld = _row_pitch(x, rows, K, "the matrix")
        if offsets is None:
            groups, table = 1, None
        else:
            groups, table = offsets.numel() - 1, offsets.data_ptr()
            if offsets.dtype != _I32 or offsets.dim() != 1 or groups < 0 or not offsets.is_contiguous():
                _bad_offsets(what)
        fits = packed.shape == (rows, K // 2) and scales.numel() >= mxfp4_scale_bytes(rows, K, groups)
    elif len(shape) == 3:
        if offsets is not None:
            raise ValueError(f"{what}: offsets go with 2-D tensors; the groups of a 3-D one are its first dimension")
        if not x.is_contiguous():
            raise ValueError(f"{what}: a 3-D tensor must be contiguous")
        groups, N, K = shape
        rows, ld, table = groups * N, K, None
        fits = packed.shape == (groups, N, K // 2) and scales.numel() >= groups * mxfp4_scale_bytes(N, K)
    else:
        raise ValueError(f"{what} takes 2-D or 3-D tensors")
    if not fits or K % 32 or packed.dtype != _U8 or scales.dtype != _U8 or not packed.is_contiguous() or not scales.is_contiguous():
        _bad_mxfp4(packed, scales, K, what, fits)
    if (rows | K | groups) >> 31:
        _too_large(what)
    cur = dev if _ONE_GPU else _current_device()
    if quantize:
        rc = fn(dev, _raw_stream(dev), dt, groups, rows, K, table, x.data_ptr(), ld, packed.data_ptr(), scales.data_ptr())
    else:
        rc = fn(dev, _raw_stream(dev), dt, groups, rows, K, table, packed.data_ptr(), scales.data_ptr(), x.data_ptr(), ld)
    if cur != dev:
        _set_device(cur)
    if rc:
        raise_for_status(rc)


def quantize_mxfp4_gpu(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
    """Microscaled 4-bit values of x: E2M1 codes, two per byte, and one power-of-two scale for 32 consecutive k.

    x [rows,K] (fp32/fp16/bf16) -> packed [rows,K/2]; with `offsets` the scales are laid out for those groups of rows
    (what grouped_matmul_mxfp4_gpu takes). x [groups,N,K] -> packed [groups,N,K/2], the weights of all experts.
    scales: mxfp4_scale_bytes(rows, K, groups) bytes, or groups * mxfp4_scale_bytes(N, K) for a 3-D x, in the block
    order that include/btm.h defines."""
    _mxfp4_convert(_LIB().btm_mxfp4_quantize, x, packed, scales, offsets, "quantize_mxfp4_gpu", True)


def dequant_mxfp4_gpu(packed: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
    """The values that quantize_mxfp4_gpu's output stands for, rounded once to out's dtype; shapes as there."""
    _mxfp4_convert(_LIB().btm_mxfp4_dequant, out, packed, scales, offsets, "dequant_mxfp4_gpu", False)


def _mxfp4_product_dtype(what: str, act, act_scales, w, w_scales, out, K: int) -> int:
    dt = _DT16.get(out.dtype)
    if dt is None:
        _not_supported(what, out.dtype)
    if act.dtype != _U8 or act_scales.dtype != _U8 or not act.is_contiguous() or not act_scales.is_contiguous() or K % 32:
        _bad_mxfp4(act, act_scales, K, what)
    if w.dtype != _U8 or w_scales.dtype != _U8 or not w.is_contiguous() or not w_scales.is_contiguous():
        _bad_mxfp4(w, w_scales, K, what)
    return dt


def matmul_mxfp4_gpu(act: torch.Tensor, act_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: torch.Tensor) -> None:
    """out[M,N] = act[M,K] . w[N,K]^T for operands that quantize_mxfp4_gpu wrote (packed [.., K/2]); out fp16/bf16."""
    dev = out.get_device()
    if dev < 0 or act.get_device() != dev or act_scales.get_device() != dev or w.get_device() != dev or w_scales.get_device() != dev:
        _same_gpu(act, act_scales, w, w_scales, out)
    sa, sw = act.shape, w.shape
    if len(sa) != 2 or len(sw) != 2 or out.dim() != 2:
        raise ValueError("matmul_mxfp4_gpu takes 2-D operands")
    M, half = sa
    N, half2 = sw
    K = 2 * half
    if half != half2 or out.shape != (M, N) or act_scales.numel() < mxfp4_scale_bytes(M, K) or w_scales.numel() < mxfp4_scale_bytes(N, K):
        raise ValueError("matmul_mxfp4_gpu: shape mismatch")
    if (M | N | K) >> 31:
        _too_large("matmul_mxfp4_gpu")
    dt = _mxfp4_product_dtype("matmul_mxfp4_gpu", act, act_scales, w, w_scales, out, K)
    cur = dev if _ONE_GPU else _current_device()
    rc = _LIB().btm_mxfp4_matmul(dev, _raw_stream(dev), dt, M, N, K, act.data_ptr(), act_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(),
                                 out.data_ptr(), _row_pitch(out, M, N, "out"))
    if cur != dev:
        _set_device(cur)
    if rc:
        raise_for_status(rc)


def grouped_matmul_mxfp4_gpu(act: torch.Tensor, act_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, offsets: torch.Tensor,
                             out: torch.Tensor) -> None:
    """out[r] = act[r] . w[g]^T for the rows r of group g; act [rows,K/2] quantised with these offsets, w [groups,N,K/2]."""
    dev = out.get_device()
    if (dev < 0 or act.get_device() != dev or act_scales.get_device() != dev or w.get_device() != dev or w_scales.get_device() != dev
            or offsets.get_device() != dev):
        _same_gpu(act, act_scales, w, w_scales, offsets, out)
    sa, sw = act.shape, w.shape
    if len(sa) != 2 or len(sw) != 3 or out.dim() != 2:
        raise ValueError("grouped_matmul_mxfp4_gpu takes act 2-D, w 3-D and out 2-D")
    rows, half = sa
    G, N, half2 = sw
    K = 2 * half
    if half != half2 or out.shape != (rows, N) or act_scales.numel() < mxfp4_scale_bytes(rows, K, G) or w_scales.numel() < G * mxfp4_scale_bytes(N, K):
        raise ValueError("grouped_matmul_mxfp4_gpu: shape mismatch")
    if offsets.dtype != _I32 or offsets.shape != (G + 1,) or not offsets.is_contiguous():
        _bad_offsets("grouped_matmul_mxfp4_gpu")
    if (rows | N | K | G) >> 31:
        _too_large("grouped_matmul_mxfp4_gpu")
    dt = _mxfp4_product_dtype("grouped_matmul_mxfp4_gpu", act, act_scales, w, w_scales, out, K)
    cur = dev if _ONE_GPU else _current_device()
    rc = _LIB().btm_mxfp4_matmul_grouped(dev, _raw_stream(dev), dt, G, rows, N, K, offsets.data_ptr(), act.data_ptr(), act_scales.data_ptr(),
                                         w.data_ptr(), w_scales.data_ptr(), out.data_ptr(), _row_pitch(out, rows, N, "out"))
    if cur != dev:
        _set_device(cur)
    if rc:
        raise_for_status(rc)


def convert_gpu(src: torch.Tensor, dst: torch.Tensor) -> None:
    """dst = dtype conversion of src (Float32 / Float16 / BFloat16, round to nearest even); the matmul-side
    counterpart of the reference's convert_gpu (Tensor/TensorOps.cu:315-365), out of place."""
    dev = _require_gpu(src, dst)
    if src.shape != dst.shape or not src.is_contiguous() or not dst.is_contiguous():
        raise ValueError("convert_gpu: shapes differ or tensors are not contiguous")
    if src.dtype not in _DT or dst.dtype not in _DT:
        from .errors import NotImplementedOp
        raise NotImplementedOp(f"convert_gpu: {src.dtype} -> {dst.dtype} is not supported")
    cur = dev if _ONE_GPU else _current_device()
    rc = _lib.lib().btm_convert(dev, _stream(dev), _DT[src.dtype], _DT[dst.dtype], src.numel(), src.data_ptr(), dst.data_ptr())
    if cur != dev:
        _set_device(cur)
    raise_for_status(rc)


def matmul(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """User-level wrapper in the style of the reference's Ops::add sketch
    (Ops/Elementwise/Add/Add.h:28-73): checks, allocates the result, dispatches by rank."""
    if a.dim() == 3:
        out = torch.empty((a.shape[0], a.shape[1], b.shape[2]), dtype=a.dtype, device=a.device)
        bmm_gpu(a, b, out)
        return out
    out = torch.empty((a.shape[0], b.shape[1]), dtype=a.dtype, device=a.device)
    matmul_gpu(a, b, out)
    return out
