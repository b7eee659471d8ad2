"""Refusals of the grouped and microscaled entry points, and what they answer without a device: nothing here computes."""
import ctypes

import pytest
import torch

from beantensor_b200 import _lib, ops
from beantensor_b200.errors import GPUTaskOnCPUBuild

P = ctypes.c_void_p(64)
ODD = ctypes.c_void_p(65)
OFF = ctypes.c_void_p(128)


def refused(rc, status, text):
    assert rc == status
    assert text in _lib.last_error(), _lib.last_error()


def test_grouped_product_arguments():
    L = _lib.lib()
    good = dict(dtype=_lib.F16, groups=2, rows=8, N=16, K=32, off=OFF, A=P, lda=32, B=P, strideB=512, ldb=16, t=0, C=P, ldc=16)

    def call(**kw):
        a = {**good, **kw}
        return L.btm_gemm_grouped(0, None, a["dtype"], a["groups"], a["rows"], a["N"], a["K"], a["off"], a["A"], a["lda"], a["B"], a["strideB"],
                                  a["ldb"], a["t"], a["C"], a["ldc"])

    refused(call(dtype=_lib.F32), _lib.ERR_UNSUPPORTED, "dtype")
    refused(call(groups=-1), _lib.ERR_INVALID, "negative")
    refused(call(rows=-1), _lib.ERR_INVALID, "negative")
    refused(call(N=-1), _lib.ERR_INVALID, "negative")
    refused(call(K=-1), _lib.ERR_INVALID, "negative")
    refused(call(off=None), _lib.ERR_INVALID, "offsets")
    refused(call(off=ctypes.c_void_p(130)), _lib.ERR_INVALID, "offsets")
    refused(call(A=None), _lib.ERR_INVALID, "null")
    refused(call(B=None), _lib.ERR_INVALID, "null")
    refused(call(C=None), _lib.ERR_INVALID, "null")
    refused(call(lda=31), _lib.ERR_INVALID, "leading dimension")
    refused(call(ldb=15), _lib.ERR_INVALID, "leading dimension")
    refused(call(ldb=31, t=1), _lib.ERR_INVALID, "leading dimension")
    refused(call(ldc=15), _lib.ERR_INVALID, "leading dimension")
    refused(call(strideB=511), _lib.ERR_INVALID, "strideB")
    refused(call(A=ODD), _lib.ERR_INVALID, "aligned")


def test_grouped_weight_gradient_arguments():
    L = _lib.lib()
    good = dict(dtype=_lib.BF16, groups=2, rows=8, M=32, N=16, off=OFF, A=P, lda=32, D=P, ldd=16, C=P, strideC=512, ldc=16)

    def call(**kw):
        a = {**good, **kw}
        return L.btm_gemm_grouped_wgrad(0, None, a["dtype"], a["groups"], a["rows"], a["M"], a["N"], a["off"], a["A"], a["lda"], a["D"], a["ldd"],
                                        a["C"], a["strideC"], a["ldc"])

    refused(call(dtype=_lib.I32), _lib.ERR_UNSUPPORTED, "dtype")
    refused(call(M=-1), _lib.ERR_INVALID, "negative")
    refused(call(off=None), _lib.ERR_INVALID, "offsets")
    refused(call(D=None), _lib.ERR_INVALID, "null")
    refused(call(C=None), _lib.ERR_INVALID, "null")
    refused(call(lda=31), _lib.ERR_INVALID, "leading dimension")
    refused(call(ldd=15), _lib.ERR_INVALID, "leading dimension")
    refused(call(strideC=511), _lib.ERR_INVALID, "strideC")
    refused(call(C=ODD), _lib.ERR_INVALID, "aligned")


def test_mxfp4_arguments():
    L = _lib.lib()
    q = L.btm_mxfp4_quantize
    refused(q(0, None, _lib.I8, 1, 8, 32, None, P, 32, P, P), _lib.ERR_UNSUPPORTED, "dtype")
    refused(q(0, None, _lib.F16, 1, 8, 48, None, P, 48, P, P), _lib.ERR_INVALID, "multiple of 32")
    refused(q(0, None, _lib.F16, 3, 8, 32, None, P, 32, P, P), _lib.ERR_INVALID, "equal groups")
    refused(q(0, None, _lib.F16, 1, -8, 32, None, P, 32, P, P), _lib.ERR_INVALID, "negative")
    refused(q(0, None, _lib.F16, 1, 8, 32, None, P, 31, P, P), _lib.ERR_INVALID, "leading dimension")
    refused(q(0, None, _lib.F16, 1, 8, 32, None, None, 32, P, P), _lib.ERR_INVALID, "null")
    refused(q(0, None, _lib.F16, 1, 8, 32, None, P, 32, None, P), _lib.ERR_INVALID, "null")
    refused(q(0, None, _lib.F16, 1, 8, 32, None, P, 32, P, ctypes.c_void_p(72)), _lib.ERR_INVALID, "16-byte")
    refused(q(0, None, _lib.F32, 1, 8, 32, None, ctypes.c_void_p(66), 32, P, P), _lib.ERR_INVALID, "aligned")
    refused(q(0, None, _lib.F16, 2, 9, 32, ctypes.c_void_p(130), P, 32, P, P), _lib.ERR_INVALID, "offsets")
    d = L.btm_mxfp4_dequant
    refused(d(0, None, _lib.F64, 1, 8, 32, None, P, P, P, 32), _lib.ERR_UNSUPPORTED, "dtype")
    refused(d(0, None, _lib.F16, 1, 8, 32, None, P, P, None, 32), _lib.ERR_INVALID, "null")
    m = L.btm_mxfp4_matmul
    refused(m(0, None, _lib.F32, 4, 8, 32, P, P, P, P, P, 8), _lib.ERR_UNSUPPORTED, "dtype")
    refused(m(0, None, _lib.F16, 4, 8, 40, P, P, P, P, P, 8), _lib.ERR_INVALID, "multiple of 32")
    refused(m(0, None, _lib.F16, -4, 8, 32, P, P, P, P, P, 8), _lib.ERR_INVALID, "negative")
    refused(m(0, None, _lib.F16, 4, -8, 32, P, P, P, P, P, 8), _lib.ERR_INVALID, "negative")
    refused(m(0, None, _lib.F16, 4, 8, 32, P, P, None, P, P, 8), _lib.ERR_INVALID, "null")
    refused(m(0, None, _lib.F16, 4, 8, 32, P, P, P, P, None, 8), _lib.ERR_INVALID, "null")
    refused(m(0, None, _lib.F16, 4, 8, 32, P, P, P, P, P, 7), _lib.ERR_INVALID, "leading dimension")
    refused(m(0, None, _lib.F16, 4, 8, 32, P, P, ctypes.c_void_p(72), P, P, 8), _lib.ERR_INVALID, "16-byte")
    g = L.btm_mxfp4_matmul_grouped
    refused(g(0, None, _lib.F16, 2, 4, 8, 32, None, P, P, P, P, P, 8), _lib.ERR_INVALID, "offsets")


def test_scale_bytes():
    n = _lib.lib().btm_mxfp4_scale_bytes
    assert n(1, 1, 32) == 512 and n(1, 128, 128) == 512 and n(1, 129, 128) == 1024 and n(1, 128, 160) == 1024
    assert n(0, 5, 32) == 0 and n(1, 0, 32) == 0 and n(1, 5, 0) == 0
    # however the rows are divided: a group of m rows takes ceil(m / 128) blocks
    for groups, rows in ((3, 2), (4, 4), (2, 130), (5, 1000), (64, 256)):
        worst = 0
        first = min(groups, rows)
        sizes = [1] * first + [0] * (groups - first)
        left = rows - first
        for i in range(first):  # one row more than a multiple of 128 wastes most
            take = left // 128 * 128 if i == 0 else 0
            sizes[i] += take
            left -= take
        sizes[0] += left
        worst = sum((s + 127) // 128 for s in sizes)
        assert n(groups, rows, 32) >= worst * 512
    assert n(2, 2 ** 31 - 1, 4096) == ((2 ** 31 - 1 + 254) // 128) * 32 * 512


def test_cpu_tensors_are_refused():
    if torch.cuda.is_available():
        pytest.skip("has a GPU")
    a, b = torch.zeros((4, 32), dtype=torch.float16), torch.zeros((2, 32, 16), dtype=torch.float16)
    off, out = torch.zeros(3, dtype=torch.int32), torch.zeros((4, 16), dtype=torch.float16)
    by = torch.zeros(1024, dtype=torch.uint8)
    with pytest.raises(GPUTaskOnCPUBuild):
        ops.grouped_matmul_gpu(a, b, off, out)
    with pytest.raises(GPUTaskOnCPUBuild):
        ops.grouped_matmul_wgrad_gpu(a, out, off, b)
    with pytest.raises(GPUTaskOnCPUBuild):
        ops.quantize_mxfp4_gpu(a, by[:64].reshape(4, 16), by)
    with pytest.raises(GPUTaskOnCPUBuild):
        ops.matmul_mxfp4_gpu(by[:64].reshape(4, 16), by, by[:256].reshape(16, 16), by, out)


def test_scale_bytes_of_both_sides_agree():
    n = _lib.lib().btm_mxfp4_scale_bytes
    for groups in (0, 1, 2, 7, 64, 300):
        for rows in (0, 1, 5, 127, 128, 129, 1000, 2 ** 31 - 1):
            for K in (0, 32, 128, 160, 4096):
                assert ops.mxfp4_scale_bytes(rows, K, groups) == n(groups, rows, K)


def test_sizes_beyond_the_kernels_are_refused():
    L = _lib.lib()
    big = 2 ** 31 - 1
    refused(L.btm_gemm_grouped(0, None, _lib.F16, 2, big, 16, 32, OFF, P, 32, P, 512, 16, 0, P, 16), _lib.ERR_UNSUPPORTED, "dimensions")
    refused(L.btm_gemm_grouped(0, None, _lib.F16, 2 ** 21, 8, 16, 32, OFF, P, 32, P, 512, 16, 0, P, 16), _lib.ERR_UNSUPPORTED, "groups")
    refused(L.btm_gemm_grouped_wgrad(0, None, _lib.F16, 2, big, 32, 16, OFF, P, 32, P, 16, P, 512, 16), _lib.ERR_UNSUPPORTED, "dimensions")
    refused(L.btm_mxfp4_quantize(0, None, _lib.F16, 1, big, 32, None, P, 32, P, P), _lib.ERR_UNSUPPORTED, "dimensions")
    refused(L.btm_mxfp4_quantize(0, None, _lib.F16, 2 ** 21, 2 ** 21, 32, None, P, 32, P, P), _lib.ERR_UNSUPPORTED, "groups")
    refused(L.btm_mxfp4_matmul(0, None, _lib.F16, big, 8, 32, P, P, P, P, P, 8), _lib.ERR_UNSUPPORTED, "dimensions")
    refused(L.btm_mxfp4_matmul(0, None, _lib.F16, 8, big, 32, P, P, P, P, P, big), _lib.ERR_UNSUPPORTED, "dimensions")
