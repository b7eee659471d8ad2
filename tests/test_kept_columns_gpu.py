"""Dense products into views whose width ends inside 16 bytes of a wider, aligned pitch: the columns behind the width belong to
somebody else (a neighbour's results, another rank's block) and keep what they held."""
import ctypes as C

import pytest
import torch

from beantensor_b200 import _lib
from tests import ragged

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DT = {F16: _lib.F16, BF16: _lib.BF16, F32: _lib.F32}
WIDTHS = [1, 5, 37, 61, 66, 130, 325]
M, K = 300, 128


def normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def operands(N, dtype):
    """a, b in pitches of whole 16 bytes, the output's wider buffer (guard rows behind it) and what that held."""
    unit = 128 // torch.finfo(dtype).bits
    pitch = (N + unit - 1) // unit * unit + (unit if N % unit == 0 else 0)
    wide = normal((M + 3, pitch), dtype, 3)
    return normal((M, K), dtype, 1), normal((K, pitch), dtype, 2)[:, :N], wide, wide.clone()


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def expect(wide, kept, N, a, b, relu_bias=None):
    exact, mass = ragged.product(a, b)
    out = wide[:M, :N]
    if relu_bias is not None:
        exact, mass = exact + relu_bias.double(), mass + relu_bias.double().abs()
        # max(., 0) moves no value away from the exact one's maximum with 0
        exact = exact.clamp(min=0)
    if out.dtype == F32:
        # Three products of TF32 halves, the low half below 2^-10 of the value: lo . lo is left out, and the tensor core cuts each
        # low half at 2^-10 of itself, so three times 2^-20 of the mass; beside that the additions.
        assert ((out.double() - exact).abs() <= (3 * 2.0 ** -20 + 3 * (K + 1) * 2.0 ** -23) * mass).all()
    else:
        ragged.check(out, exact, mass, K + 1)
    assert torch.equal(wide[:M, N:], kept[:M, N:]), "columns behind the width"
    assert torch.equal(wide[M:], kept[M:]), "rows behind the last"


@pytest.fixture(params=["1cta", "2cta"])
def kernel(request, monkeypatch):
    monkeypatch.setenv("BTM_FORCE_KERNEL", request.param)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N", WIDTHS)
def test_matmul(btm, kernel, N, dtype):
    a, b, wide, kept = operands(N, dtype)
    btm.matmul_gpu(a, b, wide[:M, :N])
    btm.check_device_status(0)
    expect(wide, kept, N, a, b)


@pytest.mark.parametrize("N", WIDTHS)
def test_bias_and_relu(btm, kernel, N):
    a, b, wide, kept = operands(N, BF16)
    bias = normal((N,), BF16, 4)
    btm.matmul_gpu(a, b, wide[:M, :N], bias=bias, relu=True)
    btm.check_device_status(0)
    expect(wide, kept, N, a, b, bias)


@pytest.mark.parametrize("N", WIDTHS)
def test_transposed_operands(btm, N):
    a, b, wide, kept = operands(N, F16)
    bt = b.t().contiguous()
    assert _lib.lib().btm_gemm_bt(0, stream(), _lib.F16, M, N, K, a.data_ptr(), K, bt.data_ptr(), K, wide.data_ptr(), wide.stride(0)) == _lib.OK
    btm.check_device_status(0)
    expect(wide, kept, N, a, b)
    wide.copy_(kept)
    at = normal((K, 304), F16, 5)[:, :M].t()
    btm.matmul_gpu(at, b, wide[:M, :N])
    btm.check_device_status(0)
    expect(wide, kept, N, at, b)


@pytest.mark.parametrize("form", ["plain", "workspace", "static", "transposed"])
@pytest.mark.parametrize("N", WIDTHS)
def test_fp32(btm, N, form):
    a, b, wide, kept = operands(N, F32)
    out, L, args = wide[:M, :N], _lib.lib(), None
    if form == "plain":
        btm.matmul_gpu(a, b, out)
    elif form == "transposed":
        btm.matmul_gpu(a.t().contiguous().t(), b, out)
    else:
        args = (0, stream(), M, N, K, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), wide.data_ptr(), wide.stride(0))
        if form == "static":
            assert L.btm_gemm_f32_static(*args) == _lib.OK
        else:
            need = L.btm_gemm_f32_workspace_bytes(M, N, K)
            ws = torch.empty(need, dtype=torch.uint8, device="cuda")
            assert L.btm_gemm_f32_ws(*args, ws.data_ptr(), need) == _lib.OK
    btm.check_device_status(0)
    expect(wide, kept, N, a, b)


@pytest.mark.parametrize("world,Nloc", [(1, 61), (2, 61), (2, 130), (3, 325), (8, 5)])
def test_blocks_of_the_other_ranks(btm, kernel, world, Nloc):
    # All ranks' calls on one GPU, one after the other, the first rank last: what the others wrote has to be there still.
    N = world * Nloc
    pitch = (N + 7) // 8 * 8
    a = normal((M, K), BF16, 1)
    b = normal((world, K, (Nloc + 7) // 8 * 8), BF16, 2)
    copies = [normal((M, pitch), BF16, 3) for _ in range(world)]
    kept = copies[0].clone()
    table = (C.c_void_p * world)(*[c.data_ptr() for c in copies])
    for r in reversed(range(world)):
        assert _lib.lib().btm_gemm_nshard(0, stream(), _lib.BF16, M, Nloc, K, a.data_ptr(), K, b[r].data_ptr(), b.stride(1), table, pitch, r, world) == _lib.OK
    btm.check_device_status(0)
    exact, mass = ragged.product(a, torch.cat([b[r, :, :Nloc] for r in range(world)], dim=1))
    for c in copies:
        ragged.check(c[:, :N], exact, mass, K)
        assert torch.equal(c[:, N:], kept[:, N:])


@pytest.mark.parametrize("kernel_name", ["1cta", "2cta"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_bounds_check_sees_the_last_columns(btm, monkeypatch, kernel_name, dtype):
    # Stores of a width that ends inside 16 bytes have hand-computed addresses: a clean run stays clean, and an extent that
    # ends one row earlier stops the last row's.
    from beantensor_b200.errors import CudaError
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel_name)
    L, N = _lib.lib(), 37
    a, b, wide, kept = operands(N, dtype)
    try:
        assert L.btm_debug_set(b"bounds", 1) == _lib.OK
        btm.matmul_gpu(a, b, wide[:M, :N])
        btm.check_device_status(0)
        expect(wide, kept, N, a, b)
        wide.copy_(kept)
        assert L.btm_debug_set(b"bounds_shrink", wide.stride(0)) == _lib.OK
        btm.matmul_gpu(a, b, wide[:M, :N])
        with pytest.raises(CudaError, match="bounds"):
            btm.check_device_status(0)
        last = N // 32 * 32 if dtype == F32 else 0  # whole boxes in front of them leave by TMA, whose extent is the tensor map's
        assert torch.equal(wide[M - 1, last:], kept[M - 1, last:])
    finally:
        assert L.btm_debug_set(b"bounds_shrink", 0) == _lib.OK
        assert L.btm_debug_set(b"bounds", 0) == _lib.OK
