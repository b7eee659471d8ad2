"""Infinities in the fp32 product beside values that the first TF32 half holds whole (small whole numbers, halves): an
infinite element makes its row or column infinite with the product's sign, and NaN only where the definition says so."""
import ctypes as C

import pytest
import torch

from beantensor_b200 import _lib

pytestmark = pytest.mark.gpu


def inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-3, 4, (150, 136), generator=g, device="cuda").float()
    b = torch.randint(-3, 4, (136, 140), generator=g, device="cuda").float()
    inf = float("inf")
    a[3, 5], a[17, 100], a[20, 0], a[20, 1], a[90, 7] = inf, -inf, inf, -inf, inf
    b[7, 9], b[100, 11], b[5, 30], b[5, 31] = -inf, inf, inf, 0.5
    a[101, 2] = float("nan")
    a[40] += 1e-3  # values with both halves
    return a, b


def expect(out, a, b):
    ref = a.double() @ b.double()
    assert torch.equal(out.isnan(), ref.isnan())
    assert torch.equal(out.isposinf(), ref.isposinf())
    assert torch.equal(out.isneginf(), ref.isneginf())
    rest = torch.isfinite(ref)
    rest[40] = False
    assert torch.equal(out.double()[rest], ref[rest])  # sums of small whole numbers are exact


@pytest.mark.parametrize("form", ["plain", "transposed", "static"])
@pytest.mark.parametrize("seed", range(4))
def test_infinities_beside_whole_numbers(btm, seed, form):
    a, b = inputs(seed)
    out = torch.empty((150, 140), device="cuda")
    if form == "plain":
        btm.matmul_gpu(a, b, out)
    elif form == "transposed":
        btm.matmul_gpu(a.t().contiguous().t(), b.t().contiguous().t(), out)
    else:
        st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert _lib.lib().btm_gemm_f32_static(0, st, 150, 140, 136, a.data_ptr(), 136, b.data_ptr(), 140, out.data_ptr(), 140) == _lib.OK
    btm.check_device_status(0)
    expect(out, a, b)
