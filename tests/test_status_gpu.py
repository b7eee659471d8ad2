"""The device status: a repaired table of row offsets never hides that a kernel gave up, nor the other way round."""
import pytest
import torch

from beantensor_b200 import _lib
from beantensor_b200.errors import CudaError, DeviceTimeout

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture
def hooks(btm):
    L = _lib.lib()
    btm.check_device_status(0)
    yield L
    for key in (b"skip_loads", b"wait_limit_cycles", b"bounds_shrink", b"bounds"):
        assert L.btm_debug_set(key, 0) == _lib.OK


def operands():
    g = torch.Generator(device="cuda").manual_seed(1)
    a, b = torch.randn((300, 128), generator=g, device="cuda").to(BF16), torch.randn((2, 128, 264), generator=g, device="cuda").to(BF16)
    return a, b, torch.zeros((300, 264), dtype=BF16, device="cuda")


def table(*bounds):
    return torch.tensor(bounds, dtype=torch.int32, device="cuda")


def repaired(btm, what):
    a, b, out = operands()
    t = table(0, 200, 100)
    if what == "product":
        btm.grouped_matmul_gpu(a, b, t, out)
    elif what == "general":
        btm.grouped_matmul_gpu(a[:, :65], b[:, :65, :33], t, torch.zeros((300, 33), dtype=BF16, device="cuda"))
    else:
        packed, scales = torch.empty((300, 64), dtype=torch.uint8, device="cuda"), torch.empty(btm.mxfp4_scale_bytes(300, 128, 2), dtype=torch.uint8, device="cuda")
        btm.quantize_mxfp4_gpu(a, packed, scales, t)


def gives_up(btm, L):
    a, b, out = operands()
    good = table(0, 100, 300)
    assert L.btm_debug_set(b"wait_limit_cycles", 200_000) == _lib.OK
    assert L.btm_debug_set(b"skip_loads", 1) == _lib.OK
    btm.grouped_matmul_gpu(a, b, good, out)
    torch.cuda.synchronize()
    assert L.btm_debug_set(b"skip_loads", 0) == _lib.OK
    assert L.btm_debug_set(b"wait_limit_cycles", 0) == _lib.OK


@pytest.mark.parametrize("what", ["product", "general", "quantise"])
def test_a_wait_that_ran_out_behind_a_repaired_table(btm, hooks, what):
    repaired(btm, what)
    gives_up(btm, hooks)
    with pytest.raises(DeviceTimeout):
        btm.check_device_status(0)
    with pytest.raises(ValueError, match="offsets"):  # both are reported, the graver one first
        btm.check_device_status(0)
    btm.check_device_status(0)


def test_a_repaired_table_behind_a_wait_that_ran_out(btm, hooks):
    gives_up(btm, hooks)
    repaired(btm, "product")
    with pytest.raises(DeviceTimeout):
        btm.check_device_status(0)
    with pytest.raises(ValueError, match="offsets"):
        btm.check_device_status(0)
    btm.check_device_status(0)


def test_a_stopped_store_behind_a_repaired_table(btm, hooks):
    repaired(btm, "product")
    a, b, _ = operands()
    wide = torch.zeros((300, 267), dtype=BF16, device="cuda")
    assert hooks.btm_debug_set(b"bounds", 1) == _lib.OK
    assert hooks.btm_debug_set(b"bounds_shrink", 267) == _lib.OK
    btm.grouped_matmul_gpu(a, b, table(0, 100, 300), wide[:, :264])
    with pytest.raises(CudaError, match="bounds"):
        btm.check_device_status(0)
    with pytest.raises(ValueError, match="offsets"):
        btm.check_device_status(0)
    btm.check_device_status(0)
