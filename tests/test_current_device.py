"""Operators on tensors of another GPU than the current one: they go to the tensors' GPU and its stream, and the calling thread's current
GPU is the same afterwards, also when the call fails. The library and the devices are stand-ins, no GPU is needed."""
import pytest
import torch

from beantensor_b200 import _lib, ops

F16, U8 = torch.float16, torch.uint8


class OnGpu(torch.Tensor):
    """A CPU tensor that says it lies on GPU 1."""

    device = property(lambda self: torch.device("cuda", 1))
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 1

    def data_ptr(self):
        return 4096


def t(*shape, dtype=F16):
    return torch.Tensor._make_subclass(OnGpu, torch.zeros(shape, dtype=dtype))


class Machine:
    """The current device, and a library whose every call makes its device current, as the real one does."""

    def __init__(self):
        self.current, self.calls, self.status = 0, [], 0

    def set(self, dev):
        self.current = dev

    def __getattr__(self, name):
        def call(dev, stream, *args):
            self.calls.append((name, dev, stream))
            self.current = dev
            return self.status

        if not name.startswith("btm_"):
            raise AttributeError(name)
        return call


@pytest.fixture
def machine(monkeypatch):
    m = Machine()
    monkeypatch.setattr(_lib, "_lib", m)
    monkeypatch.setattr(_lib, "lib", lambda: m)
    monkeypatch.setattr(_lib, "last_error", lambda: "refused")
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: 1)
    for name, value in (("_current_device", lambda: m.current), ("_set_device", m.set), ("_ONE_GPU", False)):
        monkeypatch.setattr(ops, name, value, raising=False)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 1000 + dev)
    monkeypatch.setattr(ops, "_stream", lambda dev=None: 1000 + dev)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 1000 + dev)
    return m


OFF = t(3, dtype=torch.int32)
BYTES = t(4096, dtype=U8)
CALLS = {
    "btm_gemm": lambda: ops.matmul_gpu(t(4, 8), t(8, 16), t(4, 16)),
    "btm_gemm_bias_act": lambda: ops.matmul_gpu(t(4, 8), t(8, 16), t(4, 16), bias=t(16)),
    "btm_gemm_strided": lambda: ops.matmul_gpu(t(8, 4).t(), t(8, 16), t(4, 16)),
    "btm_bmm": lambda: ops.bmm_gpu(t(2, 4, 8), t(2, 8, 16), t(2, 4, 16)),
    "btm_int4_matmul": lambda: ops.matmul_int4_gpu(t(1, 128), t(8, 64, dtype=U8), t(8, 1), t(1, 8)),
    "btm_int4_dequant": lambda: ops.dequant_int4_gpu(t(8, 64, dtype=U8), t(8, 1), t(8, 128)),
    "btm_int4_unpack": lambda: ops.unpack_int4_gpu(t(8, 64, dtype=U8), t(8, 128, dtype=torch.int8)),
    "btm_int4_quantize": lambda: ops.quantize_int4_gpu(t(8, 128), t(8, 64, dtype=U8), t(8, 1)),
    "btm_gemm_grouped": lambda: ops.grouped_matmul_gpu(t(4, 8), t(2, 8, 16), OFF, t(4, 16)),
    "btm_gemm_grouped_wgrad": lambda: ops.grouped_matmul_wgrad_gpu(t(4, 8), t(4, 16), OFF, t(2, 8, 16)),
    "btm_mxfp4_quantize": lambda: ops.quantize_mxfp4_gpu(t(4, 32), t(4, 16, dtype=U8), BYTES, OFF),
    "btm_mxfp4_dequant": lambda: ops.dequant_mxfp4_gpu(t(4, 16, dtype=U8), BYTES, t(4, 32), OFF),
    "btm_mxfp4_matmul": lambda: ops.matmul_mxfp4_gpu(t(4, 16, dtype=U8), BYTES, t(8, 16, dtype=U8), BYTES, t(4, 8)),
    "btm_mxfp4_matmul_grouped": lambda: ops.grouped_matmul_mxfp4_gpu(t(4, 16, dtype=U8), BYTES, t(2, 8, 16, dtype=U8), BYTES, OFF, t(4, 8)),
    "btm_convert": lambda: ops.convert_gpu(t(4, 8), t(4, 8, dtype=torch.float32)),
    "btm_check_device_status": lambda: ops.check_device_status(1),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("current", [0, 1, 3])
def test_the_current_device_is_put_back(machine, name, current):
    machine.current = current
    CALLS[name]()
    assert machine.calls == [(name, 1, 1001)]
    assert machine.current == current


@pytest.mark.parametrize("name", CALLS)
def test_also_when_the_call_is_refused(machine, name):
    machine.current, machine.status = 2, _lib.ERR_INVALID
    with pytest.raises(ValueError, match="refused"):
        CALLS[name]()
    assert machine.current == 2
