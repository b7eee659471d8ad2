"""Chains of calls over the same few buffers with changing data, every call fed by the one before it: back to back they give the
bits of a run that waits after every call."""
import pytest
import torch

from tests import ragged

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def both_ways(chain):
    """chain(wait) twice; wait() is called between the calls."""
    apart = chain(torch.cuda.synchronize)
    torch.cuda.synchronize()
    together = chain(lambda: None)
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(apart, together)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), f"step {i}"
    return apart


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_product_quantise_dequantise(btm, pad, rows, dtype):
    # pad: the plain side's rows start on 32 bytes, on 16, anywhere
    K, steps = 416, 12
    a = [normal((rows, 64), dtype, i) for i in range(steps)]
    w = normal((64, K), dtype, 99)
    h, y = torch.zeros((rows, K + pad), dtype=dtype, device="cuda"), torch.zeros((rows, K + pad), dtype=dtype, device="cuda")
    packed, scales = torch.empty((rows, K // 2), dtype=torch.uint8, device="cuda"), torch.empty(btm.mxfp4_scale_bytes(rows, K), dtype=torch.uint8, device="cuda")

    def chain(wait):
        kept = []
        for x in a:
            for call in (lambda: btm.matmul_gpu(x, w, h[:, :K]), lambda: btm.quantize_mxfp4_gpu(h[:, :K], packed, scales),
                         lambda: btm.dequant_mxfp4_gpu(packed, scales, y[:, :K]), lambda: btm.quantize_mxfp4_gpu(y[:, :K], packed, scales),
                         lambda: btm.dequant_mxfp4_gpu(packed, scales, h[:, :K])):
                call()
                wait()
            kept += [h[:, :K].clone(), y[:, :K].clone()]
        return kept

    kept = both_ways(chain)
    btm.check_device_status(0)
    out = torch.empty((rows, K), dtype=dtype, device="cuda")
    btm.matmul_gpu(a[-1], w, out)
    assert torch.equal(kept[-1], ragged.quantize(out)[0].to(dtype))


@pytest.mark.parametrize("M", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("form", ["regs", "stream", "slab"])
def test_int4_behind_grouped_and_int4_products(btm, monkeypatch, form, M):
    monkeypatch.setenv("BTM_FORCE_GEMV", form)
    K, steps = 2048, 12
    x = [normal((M, K), F16, i) for i in range(steps)]
    w = normal((2, K, K), F16, 50, K ** -0.5)
    t = torch.tensor([0, M // 2, M], dtype=torch.int32, device="cuda")
    q, s = [], []
    for i in range(2):
        q.append(torch.empty((K, K // 2), dtype=torch.uint8, device="cuda"))
        s.append(torch.empty((K, K // 128), dtype=F16, device="cuda"))
        btm.quantize_int4_gpu(normal((K, K), F16, 60 + i, K ** -0.5), q[i], s[i])
    h, y = torch.zeros((M, K), dtype=F16, device="cuda"), torch.zeros((M, K), dtype=F16, device="cuda")
    torch.cuda.synchronize()

    def chain(wait):
        kept = []
        for a in x:
            for call in (lambda: btm.grouped_matmul_gpu(a, w, t, h), lambda: btm.matmul_int4_gpu(h, q[0], s[0], y),
                         lambda: btm.matmul_int4_gpu(y, q[1], s[1], h), lambda: btm.matmul_int4_gpu(h, q[0], s[0], y)):
                call()
                wait()
            kept += [h.clone(), y.clone()]
        return kept

    kept = both_ways(chain)
    btm.check_device_status(0)
    assert all(torch.isfinite(k).all() and (k != 0).any() for k in kept)
