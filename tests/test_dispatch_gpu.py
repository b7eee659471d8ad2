"""The grouped and microscaled products as they are dispatched by themselves, on both sides of every rule: the decode form (tiles that
fit the machine at once), one CTA, pairs of CTAs, the general kernel; equal groups and one that holds nearly all rows."""
import pytest
import torch

from tests import ragged

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def unforced(monkeypatch):
    monkeypatch.delenv("BTM_FORCE_KERNEL", raising=False)


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def bounds_of(rows, groups, uneven):
    if uneven and groups > 1:  # the last group takes what one row each of the others leaves
        return list(range(groups)) + [rows]
    return [rows * g // groups for g in range(groups + 1)]


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def decode_width(rows, groups):
    """Widest output whose 64-row slots times 128-column tiles are all resident at once (two per SM)."""
    return 2 * sms() // ((rows + 63 * min(groups, rows)) // 64) * 128


# rows, groups, K: height * K on both sides of 2^19, heights on both sides of 256; N as wide as four tiles
SIZES = [(4096, 4, 1024), (2048, 4, 1024), (2048, 4, 1032), (1020, 4, 4096), (1024, 4, 4096), (4100, 9, 776), (3000, 1, 512)]


@pytest.mark.parametrize("uneven", [False, True])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("rows,groups,K", SIZES)
def test_grouped_product(btm, rows, groups, K, trans, uneven):
    N, bounds = 2048, bounds_of(rows, groups, uneven)
    a = normal((rows, K), BF16, 1)
    b = normal((groups, N, K), BF16, 2, K ** -0.5).transpose(1, 2) if trans else normal((groups, K, N), BF16, 2, K ** -0.5)
    out = torch.full((rows, N), float("nan"), dtype=BF16, device="cuda")
    btm.grouped_matmul_gpu(a, b, torch.tensor(bounds, dtype=torch.int32, device="cuda"), out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        ragged.check(out[lo:hi], *ragged.product(a[lo:hi], b[g]), K)


@pytest.mark.parametrize("over", [0, 1])
@pytest.mark.parametrize("rows,groups", [(1, 1), (64, 8), (40, 24), (200, 3), (65, 1)])
def test_grouped_product_at_the_end_of_the_decode_form(btm, rows, groups, over):
    K, N, bounds = 200, min(decode_width(rows, groups) + over, 40000), bounds_of(rows, groups, True)
    a, b = normal((rows, K), F16, 1), normal((groups, N, K), F16, 2, K ** -0.5).transpose(1, 2)
    out = torch.full((rows, N), float("nan"), dtype=F16, device="cuda")
    btm.grouped_matmul_gpu(a, b, torch.tensor(bounds, dtype=torch.int32, device="cuda"), out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        ragged.check(out[lo:hi], *ragged.product(a[lo:hi], b[g]), K)


def microscaled(btm, rows, groups, K, N, bounds, dtype):
    x, w = normal((rows, K), BF16, 1), normal((groups * N, K), BF16, 2, K ** -0.5).reshape(groups, N, K)
    t = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    xq = torch.empty((rows, K // 2), dtype=torch.uint8, device="cuda")
    xs = torch.empty(btm.mxfp4_scale_bytes(rows, K, groups), dtype=torch.uint8, device="cuda")
    wq = torch.empty((groups, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((groups, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(x, xq, xs, t)
    btm.quantize_mxfp4_gpu(w, wq, ws)
    xv, wv = torch.empty_like(x), torch.empty_like(w)  # 16-bit values hold the 4-bit ones exactly
    btm.dequant_mxfp4_gpu(xq, xs, xv, t)
    btm.dequant_mxfp4_gpu(wq, ws, wv)
    out = torch.full((rows, N), float("nan"), dtype=dtype, device="cuda")
    if t is None:
        btm.matmul_mxfp4_gpu(xq, xs, wq[0], ws[0], out)
    else:
        btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds or [0, rows], rows)):
        ragged.check(out[lo:hi], *ragged.product(xv[lo:hi], wv[g].t()), K)


@pytest.mark.parametrize("rows,K,N", [(2048, 2048, 4096), (2048, 2016, 4096), (2047, 2048, 4096), (512, 2048, 16384), (511, 2048, 16520), (8192, 2080, 1000)])
def test_microscaled_product(btm, rows, K, N):
    microscaled(btm, rows, 1, K, N, None, BF16)


@pytest.mark.parametrize("uneven", [False, True])
@pytest.mark.parametrize("rows,groups,K,N", [(4096, 4, 2048, 2048), (2048, 4, 2080, 4096), (2044, 4, 2048, 4200), (3001, 24, 1440, 1001), (300, 130, 256, 512)])
def test_microscaled_experts(btm, rows, groups, K, N, uneven):
    microscaled(btm, rows, groups, K, N, bounds_of(rows, groups, uneven), F16)


@pytest.mark.parametrize("over", [0, 1])
@pytest.mark.parametrize("rows,groups", [(1, 1), (64, 8), (200, 3), (65, 1)])
def test_microscaled_product_at_the_end_of_the_decode_form(btm, rows, groups, over):
    microscaled(btm, rows, groups, 288, min(decode_width(rows, groups) + over, 40000), bounds_of(rows, groups, True), BF16)


@pytest.mark.parametrize("rows,groups,M,N", [(4096, 4, 512, 1024), (515, 16, 512, 1024), (130, 64, 200, 72), (2000, 3, 65, 33)])
@pytest.mark.parametrize("uneven", [False, True])
def test_grouped_gradient(btm, rows, groups, M, N, uneven):
    bounds = bounds_of(rows, groups, uneven)
    a, d = normal((rows, M), F16, 1), normal((rows, N), F16, 2)
    out = torch.full((groups, M, N), float("nan"), dtype=F16, device="cuda")
    btm.grouped_matmul_wgrad_gpu(a, d, torch.tensor(bounds, dtype=torch.int32, device="cuda"), out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        ragged.check(out[g], *ragged.product(a[lo:hi].t(), d[lo:hi]), hi - lo)
