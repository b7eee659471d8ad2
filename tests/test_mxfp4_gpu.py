"""Microscaled 4-bit operands: quantisation, its inverse and the products against plain 64-bit forms."""
import numpy as np
import pytest
import torch

from beantensor_b200.errors import NotImplementedOp
from tests import ragged

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda") * scale
    x = x * torch.exp2(torch.randint(-6, 7, shape[:-1] + (1,), generator=g, device="cuda").float())  # rows of very different size
    return x.to(dtype)


def table(bounds):
    return torch.tensor(bounds, dtype=torch.int32, device="cuda")


@pytest.fixture(params=["1cta", "2cta", "decode"])
def kernel(request, monkeypatch):
    """Every form of the tensor-core product on every shape."""
    monkeypatch.setenv("BTM_FORCE_KERNEL", request.param)


def quantized(btm, x, offsets=None, groups=1):
    rows, K = x.shape
    packed = torch.full((rows, K // 2), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((btm.mxfp4_scale_bytes(rows, K, groups),), 0x5A, dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(x, packed, scales, offsets)
    return packed, scales


def expect_quantized(x, packed, scales, group_spans):
    """Codes and scales bit by bit, padding bytes of the scale blocks included; rows outside the groups as they were."""
    rows, K = x.shape
    at, slot, place, n_slots = ragged.slots(group_spans)
    val, X = ragged.quantize(x[torch.from_numpy(at).cuda()])
    codes = ragged.codes_of(packed).cpu()
    mag = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
    unit = torch.ldexp(torch.ones_like(X, dtype=torch.float64), X.clamp(max=127)).repeat_interleave(32, dim=1)
    want = torch.where(X.repeat_interleave(32, dim=1) == 128, torch.zeros_like(val), val / unit).cpu()
    got = mag[codes[torch.from_numpy(at)].long()]
    assert torch.equal(got, want)
    finite = (X != 128).repeat_interleave(32, dim=1).cpu()
    assert torch.equal(torch.signbit(got)[finite], torch.signbit(want)[finite])
    need = np.zeros(n_slots * ((K + 127) // 128) * 512, dtype=np.uint8)
    need[ragged.scale_index(slot, place, K)] = (X + 127).cpu().numpy().astype(np.uint8)
    assert np.array_equal(scales.cpu().numpy()[:need.size], need)
    assert (scales[need.size:] == 0x5A).all()
    outside = np.ones(rows, dtype=bool)
    outside[at] = False
    assert (packed[torch.from_numpy(outside).cuda()] == 0xA5).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 64), (128, 128), (129, 160), (257, 96), (40, 4096), (1000, 416)])
def test_quantize(btm, rows, K, dtype):
    x = normal((rows, K), dtype, rows + K)
    packed, scales = quantized(btm, x)
    expect_quantized(x, packed, scales, [(0, rows)])
    for to in (F16, BF16, F32):
        out = torch.empty((rows, K), dtype=to, device="cuda")
        btm.dequant_mxfp4_gpu(packed, scales, out)
        assert torch.equal(out, ragged.quantize(x)[0].to(to))


def test_quantize_ties_and_edges(btm):
    # All multiples of 1/8 from -8 to 8 beside a largest value that fixes the scale: ties, saturation, signed zeros.
    v = torch.arange(-64, 65, device="cuda").float() / 8
    rows = []
    for top in (4.0, 5.0, 6.0, 7.0, 7.875):
        for part in v[v.abs() <= top].split(31):
            row = torch.zeros(32, device="cuda")
            row[0] = top
            row[1:1 + part.numel()] = part
            rows.append(row)
    x = torch.stack(rows)
    for scale in (0, -100, 90, -126, 120):
        y = torch.ldexp(x, torch.tensor(scale, device="cuda"))
        packed, scales = quantized(btm, y)
        expect_quantized(y, packed, scales, [(0, y.shape[0])])
    # zeros of both signs, subnormals, the smallest and the largest numbers
    tiny = torch.tensor([[0.0] * 32, [-0.0] * 32, [1e-45] * 32, [2.0 ** -126] * 32, [2.0 ** -127] * 16 + [-2.0 ** -128] * 16,
                         [3.4028234e38] * 31 + [-1.0]], device="cuda")
    packed, scales = quantized(btm, tiny)
    expect_quantized(tiny, packed, scales, [(0, 6)])


def test_infinities_and_nan(btm):
    x = normal((70, 96), F32, 3)
    x[5, 40], x[6, 0], x[69, 95] = float("inf"), float("nan"), float("-inf")
    packed, scales = quantized(btm, x)
    expect_quantized(x, packed, scales, [(0, 70)])
    out = torch.empty((70, 96), dtype=BF16, device="cuda")
    btm.dequant_mxfp4_gpu(packed, scales, out)
    bad = out.isnan()
    assert bad[5, 32:64].all() and bad[6, :32].all() and bad[69, 64:].all() and int(bad.sum()) == 96


BOUNDS = [[0, 5, 5, 133, 134, 390, 390, 421], [7, 40, 168, 168, 297], [3, 3, 3], sorted([0] + [(i * i * 7) % 613 for i in range(75)] + [613])]


@pytest.mark.parametrize("bounds", BOUNDS)
@pytest.mark.parametrize("K", [32, 416])
def test_quantize_groups(btm, bounds, K):
    rows = bounds[-1] + 9
    x = normal((rows, K), BF16, K)
    x[bounds[-1]:] = float("nan")
    packed, scales = quantized(btm, x, table(bounds), len(bounds) - 1)
    btm.check_device_status(0)
    if bounds[-1] > bounds[0]:
        expect_quantized(x, packed, scales, ragged.spans(bounds, rows))
    out = torch.full((rows, K), 9.0, dtype=F32, device="cuda")
    btm.dequant_mxfp4_gpu(packed, scales, out, table(bounds))
    btm.check_device_status(0)
    want = torch.full((rows, K), 9.0, dtype=F32, device="cuda")
    lo, hi = bounds[0], bounds[-1]
    if hi > lo:
        want[lo:hi] = ragged.quantize(x[lo:hi])[0].float()
    assert torch.equal(out, want)


def test_quantize_strided_and_unaligned(btm):
    wide = normal((50, 200), F16, 1)
    for at in (0, 8, 3):
        x = wide[:, at:at + 160]
        packed, scales = quantized(btm, x)
        expect_quantized(x, packed, scales, [(0, 50)])
        out = torch.zeros((50, 200), dtype=F16, device="cuda")
        btm.dequant_mxfp4_gpu(packed, scales, out[:, at:at + 160])
        assert torch.equal(out[:, at:at + 160], ragged.quantize(x)[0].to(F16)) and (out[:, :at] == 0).all() and (out[:, at + 160:] == 0).all()


def test_weights_of_all_experts(btm):
    G, N, K = 5, 200, 160
    w = normal((G * N, K), BF16, 2).reshape(G, N, K)
    packed = torch.empty((G, N, K // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((G, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(w, packed, scales)
    for g in range(G):
        p1, s1 = quantized(btm, w[g])
        assert torch.equal(p1, packed[g]) and torch.equal(s1, scales[g])
    out = torch.empty_like(w)
    btm.dequant_mxfp4_gpu(packed, scales, out)
    assert torch.equal(out, ragged.quantize(w.reshape(G * N, K))[0].to(BF16).reshape(G, N, K))


# ---------------------------------------------------------------- products
SHAPES = [(1, 8, 32), (1, 136, 256), (2, 64, 64), (7, 200, 96), (16, 128, 128), (17, 1001, 416), (64, 264, 1440), (65, 33, 320), (128, 256, 512),
          (130, 520, 2048), (300, 776, 224), (1, 11008, 4096), (5, 512, 16384), (1025, 640, 1056)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(btm, kernel, M, N, K, dtype):
    x, w = normal((M, K), BF16, 1), normal((N, K), BF16, 2, K ** -0.5)
    xq, xs = quantized(btm, x)
    wq, ws = quantized(btm, w)
    out = torch.full((M, N), float("nan"), dtype=dtype, device="cuda")
    btm.matmul_mxfp4_gpu(xq, xs, wq, ws, out)
    btm.check_device_status(0)
    exact, mass = ragged.product(ragged.quantize(x)[0], ragged.quantize(w)[0].t())
    ragged.check(out, exact, mass, K)


@pytest.mark.parametrize("M,N,K,pad", [(40, 100, 128, 3), (130, 264, 320, 8), (1, 264, 320, 1), (200, 128, 64, 24)])
def test_product_into_a_wider_output(btm, kernel, M, N, K, pad):
    x, w = normal((M, K), BF16, 1), normal((N, K), BF16, 2)
    wide = normal((M, N + 2 * pad), F16, 3)
    before = wide.clone()
    btm.matmul_mxfp4_gpu(*quantized(btm, x), *quantized(btm, w), wide[:, pad:pad + N])
    btm.check_device_status(0)
    exact, mass = ragged.product(ragged.quantize(x)[0], ragged.quantize(w)[0].t())
    ragged.check(wide[:, pad:pad + N], exact, mass, K)
    assert torch.equal(wide[:, :pad], before[:, :pad]) and torch.equal(wide[:, pad + N:], before[:, pad + N:])


def test_nan_blocks_spoil_their_row_and_column_only(btm, kernel):
    M, N, K = 150, 140, 288
    x, w = normal((M, K), F32, 1), normal((N, K), F32, 2)
    x[3, 200], w[137, 287] = float("nan"), float("inf")
    out = torch.empty((M, N), dtype=BF16, device="cuda")
    btm.matmul_mxfp4_gpu(*quantized(btm, x), *quantized(btm, w), out)
    btm.check_device_status(0)
    bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
    bad[3], bad[:, 137] = True, True
    assert torch.equal(out.isnan(), bad)
    exact, mass = ragged.product(ragged.quantize(x)[0].nan_to_num(nan=0.0), ragged.quantize(w)[0].nan_to_num(nan=0.0).t())
    ragged.check(torch.where(bad, 0, out), torch.where(bad, 0.0, exact), mass, K)


def test_extreme_scales(btm, kernel):
    # 2^-127 and 2^125 in one product: the factors meet exactly, nothing is flushed in between.
    M, N, K = 20, 24, 64
    x, w = torch.zeros((M, K), device="cuda"), torch.zeros((N, K), device="cuda")
    x[:, :32], w[:, :32] = 6.0 * 2.0 ** 120, 3.0 * 2.0 ** -122
    x[:, 32:], w[:, 32:] = 1.5 * 2.0 ** -126, 2.0 ** 120
    out = torch.empty((M, N), dtype=BF16, device="cuda")
    btm.matmul_mxfp4_gpu(*quantized(btm, x), *quantized(btm, w), out)
    exact, mass = ragged.product(ragged.quantize(x)[0], ragged.quantize(w)[0].t())
    ragged.check(out, exact, mass, K)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,K", [(8, 32), (136, 256), (1001, 416), (264, 1440), (640, 96)])
@pytest.mark.parametrize("bounds", BOUNDS + [[0, 0, 1, 1, 1, 2], [0, 1], [0, 700, 701, 1500]])
def test_grouped_product(btm, kernel, bounds, N, K, dtype):
    rows, groups = bounds[-1] + 11, len(bounds) - 1
    x = normal((rows, K), BF16, 1)
    w = normal((groups * N, K), BF16, 2, K ** -0.5).reshape(groups, N, K)
    t = table(bounds)
    x[bounds[-1]:], x[:bounds[0]] = float("nan"), float("inf")
    xq, xs = quantized(btm, x, t, groups)
    wq = torch.empty((groups, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((groups, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(w, wq, ws)
    out = normal((rows, N), dtype, 3)
    before = out.clone()
    btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        if hi > lo:
            exact, mass = ragged.product(ragged.quantize(x[lo:hi])[0], ragged.quantize(w[g])[0].t())
            ragged.check(out[lo:hi], exact, mass, K)
    for part in (slice(0, bounds[0]), slice(bounds[-1], rows)):
        assert torch.equal(out[part].view(torch.int16), before[part].view(torch.int16))


def test_empty_calls(btm, kernel):
    by = lambda *s: torch.empty(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    wq, ws = quantized(btm, normal((40, 64), BF16, 1))
    btm.quantize_mxfp4_gpu(torch.empty((0, 64), dtype=F16, device="cuda"), by(0, 32), by(0))
    btm.matmul_mxfp4_gpu(by(0, 32), by(0), wq, ws, torch.empty((0, 40), dtype=F16, device="cuda"))
    xq, xs = quantized(btm, normal((3, 64), BF16, 1))
    btm.matmul_mxfp4_gpu(xq, xs, by(0, 32), by(0), torch.empty((3, 0), dtype=F16, device="cuda"))
    out = torch.ones((3, 40), dtype=F16, device="cuda")
    btm.matmul_mxfp4_gpu(by(3, 0), by(0), by(40, 0), by(0), out)  # no reduction: an empty sum
    btm.check_device_status(0)
    assert (out == 0).all()


def test_captured_experts_with_another_table(btm, kernel):
    rows, groups, N, K = 200, 6, 264, 192
    x, w = normal((rows, K), BF16, 1), normal((groups * N, K), BF16, 2).reshape(groups, N, K)
    wq = torch.empty((groups, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((groups, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(w, wq, ws)
    t = table([0, 10, 20, 30, 40, 50, 200])
    xq, xs = quantized(btm, x, t, groups)
    out = torch.zeros((rows, N), dtype=BF16, device="cuda")
    btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        btm.quantize_mxfp4_gpu(x, xq, xs, t)
        btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, out)
    for bounds in ([0, 10, 20, 30, 40, 50, 200], [0, 0, 0, 150, 150, 151, 190], [9, 9, 9, 9, 9, 9, 9]):
        t.copy_(table(bounds))
        x.copy_(normal((rows, K), BF16, bounds[3]))
        out.zero_()
        graph.replay()
        btm.check_device_status(0)
        for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
            exact, mass = ragged.product(ragged.quantize(x[lo:hi])[0], ragged.quantize(w[g])[0].t())
            ragged.check(out[lo:hi], exact, mass, K)
        assert (out[bounds[-1]:] == 0).all()


def test_two_layers_in_4_bits(btm, kernel):
    # quantise -> product -> quantise -> product, back to back, every launch fed by the one before; twenty times the same bits
    M, K, H = 33, 512, 1056
    x, w1, w2 = normal((M, K), BF16, 1), normal((H, K), BF16, 2, K ** -0.5), normal((K, H), BF16, 3, H ** -0.5)
    q1, q2 = quantized(btm, w1), quantized(btm, w2)
    first = None
    for i in range(20):
        h, y = torch.empty((M, H), dtype=BF16, device="cuda"), torch.empty((M, K), dtype=BF16, device="cuda")
        btm.matmul_mxfp4_gpu(*quantized(btm, x), *q1, h)
        btm.matmul_mxfp4_gpu(*quantized(btm, h), *q2, y)
        if first is None:
            btm.check_device_status(0)
            exact, mass = ragged.product(ragged.quantize(x)[0], ragged.quantize(w1)[0].t())
            ragged.check(h, exact, mass, K)
            exact, mass = ragged.product(ragged.quantize(h)[0], ragged.quantize(w2)[0].t())
            ragged.check(y, exact, mass, H)
            first = (h, y)
        assert torch.equal(h, first[0]) and torch.equal(y, first[1])


def test_experts_quantised_and_dense_agree(btm, kernel):
    # The 4-bit product of experts against the 16-bit grouped product of the same values: both sum the same exact products.
    bounds, rows, groups, N, K = [0, 50, 50, 181, 200], 200, 4, 136, 256
    x, w = normal((rows, K), BF16, 1, 0.1), normal((groups * N, K), BF16, 2, 0.1).reshape(groups, N, K)
    t = table(bounds)
    xq, xs = quantized(btm, x, t, groups)
    wq = torch.empty((groups, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((groups, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(w, wq, ws)
    xd, wd = torch.empty_like(x), torch.empty_like(w)
    btm.dequant_mxfp4_gpu(xq, xs, xd, t)
    btm.dequant_mxfp4_gpu(wq, ws, wd)
    o4, o16 = torch.empty((rows, N), dtype=BF16, device="cuda"), torch.empty((rows, N), dtype=BF16, device="cuda")
    btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, o4)
    btm.grouped_matmul_gpu(xd, wd.transpose(1, 2), t, o16)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        exact, mass = ragged.product(xd[lo:hi], wd[g].t())
        ragged.check(o4[lo:hi], exact, mass, K)
        ragged.check(o16[lo:hi], exact, mass, K)


def test_refusals_on_the_gpu(btm):
    x = normal((4, 64), F16, 1)
    xq, xs = quantized(btm, x)
    out = torch.zeros((4, 4), dtype=F16, device="cuda")
    with pytest.raises(ValueError, match="shape mismatch"):
        btm.quantize_mxfp4_gpu(x, xq[:, :16], xs)
    with pytest.raises(ValueError, match="multiple of 32"):
        btm.quantize_mxfp4_gpu(x[:, :48], torch.empty((4, 24), dtype=torch.uint8, device="cuda"), xs)
    with pytest.raises(ValueError, match="shape mismatch"):
        btm.quantize_mxfp4_gpu(x, xq, xs[:511])
    with pytest.raises(ValueError, match="bytes"):
        btm.quantize_mxfp4_gpu(x, xq.char(), xs)
    with pytest.raises(ValueError, match="offsets"):
        btm.quantize_mxfp4_gpu(x, xq, xs, torch.tensor([0, 4], device="cuda"))
    with pytest.raises(NotImplementedOp):
        btm.quantize_mxfp4_gpu(x.double(), xq, xs)
    with pytest.raises(ValueError, match="not on the GPU"):
        btm.quantize_mxfp4_gpu(x, xq.cpu(), xs)
    with pytest.raises(ValueError, match="shape mismatch"):
        btm.matmul_mxfp4_gpu(xq, xs, xq[:, :16], xs, out)
    with pytest.raises(ValueError, match="contiguous"):
        btm.matmul_mxfp4_gpu(xq.t().contiguous().t(), xs, xq, xs, out)
    with pytest.raises(NotImplementedOp):
        btm.matmul_mxfp4_gpu(xq, xs, xq, xs, out.float())
    with pytest.raises(ValueError, match="16-byte"):
        flat = torch.zeros(4 * 32 + 8, dtype=torch.uint8, device="cuda")
        btm.matmul_mxfp4_gpu(flat[8:].reshape(4, 32), xs, xq, xs, out)
    with pytest.raises(ValueError, match="shape mismatch"):
        btm.grouped_matmul_mxfp4_gpu(xq, xs, xq.reshape(2, 2, 32), xs, torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), out)
    torch.cuda.synchronize()
    assert (out == 0).all()
