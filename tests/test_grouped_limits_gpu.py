"""The grouped and microscaled operators at their edges: bounded waits that run out, bounds checks of hand-computed stores, operands
longer than 32-bit offsets reach, many groups, tensors of another stream."""
import pytest
import torch

from beantensor_b200 import _lib
from beantensor_b200.errors import CudaError, DeviceTimeout
from tests import ragged
from tests.test_mxfp4_gpu import quantized

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def table(bounds):
    return torch.tensor(bounds, dtype=torch.int32, device="cuda")


@pytest.fixture
def hooks():
    L = _lib.lib()
    yield L
    for key in (b"skip_loads", b"wait_limit_cycles", b"bounds_shrink", b"bounds"):
        assert L.btm_debug_set(key, 0) == _lib.OK


def products(btm, rows, K, N):
    """Calls of both products on the same table, with what they have to give."""
    bounds, groups = [0, 40, 40, rows], 3
    t = table(bounds)
    a, b = normal((rows, K), BF16, 1), normal((groups, K, N), BF16, 2)
    xq, xs = quantized(btm, a, t, groups)
    wq = torch.empty((groups, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((groups, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    w = b.transpose(1, 2).contiguous()
    btm.quantize_mxfp4_gpu(w, wq, ws)

    def check(out, lhs, rhs):
        for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
            exact, mass = ragged.product(lhs[lo:hi], rhs[g])
            ragged.check(out[lo:hi], exact, mass, K)

    values = ragged.quantize(w.reshape(groups * N, K))[0].reshape(groups, N, K).transpose(1, 2)
    return {"16 bit": (lambda out: btm.grouped_matmul_gpu(a, b, t, out), lambda out: check(out, a, b)),
            "4 bit": (lambda out: btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, out), lambda out: check(out, ragged.quantize(a)[0], values))}


@pytest.mark.parametrize("which", ["16 bit", "4 bit"])
@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
def test_wait_runs_out_and_the_device_stays_usable(btm, hooks, monkeypatch, kernel, which):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    run, check = products(btm, 300, 512, 264)[which]
    out = torch.zeros((300, 264), dtype=BF16, device="cuda")
    btm.check_device_status(0)
    assert hooks.btm_debug_set(b"wait_limit_cycles", 200_000) == _lib.OK
    assert hooks.btm_debug_set(b"skip_loads", 1) == _lib.OK
    run(out)
    torch.cuda.synchronize()
    with pytest.raises(DeviceTimeout):
        btm.check_device_status(0)
    btm.check_device_status(0)
    assert hooks.btm_debug_set(b"skip_loads", 0) == _lib.OK
    assert hooks.btm_debug_set(b"wait_limit_cycles", 0) == _lib.OK
    run(out)
    btm.check_device_status(0)
    check(out)


def test_gradient_wait_runs_out(btm, hooks):
    a, d = normal((300, 264), BF16, 1), normal((300, 136), BF16, 2)
    t, out = table([0, 40, 40, 300]), torch.zeros((3, 264, 136), dtype=BF16, device="cuda")
    assert hooks.btm_debug_set(b"wait_limit_cycles", 200_000) == _lib.OK
    assert hooks.btm_debug_set(b"skip_loads", 1) == _lib.OK
    btm.grouped_matmul_wgrad_gpu(a, d, t, out)
    torch.cuda.synchronize()
    with pytest.raises(DeviceTimeout):
        btm.check_device_status(0)
    assert hooks.btm_debug_set(b"skip_loads", 0) == _lib.OK
    assert hooks.btm_debug_set(b"wait_limit_cycles", 0) == _lib.OK
    btm.grouped_matmul_wgrad_gpu(a, d, t, out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans([0, 40, 40, 300], 300)):
        exact, mass = ragged.product(a[lo:hi].t(), d[lo:hi])
        ragged.check(out[g], exact, mass, hi - lo)


@pytest.mark.parametrize("which", ["16 bit", "4 bit"])
@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
@pytest.mark.parametrize("pad", [0, 3])
def test_bounds_checks(btm, hooks, monkeypatch, kernel, which, pad):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    rows, N = 310, 264
    run, check = products(btm, rows, 256, N)[which]
    wide = torch.zeros((rows, N + pad), dtype=BF16, device="cuda")
    assert hooks.btm_debug_set(b"bounds", 1) == _lib.OK
    run(wide[:, :N])
    btm.check_device_status(0)
    check(wide[:, :N])
    # pretend the output ends one row earlier: the last row's stores are stopped and reported
    last = wide[-1].clone()
    wide.zero_()
    assert hooks.btm_debug_set(b"bounds_shrink", N + pad) == _lib.OK
    run(wide[:, :N])
    with pytest.raises(CudaError, match="bounds"):
        btm.check_device_status(0)
    assert (wide[-1] == 0).all() and not (last == 0).all()


@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
def test_operands_longer_than_32_bit_offsets(btm, monkeypatch, kernel):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    rows = 1_100_000
    bounds = [rows - 210, rows - 77, rows - 77, rows - 5]
    t = table(bounds)
    for K, N in ((2048, 64), (64, 2048)):
        a = torch.empty((rows, K), dtype=BF16, device="cuda")
        a[-300:] = normal((300, K), BF16, 1)
        b = normal((3, K, N), BF16, 2)
        out = torch.empty((rows, N), dtype=BF16, device="cuda")
        out[-300:] = 9
        btm.grouped_matmul_gpu(a, b, t, out)
        btm.check_device_status(0)
        for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            if hi > lo:
                exact, mass = ragged.product(a[lo:hi], b[g])
                ragged.check(out[lo:hi], exact, mass, K)
        assert (out[-300:-210] == 9).all() and (out[-5:] == 9).all()
        db = torch.empty((3, K, N), dtype=BF16, device="cuda")
        btm.grouped_matmul_wgrad_gpu(a, out, t, db)
        btm.check_device_status(0)
        for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            exact, mass = ragged.product(a[lo:hi].t(), out[lo:hi])
            ragged.check(db[g], exact, mass, hi - lo)
        del a, out
    K, N = 4096, 72
    x = torch.empty((rows, K), dtype=BF16, device="cuda")
    x[-300:] = normal((300, K), BF16, 3)
    w = normal((3 * N, K), BF16, 4).reshape(3, N, K)
    xq = torch.empty((rows, K // 2), dtype=torch.uint8, device="cuda")
    xs = torch.empty(btm.mxfp4_scale_bytes(rows, K, 3), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(x, xq, xs, t)
    wq = torch.empty((3, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((3, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(w, wq, ws)
    out = torch.empty((rows, N), dtype=BF16, device="cuda")
    btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if hi > lo:
            exact, mass = ragged.product(ragged.quantize(x[lo:hi])[0], ragged.quantize(w[g])[0].t())
            ragged.check(out[lo:hi], exact, mass, K)


@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
def test_many_groups(btm, monkeypatch, kernel):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    groups, K, N = 1500, 64, 72
    g = torch.Generator().manual_seed(5)
    sizes = torch.randint(0, 5, (groups,), generator=g)
    sizes[1400] = 300
    bounds = [0] + sizes.cumsum(0).tolist()
    rows, t = bounds[-1], table(bounds)
    a, b, d = normal((rows, K), F16, 1), normal((groups, K, N), F16, 2), normal((rows, N), F16, 3)
    out, db = torch.zeros((rows, N), dtype=F16, device="cuda"), torch.empty((groups, K, N), dtype=F16, device="cuda")
    btm.grouped_matmul_gpu(a, b, t, out)
    btm.grouped_matmul_wgrad_gpu(a, d, t, db)
    xq, xs = quantized(btm, a, t, groups)
    wq = torch.empty((groups, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((groups, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    w = b.transpose(1, 2).contiguous()
    btm.quantize_mxfp4_gpu(w, wq, ws)
    o4 = torch.zeros_like(out)
    btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, o4)
    btm.check_device_status(0)
    of = torch.repeat_interleave(torch.arange(groups), sizes).cuda()
    exact, mass = torch.einsum("rk,rkn->rn", a.double(), b.double()[of]), torch.einsum("rk,rkn->rn", a.double().abs(), b.double().abs()[of])
    ragged.check(out, exact, mass, K)
    aq, wv = ragged.quantize(a)[0], ragged.quantize(w.reshape(groups * N, K))[0].reshape(groups, N, K)[of]
    ragged.check(o4, torch.einsum("rk,rnk->rn", aq, wv), torch.einsum("rk,rnk->rn", aq.abs(), wv.abs()), K)
    full = torch.zeros((groups, K, N), dtype=torch.float64, device="cuda").index_add_(0, of, a.double()[:, :, None] * d.double()[:, None, :])
    amass = torch.zeros_like(full).index_add_(0, of, a.double().abs()[:, :, None] * d.double().abs()[:, None, :])
    ragged.check(db, full, amass, 300)


def test_side_stream_orders_by_itself(btm):
    # The calls go to the current stream: inputs written on it just before, outputs read on it just after.
    s = torch.cuda.Stream()
    bounds, K, N = [0, 100, 100, 333], 256, 264
    t = table(bounds)
    b = normal((3, K, N), BF16, 2)
    wq = torch.empty((3, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((3, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for seed in range(5):
            a = normal((333, K), BF16, seed)
            out = torch.empty((333, N), dtype=BF16, device="cuda")
            btm.grouped_matmul_gpu(a, b, t, out)
            twice = out + out
            btm.quantize_mxfp4_gpu(b.transpose(1, 2).contiguous(), wq, ws)
            xq, xs = quantized(btm, a, t, 3)
            o4 = torch.empty_like(out)
            btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, o4)
            s.synchronize()
            assert torch.equal(twice, out + out)
            for g, (lo, hi) in enumerate(ragged.spans(bounds, 333)):
                exact, mass = ragged.product(a[lo:hi], b[g])
                ragged.check(out[lo:hi], exact, mass, K)
                exact, mass = ragged.product(ragged.quantize(a[lo:hi])[0], ragged.quantize(b[g].t().contiguous())[0].t())
                ragged.check(o4[lo:hi], exact, mass, K)
    btm.check_device_status(0)


@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
@pytest.mark.parametrize("N", [1, 5, 37, 61, 66, 130, 325])
def test_columns_behind_an_odd_width_are_kept(btm, monkeypatch, kernel, N):
    # The output's pitch is a multiple of 16 bytes, its width is not: what lies between belongs to somebody else.
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    rows, K, pitch = 200, 128, (N + 7) // 8 * 8
    bounds = [0, 64, 64, 190]
    t = table(bounds)
    a, d = normal((rows, K), BF16, 1), normal((rows, pitch), BF16, 2)[:, :N]
    b = normal((3, K, pitch), BF16, 3)[:, :, :N]
    wide, grad = normal((rows, pitch), BF16, 4), normal((3, K, pitch), BF16, 5)
    kept, kept_grad = wide.clone(), grad.clone()
    btm.grouped_matmul_gpu(a, b, t, wide[:, :N])
    btm.grouped_matmul_wgrad_gpu(a, d, t, grad[:, :, :N])
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        if hi > lo:
            ragged.check(wide[lo:hi, :N], *ragged.product(a[lo:hi], b[g]), K)
        ragged.check(grad[g, :, :N], *ragged.product(a[lo:hi].t(), d[lo:hi]), hi - lo)
    assert torch.equal(wide[:, N:], kept[:, N:]) and torch.equal(grad[:, :, N:], kept_grad[:, :, N:]) and torch.equal(wide[190:], kept[190:])
    xq, xs = quantized(btm, a, t, 3)
    w = b.transpose(1, 2).contiguous()
    wq = torch.empty((3, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.empty((3, btm.mxfp4_scale_bytes(N, K)), dtype=torch.uint8, device="cuda")
    btm.quantize_mxfp4_gpu(w, wq, ws)
    wide = kept.clone()
    btm.grouped_matmul_mxfp4_gpu(xq, xs, wq, ws, t, wide[:, :N])
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        if hi > lo:
            ragged.check(wide[lo:hi, :N], *ragged.product(ragged.quantize(a[lo:hi])[0], ragged.quantize(w[g])[0].t()), K)
    assert torch.equal(wide[:, N:], kept[:, N:]) and torch.equal(wide[190:], kept[190:])
