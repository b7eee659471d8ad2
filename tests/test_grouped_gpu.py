"""Products grouped by expert and their weight gradients against plain 64-bit forms."""
import pytest
import torch

from tests import ragged
from beantensor_b200 import _lib
from beantensor_b200.errors import NotImplementedOp

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16

# (bounds, rows of the buffers): empty groups, one row, tiles that end inside a 128-row slot, rows in front and behind
TABLES = {
    "one": ([0, 130], 130),
    "single_row": ([0, 1], 1),
    "two_tokens": ([0, 0, 1, 1, 1, 2, 2, 2, 2], 2),
    "ragged": ([0, 5, 5, 133, 134, 390, 390, 421], 421),
    "inside": ([7, 40, 168, 168, 297], 331),
    "all_empty": ([3, 3, 3, 3], 9),
    "many": (sorted([0] + [(i * i * 7) % 613 for i in range(75)] + [613]), 640),
}
DENSE = [(64, 64), (72, 8), (8, 136), (520, 264), (200, 1000)]  # (K, N), 16-byte pitches
ODD = [(65, 33), (7, 130), (1, 1), (64, 31), (130, 128 + 5)]


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def table(bounds):
    return torch.tensor(bounds, dtype=torch.int32, device="cuda")


@pytest.fixture(params=["1cta", "2cta", "decode"])
def kernel(request, monkeypatch):
    """Every tensor-core kernel on every shape; operands that they cannot address take the general one either way."""
    monkeypatch.setenv("BTM_FORCE_KERNEL", request.param)


def expect_product(a, b, bounds, rows, out, before):
    """out against the plain form; what no group owns has to be as before."""
    touched = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        if hi > lo:
            exact, mass = ragged.product(a[lo:hi], b[g])
            ragged.check(out[lo:hi], exact, mass, a.shape[1])
            touched[lo:hi] = True
    assert torch.equal(out[~touched].view(torch.int16), before[~touched].view(torch.int16))


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", TABLES)
@pytest.mark.parametrize("K,N", DENSE + ODD)
def test_product(btm, kernel, name, dtype, K, N, trans):
    bounds, rows = TABLES[name]
    a = normal((rows, K), dtype, 1)
    groups = len(bounds) - 1
    b = normal((groups, N, K), dtype, 2).transpose(1, 2) if trans else normal((groups, K, N), dtype, 2)
    out = normal((rows, N), dtype, 3)
    before = out.clone()
    btm.grouped_matmul_gpu(a, b, table(bounds), out)
    btm.check_device_status(0)
    expect_product(a, b, bounds, rows, out, before)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", TABLES)
@pytest.mark.parametrize("K,N", DENSE + ODD)
def test_wgrad(btm, kernel, name, dtype, K, N):
    bounds, rows = TABLES[name]
    a, d = normal((rows, K), dtype, 1), normal((rows, N), dtype, 2)
    out = normal((len(bounds) - 1, K, N), dtype, 3)
    btm.grouped_matmul_wgrad_gpu(a, d, table(bounds), out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        exact, mass = ragged.product(a[lo:hi].t(), d[lo:hi])
        ragged.check(out[g], exact, mass, hi - lo)


@pytest.mark.parametrize("rows,groups,K,N", [(1500, 3, 1024, 2048), (4100, 9, 776, 1544), (300, 130, 256, 512)])
def test_larger_products_and_gradients(btm, kernel, rows, groups, K, N):
    g = torch.Generator().manual_seed(rows)
    cuts = sorted(torch.randint(0, rows + 1, (groups - 1,), generator=g).tolist())
    bounds = [0] + cuts + [rows]
    a, d = normal((rows, K), BF16, 1), normal((rows, N), BF16, 2)
    b = normal((groups, K, N), BF16, 3, K ** -0.5)
    out, da, db = torch.zeros_like(d), torch.zeros_like(a), torch.zeros_like(b)
    t = table(bounds)
    btm.grouped_matmul_gpu(a, b, t, out)
    btm.grouped_matmul_gpu(d, b.transpose(1, 2), t, da)
    btm.grouped_matmul_wgrad_gpu(a, d, t, db)
    btm.check_device_status(0)
    expect_product(a, b, bounds, rows, out, torch.zeros_like(out))
    expect_product(d, b.transpose(1, 2), bounds, rows, da, torch.zeros_like(da))
    for i, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        exact, mass = ragged.product(a[lo:hi].t(), d[lo:hi])
        ragged.check(db[i], exact, mass, hi - lo)


def test_gradients_against_differences(btm, kernel):
    # L = sum(out * d) is linear in a and in b: L(x + step) - L(x - step) is <gradient, 2 step> but for the roundings of the
    # outputs and of the gradient, each within its bound.
    bounds, rows, K, N = [0, 33, 33, 170, 201], 201, 136, 72
    a, d = normal((rows, K), F16, 1), normal((rows, N), F16, 2)
    b = normal((4, K, N), F16, 3)
    t = table(bounds)
    groups = list(enumerate(ragged.spans(bounds, rows)))
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    btm.grouped_matmul_gpu(d, b.transpose(1, 2), t, da)
    btm.grouped_matmul_wgrad_gpu(a, d, t, db)
    lim_a, lim_b = torch.zeros_like(a, dtype=torch.float64), torch.zeros_like(b, dtype=torch.float64)
    for g, (lo, hi) in groups:
        lim_a[lo:hi] = ragged.bound(*ragged.product(d[lo:hi], b[g].t()), N, F16)
        lim_b[g] = ragged.bound(*ragged.product(a[lo:hi].t(), d[lo:hi]), hi - lo, F16)

    def loss(a_, b_):
        o = torch.zeros((rows, N), dtype=F16, device="cuda")
        btm.grouped_matmul_gpu(a_, b_, t, o)
        off = sum((ragged.bound(*ragged.product(a_[lo:hi], b_[g]), K, F16) * d[lo:hi].double().abs()).sum() for g, (lo, hi) in groups)
        return (o.double() * d.double()).sum(), off

    for x, grad, lim, at in ((a, da, lim_a, lambda v: loss(v, b)), (b, db, lim_b, lambda v: loss(a, v))):
        step = normal(x.shape, F16, 7)
        xp, xm = x + step, x - step
        (lp, op), (lm, om) = at(xp), at(xm)
        real = xp.double() - xm.double()  # x +- step are rounded; this is what was taken
        want = (grad.double() * real).sum()
        assert want.abs() > 100 * 2.0 ** -11  # the quotient says something
        assert (lp - lm - want).abs() <= op + om + (lim * real.abs()).sum()


def test_foreign_rows_never_enter(btm, kernel):
    # Infinities and NaN in rows of other groups, behind the last group and in front of the first one.
    bounds, rows, K, N = [3, 20, 41, 41, 200], 230, 200, 136
    for dtype in (F16, BF16):
        a, d = normal((rows, K), dtype, 1), normal((rows, N), dtype, 2)
        b = normal((4, K, N), dtype, 3)
        for t in (a, d):
            t[:3] = float("nan")
            t[200:] = float("inf")
            t[20:41] = float("nan")
        out, db = torch.zeros_like(d), torch.zeros_like(b)
        tb = table(bounds)
        btm.grouped_matmul_gpu(a, b, tb, out)
        btm.grouped_matmul_wgrad_gpu(a, d, tb, db)
        btm.check_device_status(0)
        assert out[20:41].isnan().all() and db[1].isnan().all()
        assert (out[:3] == 0).all() and (out[200:] == 0).all() and (db[2] == 0).all()
        for g, (lo, hi) in ((0, (3, 20)), (3, (41, 200))):
            exact, mass = ragged.product(a[lo:hi], b[g])
            ragged.check(out[lo:hi], exact, mass, K)
            exact, mass = ragged.product(a[lo:hi].t(), d[lo:hi])
            ragged.check(db[g], exact, mass, hi - lo)


@pytest.mark.parametrize("pad", [0, 8, 3])
def test_strided_operands(btm, kernel, pad):
    # Column ranges of wider buffers, groups of b apart from each other, an output inside a wider one whose rest is kept.
    bounds, rows, K, N = [0, 50, 179, 260], 260, 128, 200
    a_all, b_all, c_all = normal((rows, K + pad), F16, 1), normal((3, K + 5, N + pad), F16, 2), normal((rows, N + 2 * pad), F16, 3)
    a, b, out = a_all[:, :K], b_all[:, :K, :N], c_all[:, pad:pad + N]
    before = c_all.clone()
    btm.grouped_matmul_gpu(a, b, table(bounds), out)
    btm.check_device_status(0)
    expect_product(a, b, bounds, rows, out, out)
    assert torch.equal(c_all[:, :pad], before[:, :pad]) and torch.equal(c_all[:, pad + N:], before[:, pad + N:])
    w_all = normal((3, K + 2, N + 2 * pad), F16, 4)
    before = w_all.clone()
    w = w_all[:, :K, pad:pad + N]
    d = normal((rows, N + pad), F16, 5)[:, :N]
    btm.grouped_matmul_wgrad_gpu(a, d, table(bounds), w)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        exact, mass = ragged.product(a[lo:hi].t(), d[lo:hi])
        ragged.check(w[g], exact, mass, hi - lo)
    assert torch.equal(w_all[:, K:], before[:, K:]) and torch.equal(w_all[:, :, pad + N:], before[:, :, pad + N:])


def test_empty_calls(btm, kernel):
    e = torch.empty((0, 64), dtype=F16, device="cuda")
    b = normal((2, 64, 32), F16, 1)
    btm.grouped_matmul_gpu(e, b, table([0, 0, 0]), torch.empty((0, 32), dtype=F16, device="cuda"))
    db = normal((2, 64, 32), F16, 2)
    btm.grouped_matmul_wgrad_gpu(e, torch.empty((0, 32), dtype=F16, device="cuda"), table([0, 0, 0]), db)
    assert (db == 0).all()
    # no reduction: the rows of the groups become zero, the others stay
    out = normal((5, 32), F16, 3)
    before = out.clone()
    btm.grouped_matmul_gpu(torch.empty((5, 0), dtype=F16, device="cuda"), torch.empty((2, 0, 32), dtype=F16, device="cuda"), table([1, 2, 4]), out)
    assert (out[1:4] == 0).all() and torch.equal(out[0], before[0]) and torch.equal(out[4], before[4])
    btm.grouped_matmul_gpu(normal((5, 8), F16, 1), torch.empty((0, 8, 32), dtype=F16, device="cuda"), table([0]), out)
    btm.check_device_status(0)


@pytest.mark.parametrize("bounds", [[0, 50, 20, 60], [0, 70, 500, 600], [-5, 10, 20, 60], [90, 80, 70, 60], [2 ** 31 - 1, -2 ** 31, 0, 2 ** 31 - 1]])
@pytest.mark.parametrize("K,N", [(64, 72), (33, 21)])
def test_bad_offsets_are_clamped_and_reported(btm, kernel, bounds, K, N):
    rows = 75
    a, d = normal((rows, K), BF16, 1), normal((rows, N), BF16, 4)
    b = normal((3, K, N), BF16, 2)
    out = normal((rows, N), BF16, 3)
    before = out.clone()
    btm.grouped_matmul_gpu(a, b, table(bounds), out)
    with pytest.raises(ValueError, match="offsets"):
        btm.check_device_status(0)
    btm.check_device_status(0)
    expect_product(a, b, bounds, rows, out, before)
    db = torch.empty_like(b)
    btm.grouped_matmul_wgrad_gpu(a, d, table(bounds), db)
    with pytest.raises(ValueError, match="offsets"):
        btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        exact, mass = ragged.product(a[lo:hi].t(), d[lo:hi])
        ragged.check(db[g], exact, mass, hi - lo)


def test_captured_and_replayed_with_another_table(btm, kernel):
    rows, K, N = 300, 192, 264
    a, d, b = normal((rows, K), BF16, 1), normal((rows, N), BF16, 2), normal((4, K, N), BF16, 3)
    out, da, db = torch.zeros_like(d), torch.zeros_like(a), torch.zeros_like(b)
    t = table([0, 10, 20, 30, 300])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        btm.grouped_matmul_gpu(a, b, t, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        btm.grouped_matmul_gpu(a, b, t, out)
        btm.grouped_matmul_gpu(d, b.transpose(1, 2), t, da)
        btm.grouped_matmul_wgrad_gpu(a, d, t, db)
    for bounds in ([0, 10, 20, 30, 300], [0, 150, 150, 290, 299], [5, 5, 5, 5, 5]):
        t.copy_(table(bounds))
        for x in (out, da):
            x.zero_()
        db.fill_(7)
        graph.replay()
        btm.check_device_status(0)
        expect_product(a, b, bounds, rows, out, torch.zeros_like(out))
        expect_product(d, b.transpose(1, 2), bounds, rows, da, torch.zeros_like(da))
        for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
            exact, mass = ragged.product(a[lo:hi].t(), d[lo:hi])
            ragged.check(db[g], exact, mass, hi - lo)


def test_two_streams_and_repeated_calls_give_the_same_bits(btm, kernel):
    rows, K, N = 700, 520, 776
    a, b = normal((rows, K), F16, 1), normal((6, K, N), F16, 2)
    t = table([0, 3, 300, 301, 500, 500, 699])
    first = torch.zeros((rows, N), dtype=F16, device="cuda")
    btm.grouped_matmul_gpu(a, b, t, first)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros_like(first) for _ in range(10)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                btm.grouped_matmul_gpu(a, b, t, o[i])
    torch.cuda.synchronize()
    btm.check_device_status(0)
    for o in outs:
        for x in o:
            assert torch.equal(x, first)


def test_chain_behind_the_router(btm, kernel):
    # The table and the rows come from work queued just before, the products feed one another back to back.
    tokens, groups, K, H = 200, 8, 256, 384
    x = normal((tokens, K), BF16, 1)
    w1, w2 = normal((groups, K, H), BF16, 2, K ** -0.5), normal((groups, H, K), BF16, 3, H ** -0.5)
    for seed in range(10):
        expert = torch.randint(0, groups, (tokens,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        order = expert.argsort(stable=True)
        t = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
        t[1:] = torch.bincount(expert, minlength=groups).cumsum(0)
        rows = x[order].contiguous()
        h, y = torch.empty((tokens, H), dtype=BF16, device="cuda"), torch.empty((tokens, K), dtype=BF16, device="cuda")
        btm.grouped_matmul_gpu(rows, w1, t, h)
        btm.grouped_matmul_gpu(h, w2, t, y)
        btm.check_device_status(0)
        bounds = t.tolist()
        expect_product(rows, w1, bounds, tokens, h, h)
        expect_product(h, w2, bounds, tokens, y, y)


def test_refusals_on_the_gpu(btm):
    a, b, out = normal((10, 64), F16, 1), normal((2, 64, 32), F16, 2), torch.zeros((10, 32), dtype=F16, device="cuda")
    t = table([0, 4, 10])
    with pytest.raises(ValueError, match="offsets"):
        btm.grouped_matmul_gpu(a, b, t.long(), out)
    with pytest.raises(ValueError, match="offsets"):
        btm.grouped_matmul_gpu(a, b, t[:2], out)
    with pytest.raises(ValueError, match="not on the GPU"):
        btm.grouped_matmul_gpu(a, b, t.cpu(), out)
    with pytest.raises(ValueError, match="shape mismatch"):
        btm.grouped_matmul_gpu(a, b.transpose(1, 2), t, out)
    with pytest.raises(ValueError, match="dtypes differ"):
        btm.grouped_matmul_gpu(a, b, t, out.bfloat16())
    with pytest.raises(NotImplementedOp):
        btm.grouped_matmul_gpu(a.float(), b.float(), t, out.float())
    with pytest.raises(ValueError, match="row-major"):
        btm.grouped_matmul_gpu(normal((64, 10), F16, 1).t(), b, t, out)
    with pytest.raises(ValueError, match="row-major"):
        btm.grouped_matmul_gpu(a, normal((2, 64, 64), F16, 2)[:, :, ::2], t, out)
    with pytest.raises(ValueError, match="leading dimension"):
        btm.grouped_matmul_gpu(a[:1].expand(10, 64), b, t, out)
    with pytest.raises(ValueError, match="strideB"):
        btm.grouped_matmul_gpu(a, b[:1].expand(2, 64, 32), t, out)
    with pytest.raises(ValueError, match="shape mismatch"):
        btm.grouped_matmul_wgrad_gpu(a, out, t, torch.zeros((2, 32, 64), dtype=F16, device="cuda"))
    with pytest.raises(ValueError, match="strideC"):
        btm.grouped_matmul_wgrad_gpu(a, out, t, torch.zeros((1, 64, 32), dtype=F16, device="cuda").expand(2, 64, 32))
    torch.cuda.synchronize()
    assert (out == 0).all()
