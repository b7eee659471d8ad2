"""Ragged products grouped by expert and microscaled 4-bit products: the calls, their plain forms and their sizes.

Four operators. `groups` below are the experts of a mixture-of-experts layer: the rows of the activations are sorted by
expert, `offsets[g] .. offsets[g + 1]` are the rows of group g, and rows behind `offsets[groups]` belong to nobody.

grouped          out[r, :] = a[r, :] . b[g]                      for the rows r of group g; b is [groups, K, N]
grouped_train    the same product with both gradients: da[r, :] = dout[r, :] . b[g]^T and
                 db[g] = a[rows of g]^T . dout[rows of g]
mxfp4_quantize   x -> 4-bit E2M1 values with one power-of-two scale (E8M0) for 32 consecutive k, and back:
                 X = floor(log2(max |x|)) - 2 per block, q = round(x / 2^X) to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6
                 (ties to the even code, saturating), value q 2^X
mxfp4_linear     out[r, :] = Q(x[r, :]) . w[g]^T with x quantised as above inside the call and w [groups, N, K] held in
                 4 bits; a plain layer is one group that owns every row

With `own` false `run` computes these in elementary torch operations, with `own` true it calls the framework.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One token of a small layer that takes two of eight experts: the smallest call, latency counts.
        dict(name="grouped_token", op="grouped", dtype="bf16", groups=8, rows=2, spare=0, pad=0, K=1024, N=1024, skew=0.0),
        # A decoding batch of 32 tokens with eight experts each: a few rows per expert, all weights are read.
        dict(name="grouped_batch", op="grouped", dtype="f16", groups=64, rows=256, spare=0, pad=0, K=2048, N=2048, skew=0.5),
        # A short prompt over many experts of odd width, unevenly loaded, some without a row; the activations are a column
        # range of a wider buffer that has spare rows at its end.
        dict(name="grouped_ragged", op="grouped", dtype="bf16", groups=40, rows=5003, spare=117, pad=88, K=1416, N=1000, skew=1.5),
        # A long prompt through eight wide experts.
        dict(name="grouped_prompt", op="grouped", dtype="bf16", groups=8, rows=16384, spare=0, pad=0, K=4096, N=4096, skew=0.7),
        # A training step of a small layer: every expert holds a few dozen rows.
        dict(name="train_small", op="grouped_train", dtype="f16", groups=16, rows=515, spare=0, pad=0, K=512, N=1024, skew=0.7),
        # A training step of a large layer.
        dict(name="train_large", op="grouped_train", dtype="bf16", groups=16, rows=16384, spare=0, pad=0, K=4096, N=2048, skew=0.7),
        # The activations of a few tokens.
        dict(name="quantize_tokens", op="mxfp4_quantize", dtype="f16", rows=5, K=4096),
        # The activations of a long prompt behind the wide layer of a feed-forward block.
        dict(name="quantize_prompt", op="mxfp4_quantize", dtype="bf16", rows=16384, K=11008),
        # A wide layer for a single token.
        dict(name="linear_token", op="mxfp4_linear", dtype="bf16", groups=1, rows=1, spare=0, K=4096, N=11008, skew=0.0),
        # Experts in 4 bits for a decoding batch.
        dict(name="linear_experts", op="mxfp4_linear", dtype="bf16", groups=64, rows=256, spare=0, K=2048, N=2048, skew=0.5),
        # Experts in 4 bits for a short prompt: odd sizes, uneven load, spare rows.
        dict(name="linear_ragged", op="mxfp4_linear", dtype="f16", groups=24, rows=3001, spare=71, K=1440, N=1001, skew=1.5),
        # A wide layer for a long prompt.
        dict(name="linear_prompt", op="mxfp4_linear", dtype="bf16", groups=1, rows=8192, spare=0, K=4096, N=11008, skew=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["grouped", "grouped_train", "mxfp4_quantize", "mxfp4_linear"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "mxfp4_quantize":
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 16000), K=32 * _log(rng, 4, 340))
    groups = _log(rng, 2, 96)
    rows = _log(rng, 1, 12000)
    spare = rng.choice([0, 0, rng.randrange(1, 200)])
    skew = rng.choice([0.0, 0.5, 1.0, 2.0])
    if op == "mxfp4_linear":
        if rng.random() < 0.5:
            groups, spare, skew = 1, 0, 0.0
        width = 8000 if groups == 1 else 3000
        N = _log(rng, 256, width)
        return dict(op=op, dtype=dtype, groups=groups, rows=rows, spare=spare, K=32 * _log(rng, 8, 128 if groups == 1 else 64),
                    N=N if rng.random() < 0.3 else 8 * (N // 8), skew=skew)
    return dict(op=op, dtype=dtype, groups=groups, rows=rows, spare=spare, pad=rng.choice([0, 0, 8 * rng.randrange(1, 32)]) if op == "grouped" else 0,
                K=8 * _log(rng, 16, 320), N=8 * _log(rng, 16, 320), skew=skew)


# ------------------------------------------------------------------------------------------------ inputs
def _sizes(case, seed):
    """Rows per group: drawn with a load of 1 / rank^skew over the groups in random order."""
    rng = np.random.default_rng([seed, 7])
    g = case["groups"]
    load = 1.0 / np.arange(1, g + 1) ** case["skew"]
    rng.shuffle(load)
    return [int(n) for n in rng.multinomial(case["rows"], load / load.sum())]


def _normal(shape, std, gen, dtype):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _activations(shape, gen, dtype):
    """Normal values with some channels ten times larger than the rest, as hidden states have them."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    wide = torch.rand(shape[-1], generator=gen, device="cuda") < 0.02
    return (x * torch.where(wide, 10.0, 1.0)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DT[case["dtype"]]
    st = {"op": case["op"], "dt": dt}
    if case["op"] == "mxfp4_quantize":
        st["x"] = _activations((case["rows"], case["K"]), gen, dt)
        return st
    rows, K, N, groups = case["rows"], case["K"], case["N"], case["groups"]
    total = rows + case["spare"]
    sizes = _sizes(case, seed)
    bounds = [0]
    for n in sizes:
        bounds.append(bounds[-1] + n)
    st["bounds"] = bounds  # the same numbers on the host: the plain forms walk over the groups
    st["offsets"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    if case["op"] == "mxfp4_linear":
        st["x"] = _activations((total, K), gen, dt)
        codes, scales = [], []
        for _ in range(groups):
            c, e = _plain_quantize(torch.randn((N, K), generator=gen, device="cuda") * (1.0 / math.sqrt(K)))
            codes.append(c[:, 0::2] | (c[:, 1::2] << 4))
            scales.append(_scale_blocks(e))
        st["w"] = torch.stack(codes)
        st["w_scales"] = torch.stack(scales)
    else:
        st["a"] = _normal((total, K + case["pad"]), 1.0, gen, dt)[:, :K]
        st["b"] = _normal((groups, K, N), 1.0 / math.sqrt(K), gen, dt)
    st["out"] = torch.zeros((total, N), dtype=dt, device="cuda")
    if case["op"] == "grouped_train":
        st["dout"] = _normal((total, N), 1.0, gen, dt)
        st["da"] = torch.zeros((total, K), dtype=dt, device="cuda")
        st["db"] = torch.zeros((groups, K, N), dtype=dt, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ plain forms
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_quantize(x):
    """[rows, K] -> codes [rows, K] (sign in bit 3) and scale bytes [rows, K / 32] (exponent + 127)."""
    rows, K = x.shape
    b = x.float().reshape(rows, K // 32, 32)
    amax = b.abs().amax(dim=2)
    e = (torch.frexp(amax)[1] - 1 - 2).clamp(-127, 127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    m = torch.ldexp(b, -e.unsqueeze(2)).abs()
    # Half-way points between neighbours; a tie goes to the even code.
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8) + (m >= 1.75).to(torch.uint8) +
            (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8) + (m > 5.0).to(torch.uint8))
    code = code | (torch.signbit(b).to(torch.uint8) << 3)
    return code.reshape(rows, K), (e + 127).to(torch.uint8)


def _scale_blocks(e):
    """Scale bytes [rows, K / 32] in the order the framework keeps them: blocks of 128 rows x 4 scales, 512 bytes each,
    the block of rows R and scales C at index R * ceil(K / 128) + C; within a block the scale c of row r is byte
    (r % 32) * 16 + (r // 32) * 4 + c. What lies outside the matrix is 0."""
    rows, cols = e.shape
    rb, cb = (rows + 127) // 128, (cols + 3) // 4
    p = torch.zeros((rb * 128, cb * 4), dtype=torch.uint8, device=e.device)
    p[:rows, :cols] = e
    return p.reshape(rb, 4, 32, cb, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _plain_values(code, e):
    rows, K = code.shape
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=code.device)
    v = table[code.long()].reshape(rows, K // 32, 32)
    return torch.ldexp(v, e.int().unsqueeze(2) - 127).reshape(rows, K)


def _plain_weight(w, blocks):
    """One group's packed weights [N, K / 2] and scale blocks -> float values [N, K]."""
    N, K = w.shape[0], w.shape[1] * 2
    cols, cb = K // 32, (K // 32 + 3) // 4
    e = blocks.reshape(-1, cb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, cb * 4)[:N, :cols]
    code = torch.stack((w & 15, w >> 4), dim=2).reshape(N, K)
    return _plain_values(code, e)


def _run_plain(st):
    op, dt = st["op"], st["dt"]
    if op == "mxfp4_quantize":
        return _plain_values(*_plain_quantize(st["x"])).to(dt)
    bounds = st["bounds"]
    groups = len(bounds) - 1
    out = torch.zeros_like(st["out"])
    if op == "mxfp4_linear":
        x = _plain_values(*_plain_quantize(st["x"]))
        for g in range(groups):
            lo, hi = bounds[g], bounds[g + 1]
            if hi > lo:
                out[lo:hi] = (x[lo:hi] @ _plain_weight(st["w"][g], st["w_scales"][g]).t()).to(dt)
        return out
    a, b = st["a"], st["b"]
    for g in range(groups):
        lo, hi = bounds[g], bounds[g + 1]
        if hi > lo:
            out[lo:hi] = (a[lo:hi].float() @ b[g].float()).to(dt)
    if op == "grouped":
        return out
    dout = st["dout"]
    da, db = torch.zeros_like(st["da"]), torch.zeros_like(st["db"])
    for g in range(groups):
        lo, hi = bounds[g], bounds[g + 1]
        if hi > lo:
            d = dout[lo:hi].float()
            da[lo:hi] = (d @ b[g].float().t()).to(dt)
            db[g] = (a[lo:hi].float().t() @ d).to(dt)
    return {"out": out, "da": da, "db": db}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(st):
    from beantensor_b200 import ops

    op, dt = st["op"], st["dt"]
    if op in ("mxfp4_quantize", "mxfp4_linear"):
        x = st["x"]
        rows, K = x.shape
        packed = torch.empty((rows, K // 2), dtype=torch.uint8, device=x.device)
        if op == "mxfp4_quantize":
            scales = torch.empty(ops.mxfp4_scale_bytes(rows, K), dtype=torch.uint8, device=x.device)
            ops.quantize_mxfp4_gpu(x, packed, scales)
            values = torch.empty((rows, K), dtype=dt, device=x.device)
            ops.dequant_mxfp4_gpu(packed, scales, values)
            return values
        groups = st["w"].shape[0]
        out = st["out"]
        if groups == 1:
            scales = torch.empty(ops.mxfp4_scale_bytes(rows, K), dtype=torch.uint8, device=x.device)
            ops.quantize_mxfp4_gpu(x, packed, scales)
            ops.matmul_mxfp4_gpu(packed, scales, st["w"][0], st["w_scales"][0], out)
        else:
            scales = torch.empty(ops.mxfp4_scale_bytes(rows, K, groups), dtype=torch.uint8, device=x.device)
            ops.quantize_mxfp4_gpu(x, packed, scales, offsets=st["offsets"])
            ops.grouped_matmul_mxfp4_gpu(packed, scales, st["w"], st["w_scales"], st["offsets"], out)
        return out
    a, b, offsets, out = st["a"], st["b"], st["offsets"], st["out"]
    ops.grouped_matmul_gpu(a, b, offsets, out)
    if op == "grouped":
        return out
    ops.grouped_matmul_gpu(st["dout"], b.transpose(1, 2), offsets, st["da"])
    ops.grouped_matmul_wgrad_gpu(a, st["dout"], offsets, st["db"])
    return {"out": out, "da": st["da"], "db": st["db"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    rows, K = case["rows"], case["K"]
    if case["op"] == "mxfp4_quantize":
        held = rows * (K // 2 + K // 32)
        # read x, write the 4-bit form, read it, write the values
        return {"bytes": 2 * rows * K + 2 * held + 2 * rows * K, "flops": 4 * rows * K}
    N = case["N"]
    touched = min(case["groups"], rows)  # an expert without a row is not read
    flops = 2 * rows * K * N
    if case["op"] == "mxfp4_linear":
        return {"bytes": 2 * rows * K + touched * N * (K // 2 + K // 32) + 2 * rows * N, "flops": flops}
    forward = 2 * (rows * K + touched * K * N + rows * N)
    if case["op"] == "grouped":
        return {"bytes": forward, "flops": flops}
    # a, b, dout read once; out, da and all of db written once
    return {"bytes": 2 * (2 * rows * K + touched * K * N + case["groups"] * K * N + 2 * rows * N), "flops": 3 * flops}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_quantized(x):
    """The values Q(x) in 64 bits: nearest grid point by distance, ties to the point whose code is even."""
    rows, K = x.shape
    v = x.double().reshape(rows, K // 32, 32)
    top = v.abs().max(dim=2, keepdim=True).values
    X = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    # log2 may round up across a power of two
    X = torch.where(torch.pow(2.0, X) > top, X - 1, X)
    X = torch.where(torch.pow(2.0, X + 1) <= top, X + 1, X) - 2
    X = torch.where(top > 0, X.clamp(-127, 127), torch.full_like(X, -127))
    unit = torch.pow(torch.full_like(X, 2.0), X)
    m = (v / unit).abs()
    # The grid is uniform with step 1/2 up to 2, step 1 up to 4 and step 2 up to 6; torch.round takes ties to even
    # multiples of the step, which are the even codes.
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).double()
    q = (torch.round(m / step) * step).clamp(max=6.0)
    return (torch.copysign(q, v) * unit).reshape(rows, K)


def _exact_weight(packed, blocks):
    N, half = packed.shape
    K = 2 * half
    n = torch.arange(N, device=packed.device).unsqueeze(1)
    k = torch.arange(K, device=packed.device).unsqueeze(0)
    byte = packed.long()[n, k // 2]
    code = torch.where(k % 2 == 0, byte % 16, byte // 16)
    c = k // 32
    where = ((n // 128) * ((K + 127) // 128) + c // 4) * 512 + (n % 32) * 16 + ((n % 128) // 32) * 4 + c % 4
    exponent = blocks.long()[where].double() - 127
    mag = code % 8
    ex, man = mag // 2, (mag % 2).double()
    val = torch.where(ex == 0, man / 2, (1 + man / 2) * torch.pow(2.0, (ex - 1).double()))
    return torch.where(code >= 8, -val, val) * torch.pow(torch.full_like(exponent, 2.0), exponent)


def exact(case, seed):
    st = prepare(case, seed)
    op = st["op"]
    if op == "mxfp4_quantize":
        return torch.cat([_exact_quantized(part) for part in st["x"].split(2048)])
    spans = [(g, lo, hi) for g, (lo, hi) in enumerate(zip(st["bounds"][:-1], st["bounds"][1:])) if hi > lo]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    if op == "mxfp4_linear":
        for g, lo, hi in spans:
            w = torch.cat([_exact_weight(st["w"][g][n:n + 1024], st["w_scales"][g][n // 128 * ((case["K"] + 127) // 128) * 512:])
                           for n in range(0, case["N"], 1024)])
            out[lo:hi] = torch.mm(_exact_quantized(st["x"][lo:hi]), w.T)
        return out
    a, b = st["a"], st["b"]
    for g, lo, hi in spans:
        out[lo:hi] = torch.mm(a[lo:hi].double(), b[g].double())
    if op == "grouped":
        return out
    da = torch.zeros(st["da"].shape, dtype=torch.float64, device="cuda")
    db = torch.zeros(st["db"].shape, dtype=torch.float64, device="cuda")
    for g, lo, hi in spans:
        d = st["dout"][lo:hi].double()
        da[lo:hi] = torch.mm(d, b[g].double().T)
        db[g] = torch.mm(a[lo:hi].double().T, d)
    return {"out": out, "da": da, "db": db}
