"""Plain 64-bit forms of the grouped and microscaled operators, and the error bounds their kernels have to keep."""
from __future__ import annotations

import numpy as np
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def spans(bounds, rows):
    """Rows of each group as the operators read a table: clamped, an entry below an earlier one counts as that one."""
    out, at = [], min(max(bounds[0], 0), rows)
    for b in bounds[1:]:
        nxt = max(at, min(max(b, 0), rows))
        out.append((at, nxt))
        at = nxt
    return out


def bound(exact: torch.Tensor, mass: torch.Tensor, terms: int, dtype) -> torch.Tensor:
    """Largest error of a sum of `terms` exact products accumulated in fp32 and rounded once to `dtype`.

    mass = sum of |products|. Each of the fp32 additions is off by at most one unit in the last place of a partial sum,
    which is at most 2^-23 of the mass (the tensor core truncates where IEEE would round); the final rounding by half a
    step of the type, or half its smallest subnormal."""
    acc = (terms + 1) * 2.0 ** -23 * mass
    half = torch.finfo(dtype).eps / 2
    return half * (exact.abs() + acc) + acc + torch.finfo(dtype).smallest_normal * half


def check(got: torch.Tensor, exact: torch.Tensor, mass: torch.Tensor, terms: int) -> None:
    err = (got.double() - exact).abs()
    lim = bound(exact, mass, terms, got.dtype)
    bad = ~(err <= lim)
    # Round to nearest gives an infinity from half a step behind the type's largest number on: that step is eps / 2 times
    # the power of two above it. A sum that may reach this border within its accumulated error may come out infinite.
    fi = torch.finfo(got.dtype)
    top = 2.0 ** np.ceil(np.log2(fi.max))
    border = fi.max + top * fi.eps / 4
    over = (exact.abs() + (terms + 1) * 2.0 ** -23 * mass >= border) & got.isinf() & (got.sign() == exact.sign())
    bad &= ~over
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((err / lim).nan_to_num(nan=float('inf')).max()):.3g} of the bound, first at {bad.nonzero()[0].tolist()}"


def product(a, b):
    """(a . b, |a| . |b|) in 64 bits."""
    a, b = a.double(), b.double()
    return a @ b, a.abs() @ b.abs()


# ---------------------------------------------------------------- microscaled 4-bit values
def quantize(x: torch.Tensor):
    """[rows, K] -> (values, exponents X [rows, K/32]) in 64 bits; NaN values for a block that is not finite."""
    rows, K = x.shape
    v = x.double().reshape(rows, K // 32, 32)
    top = v.abs().amax(dim=2)
    finite = torch.isfinite(v).all(dim=2)
    m, e = torch.frexp(torch.where(finite, top, torch.ones_like(top)))
    X = torch.where(top > 0, (e - 3).clamp(-127, 127), torch.full_like(e, -127))
    unit = torch.ldexp(torch.ones_like(top), X).unsqueeze(2)
    s = (v / unit).nan_to_num(nan=0.0, posinf=0.0, neginf=0.0)
    grid = GRID.to(x.device)
    d = (s.abs().unsqueeze(-1) - grid).abs()
    # nearest code; of two equally near ones the even code
    near = d == d.amin(dim=-1, keepdim=True)
    codes = torch.arange(8, device=x.device)
    rank = torch.where(near, codes % 2, 2)
    code = rank.argmin(dim=-1)
    val = torch.copysign(grid[code], v) * unit
    val = torch.where(finite.unsqueeze(2), val, torch.nan)
    return val.reshape(rows, K), torch.where(finite, X, torch.full_like(X, 128))


def codes_of(packed: torch.Tensor) -> torch.Tensor:
    return torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)


def scale_index(slot_of_row, row_in_slot, K: int) -> np.ndarray:
    """Byte position of every scale [rows, K/32] of rows whose slot and place in it are given."""
    c = np.arange(K // 32)[None, :]
    r = np.asarray(row_in_slot)[:, None]
    s = np.asarray(slot_of_row)[:, None].astype(np.int64)
    return (s * ((K + 127) // 128) + c // 4) * 512 + (r % 32) * 16 + (r // 32) * 4 + c % 4


def slots(group_spans):
    """(rows, slot, place) of all rows of all groups: a group starts a new slot of 128 rows."""
    rows, slot, place, at = [], [], [], 0
    for lo, hi in group_spans:
        n = np.arange(hi - lo)
        rows.append(lo + n)
        slot.append(at + n // 128)
        place.append(n % 128)
        at += (hi - lo + 127) // 128
    return np.concatenate(rows), np.concatenate(slot), np.concatenate(place), at
