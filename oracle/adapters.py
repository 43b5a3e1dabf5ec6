"""Low-rank adapters beside a projection and counter-based dropout in float64, forward and
gradients, with the error that the kernels' roundings allow for each element (test
infrastructure).

Roundings counted, u = half a step of the 16-bit type relative to the value:
* out, dx, da, db rounded once: u |result|, and half the type's smallest step;
* h = A d(x) and dh = B^T g summed in float32: n 2^-23 of the sum of absolute values for n terms
  (each partial sum is at most that sum, rounded by 2^-24; the factors s_a and 1 / kept share are
  rounded twice more);
* h and dh enter products as two 16-bit parts: u^2 |h|, and in fp16, whose operands are scaled
  to the largest of their row (or of 32 rows' column), what falls below its smallest step: 2^-37 of
  that largest;
* the second products summed in float32: n 2^-23 of the sum of absolute values for n terms.
"""
from __future__ import annotations

import torch

STEP = 2.0 ** -23
# wide features: rows, k, n, rank, adapters, order of the rows' adapters
WIDE = [(1, 4096, 64, 16, 1, "one"), (31, 4168, 1096, 8, 3, "mixed"), (65, 8200, 520, 72, 2, "runs"), (96, 64, 4360, 128, 3, "runs")]
WORD = 0xFFFFFFFF


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def philox(counter, key):
    """Philox 4x32 with 10 rounds in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & WORD, (a >> 32) ^ c[3] ^ k[1], a & WORD]
        k = [(k[0] + 0x9E3779B9) & WORD, (k[1] + 0xBB67AE85) & WORD]
    return c


def kept(rows: int, cols: int, drop: int, seed: int, offset: int) -> torch.Tensor:
    """bool [rows, cols]: the elements that dropout with drop / 65536 keeps."""
    out = torch.empty(rows, -(-cols // 8) * 8, dtype=torch.bool)
    key = (seed & WORD, (seed >> 32) & WORD)
    for r in range(rows):
        bits = []
        for unit in range(-(-cols // 8)):
            for w in philox((unit, r, offset & WORD, (offset >> 32) & WORD), key):
                bits += [(w & 0xFFFF) >= drop, (w >> 16) >= drop]
        out[r] = torch.tensor(bits)
    return out[:, :cols]


def floor(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def low_rank(x, base, a, b, scaling, index, dout=None, mask=None, drop: int = 0):
    """All on the CPU.  -> (out, its error), or with dout ((out, dx, da, db), their errors)."""
    dtype = x.dtype
    u, tiny = half_step(dtype), floor(dtype)
    low = 0.0 if dtype == torch.bfloat16 else 2.0 ** -37
    x, base, a, b, s = x.double(), base.double(), a.double(), b.double(), scaling.double()
    share = 65536 / (65536 - drop) if drop < 65536 else 0.0
    if mask is not None:
        x = torch.where(mask, x, 0.0)
    out, err = base.clone(), torch.zeros_like(base)
    k, n, r = x.shape[1], base.shape[1], a.shape[1]
    if dout is not None:
        g = dout.double()
        dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
        edx, eda, edb = (torch.zeros_like(t) for t in (dx, da, db))
    for i in range(a.shape[0]):
        t = (index == i).nonzero()[:, 0]
        if not len(t):
            continue
        f = float(s[i]) * share
        h, habs = f * (x[t] @ a[i].T), f * (x[t].abs() @ a[i].abs().T)
        eh = (k + 4) * STEP * habs + u * u * h.abs()
        erow = eh + low * h.abs().amax(1, keepdim=True)
        out[t] += h @ b[i].T
        err[t] = erow @ b[i].abs().T + (r + 2) * STEP * (h.abs() @ b[i].abs().T + base[t].abs())
        if dout is None:
            continue
        ecol = eh + low * h.abs().amax(0, keepdim=True)
        m = len(t) + 2
        db[i] = g[t].T @ h
        edb[i] = g[t].abs().T @ ecol + m * STEP * (g[t].abs().T @ h.abs())
        dh, dhabs = f * (g[t] @ b[i]), f * (g[t].abs() @ b[i].abs())
        edh = (n + 4) * STEP * dhabs + u * u * dh.abs()
        dx[t] = dh @ a[i]
        edx[t] = (edh + low * dh.abs().amax(1, keepdim=True)) @ a[i].abs() + (r + 2) * STEP * (dh.abs() @ a[i].abs())
        da[i] = dh.T @ x[t]
        eda[i] = (edh + low * dh.abs().amax(0, keepdim=True)).T @ x[t].abs() + m * STEP * (dh.abs().T @ x[t].abs())
    if dout is None:
        return out, err + u * (out.abs() + err) + tiny
    if mask is not None:
        dx, edx = torch.where(mask, dx, 0.0), torch.where(mask, edx, 0.0)
    values, errors = (out, dx, da, db), (err, edx, eda, edb)
    return values, tuple(e + u * (v.abs() + e) + tiny for v, e in zip(values, errors))


def whole_case(rows, k, n, rank, adapters, dtype, seed):
    """(x, base, a, b, scaling, dout) of whole numbers, small enough that with a dropout of one half every sum
    stays below 2^24 of its units in any order: float32 holds it exactly, two 16-bit parts hold h and dh (one
    does not, where the features are wide), and results equal the formulas' rounded once."""
    g = torch.Generator().manual_seed(seed)

    def ints(most, *shape):
        return torch.randint(-most, most + 1, shape, generator=g).to(dtype)

    scaling = 2.0 ** -torch.randint(7, 10, (adapters,), generator=g).float()
    return ints(31, rows, k), ints(100, rows, n), ints(3, adapters, rank, k), ints(1, adapters, n, rank), scaling, ints(63, rows, n)
