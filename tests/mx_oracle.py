"""Microscaled 4-bit operands on the CPU in 64 bits, element by element from the definition."""
import torch

# magnitudes and the borders between them; a value on a border goes to the neighbour with the even code
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise(x):
    """Values that ``x`` (any float type, CPU) stands for, blocks of 32 along the last axis, float64."""
    K = x.shape[-1]
    full = torch.zeros(*x.shape[:-1], (K + 31) // 32 * 32, dtype=torch.float64)
    full[..., :K] = x.double()
    b = full.view(*x.shape[:-1], full.shape[-1] // 32, 32)
    a = b.abs().amax(-1, keepdim=True)                     # (NaN if there is one)
    m, e = torch.frexp(torch.where(a.isfinite(), a, 1.0))  # a = m 2^e, m in [0.5, 1)
    e = torch.where(a > 0, e - 3, -127).clamp(-127, 127)
    unit = torch.ldexp(torch.ones_like(a), e)
    q = b / unit
    mag = q.abs()
    out = torch.zeros_like(mag)
    for i, (lo, hi) in enumerate(zip(_VALUES, _VALUES[1:])):
        border = (lo + hi) / 2
        up = mag > border if i % 2 == 0 else mag >= border  # (code i is even: the tie stays)
        out = torch.where(up, torch.full_like(out, hi), out)
    val = torch.copysign(out, q) * unit
    val = torch.where(a.isfinite(), val, torch.full_like(val, float("nan")))
    return val.reshape(full.shape)[..., :K]


def groups(ends):
    start = 0
    for g, e in enumerate(ends):
        yield g, start, e
        start = e


def product(a, w, ends):
    """``a`` [rows, K] and ``w`` [G, N, K] of values: rows of each group times its matrix, and the sum of magnitudes."""
    y = torch.zeros(a.shape[0], w.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(y)
    for g, s, e in groups(ends):
        y[s:e] = a[s:e] @ w[g].T
        mag[s:e] = a[s:e].abs() @ w[g].abs().T
    return y, mag
