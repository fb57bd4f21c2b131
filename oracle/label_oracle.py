"""MX4 label matrices and the preference loss from their definitions, in 64 bits on the CPU, for the tests."""
from __future__ import annotations

import torch


def _short_floats(exponents, mantissa_bits, bias, most):
    """The numbers >= 0 of a format, ascending, by their codes."""
    v = []
    for code in range(exponents << mantissa_bits):
        e, m = code >> mantissa_bits, (code & ((1 << mantissa_bits) - 1)) / (1 << mantissa_bits)
        x = (1 + m) * 2.0 ** (e - bias) if e else m * 2.0 ** (1 - bias)
        if x <= most:
            v.append(x)
    return torch.tensor(v, dtype=torch.float64)


E2M1 = _short_floats(4, 1, 1, 6.0)
E4M3 = _short_floats(16, 3, 7, 448.0)


def round_to(x, grid):
    """The nearest of the grid by magnitude, ties to an even code, the largest beyond; as codes (without the sign)."""
    a = x.abs().double().contiguous()
    hi = torch.searchsorted(grid, a).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - grid[lo], grid[hi] - a
    return torch.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)) | (a >= grid[-1]), hi, lo)


def blocks(x, bits):
    """Signed numbers (rows, blocks, 32) and scale bytes (rows, blocks) of a (rows, dims) matrix: NaN and 255 for blocks with
    anything that is not finite."""
    grid, emax = (E2M1, 2) if bits == 4 else (E4M3, 8)
    x = x.double()
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32)
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    top = torch.where(bad, 1.0, top)
    s = torch.where(top > 0, torch.frexp(top).exponent.double() - 1 - emax, -127.0).clamp(-127, 127)
    y = torch.where(bad[..., None], 0.0, x) * torch.exp2(-s)[..., None]
    v = grid[round_to(y, grid)] * torch.where(y < 0, -1.0, 1.0)
    return torch.where(bad[..., None], torch.nan, v), torch.where(bad, 255, (s + 127).long())


def rounded(x, bits):
    """The matrix that a (rows, dims) matrix becomes."""
    v, s = blocks(x, bits)
    return (v * torch.exp2(s.double() - 127)[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def pack(w):
    """codes and scales as the header lays them out, byte by byte."""
    L, d = w.shape
    v, s = blocks(w, 4)
    nb = v.shape[1]
    code = round_to(torch.nan_to_num(v), E2M1) + 8 * (torch.signbit(v) & ~torch.isnan(v))
    units, steps = -(-L // 64), -(-nb // 4)
    codes = torch.zeros(units, 1024 * nb, dtype=torch.uint8)
    scales = torch.zeros(units, 256 * steps, dtype=torch.uint8)
    for label in range(L):
        u, at = divmod(label, 64)
        p, q, t, r = at >> 5, (at >> 3) & 3, (at >> 2) & 1, at & 3
        tile, row = 2 * p + t, 4 * q + r
        for b in range(nb):
            step = b // 4
            wide = min(4, nb - 4 * step)
            first = step * 4096 + ((tile * 16 + row) * wide + b % 4) * 16
            codes[u, first:first + 16] = (code[label, b, 0::2] + 16 * code[label, b, 1::2]).byte()
            scales[u, step * 256 + (b % 4) * 64 + row * 4 + tile] = int(s[label, b])
    return codes, scales


def topk(z, K):
    """The K largest of each row, the lower label first where they are equal; NaN never: (-inf, -1) where there are fewer."""
    v = torch.where(torch.isnan(z), -torch.inf, z)
    bad = torch.isnan(z)
    order = torch.sort(torch.where(bad, 1, 0), dim=1, stable=True).indices
    v, bad = v.gather(1, order), bad.gather(1, order)
    by = torch.sort(v, dim=1, descending=True, stable=True).indices
    # numbers that are -inf still rank before what is no number
    by = by.gather(1, torch.sort(bad.gather(1, by).long(), dim=1, stable=True).indices)[:, :K]
    label, none = order.gather(1, by), bad.gather(1, by)
    return torch.where(none, -torch.inf, v.gather(1, by)), torch.where(none, -1, label)


def preference(x, w, rowptr, chosen, rejected, reference=None, weight=None, beta=0.1, smoothing=0.0):
    """loss, margins, slopes, gradient of x, and the pairs' rows, by autograd-free formulas in float64."""
    x, w = x.double(), w.double()
    P, B, L = chosen.numel(), x.shape[0], w.shape[0]
    margin, slope = torch.zeros(P, dtype=torch.float64), torch.zeros(P, dtype=torch.float64)
    loss, grad = torch.zeros((), dtype=torch.float64), torch.zeros_like(x)
    row = torch.full((P,), -1)
    for b in range(B):
        for p in range(max(0, int(rowptr[b])), min(P, int(rowptr[b + 1]))):
            c, r = int(chosen[p]), int(rejected[p])
            a = 1.0 if weight is None else float(weight[p])
            if not (0 <= c < L and 0 <= r < L) or a == 0.0:
                continue
            row[p] = b
            diff = w[c] - w[r]
            m = x[b] @ diff - (0.0 if reference is None else float(reference[p]))
            margin[p] = m
            t = beta * m
            loss += a * (-(1 - smoothing) * torch.nn.functional.logsigmoid(t) - smoothing * torch.nn.functional.logsigmoid(-t))
            slope[p] = a * beta * ((1 - smoothing) * -torch.sigmoid(-t) + smoothing * torch.sigmoid(t))
            grad[b] += slope[p] * diff
    return loss, margin, slope, grad, row


def add_to_g(g, row, chosen, rejected, slope):
    """G with the pairs' slopes, in float64."""
    g = g.double().clone()
    for p in range(row.numel()):
        if row[p] >= 0:
            g[row[p], chosen[p]] += slope[p]
            g[row[p], rejected[p]] -= slope[p]
    return g
