"""Rotary positions from the definition, in float64 on the CPU: every pair as a complex number."""

import torch


def rotate64(x, positions, table, axes, gain, layout, *, inverse=False):
    """(y, bound): x (B, H, N, D) turned, and |x0| + |x1| of each entry's pair times gain (0 past rotary_dim)."""
    x = x.detach().cpu().double()
    pos = positions.detach().cpu().double()
    pos = pos[..., None] if pos.ndim == 2 else pos
    table = table.cpu()
    per = table.numel() // axes
    angle = torch.stack([pos[..., p // per] * table[p] for p in range(table.numel())], dim=-1)[:, None]
    if inverse:
        angle = -angle
    turn = torch.polar(torch.full_like(angle, gain), angle)
    R = 2 * table.numel()
    a, b = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    y, bound = x.clone(), torch.zeros_like(x)
    z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
    y[..., a], y[..., b] = z.real, z.imag
    size = (x[..., a].abs() + x[..., b].abs()) * abs(gain)
    bound[..., a], bound[..., b] = size, size
    return y, bound


def assert_turned(got, want, bound, what):
    """|got - want| <= bound * 7 * 2^-24 + half a step of got's dtype.

    cos and sin come within 4 units of 2^-24 (the rounded rest of the angle, their sums' cut and roundings), the product
    with gain adds one more, and y = x0 c - x1 s rounds twice: in all (|x0| + |x1|) gain (4 + 1 + 2) 2^-24.  Then one rounding to the output's type, half a step relative (or half the
    smallest subnormal)."""
    fi = torch.finfo(got.dtype)
    tol = bound * 7 * 2.0 ** -24 + want.abs() * fi.eps / 2 * (1 + 2.0 ** -20) + fi.smallest_normal * fi.eps / 2
    err = (got.detach().cpu().double() - want).abs()
    worst = float((err - tol).max()) if err.numel() else 0.0
    assert torch.all(err <= tol), f"{what}: off by {float(err.max()):.3e}, {worst:.3e} past the bound"
