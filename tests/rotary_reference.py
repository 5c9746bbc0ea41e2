"""Norms and rotations of query and key heads from their definitions in 64 bits, with
the bounds on how far a kernel may be off.

Bounds. H = 2^-8 is half a bf16 step relative to the value. Everything up to the one
rounding is in 32 bits: the sum of at most 128 squares is off by 2^-17 of itself at
most and r by half of that, sine and cosine by 2^-20 of one (the instructions are
within 2^-22 over a whole turn, and an angle below half a turn is rounded by 2^-26 of
a turn, 2^-23), each product and sum by 2^-24. S = 2^-16 of the sum of a value's terms
covers them all together.
  y    H |y| + S (|z_a| + |z_b|) for a pair's z = x r w
  dz   S (|dy_a| + |dy_b|)
  dw   S sum (|dy_a| + |dy_b|) |x r|, and its own rounding
  dx   H |dx| + S r (G + |x r| mean(G |x r|)), G = (|dy_a| + |dy_b|) |w|
A row's sum of as many as T H terms, in 32 bits, is a tree with at most 2^10 terms to a
lane and then some 30 joins of partial sums: off by 2^-14 of the sum of magnitudes.
"""

from __future__ import annotations

import torch

H = 2.0 ** -8
S = 2.0 ** -16
LONG = 2.0 ** -13


def angles(positions, rotary, rows):
    """[rows, 1, pairs] radians."""
    if rotary is None:
        return None
    p = positions.double()
    if p.dim() == 1:
        p = p[:, None].expand(rows, rotary.n_axes)
    return (p[:, rotary.axes.long()] * rotary.turns * (2 * torch.pi))[:, None]


def turn(z, angle, adjacent):
    """The rotation of z [rows, heads, D] by the angles of its pairs."""
    if angle is None:
        return z
    n = angle.shape[-1]
    j = torch.arange(n, device=z.device)
    a, b = (2 * j, 2 * j + 1) if adjacent else (j, j + n)
    y = z.clone()
    y[..., a] = z[..., a] * angle.cos() - z[..., b] * angle.sin()
    y[..., b] = z[..., b] * angle.cos() + z[..., a] * angle.sin()
    return y


def both(z, angle, adjacent):
    """|z_a| + |z_b| of a pair at either of its dims, |z| of the dims of no pair."""
    if angle is None:
        return z.abs()
    n = angle.shape[-1]
    j = torch.arange(n, device=z.device)
    a, b = (2 * j, 2 * j + 1) if adjacent else (j, j + n)
    y = z.abs().clone()
    y[..., a] = y[..., b] = z[..., a].abs() + z[..., b].abs()
    return y


def norm_rotate(x, positions, rotary, weight, eps):
    """(y, bound)."""
    x = x.detach().double()
    angle, adjacent = angles(positions, rotary, x.shape[0]), rotary is not None and rotary.interleaved
    z = x
    if eps is not None:
        z = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        if weight is not None:
            z = z * weight.detach().double()
    y = turn(z, angle, adjacent)
    return y, H * y.abs() + S * both(z, angle, adjacent) + 1e-38


def gradients(x, positions, rotary, weight, eps, dy):
    """dict of dx, dw and their bounds."""
    x, dy = x.detach().double(), dy.double()
    angle, adjacent = angles(positions, rotary, x.shape[0]), rotary is not None and rotary.interleaved
    back = None if angle is None else -angle
    dz, reach = turn(dy, back, adjacent), both(dy, back, adjacent)
    if eps is None:
        return dict(dx=dz, dx_tol=H * dz.abs() + S * reach + 1e-38)
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.detach().double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    normal = x * r
    dx = r * (dz * w - normal * (dz * w * normal).mean(-1, keepdim=True))
    big = reach * w.abs()
    tol = S * r * (big + normal.abs() * (big * normal.abs()).mean(-1, keepdim=True))
    dw, most = (dz * normal).sum((0, 1)), (reach * normal.abs()).sum((0, 1))
    unit = 2.0 ** -24 if weight is None or weight.dtype == torch.float32 else H
    return dict(dx=dx, dx_tol=H * dx.abs() + tol + 1e-38, dw=dw, dw_tol=unit * dw.abs() + (S + LONG) * most + 1e-38)


def within(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - tol
    assert not torch.isnan(off).any() and off.max() <= 0 if off.numel() else True, \
        f'off by {off.max().item():.3e} past the bound'
