"""Attention of packed sequences and the paged cache from their definitions in
64 bits, a sequence and a head at a time, with the bounds on how far a kernel
may be off.

Bounds. H = 2^-8 is half a bf16 step relative to the value (finfo.eps / 2). The
kernels round the probabilities P, and in the backward dS, to bf16 for the
matrix products, and the results; everything else is held in 32 bits.
  out   P off by H of itself: H sum_j P_j |v_j|, and H |out| for the result
  dv    H sum_i P_ij |dout_i| + H |dv|
  dS    H |dS| from its rounding; D = dout . out is formed from the rounded
        out, off by E_i = sum_d |dout_d| (bound of out)_d, which moves dS_ij by
        P_ij E_i
  dq    scale sum_j (bound of dS_ij) |k_j| + H |dq|, and dk likewise over i
FP32 work (exponentials, sums of products) is off by far less: a score off by e
moves P by the factor exp(e), and e <= 128 2^-24 sum_d |q_d k_d| scale, below
2^-12 at these inputs (sums up to 30), so R = 2^-11 of the same sums covers it.
"""

from __future__ import annotations

import math

import torch

H = 2.0 ** -8
R = 2.0 ** -11
# A gradient's distance from 64 bits by its norm, a head's: those bounds are worst
# cases of every value, and leave room for a D that is off. A bf16 rounding is even
# over a step of 2^-7 2^e, 2^-7 / sqrt(12) by its square mean, of values m 2^e whose
# square mean is 1.47 2^e where log m is even: 1.5e-3. Two are in a gradient, dS's
# and its own, of which dS's meets terms that may cancel: 2.1e-3 to 2.7e-3 by
# `gradients_as_rounded` at thousands of keys, and 1.5 times the two together here.
# An out has P's, whose terms do not cancel more, and its own.
# With D from the bf16 out as it is, or without what the rounded dS sum to taken off,
# keys with a direction in common give 4e-3 to 2e-2.
NORM = 3.5e-3


def offsets(lens, device='cuda'):
    return torch.tensor([0] + list(torch.tensor(lens, dtype=torch.int64).cumsum(0)),
                        dtype=torch.int32, device=device)


def attend(q, k, v, lens_q, lens_k, causal=True, scale=None, dout=None, dlse=None):
    """dict of out, lse and their bounds (and dq, dk, dv with dout) in 64 bits;
    rows of no sequence: out 0, lse -inf, gradients 0."""
    q, k, v = (t.detach().double() for t in (q, k, v))
    heads, d = q.shape[1:]
    group = heads // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    res = dict(out=torch.zeros_like(q), out_tol=torch.zeros_like(q),
               lse=torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device),
               lse_tol=torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device))
    if dout is not None:
        dout = dout.double()
        for name, t in (('dq', q), ('dk', k), ('dv', v)):
            res[name], res[name + '_tol'] = torch.zeros_like(t), torch.zeros_like(t)
    i0 = j0 = 0
    for m, n in zip(lens_q, lens_k):
        rows, keys = slice(i0, i0 + m), slice(j0, j0 + n)
        i0, j0 = i0 + m, j0 + n
        if m == 0 or n == 0:
            continue
        see = torch.ones(m, n, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril(n - m)
        some = see.any(-1)
        for h in range(heads):
            g = h // group
            a = (q[rows, h] @ k[keys, g].t()) * scale
            a = a.masked_fill(~see, -math.inf)
            lse = torch.logsumexp(a, -1)
            p = torch.where(see, torch.exp(a - torch.where(some, lse, 0.0)[:, None]), 0.0)
            out = p @ v[keys, g]
            spread = p @ v[keys, g].abs()
            tol = (H + R) * spread + H * out.abs() + 1e-30
            res['out'][rows, h], res['out_tol'][rows, h] = out, tol
            res['lse'][rows, h] = lse
            reach = ((q[rows, h].abs() @ k[keys, g].abs().t()) * scale).amax(-1)
            res['lse_tol'][rows, h] = (reach * 2.0 ** -17 + n * 2.0 ** -24
                                       + 2.0 ** -20 * (1 + torch.where(some, lse, 0.0).abs()))
            if dout is None:
                continue
            go = dout[rows, h]
            dd = (go * out).sum(-1)
            if dlse is not None:
                dd = dd - dlse[rows, h].double()
            ds = p * (go @ v[keys, g].t() - dd[:, None])
            off = (H + R) * ds.abs() + p * ((go.abs() * tol).sum(-1) + R * (go.abs() @ v[keys, g].abs().t()).amax(-1))[:, None]
            res['dv'][keys, g] += p.t() @ go
            res['dv_tol'][keys, g] += (H + R) * (p.t() @ go.abs())
            res['dq'][rows, h] = scale * (ds @ k[keys, g])
            res['dq_tol'][rows, h] = scale * (off @ k[keys, g].abs())
            res['dk'][keys, g] += scale * (ds.t() @ q[rows, h])
            res['dk_tol'][keys, g] += scale * (off.t() @ q[rows, h].abs())
    if dout is not None:
        for name in ('dq', 'dk', 'dv'):
            res[name + '_tol'] += H * res[name].abs() + 1e-30
    return res


def leaning(n, heads, kv, d, seed, device='cuda'):
    """q, k, v, dout in bf16 and dlse of n tokens, queries and keys with a direction in
    common, as they have it after normalisation."""
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g)

    shared = rand(1, 1, d)
    ts = (rand(n, heads, d) + 0.7 * shared, rand(n, kv, d) + 0.7 * rand(n, kv, 1) * shared,
          rand(n, kv, d), rand(n, heads, d))
    return [t.to(torch.bfloat16).to(device) for t in ts] + [rand(n, heads).to(device)]


def gradients_as_rounded(q, k, v, dout, dlse=None, take_off=True, mend=True, sign=1):
    """(dq, dk) of one causal sequence in 64 bits but for the roundings to bf16 of P, dS,
    out and the results. take_off: what the rounded dS of a row sum to beside dlse is
    taken off its dq, times P K; mend: D of dk is mended by what the exact ones sum to;
    sign: of dlse in that sum."""
    def bf16(x):
        return x.to(torch.bfloat16).double()

    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    n, heads, d = q.shape
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    see = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
    for h in range(heads):
        kh, vh = (t[:, h // (heads // k.shape[1])] for t in (k, v))
        a = (q[:, h] @ kh.t() * d ** -0.5).masked_fill(~see, -math.inf)
        p = torch.softmax(a, -1)
        dl = 0.0 * p[:, 0] if dlse is None else dlse[:, h].double()
        dd = (dout[:, h] * bf16(bf16(p) @ vh)).sum(-1) - dl
        dp = dout[:, h] @ vh.t()
        ds = p * (dp - dd[:, None])
        x = bf16(ds) @ kh
        if take_off:
            x += (sign * dl - bf16(ds).sum(-1))[:, None] * (bf16(p) @ kh)
        dq[:, h] = bf16(d ** -0.5 * x)
        if mend:
            ds = p * (dp - (dd + ds.sum(-1) - dl)[:, None])
        dk[:, h // (heads // k.shape[1])] += d ** -0.5 * (bf16(ds).t() @ q[:, h])
    return dq, bf16(dk)


def distance(got, want):
    """The largest of the heads' distances by norm, relative."""
    off = (got.double() - want).norm(dim=(0, 2)) / want.norm(dim=(0, 2))
    return off.max().item()


def check(got, ref, name):
    """Every value of `got` within the bound of ref[name]."""
    want, tol = ref[name], ref[name + '_tol']
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), f'{name}: {(fine != torch.isfinite(got)).sum()} not finite'
    assert torch.equal(got[~fine], want[~fine]), name
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or over.max() <= 0, (
        f'{name}: {(over > 0).sum()} of {over.numel()} values past their bound, by up to '
        f'{over.max():.3g}')


def held(x):
    """What an e4m3 cache holds of rows [.., D]: (values, exponent bytes), from
    the definition in 64 bits."""
    x = x.double()
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448))
    e = torch.where(top > 0, e, -127.0).clamp(min=-127)
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    y = torch.round(y / step) * step * torch.exp2(e)
    return torch.where(torch.isfinite(x), y, math.nan), (e + 127)[..., 0].to(torch.uint8)
