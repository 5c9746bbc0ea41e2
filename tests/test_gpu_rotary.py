"""Norms and rotations of query and key heads (kernels.norm_rotate,
cache_append_rotated_) against their definitions in 64 bits."""

import math

import pytest
import torch

from miowtion_amd import kernels
from tests import packed_reference as pr
from tests import rotary_reference as rr

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _inputs(rows, heads, kv, d, seed=0, wide=False):
    """q and k as views of one projection, weights, and positions."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, heads + 2 * kv, d, generator=g) * torch.exp(torch.randn(rows, heads + 2 * kv, 1, generator=g))
    x = x.to(BF16).cuda()
    wq, wk = (1 + 0.3 * torch.randn(d, generator=g) for _ in range(2))
    dtype = torch.float32 if wide else BF16
    return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], wq.to(dtype).cuda(), wk.to(dtype).cuda()


def _positions(rows, axes, kind, seed=0, far=1 << 20):
    g = torch.Generator().manual_seed(seed + 1)
    p = torch.randint(0, far, (rows, axes), generator=g)
    if kind == torch.float32:
        p = p / 7.0
    return p.to(kind).cuda()


def _both(q, k, pos, rot, wq, wk, eps):
    got = kernels.norm_rotate(q, k, pos, rot, wq, wk, eps)
    for y, x, w in zip(got, (q, k), (wq, wk)):
        assert y.is_contiguous() and y.dtype == BF16
        rr.within(y, *rr.norm_rotate(x, pos, rot, w, eps))


@pytest.mark.parametrize('d,sections', [(128, [64]), (128, [16, 24, 24]), (128, [8]), (128, [40]), (64, [32]),
                                        (64, [8, 12, 12]), (64, [8, 8])])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('rows,heads,kv', [(1, 1, 1), (7, 5, 5), (77, 40, 8), (300, 3, 1), (4500, 8, 2)])
def test_sizes(rows, heads, kv, interleaved, d, sections):
    q, k, _, wq, wk = _inputs(rows, heads, kv, d)
    _both(q, k, _positions(rows, len(sections), torch.int32), kernels.rotary(sections, interleaved=interleaved),
          wq, wk, 1e-6)


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('kind', [torch.int32, torch.int64, torch.float32])
def test_positions_of_every_kind(kind, interleaved):
    rot = kernels.rotary([16, 24, 24], interleaved=interleaved)
    q, k, _, wq, wk = _inputs(50, 6, 2, 128, wide=True)
    pos = _positions(50, 3, kind)
    _both(q, k, pos, rot, wq, wk, 1e-6)
    _both(q, k, pos.t().contiguous().t(), rot, wq, wk, 1e-6)  # axes first
    _both(q, k, pos[:, 0], rot, wq, wk, 1e-6)                 # one for every axis, strided
    _both(q, k, -pos, rot, wq, wk, 1e-6)


@pytest.mark.parametrize('pairs', [1, 3, 31, 33, 64])
def test_few_and_odd_numbers_of_adjacent_pairs(pairs):
    q, k, _, wq, wk = _inputs(20, 3, 2, 128)
    _both(q, k, _positions(20, 1, torch.int32), kernels.rotary(pairs, interleaved=True), wq, wk, 1e-6)


def test_far_positions():
    q, k, *_ = _inputs(64, 4, 1, 128)
    pos = _positions(64, 1, torch.int64, far=(1 << 31) - 1)
    rot = kernels.rotary(64, base=1e6)
    got = kernels.norm_rotate(q, k, pos, rot)
    for y, x in zip(got, (q, k)):
        want, tol = rr.norm_rotate(x, pos, rot, None, None)
        # the product of a position of 31 bits and a rate is off by 2^-53 of itself on either side
        rr.within(y, want, tol + 2.0 ** -18 * rr.both(x.double(), rr.angles(pos, rot, 64), False))


@pytest.mark.parametrize('d', [64, 128])
def test_norm_alone_rotation_alone_and_neither(d):
    q, k, _, wq, wk = _inputs(33, 5, 2, d)
    pos, rot = _positions(33, 1, torch.int32), kernels.rotary(d // 2)
    _both(q, k, None, None, wq, wk, 1e-5)
    _both(q, k, None, None, None, wk, 1e-5)
    _both(q, k, pos, rot, None, None, None)
    _both(q, k, pos, rot, wq, None, 1e-3)
    y, z = kernels.norm_rotate(q, k)
    assert torch.equal(y, q) and torch.equal(z, k)
    y, z = kernels.norm_rotate(q, None, pos, rot, wq, eps=1e-6)
    assert z is None and torch.equal(y, kernels.norm_rotate(q, k, pos, rot, wq, wk, 1e-6)[0])


def test_no_rows():
    q, k, _, wq, wk = _inputs(0, 5, 2, 128)
    y, z = kernels.norm_rotate(q, k, _positions(0, 1, torch.int32), kernels.rotary(64), wq, wk, 1e-6)
    assert y.shape == q.shape and z.shape == k.shape


def test_large_small_and_not_finite_rows():
    q, k, _, wq, _ = _inputs(40, 4, 1, 128)
    q = q.clone()
    q[0] = 3e38          # squares past 32 bits
    q[1] *= 1e30
    q[2] = 0
    q[3] = 1e-30
    q[4, 0, 5], q[5, 1, 70], q[6, 2, 0] = math.inf, math.nan, -math.inf
    pos, rot = _positions(40, 1, torch.int32), kernels.rotary(64)
    got = kernels.norm_rotate(q, None, pos, rot, wq, eps=1e-6)[0]
    want, tol = rr.norm_rotate(q, pos, rot, wq, 1e-6)
    bad = torch.isnan(want)
    assert bad.any() and torch.equal(torch.isnan(got), bad)
    rr.within(torch.where(bad, 0.0, got.double()), torch.where(bad, 0.0, want), torch.where(bad, 1.0, tol))


@pytest.mark.parametrize('d,pairs,interleaved', [(128, 8, False), (128, 7, True), (64, 0, False), (64, 13, True)])
def test_dims_of_no_pair_are_apart(d, pairs, interleaved):
    """An infinity or a NaN in a dim of no pair, its weight or its gradient: in no other dim."""
    rot = kernels.rotary(pairs, interleaved=interleaved) if pairs else None
    q, _, _, wq, _ = _inputs(12, 3, 1, d)
    pos = _positions(12, 1, torch.int32) if pairs else None
    x, w = q.clone(), wq.clone()
    for i in range(12):
        x[i, i % 3, d - 1 - i] = (math.inf, -math.inf, math.nan)[i % 3]
    w[d - 3], w[d - 8] = math.inf, math.nan
    for a, b, eps in ((x, None, None), (x, wq, 1e-6), (q, w, 1e-6)):
        got, (want, tol) = kernels.norm_rotate(a, None, pos, rot, b, eps=eps)[0].double(), rr.norm_rotate(a, pos, rot, b, eps)
        odd = ~torch.isfinite(want)
        assert odd.any() and torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[odd].nan_to_num(7.0), want[odd].nan_to_num(7.0))
        rr.within(torch.where(odd, 0.0, got), torch.where(odd, 0.0, want), torch.where(odd, 1.0, tol))
    leaf = q.clone().requires_grad_(True)
    dx, = torch.autograd.grad(kernels.norm_rotate(leaf, None, pos, rot)[0], leaf, x)
    want = rr.gradients(q, pos, rot, None, None, x)['dx']
    assert torch.equal(torch.isnan(dx), torch.isnan(want)) and torch.equal(torch.isinf(dx), torch.isinf(want))


@pytest.mark.parametrize('d,sections,interleaved', [(128, [64], False), (128, [16, 24, 24], True), (64, [8, 8], False),
                                                    (64, [32], True), (128, None, False)])
@pytest.mark.parametrize('rows,heads,kv', [(1, 1, 1), (77, 5, 2), (611, 8, 2), (5000, 6, 6)])
@pytest.mark.parametrize('wide', [False, True])
def test_gradients(rows, heads, kv, d, sections, interleaved, wide):
    q, k, _, wq, wk = _inputs(rows, heads, kv, d, wide=wide)
    rot = None if sections is None else kernels.rotary(sections, interleaved=interleaved)
    pos = None if rot is None else _positions(rows, len(sections), torch.int32)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
    g = torch.Generator().manual_seed(9)
    dq, dk = (torch.randn(t.shape, generator=g).to(BF16).cuda() for t in (q, k))
    out = kernels.norm_rotate(leaves[0], leaves[1], pos, rot, leaves[2], leaves[3], 1e-6)
    plain = kernels.norm_rotate(q, k, pos, rot, wq, wk, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(out, plain))
    got = torch.autograd.grad(out, leaves, (dq, dk), retain_graph=True)
    again = torch.autograd.grad(out, leaves, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        want = rr.gradients(x, pos, rot, w, 1e-6, dy)
        assert got[2 + i].dtype == w.dtype
        rr.within(got[i], want['dx'], want['dx_tol'])
        rr.within(got[2 + i], want['dw'], want['dw_tol'])


def test_gradients_of_some_inputs():
    q, k, _, wq, wk = _inputs(90, 5, 2, 128)
    pos, rot = _positions(90, 1, torch.int32), kernels.rotary(64)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
    g = torch.Generator().manual_seed(9)
    dq, dk = (torch.randn(t.shape, generator=g).to(BF16).cuda() for t in (q, k))
    whole = torch.autograd.grad(kernels.norm_rotate(*leaves[:2], pos, rot, *leaves[2:], 1e-6), leaves, (dq, dk))
    for which in range(1, 16):
        some = [t if which >> i & 1 else t.detach() for i, t in enumerate(leaves)]
        out = kernels.norm_rotate(some[0], some[1], pos, rot, some[2], some[3], 1e-6)
        mine = [t for t in some if t.requires_grad]
        found = torch.autograd.grad([t for t in out if t.requires_grad], mine,
                                    [t for t, o in zip((dq, dk), out) if o.requires_grad], allow_unused=True)
        for t, w in zip(found, [w for i, w in enumerate(whole) if which >> i & 1]):
            assert torch.equal(t, w)
    # of one result alone, and of neither weight
    out = kernels.norm_rotate(*leaves[:2], pos, rot, *leaves[2:], 1e-6)
    gq, gk, gwq, gwk = torch.autograd.grad(out[0], leaves, dq, allow_unused=True)
    assert gk is None and gwk is None and torch.equal(gq, whole[0]) and torch.equal(gwq, whole[2])
    x = q.detach().clone().requires_grad_(True)
    gx, = torch.autograd.grad(kernels.norm_rotate(x, None, pos, rot)[0], x, dq)
    want = rr.gradients(q, pos, rot, None, None, dq)
    rr.within(gx, want['dx'], want['dx_tol'])


@pytest.mark.parametrize('rows,heads,kv', [(0, 5, 2), (9, 0, 0), (9, 5, 0), (9, 0, 2), (0, 0, 0)])
def test_gradients_of_nothing(rows, heads, kv):
    """No rows, no heads: weights' gradients are zeros where no row is."""
    q, k, _, wq, wk = _inputs(rows, heads, kv, 128)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
    out = kernels.norm_rotate(*leaves[:2], _positions(rows, 1, torch.int32), kernels.rotary(64), *leaves[2:], 1e-6)
    got = torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])
    for x, n, g, w in zip(leaves, (heads, kv), got, got[2:]):
        assert g.shape == x.shape and bool(w.any()) == (rows * n > 0)


def test_gradients_that_are_views():
    """Output gradients in strides of their own, expanded ones among them."""
    q, k, _, wq, wk = _inputs(65, 4, 2, 64)
    pos, rot = _positions(65, 1, torch.int32), kernels.rotary(32)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
    out = kernels.norm_rotate(*leaves[:2], pos, rot, *leaves[2:], 1e-6)
    g = torch.Generator().manual_seed(9)
    dq = torch.randn(4, 65, 64, generator=g).to(BF16).cuda().transpose(0, 1)
    dk = torch.randn(64, generator=g).to(BF16).cuda().expand(65, 2, 64)
    odd = torch.empty(65 * 4 * 64 + 1, dtype=BF16, device='cuda')[1:].view(65, 4, 64).copy_(dq)
    one = torch.ones((), dtype=BF16, device='cuda').expand(65, 4, 64)
    for a in (dq, odd, one):
        got = torch.autograd.grad(out, leaves, (a, dk), retain_graph=True)
        want = torch.autograd.grad(out, leaves, (a.contiguous().clone(), dk.contiguous()), retain_graph=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gradients_against_differences():
    """A step along a direction moves the loss as the gradients say, all in 64 bits on
    the reference's side."""
    q, k, _, wq, _ = _inputs(17, 3, 1, 64, wide=True)
    pos, rot = _positions(17, 1, torch.int32), kernels.rotary(32)
    x, w = q.detach().clone().requires_grad_(True), wq.clone().requires_grad_(True)
    g = torch.Generator().manual_seed(4)
    dy, vx, vw = (torch.randn(s, generator=g).cuda() for s in (q.shape, q.shape, wq.shape))
    dy = dy.to(BF16)
    gx, gw = torch.autograd.grad(kernels.norm_rotate(x, None, pos, rot, w, eps=1e-6)[0], (x, w), dy)

    def loss(h):
        a = q.double() + h * vx.double()
        z = a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (wq.double() + h * vw.double())
        return (rr.turn(z, rr.angles(pos, rot, 17), False) * dy.double()).sum()

    h = 1e-4
    moved = ((loss(h) - loss(-h)) / (2 * h)).item()
    said = (gx.double() * vx.double()).sum().item() + (gw.double() * vw.double()).sum().item()
    # dx is rounded to bf16: each term by H of itself
    tol = rr.H * (gx.double() * vx.double()).abs().sum().item() + 1e-4 * abs(moved) + 1e-4
    assert abs(moved - said) <= tol


# ---------------------------------------------------------------------------
# into a cache


def _cache(lens, page, kv, d, dtype, seed=0):
    """(cache, table): pages in no order, what is not written not finite."""
    need = sum(-(-n // page) for n in lens) + 2
    g = torch.Generator().manual_seed(seed)
    order, at = torch.randperm(need, generator=g).to(torch.int32), 0
    table = torch.full((len(lens), max(1, max(-(-n // page) for n in lens))), 1 << 30, dtype=torch.int32)
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order[at:at + m]
        at += m
    cache = kernels.paged_cache(need, page, kv, d, dtype)
    for t in cache[:2]:
        (t.view(torch.uint8) if dtype == E4M3 else t).fill_(0x7f if dtype == E4M3 else math.nan)
    return cache, table.cuda()


def _starts(lens, new):
    return torch.tensor([n - m for n, m in zip(lens, new)], dtype=torch.int32, device='cuda')


@pytest.mark.parametrize('d,sections,interleaved', [(128, [64], False), (128, [16, 24, 24], True), (64, [16], False),
                                                    (64, [32], True), (128, None, False)])
@pytest.mark.parametrize('heads,kv', [(1, 1), (40, 8), (6, 3)])
@pytest.mark.parametrize('own', [True, False])
def test_append_is_norm_rotate_then_append(heads, kv, d, sections, interleaved, own):
    """Bit for bit in bf16."""
    lens, new = [40, 1, 16, 300, 0, 33], [40, 1, 3, 17, 0, 32]
    rows = sum(new) + 5  # five rows of no sequence behind the last
    q, k, v, wq, wk = _inputs(rows, heads, kv, d)
    rot = None if sections is None else kernels.rotary(sections, interleaved=interleaved)
    pos = None if rot is None or own else _positions(rows, len(sections), torch.int64)
    cache, table = _cache(lens, 16, kv, d, BF16)
    other = kernels.PagedCache(cache.k.clone(), cache.v.clone())
    start, cu = _starts(lens, new), pr.offsets(new)
    got = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, pos, wq, wk, 1e-6)
    at = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)] + [torch.zeros(5, dtype=torch.int64)]).cuda()
    y, z = kernels.norm_rotate(q, k, None if rot is None else at if own else pos, rot, wq, wk, 1e-6)
    kernels.cache_append_(other, z, v, cu, table, start)
    assert torch.equal(got[:-5], y[:-5]) and not got[-5:].any()
    for a, b in zip(cache[:2], other[:2]):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('kv', [1, 3, 8])
@pytest.mark.parametrize('normed', [True, False])
def test_append_in_eight_bits(d, kv, normed):
    """The key's value in 32 bits rounded once; V as cache_append_ holds it."""
    lens, new = [50, 2, 130], [50, 1, 17]
    rows = sum(new)
    q, k, v, wq, wk = _inputs(rows, 2 * kv, kv, d)
    if not normed:
        wq = wk = None
    eps = 1e-6 if normed else None
    rot = kernels.rotary(d // 2)
    cache, table = _cache(lens, 16, kv, d, E4M3)
    other = kernels.PagedCache(*(t.clone() for t in cache))
    start, cu = _starts(lens, new), pr.offsets(new)
    got = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, None, wq, wk, eps)
    at = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).cuda()
    assert torch.equal(got, kernels.norm_rotate(q, None, at, rot, wq, eps=eps)[0])
    kernels.cache_append_(other, k, v, cu, table, start)
    assert torch.equal(cache.v.view(torch.uint8), other.v.view(torch.uint8))
    assert torch.equal(cache.v_exp, other.v_exp)
    want, tol = rr.norm_rotate(k, at, rot, wk, eps)
    tol = tol - rr.H * want.abs()  # what 32 bits are off by
    held = kernels.cache_gather(cache, pr.offsets(lens), table, sum(lens))[0]
    i0 = j0 = 0
    for n, m in zip(lens, new):
        w, t, y = want[i0:i0 + m], tol[i0:i0 + m], held[j0 + n - m:j0 + n].double()
        # a code is off by 2^-4 of the value, and by 2^-10 of the row's power of two below
        # 2^-6 of it; that power is at most 2^-7 of the largest value
        rr.within(y, w, 2.0 ** -4 * (w.abs() + t) + t + 2.0 ** -17 * w.abs().amax(-1, keepdim=True))
        i0, j0 = i0 + m, j0 + n


def _codes(x, e):
    """x [.., D] in 64 bits as e4m3 values at the exponents e [..], rounded once."""
    y = x / torch.exp2(e - 127)[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('normed', [True, False])
def test_append_in_eight_bits_rounds_once(d, normed):
    """Codes and exponents of the keys are those of the value in 64 bits, wherever what 32
    bits may be off by leaves no other; by way of bf16 they are not."""
    lens, new, kv = [300, 130], [300, 117], 4
    q, k, v, wq, wk = _inputs(sum(new), kv, kv, d)
    if not normed:
        wq = wk = None
    eps = 1e-6 if normed else None
    rot = kernels.rotary(d // 2)
    cache, table = _cache(lens, 32, kv, d, E4M3)
    other = kernels.PagedCache(*(t.clone() for t in cache))
    start, cu = _starts(lens, new), pr.offsets(new)
    kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, None, wq, wk, eps)
    at = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).cuda()
    kernels.cache_append_(other, kernels.norm_rotate(q, k, at, rot, wq, wk, eps)[1], v, cu, table, start)

    want, tol = rr.norm_rotate(k, at, rot, wk, eps)
    tol = tol - rr.H * want.abs()  # what 32 bits are off by
    top, off = want.abs().amax(-1), tol.amax(-1)
    lo, e, up = (127 + torch.ceil(torch.log2(t / 448)) for t in (top - off, top, top + off))
    sure_row = (lo == e) & (e == up)
    codes = _codes(want, e)
    sure = sure_row[..., None] & (_codes(want - tol, e) == codes) & (_codes(want + tol, e) == codes)
    # a row is at a power's border in one of 2^13 cases, a value of a code's step, 2^-4 to
    # 2^-3 of it, in one of 2^11 where it is as large as its pair's other
    assert sure_row.float().mean() > 0.99 and sure.float().mean() > 0.98
    seq = torch.cat([torch.full((m,), b) for b, m in enumerate(new)]).cuda()
    page = table[seq, at // 32].long()

    def found(c):
        return c.k[page, at % 32].double(), c.k_exp[page, at % 32]

    held, power = found(cache)
    assert torch.equal(power[sure_row].double(), e[sure_row])
    assert torch.equal(held[sure], codes[sure])
    held, power = found(other)
    assert (held[sure] != codes[sure]).any()


@pytest.mark.parametrize('dtype', [BF16, E4M3])
def test_append_leaves_out_what_has_no_page(dtype):
    lens = [20, 20, 20]
    q, k, v, wq, wk = _inputs(15, 4, 2, 128)
    cache, table = _cache(lens, 16, 2, 128, dtype)
    table[0, 1] = -1                      # a page outside the cache
    start = torch.tensor([14, 30, -3], dtype=torch.int32, device='cuda')  # past the table; before it
    before = [t.view(torch.uint8).clone() if t is not None else None for t in cache]
    cu = torch.tensor([0, 5, 10, 15], dtype=torch.int32, device='cuda')
    rot = kernels.rotary(64)
    got = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, None, wq, wk, 1e-6)
    at = (start[:, None] + torch.arange(5, device='cuda')).reshape(-1)
    assert torch.equal(got, kernels.norm_rotate(q, None, at, rot, wq, eps=1e-6)[0])
    written = {(int(table[0, 0]), 14), (int(table[0, 0]), 15), (int(table[1, 1]), 14), (int(table[1, 1]), 15),
               (int(table[2, 0]), 0), (int(table[2, 0]), 1)}
    for t, b in zip(cache[:2], before):
        changed = (t.view(torch.uint8) != b).flatten(2).any(-1).nonzero().tolist()
        assert {tuple(c) for c in changed} == written


@pytest.mark.parametrize('rows', [1, 3, 70, 5000])
def test_streams_and_graphs(rows):
    """On a stream of its own and replayed, new values in the captured tensors."""
    q, k, v, wq, wk = _inputs(rows, 8, 2, 128)
    q, k, v = (t.clone() for t in (q, k, v))
    rot = kernels.rotary(64)
    cache, table = _cache([rows + 7], 32, 2, 128, BF16)
    start, cu = torch.zeros(1, dtype=torch.int32, device='cuda'), pr.offsets([rows])
    pos = _positions(rows, 1, torch.int32)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def both():
        return (*kernels.norm_rotate(q, k, pos, rot, wq, wk, 1e-6),
                kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, None, wq, wk, 1e-6))

    with torch.cuda.stream(stream):
        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = both()
    for shift in (0, 7, 3):
        start.fill_(shift)
        pos += 11
        q.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        held = cache.k.clone()
        cache.k.zero_()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        there = cache.k.view(torch.int16) != 0
        assert torch.equal(held.view(torch.int16)[there], cache.k.view(torch.int16)[there])


def test_a_captured_training_step():
    q, k, _, wq, wk = _inputs(200, 4, 2, 64)
    pos, rot = _positions(200, 1, torch.int32), kernels.rotary(32)
    g = torch.Generator().manual_seed(9)
    dq, dk = (torch.randn(t.shape, generator=g).to(BF16).cuda() for t in (q, k))
    static = [t.detach().clone() for t in (q, k, wq, wk)]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in static]
        out = kernels.norm_rotate(*leaves[:2], pos, rot, *leaves[2:], 1e-6)
        return (*out, *torch.autograd.grad(out, leaves, (dq, dk)))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    for _ in range(3):
        static[0].mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_past_32_bits():
    """Strides that put a row more than 2^31 values on."""
    wide = torch.zeros(3, (1 << 30) + 1024, dtype=BF16, device='cuda')
    q = wide.as_strided((3, 2, 128), ((1 << 30) + 1024, 128, 1))
    g = torch.Generator().manual_seed(3)
    q.copy_(torch.randn(3, 2, 128, generator=g))
    pos, rot = _positions(3, 1, torch.int32), kernels.rotary(64)
    y, _ = kernels.norm_rotate(q, None, pos, rot, eps=1e-6)
    assert torch.equal(y, kernels.norm_rotate(q.clone(), None, pos, rot, eps=1e-6)[0])


def test_refusals():
    q, k, v, wq, wk = _inputs(20, 4, 2, 128)
    pos, rot = _positions(20, 2, torch.int32), kernels.rotary([32, 32])
    ok = dict(positions=pos, rotary=rot, q_weight=wq, k_weight=wk, eps=1e-6)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            kernels.norm_rotate(*(args or (q, k)), **{**ok, **kw})

    refused('equal rows', q, k[:10])
    refused('bfloat16', q.float(), k)
    refused('16-byte', torch.zeros(20, 4, 136, dtype=BF16, device='cuda')[..., 4:132], k)
    refused('positions', positions=pos[:10])
    refused('positions', positions=pos[:, :1])
    refused('positions', positions=pos.double())
    refused('needs positions', positions=None)
    refused('have no use', rotary=None)
    refused('no norm', eps=None)
    refused('eps', eps=0.0)
    refused('eps', eps=math.nan)
    refused('eps', eps=1e-35)
    refused('q_weight', q_weight=wq[:64])
    refused('k_weight', k_weight=wk.half())
    refused('pairs', q[..., :64].contiguous(), k[..., :64].contiguous(), q_weight=None, k_weight=None)
    refused('multiple of 8', rotary=kernels.Rotary(rot.turns[:20], rot.axes[:20], 2, False))
    refused('float64', rotary=kernels.Rotary(rot.turns.float(), rot.axes, 2, False))
    for bad in ([], [0, 8], [65], [12]):
        with pytest.raises(ValueError):
            kernels.rotary(bad)
    with pytest.raises(ValueError, match='base'):
        kernels.rotary(64, base=0.0)
    cache, table = _cache([20], 16, 2, 128, BF16)
    start, cu = torch.zeros(1, dtype=torch.int32, device='cuda'), pr.offsets([20])
    for bad, match in (((kernels.PagedCache(cache.k, cache.k), q, k, v), 'share memory'),
                       ((kernels.PagedCache(cache.k[:, :1].expand(-1, 16, -1, -1), cache.v), q, k, v), 'alike|share'),
                       ((cache, q, k, v[:, :1]), 'alike'), ((cache, q, k[:, :1], v[:, :1]), 'key heads'),
                       ((cache, q, k[:10], v[:10]), 'equal rows')):
        with pytest.raises(ValueError, match=match):
            kernels.cache_append_rotated_(*bad, cu, table, start, rot, pos, wq, wk, 1e-6)
    with pytest.raises(ValueError, match='cu'):
        kernels.cache_append_rotated_(cache, q, k, v, cu.long(), table, start, rot, pos, wq, wk, 1e-6)


def test_second_order_gradients_are_refused():
    q, k, _, wq, wk = _inputs(5, 2, 1, 64)
    x = q.detach().clone().requires_grad_(True)
    y, _ = kernels.norm_rotate(x, None, eps=1e-6)
    gx, = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable|does not require grad|twice'):
        torch.autograd.grad(gx.float().sum(), x)
