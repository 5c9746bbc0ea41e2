"""Gradients of packed attention against the formulas in 64 bits, against
differences, and through captured graphs."""

import math

import pytest
import torch

from miowtion_amd import kernels, ops_packed
from tests import packed_reference as pr
from tests.test_gpu_packed import CASES, _inputs

pytestmark = pytest.mark.gpu


def _grads(q, k, v, cu_q, cu_k, causal, dout, dlse=None):
    ts = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, lse = kernels.packed_attention(*ts, cu_q, cu_k, causal=causal, return_lse=True)
    outs, grads = ([out], [dout]) if dlse is None else ([out, lse], [dout, dlse])
    return torch.autograd.grad(outs, ts, grads)


@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}')
def test_gradients(case):
    lens_q, lens_k, heads, kv, d, causal = case
    lens_k = lens_k or lens_q
    print(f'packed gradients {case}', flush=True)
    q, k, v = _inputs(lens_q, lens_k, heads, kv, d, seed=1)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    cu_q, cu_k = pr.offsets(lens_q), pr.offsets(lens_k)
    got = _grads(q, k, v, cu_q, cu_k, causal, dout)
    ref = pr.attend(q, k, v, lens_q, lens_k, causal, dout=dout)
    for name, g in zip(('dq', 'dk', 'dv'), got):
        pr.check(g, ref, name)
    for a, b in zip(got, _grads(q, k, v, cu_q, cu_k, causal, dout)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('d', [64, 128])
def test_gradient_through_the_lse(d):
    lens = [70, 1, 200]
    q, k, v = _inputs(lens, lens, 6, 2, d, seed=4)
    g = torch.Generator().manual_seed(2)
    dout = torch.randn(q.shape, generator=g).to(torch.bfloat16).cuda()
    dlse = torch.randn(q.shape[:2], generator=g).cuda()
    cu = pr.offsets(lens)
    ref = pr.attend(q, k, v, lens, lens, dout=dout, dlse=dlse)
    for name, x in zip(('dq', 'dk', 'dv'), _grads(q, k, v, cu, None, True, dout, dlse)):
        pr.check(x, ref, name)
    # the LSE alone
    ts = [t.requires_grad_(True) for t in (q, k, v)]
    _, lse = kernels.packed_attention(*ts, cu, return_lse=True)
    got = torch.autograd.grad(lse, ts, dlse)
    ref = pr.attend(q, k, v, lens, lens, dout=torch.zeros_like(dout), dlse=dlse)
    for name, x in zip(('dq', 'dk', 'dv'), got):
        pr.check(x, ref, name)


def test_gradients_are_the_differences():
    """A step of the loss along a direction is the gradient's product with it. The
    loss in 64 bits of the exact out at both ends; the gradient within its bound."""
    lens = [33, 90]
    q, k, v = _inputs(lens, lens, 4, 2, 64, seed=6)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    got = _grads(q, k, v, pr.offsets(lens), None, True, dout)
    ref = pr.attend(q, k, v, lens, lens, dout=dout)
    g = torch.Generator(device='cuda').manual_seed(3)
    for i, name in enumerate(('dq', 'dk', 'dv')):
        way = torch.randn(got[i].shape, generator=g, device='cuda', dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            xs = [t.double() for t in (q, k, v)]
            xs[i] = xs[i] + sign * 1e-5 * way
            ends.append((pr.attend(*xs, lens, lens)['out'] * dout.double()).sum())
        diff = (ends[0] - ends[1]) / 2e-5
        mine = (got[i].double() * way).sum()
        # the central difference is off by about 1e-10 of third derivatives here
        tol = (ref[name + '_tol'] * way.abs()).sum() + 1e-6 * (1 + diff.abs())
        assert (mine - diff).abs() <= tol, (name, mine.item(), diff.item(), tol.item())


@pytest.mark.parametrize('through_lse', [False, True])
@pytest.mark.parametrize('d', [64, 128])
def test_distance_of_long_sequences_by_norm(d, through_lse):
    """Thousands of keys with a direction in common: what the rounded dS of a row sum
    to would meet their mean."""
    n, heads, kv = 3001, 4, 2
    q, k, v, dout, dlse = pr.leaning(n + 70, heads, kv, d, seed=0)
    dlse = dlse if through_lse else None
    got = _grads(q, k, v, pr.offsets([n, 70]), None, True, dout, dlse)
    ref = pr.attend(q, k, v, [n, 70], [n, 70], dout=dout, dlse=dlse)
    for name, x in zip(('dq', 'dk', 'dv'), got):
        off = pr.distance(x[:n], ref[name][:n])
        print(f'{name} {off:.2e}', flush=True)
        assert off < pr.NORM
        pr.check(x, ref, name)


def test_rows_and_keys_of_no_sequence_get_zeros():
    lens = [50, 200]
    q, k, v = _inputs(lens, lens, 4, 2, 128, pad_q=150, pad_k=140)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    k[250:], v[250:], q[250:], dout[250:] = math.nan, math.inf, math.nan, math.nan
    got = _grads(q, k, v, pr.offsets(lens), None, True, dout)
    ref = pr.attend(q[:250], k[:250], v[:250], lens, lens, dout=dout[:250])
    for name, x in zip(('dq', 'dk', 'dv'), got):
        pr.check(x[:250], ref, name)
        assert (x[250:] == 0).all()
    got = _grads(q, k, v, pr.offsets([0, 0]), None, True, dout)
    assert all((x == 0).all() for x in got)


def test_a_sequence_that_is_not_finite_stays_alone():
    lens = [60, 150, 40]
    q, k, v = _inputs(lens, lens, 4, 2, 128)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    cu = pr.offsets(lens)
    clean = _grads(q, k, v, cu, None, True, dout)
    q[100], k[110], v[120], dout[130] = math.nan, math.inf, math.nan, math.inf
    for a, b in zip(clean, _grads(q, k, v, cu, None, True, dout)):
        assert torch.equal(a[:60], b[:60]) and torch.equal(a[210:], b[210:])


def test_expanded_inputs_and_gradients():
    """Key heads shared by a stride of 0, and an output gradient of one value."""
    lens = [100, 28]
    q, k, v = _inputs(lens, lens, 4, 1, 64)
    cu = pr.offsets(lens)
    ts = [t.requires_grad_(True) for t in (q, k, v)]
    out = kernels.packed_attention(q, k.expand(-1, 2, -1), v.expand(-1, 2, -1), cu)
    out.sum().backward()
    ref = pr.attend(q, k, v, lens, lens, dout=torch.ones_like(q))
    # the two heads' gradients are rounded to bf16 before autograd adds them and
    # rounds again: up to 2^-8 more of each, of at most the sum of magnitudes
    pr.check(ts[0].grad, ref, 'dq')
    for name, t in (('dk', ts[1]), ('dv', ts[2])):
        ref[name + '_tol'] = 2 * ref[name + '_tol'] + 2.0 ** -7 * _half_sums(q, k, v, lens)[name]
        pr.check(t.grad, ref, name)


def test_output_gradients_in_any_place():
    """A transposed gradient, and one that begins off a 16-byte boundary."""
    lens = [70, 3]
    q, k, v = _inputs(lens, lens, 4, 2, 64)
    cu = pr.offsets(lens)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    want = _grads(q, k, v, cu, None, True, dout)
    turned = dout.transpose(0, 1).contiguous().transpose(0, 1)
    moved = torch.empty(dout.numel() + 8, dtype=dout.dtype, device='cuda')[1:1 + dout.numel()].view(dout.shape)
    moved.copy_(dout)
    for d in (turned, moved):
        for a, b in zip(_grads(q, k, v, cu, None, True, d), want):
            assert torch.equal(a, b)


def _half_sums(q, k, v, lens):
    """Per pair of query heads the gradient's magnitude, summed."""
    res = None
    for h in (0, 2):
        r = pr.attend(q[:, h:h + 2], k, v, lens, lens, dout=torch.ones_like(q[:, :2]))
        part = {n: r[n].abs() for n in ('dk', 'dv')}
        res = part if res is None else {n: res[n] + part[n] for n in res}
    return res


def test_graph_of_forward_and_backward():
    """Captured beside an eager graph of the same leaves that is still alive, and
    replayed for new lengths with the program's own work between."""
    q, k, v = _inputs([300], [300], 4, 2, 128)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    cu = pr.offsets([100, 200])

    def step():
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = kernels.packed_attention(a, b, c, cu)
        return (out.detach(), *torch.autograd.grad(out, (a, b, c), dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for lens in ([100, 200], [300, 0], [1, 299], [77, 130]):
        cu.copy_(pr.offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
        ref = pr.attend(q, k, v, lens, lens, dout=dout)
        for name, x in zip(('out', 'dq', 'dk', 'dv'), held):
            pr.check(x, ref, name)


FAR = [
    # heads, kv, d, row stride, head stride: past what a step's 32-bit offsets reach
    (4, 2, 64, None, 1 << 24),
    (2, 2, 128, None, (1 << 24) + 128),          # a head to a group: no head offset in a step
    (2, 1, 128, 1 << 24, None),
    (65, 1, 64, None, (1 << 24) - 64),           # in reach each, not over the group
]


@pytest.mark.parametrize('case', FAR, ids=lambda c: f'{c[0]}-{c[1]}-{c[2]}')
def test_queries_in_strides_past_32_bit_offsets(case):
    """Every layout of q that the forward takes has gradients, the same bits as a
    contiguous q's."""
    heads, kv, d, s, h = case
    lens = [7, 4] if s else [70, 33]
    q, k, v = _inputs(lens, lens, heads, kv, d, seed=9)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    s, h = s or d, h or d
    room = torch.empty((sum(lens) - 1) * s + (heads - 1) * h + d, dtype=q.dtype, device='cuda')
    far = room.as_strided(q.shape, (s, h, 1))
    far.copy_(q)
    print(f'q in strides {far.stride()}', flush=True)
    cu = pr.offsets(lens)
    want = _grads(q, k, v, cu, None, True, dout)
    for a, b in zip(_grads(far, k, v, cu, None, True, dout), want):
        assert torch.equal(a, b)
    ref = pr.attend(q, k, v, lens, lens, dout=dout)
    for name, x in zip(('dq', 'dk', 'dv'), want):
        pr.check(x, ref, name)
    # an output gradient laid out so, straight into the op
    out, lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
    far.copy_(dout)
    for a, b in zip(ops_packed.packed_bwd(q, k, v, out, far, lse, None, cu, cu, True, d ** -0.5), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('group', [65535, 65536])
def test_the_largest_groups(group):
    """Without a mask the heads of one key head are rows of one head."""
    print(f'{group} query heads to a key head', flush=True)
    lens, d = [2, 1], 64
    q, k, v = _inputs(lens, lens, group, 1, d, seed=10)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    cu = pr.offsets(lens)
    out = kernels.packed_attention(q, k, v, cu, causal=False)
    ref = pr.attend(q.view(-1, 1, d), k, v, [n * group for n in lens], lens, False, dout=dout.view(-1, 1, d))
    pr.check(out.view(-1, 1, d), ref, 'out')
    for name, x in zip(('dq', 'dk', 'dv'), _grads(q, k, v, cu, None, False, dout)):
        pr.check(x.view(-1, 1, d), ref, name)


def test_rows_too_wide_for_gradients_are_refused_by_the_forward():
    q = torch.zeros(2, 1 << 17, 128, dtype=torch.bfloat16, device='cuda')
    k = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device='cuda')
    cu = pr.offsets([2])
    assert (kernels.packed_attention(q, k, k, cu) == 0).all()
    with pytest.raises(ValueError, match='gradients need'):
        kernels.packed_attention(q.requires_grad_(), k, k, cu)


def test_only_some_inputs_require_grad_and_second_order_is_refused():
    lens = [40]
    q, k, v = _inputs(lens, lens, 2, 2, 64)
    v.requires_grad_(True)
    out = kernels.packed_attention(q, k, v, pr.offsets(lens))
    dout = torch.ones_like(out)
    ref = pr.attend(q, k, v, lens, lens, dout=dout)
    dv, = torch.autograd.grad(out, v, dout, create_graph=True)
    pr.check(dv.detach(), ref, 'dv')
    with pytest.raises(RuntimeError):
        dv.sum().backward()


def test_refusals():
    q, k, v = _inputs([16], [16], 4, 2, 128)
    cu = pr.offsets([16])
    out, lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
    f = ops_packed.packed_bwd
    for bad, match in [
            (lambda: f(q, k, v, out[:8], out, lse, None, cu, cu, True, 0.1), 'must be as q'),
            (lambda: f(q, k, v, out, out.float(), lse, None, cu, cu, True, 0.1), 'bfloat16'),
            (lambda: f(q, k, v, out, out, lse.t(), None, cu, cu, True, 0.1), 'lse must be'),
            (lambda: f(q, k, v, out, out, lse, lse.half(), cu, cu, True, 0.1), 'dlse must be'),
            (lambda: f(q, k, v, out, out, lse, None, cu, cu, True, 0.0), 'scale')]:
        with pytest.raises(ValueError, match=match):
            bad()
