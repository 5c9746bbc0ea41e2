"""Norms with rotation, appends with both and chunks over a paged cache without a GPU: the
library refuses bad arguments before any launch, the ops refuse CPU tensors and give
fake outputs of the right shapes, the rules that size a launch keep within what the
kernels take, and the 64-bit reference of the tests agrees with torch."""

import math

import pytest
import torch

from miowtion_amd import _native, kernels, ops_packed, ops_rotary
from tests import rotary_reference as rr

X = 4096  # an aligned address that no refused call reads
BF16 = torch.bfloat16


def _turn(**kw):
    a = dict(pos=X, kind=0, turns=X, axes=X, pairs=64, n_axes=1, adjacent=0, eps=1e-6)
    a.update(kw)
    return [a['pos'], a['kind'], 1, 1, a['turns'], a['axes'], a['pairs'], a['n_axes'], a['adjacent'], None, 0, None,
            0, a['eps']]


def _rotate(q=X, qs=1024, heads=8, kv=2, rows=4, d=128, out=X, **kw):
    _native.call('veda_norm_rotate', q, qs, 128, heads, X, 256, 128, kv, rows, d, *_turn(**kw), out, X, None)


def _rotate_bwd(q=X, heads=8, rows=4, d=128, dq=X, dw=None, work=None, nbytes=0, **kw):
    _native.call('veda_norm_rotate_bwd', q, 1024, 128, dq, 1024, 128, heads, X, 256, 128, X, 256, 128, 2, rows, d,
                 *_turn(**kw), X, X, dw, None, work, nbytes, None)


def _cache(**kw):
    a = dict(sp=4096, ss=128, sh=2048, f8=0, exp=None, pages=4, page=16, width=2)
    a.update(kw)
    return [X, X, a['sp'], a['ss'], a['sh'], a['f8'], a['exp'], a['exp'], 32, 1, 16, a['pages'], a['page'], X, 2,
            a['width']]


def _append(q=X, v=X, heads=8, kv=2, rows=1, d=128, n=1, out=X, turn=None, **kw):
    _native.call('veda_cache_append_rotated', q, 1024, 128, heads, X, 256, 128, v, 256, 128, rows, kv, d, X, X, n,
                 *_cache(**kw), *_turn(**(turn or {})), out, None)


def _chunk(q=X, rows=4, heads=8, kv=2, d=128, n=1, scale=0.1, split=1, units=1, work=None, nbytes=0, **kw):
    _native.call('veda_chunk_fwd', q, 1024, 128, rows, heads, kv, d, X, n, *_cache(**kw), X, 1, scale, split, units, X,
                 1024, 128, None, work, nbytes, None)


@pytest.mark.parametrize('call,kw,match', [
    (_rotate, dict(d=96), 'head_dim'), (_rotate, dict(rows=-1), '2\\^26'), (_rotate, dict(rows=1 << 26), '2\\^26'),
    (_rotate, dict(eps=0.0), 'eps'), (_rotate, dict(eps=1e-31), 'eps'), (_rotate, dict(eps=math.inf), 'eps'),
    (_rotate, dict(eps=math.nan), 'eps'), (_rotate, dict(pairs=65), 'pairs'), (_rotate, dict(pairs=40, d=64), 'pairs'),
    (_rotate, dict(pairs=-8), 'pairs'), (_rotate, dict(pairs=12), 'multiple of 8'), (_rotate, dict(n_axes=0), 'axes'),
    (_rotate, dict(pos=None), 'positions'), (_rotate, dict(turns=None), 'rates'), (_rotate, dict(axes=None), 'rates'),
    (_rotate, dict(kind=3), 'kind'), (_rotate, dict(q=X + 8), '16-byte'), (_rotate, dict(qs=1028), '16-byte'),
    (_rotate, dict(heads=65536), 'heads'), (_rotate, dict(kv=-1), 'heads'), (_rotate, dict(out=X + 2), '16-byte'),
    (_rotate_bwd, dict(d=32), 'head_dim'), (_rotate_bwd, dict(q=X + 8), '16-byte'), (_rotate_bwd, dict(dq=X + 4), '16-byte'),
    (_rotate_bwd, dict(dw=X), 'workspace'), (_rotate_bwd, dict(dw=X, work=X, nbytes=1023), 'workspace'),
    (_rotate_bwd, dict(dw=X, work=X + 4, nbytes=1 << 20), 'workspace'), (_rotate_bwd, dict(dw=X, eps=-1.0), 'weights'),
    (_append, dict(d=32), 'head_dim'), (_append, dict(kv=0), 'key heads'), (_append, dict(page=24), 'pages of'),
    (_append, dict(pages=-1), 'page count'), (_append, dict(ss=132), '16-byte'), (_append, dict(f8=1), 'exponents'),
    (_append, dict(rows=1 << 26), '2\\^26'), (_append, dict(n=1 << 20), '2\\^20'), (_append, dict(v=X + 8), '16-byte'),
    (_append, dict(q=X + 8), '16-byte'), (_append, dict(out=X + 8), '16-byte'),
    (_append, dict(turn=dict(pairs=20)), 'multiple of 8'), (_append, dict(turn=dict(turns=None)), 'rates'),
    (_append, dict(turn=dict(eps=0.0)), 'eps'),
    (_chunk, dict(d=96), 'head_dim'), (_chunk, dict(heads=7), 'multiple'), (_chunk, dict(heads=2 * 65537), 'query heads to'),
    (_chunk, dict(rows=-1), 'negative'), (_chunk, dict(rows=1 << 29), 'past 2'), (_chunk, dict(n=1 << 20), '2\\^20'),
    (_chunk, dict(width=1 << 27), '2\\^31'), (_chunk, dict(ss=1 << 22), 'stride'), (_chunk, dict(scale=0.0), 'scale'),
    (_chunk, dict(scale=math.nan), 'scale'), (_chunk, dict(q=X + 8), '16-byte'), (_chunk, dict(split=0), 'n_split'),
    (_chunk, dict(split=65), 'n_split'), (_chunk, dict(units=0), 'units'), (_chunk, dict(split=2), 'workspace'),
    (_chunk, dict(split=2, work=X, nbytes=4 * 8 * (2 * 130 + 1) * 4 - 1), 'workspace'),
    (_chunk, dict(rows=1 << 25, heads=8, split=2), 'one launch'), (_chunk, dict(f8=1), 'exponents'),
    (_chunk, dict(page=512), 'pages of'),
])
def test_the_library_refuses_before_any_launch(call, kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


def test_calls_without_work_launch_nothing():
    _rotate(rows=0)
    _rotate(heads=0, kv=0)
    _rotate(rows=0, pos=None)
    _rotate_bwd(rows=0)
    _append(rows=0)
    _chunk(rows=0)


@pytest.mark.parametrize('rows', [0, 1, 5000])
def test_gradients_of_no_heads_launch_nothing(rows):
    _native.call('veda_norm_rotate_bwd', X, 1024, 128, X, 1024, 128, 0, None, 0, 0, None, 0, 0, 0, rows, 128, *_turn(), X,
                 None, None, None, None, 0, None)


def _cpu(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    q, k, cu = _cpu(4, 4, 64), _cpu(4, 2, 64), _cpu(2, dtype=torch.int32)
    rot = kernels.rotary(32, device='cpu')
    pos = _cpu(4, dtype=torch.int32)
    cache = kernels.paged_cache(2, 16, 2, 64, device='cpu')
    table, one = _cpu(1, 2, dtype=torch.int32), _cpu(1, dtype=torch.int32)
    for call in (lambda: kernels.norm_rotate(q, k, pos, rot), lambda: kernels.norm_rotate(q, None, eps=1e-6),
                 lambda: kernels.norm_rotate(q.clone().requires_grad_(), k, pos, rot),
                 lambda: kernels.cache_append_rotated_(cache, q, k, k, cu, table, one, rot),
                 lambda: kernels.paged_chunk_attention(q, cu, cache, table, one)):
        with pytest.raises(NotImplementedError, match='no CPU fallback'):
            call()


def test_fake_outputs():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        wide, cu = _cpu(40, 12, 64), _cpu(3, dtype=torch.int32)
        q, k = wide[:, :8], wide[:, 8:10]
        turns, axes, pos = _cpu(32, dtype=torch.float64), _cpu(32, dtype=torch.int32), _cpu(40, dtype=torch.int32)
        w = _cpu(64, dtype=torch.float32)
        rot = (pos, turns, axes, 1, False)
        got = torch.ops.veda.norm_rotate(q, k, *rot, w, w, 1e-6)
        assert [(t.shape, t.is_contiguous()) for t in got] == [(q.shape, True), (k.shape, True)]
        assert len(torch.ops.veda.norm_rotate(q, None, None, None, None, 0, False, None, None, 1e-6)) == 1
        grads = torch.ops.veda.norm_rotate_bwd(q, q, k, k, *rot, w, w, 1e-6, True, False)
        assert [t.shape for t in grads] == [q.shape, k.shape, w.shape] and grads[2].dtype == torch.float32
        pages = _cpu(4, 16, 2, 64)
        table = _cpu(2, 2, dtype=torch.int32)
        out = torch.ops.veda.cache_append_rotated_(pages, pages, None, None, q, k, k, cu, table, cu[:2], *rot, w, w, None)
        assert out.shape == q.shape and out.is_contiguous()
        out, lse = torch.ops.veda.chunk_fwd(q, cu, pages, pages, None, None, table, cu[:2], True, 0.1, True)
        assert out.shape == q.shape and lse.shape == (40, 8) and lse.dtype == torch.float32


def test_caches_that_share_memory_are_not_written():
    q, k, v, cu = _cpu(4, 4, 64), _cpu(4, 2, 64), _cpu(4, 2, 64), _cpu(2, dtype=torch.int32)
    table, one = _cpu(1, 2, dtype=torch.int32), _cpu(1, dtype=torch.int32)
    append = ops_rotary.cache_append_rotated_._fn  # what runs behind the refusal of CPU tensors
    e4m3 = kernels.paged_cache(2, 16, 2, 64, torch.float8_e4m3fn, device='cpu')
    plain = kernels.paged_cache(2, 16, 2, 64, device='cpu')
    exp = e4m3.k_exp[:, :1].expand(-1, 16, -1)
    for cache in (plain._replace(v=plain.k), e4m3._replace(v=e4m3.k), e4m3._replace(v_exp=e4m3.k_exp),
                  e4m3._replace(k_exp=exp, v_exp=exp.clone().as_strided(exp.shape, exp.stride())),
                  kernels.PagedCache(*(t[:1].expand(2, -1, -1, -1) for t in plain[:2]))):
        with pytest.raises(ValueError, match='share memory'):
            append(*cache, q, k, v, cu, table, one, None, None, None, 0, False, None, None, None)


def test_plans():
    rot = kernels.rotary([16, 24, 24], base=500.0, device='cpu')
    assert rot.n_axes == 3 and not rot.interleaved and rot.turns.dtype == torch.float64
    assert rot.axes.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    want = torch.cat([500.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in (16, 24, 24)]) / (2 * math.pi)
    torch.testing.assert_close(rot.turns, want, rtol=1e-15, atol=0)
    assert torch.equal(kernels.rotary(64, device='cpu').turns, kernels.rotary([64], device='cpu').turns)
    assert kernels.rotary(3, interleaved=True, device='cpu').turns.shape == (3,)
    for bad in ([], [0, 8], [8, -8], [65], 65, [12]):
        with pytest.raises(ValueError):
            kernels.rotary(bad, device='cpu')
    for base in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match='base'):
            kernels.rotary(64, base=base, device='cpu')


def test_launch_rules_stay_within_the_kernels():
    for rows in (1, 60, 5000, 1 << 20):
        for kv in (1, 3, 8, 700):
            for group in (1, 7):
                for d in (64, 128):
                    for n in (0, 1, 126, 127, 60000):
                        for capacity in (0, 16, 255, 8192, 1 << 20, (1 << 31) - 1):
                            most, units = ops_packed._chunk_splits(rows, kv * group, kv, d, n, capacity)
                            assert 1 <= most <= 64 and 1 <= units <= 1537
                            # (a single split needs no sums)
                            assert most == 1 or 4 * rows * kv * group * most * (d + 2) <= 1 << 27


def test_the_row_divisions_are_exact_as_far_as_tiles_reach():
    """Rows of a tile past a multiple of the group: up to group + 127."""
    for group in range(2, (1 << 16) + 1):
        m = 0xffffffff // group + 1
        x = (group + 127) // group * group - 1  # the excess grows with the row
        assert x * m >> 32 == x // group and (group + 127) * m >> 32 == (group + 127) // group, group


@pytest.mark.parametrize('interleaved', [False, True])
def test_reference_agrees_with_autograd(interleaved):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(9, 3, 64, generator=g, dtype=torch.float64)
    w = 1 + 0.2 * torch.randn(64, generator=g, dtype=torch.float64)
    dy = torch.randn(9, 3, 64, generator=g, dtype=torch.float64)
    rot = kernels.rotary([8, 16], interleaved=interleaved, device='cpu')
    pos = torch.randint(0, 1000, (9, 2), generator=g)
    angle = rr.angles(pos, rot, 9)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    z = a / (a.square().mean(-1, keepdim=True) + 1e-3).sqrt() * b
    j = torch.arange(24)
    first, second = (2 * j, 2 * j + 1) if interleaved else (j, j + 24)
    pair = torch.complex(z[..., first], z[..., second]) * torch.polar(torch.ones_like(angle), angle)
    y = z.index_copy(2, first, pair.real).index_copy(2, second, pair.imag)
    torch.testing.assert_close(rr.norm_rotate(x, pos, rot, w, 1e-3)[0], y.detach())
    dx, dw = torch.autograd.grad(y, (a, b), dy)
    got = rr.gradients(x, pos, rot, w, 1e-3, dy)
    torch.testing.assert_close(got['dx'], dx)
    torch.testing.assert_close(got['dw'], dw)
