"""Packed sequences and the paged cache without a GPU: the library refuses bad
arguments before any launch, the ops refuse CPU tensors and give fake outputs of
the right shapes, the rules that size a launch keep within what the kernels
take, and the 64-bit reference of the tests agrees with torch."""

import math

import pytest
import torch

from miowtion_amd import _native, kernels, ops_packed
from tests import packed_reference as pr

X = 4096  # an aligned address that no refused call reads


def _fwd(**kw):
    a = dict(q=X, qs=1024, qh=128, k=X, ks=256, kh=128, v=X, vs=256, vh=128, rows=16, k_rows=16,
             heads=8, kv=2, d=128, n=1, scale=0.1, split=1, out=X, os=1024, oh=128, work=None, nbytes=0)
    a.update(kw)
    _native.call('veda_packed_fwd', a['q'], a['qs'], a['qh'], a['k'], a['ks'], a['kh'], a['v'], a['vs'],
                 a['vh'], a['rows'], a['k_rows'], a['heads'], a['kv'], a['d'], X, X, a['n'], 1, a['scale'],
                 a['split'], a['out'], a['os'], a['oh'], None, a['work'], a['nbytes'], None)


def _bwd(**kw):
    a = dict(d=128, heads=8, kv=2, rows=16, k_rows=16, n=1, scale=0.1, split=1, nbytes=1 << 20, q=X, qs=1024)
    a.update(kw)
    _native.call('veda_packed_bwd', a['q'], a['qs'], 128, X, 256, 128, X, 256, 128, X, 1024, 128, X, 1024, 128,
                 X, None, a['rows'], a['k_rows'], a['heads'], a['kv'], a['d'], X, X, a['n'], 1, a['scale'],
                 a['split'], X, X, X, X, a['nbytes'], None)


def _cache(**kw):
    a = dict(sp=4096, ss=128, sh=2048, f8=0, exp=None, pages=4, page=16, width=2)
    a.update(kw)
    return [X, X, a['sp'], a['ss'], a['sh'], a['f8'], a['exp'], a['exp'], 32, 1, 16, a['pages'], a['page'], X, 2,
            a['width']]


def _append(rows=1, kv=2, d=128, k=X, ks=256, n=1, **kw):
    _native.call('veda_cache_append', k, ks, 128, X, 256, 128, rows, kv, d, X, X, n, *_cache(**kw), None)


def _gather(rows=1, kv=2, d=128, n=1, **kw):
    _native.call('veda_cache_gather', *_cache(**kw), X, n, rows, kv, d, X, X, None)


def _paged(n=1, heads=8, kv=2, d=128, scale=0.1, chunk=128, work=None, nbytes=0, q=X, **kw):
    _native.call('veda_paged_fwd', q, 1024, 128, n, heads, kv, d, *_cache(**kw), X, scale, chunk, X, 1024,
                 128, None, work, nbytes, None)


@pytest.mark.parametrize('call,kw,match', [
    (_fwd, dict(d=96), 'head_dim'), (_fwd, dict(heads=7), 'multiple'), (_fwd, dict(kv=0), 'multiple'),
    (_fwd, dict(rows=-1), 'negative'), (_fwd, dict(rows=1 << 29), 'past 2'), (_fwd, dict(n=1 << 20), '2\\^20'),
    (_fwd, dict(n=(1 << 20) - 1, heads=64, kv=64), 'one launch'),
    (_fwd, dict(scale=0.0), 'scale'), (_fwd, dict(scale=math.nan), 'scale'), (_fwd, dict(scale=math.inf), 'scale'),
    (_fwd, dict(q=X + 8), '16-byte'), (_fwd, dict(ks=260), '16-byte'), (_fwd, dict(out=X + 2), '16-byte'),
    (_fwd, dict(ks=1 << 24), 'stride'), (_fwd, dict(split=0), 'n_split'), (_fwd, dict(split=65), 'n_split'),
    (_fwd, dict(split=2), 'workspace'), (_fwd, dict(split=2, work=X, nbytes=2 * 16 * 8 * 130 * 4 - 1), 'workspace'),
    (_bwd, dict(d=80), 'head_dim'), (_bwd, dict(heads=3), 'multiple'), (_bwd, dict(k_rows=-1), 'negative'),
    (_bwd, dict(scale=-1.0), 'scale'), (_bwd, dict(q=X + 4), '16-byte'), (_bwd, dict(qs=1 << 24), 'stride'),
    (_bwd, dict(split=65), 'n_split'), (_bwd, dict(nbytes=100), 'workspace'),
    (_bwd, dict(split=2, nbytes=6 * 1024 + 2 * 2 * 16 * 2 * 128 * 4 - 1), 'workspace'),
    (_append, dict(d=32), 'head_dim'), (_append, dict(kv=0), 'key heads'), (_append, dict(page=24), 'pages of'),
    (_append, dict(page=512), 'pages of'), (_append, dict(pages=-1), 'page count'),
    (_append, dict(ss=132), '16-byte'), (_append, dict(f8=1), 'exponents'), (_append, dict(f8=1, exp=X, ss=136), '16-byte'),
    (_append, dict(rows=-1), 'negative'), (_append, dict(rows=1 << 26), 'rows'), (_append, dict(k=X + 8), '16-byte'),
    (_gather, dict(d=32), 'head_dim'), (_gather, dict(rows=1 << 26), 'rows'), (_gather, dict(page=8), 'pages of'),
    (_gather, dict(width=-1), 'width'),
    (_paged, dict(heads=7), 'multiple'), (_paged, dict(n=65536), '65535'), (_paged, dict(scale=0.0), 'scale'),
    (_paged, dict(chunk=48), 'chunk'), (_paged, dict(chunk=0), 'chunk'), (_paged, dict(chunk=128 * 16 + 32), 'chunk'),
    (_paged, dict(chunk=64, page=128), 'chunk'), (_paged, dict(width=1 << 27), '2\\^31'),
    (_paged, dict(ss=1 << 22), 'stride'), (_paged, dict(width=64), 'workspace'), (_paged, dict(q=X + 8), '16-byte'),
    (_paged, dict(width=64, work=X, nbytes=8 * 8 * 132 * 4 - 1), 'workspace'),
])
def test_the_library_refuses_before_any_launch(call, kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


@pytest.mark.parametrize('group', [(1 << 16) + 1, 70000, 150000])
def test_more_heads_to_a_key_head_than_the_row_loads_divide_by_are_refused(group):
    """The forward and the backward find a row's token by a product with 2^32 / group,
    which is exact up to 65,536 and wrong for row group - 1 of the first past it."""
    with pytest.raises(ValueError, match='query heads to a key head'):
        _fwd(heads=group, kv=1, rows=1)
    with pytest.raises(ValueError, match='query heads to a key head'):
        _bwd(heads=group, kv=1, rows=1)


def test_rows_that_a_step_cannot_address_are_copied():
    at = 1 << 24
    for group, stride, copied in ((1, (64, at, 1), False), (2, (64, at, 1), True), (1, (at, 64, 1), True),
                                  (2, (64, at - 64, 1), False), (65, (64, at - 64, 1), True)):
        t = torch.empty(1, dtype=torch.bfloat16).expand(2, 65, 64).as_strided((1, 1, 1), (1, 1, 1)).expand(2, 65, 64)
        got, (_, s, h) = ops_packed._near(t, [0, *stride[:2]], group, -1)
        assert ((s, h) == (65 * 64, 64)) == copied and got.is_contiguous() == copied


def test_the_row_loads_division_is_exact_for_every_group_that_is_taken():
    """A product with ceil(2^32 / group) can only be too large, and first at the rows
    before a multiple of the group; rows go up to group + 63."""
    for group in range(2, (1 << 16) + 1):
        m = 0xffffffff // group + 1
        # the excess grows with the row, so the last such row decides
        x = (group + 63) // group * group - 1
        assert x * m >> 32 == x // group, group
    group = (1 << 16) + 1
    assert (group - 1) * (0xffffffff // group + 1) >> 32 == 1


def test_calls_without_work_launch_nothing():
    _fwd(rows=0)
    _append(rows=0)
    _append(n=0)
    _gather(rows=0)
    _paged(n=0)


def _cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    q, k, cu = _cpu(4, 4, 64), _cpu(4, 2, 64), _cpu(2, dtype=torch.int32)
    cache = kernels.paged_cache(2, 16, 2, 64, device='cpu')
    table, one = _cpu(1, 2, dtype=torch.int32), _cpu(1, dtype=torch.int32)
    for call in (lambda: kernels.packed_attention(q, k, k, cu),
                 lambda: kernels.packed_attention(q.requires_grad_(), k, k, cu),
                 lambda: kernels.cache_append_(cache, k, k, cu, table, one),
                 lambda: kernels.cache_gather(cache, cu, table, 4),
                 lambda: kernels.paged_attention(q[:1], cache, table, one)):
        with pytest.raises(NotImplementedError, match='no CPU fallback'):
            call()
    assert not kernels.supports(q, 'packed')


def test_fake_outputs():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k, cu = _cpu(40, 8, 64), _cpu(30, 2, 64), _cpu(3, dtype=torch.int32)
        out, lse = torch.ops.veda.packed_fwd(q, k, k, cu, cu, True, 0.1, True)
        assert out.shape == q.shape and out.dtype == q.dtype
        assert lse.shape == (40, 8) and lse.dtype == torch.float32
        grads = torch.ops.veda.packed_bwd(q, k, k, out, out, lse, None, cu, cu, True, 0.1)
        assert [g.shape for g in grads] == [q.shape, k.shape, k.shape]
        pages, exp = _cpu(4, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), _cpu(4, 16, 2, dtype=torch.uint8)
        table = _cpu(2, 2, dtype=torch.int32)
        got = torch.ops.veda.cache_gather(pages, pages, exp, exp, cu, table, 50)
        assert [(g.shape, g.dtype) for g in got] == [((50, 2, 64), torch.bfloat16)] * 2
        out, = torch.ops.veda.paged_fwd(q[:2], pages, pages, exp, exp, table, cu[:2], 0.1, False)
        assert out.shape == (2, 8, 64)


def test_launch_rules_stay_within_the_kernels():
    for n in (1, 3, 64, 5000):
        for kv in (1, 8):
            for group in (1, 7, 40):
                for page in ops_packed.PAGES:
                    for width in (1, 2, 9, 100, 4000):
                        c = ops_packed._chunk(n, kv, group, width * page, page)
                        assert c % 32 == 0 and c % page == 0 and page <= c <= 128 * page
    for q_rows in (1, 100, 4000, 100000):
        for k_rows in (0, 1, 5000, 200000):
            for n in (0, 1, 7, 3000):
                for heads, kv in ((1, 1), (8, 8), (40, 8)):
                    assert 1 <= ops_packed._key_splits(q_rows, k_rows, n, heads, kv) <= 32
                    assert 1 <= ops_packed._splits(k_rows, kv) <= 16


def test_reference_agrees_with_torch():
    g = torch.Generator().manual_seed(0)
    lens_q, lens_k = [5, 0, 9], [8, 3, 9]
    q, k, v, go = (torch.randn(n, h, 64, generator=g, dtype=torch.float64)
                   for n, h in ((14, 4), (20, 2), (20, 2), (14, 4)))
    ref = pr.attend(q, k, v, lens_q, lens_k, dout=go)
    ts = [t.clone().requires_grad_(True) for t in (q, k, v)]
    outs, i, j = [], 0, 0
    for m, n in zip(lens_q, lens_k):
        kk, vv = (t[j:j + n].repeat_interleave(2, 1).transpose(0, 1) for t in ts[1:])
        s = ts[0][i:i + m].transpose(0, 1) @ kk.transpose(1, 2) / 8
        s = s.masked_fill(~torch.ones(m, n, dtype=torch.bool).tril(n - m), -math.inf)
        outs.append((torch.softmax(s, -1) @ vv).transpose(0, 1))
        i, j = i + m, j + n
    out = torch.cat(outs)
    torch.testing.assert_close(ref['out'], out)
    for name, x in zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, ts, go)):
        torch.testing.assert_close(ref[name], x)


@pytest.mark.parametrize('through_lse', [False, True])
@pytest.mark.parametrize('d', [64, 128])
def test_the_bound_by_norm_tells_the_row_sums_correction(d, through_lse):
    """Gradients rounded as the kernels round them are within it, and past it without
    each part of the correction, for the long sequence that the GPU's test has."""
    n = 3001
    q, k, v, dout, dlse = (t[:n] for t in pr.leaning(n + 70, 4, 2, d, seed=0, device='cpu'))
    dlse = dlse if through_lse else None
    ref = pr.attend(q, k, v, [n], [n], dout=dout, dlse=dlse)
    dq, dk = pr.gradients_as_rounded(q, k, v, dout, dlse)
    assert pr.distance(dq, ref['dq']) < pr.NORM and pr.distance(dk, ref['dk']) < pr.NORM
    dq, _ = pr.gradients_as_rounded(q, k, v, dout, dlse, take_off=False)
    assert pr.distance(dq, ref['dq']) > pr.NORM
    _, dk = pr.gradients_as_rounded(q, k, v, dout, dlse, mend=False)
    assert pr.distance(dk, ref['dk']) > pr.NORM
    if through_lse:
        dq, _ = pr.gradients_as_rounded(q, k, v, dout, dlse, sign=-1)
        assert pr.distance(dq, ref['dq']) > pr.NORM


def test_reference_of_held_rows_agrees_with_torch():
    x = torch.randn(200, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16) * 30
    values, byte = pr.held(x)
    unit = torch.exp2(byte.double() - 127)[:, None]
    assert torch.equal((x.double() / unit).float().to(torch.float8_e4m3fn).double() * unit, values)
    top = x.double().abs().amax(-1, keepdim=True) / unit
    assert (top <= 448).all() and (top > 224).all()


def _shared_caches():
    """(cache, what of it shares memory): caches whose rows cannot all be written."""
    cache = kernels.paged_cache(2, 16, 2, 64, torch.float8_e4m3fn, device='cpu')
    heads, rows = cache.k_exp[:, :, :1].expand(-1, -1, 2), cache.k_exp[:, :1].expand(-1, 16, -1)
    for exp in (heads, rows):
        yield cache._replace(k_exp=exp, v_exp=exp.clone().as_strided(exp.shape, exp.stride()))
        yield cache._replace(v_exp=exp, k_exp=exp.clone().as_strided(exp.shape, exp.stride()))
    yield cache._replace(v_exp=cache.k_exp)
    yield cache._replace(v=cache.k)
    plain = kernels.paged_cache(2, 16, 2, 64, device='cpu')
    yield plain._replace(v=plain.k)
    yield kernels.PagedCache(*(t[:1].expand(2, -1, -1, -1) for t in plain[:2]))


def test_caches_that_share_memory_are_not_written():
    k, cu = _cpu(4, 2, 64), _cpu(2, dtype=torch.int32)
    table, one = _cpu(1, 2, dtype=torch.int32), _cpu(1, dtype=torch.int32)
    append = ops_packed.cache_append_._fn  # what runs behind the refusal of CPU tensors
    v = _cpu(4, 2, 64)
    for cache in _shared_caches():
        with pytest.raises(ValueError, match='share memory'):
            append(*cache, k, v, cu, table, one)
