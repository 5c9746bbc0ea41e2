"""Attention of a chunk of new tokens over a paged cache (kernels.paged_chunk_attention)
against its definition in 64 bits."""

import math

import pytest
import torch

from miowtion_amd import kernels, ops_packed
from tests import packed_reference as pr
from tests import rotary_reference as rr

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
TYPES = pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])


def _filled(lens, page, kv, d, dtype, seed=0, width=None, scale=1.0):
    """(cache, table, k, v): a cache of these sequences, whose pages lie in no order and
    whose other rows are not finite, and the values that it stands for, packed."""
    g = torch.Generator().manual_seed(seed)
    need = sum(-(-n // page) for n in lens) + 3
    table = torch.full((len(lens), width or max(1, max(-(-n // page) for n in lens))), 1 << 30, dtype=torch.int32)
    order, at = torch.randperm(need, generator=g).to(torch.int32), 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order[at:at + m]
        at += m
    table = table.cuda()
    cache = kernels.paged_cache(need, page, kv, d, dtype)
    for t in cache[:2]:
        (t.view(torch.uint8) if dtype == E4M3 else t).fill_(0x7f if dtype == E4M3 else math.nan)
    for t in cache[2:]:
        if t is not None:
            t.fill_(255)
    k, v = ((torch.randn(sum(lens), kv, d, generator=g) * scale).to(BF16).cuda() for _ in range(2))
    kernels.cache_append_(cache, k, v, pr.offsets(lens), table, torch.zeros(len(lens), dtype=torch.int32, device='cuda'))
    if dtype == E4M3:
        k, v = (pr.held(t)[0].to(BF16) for t in (k, v))
    return cache, table, k, v


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _queries(rows, heads, d, seed=0):
    return torch.randn(rows, heads, d, generator=torch.Generator().manual_seed(seed + 7)).to(BF16).cuda()


def _check(got, want):
    out, lse = got
    rr.within(out, want['out'], want['out_tol'])
    none = want['lse'] == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert not out[none].any()
    rr.within(torch.where(none, 0.0, lse.double()), torch.where(none, 0.0, want['lse']), want['lse_tol'])
    assert (out.double() - want['out']).norm() <= pr.NORM * want['out'].norm() + 1e-30


CASES = [  # (lengths, new), query heads, key heads
    (([1], [1]), 1, 1),
    (([16, 1, 0, 40], [1, 1, 0, 3]), 5, 1),
    (([70, 64, 65, 300], [4, 64, 1, 17]), 8, 2),
    (([513, 129, 128], [130, 129, 1]), 4, 4),
    (([1000, 3, 700], [33, 5, 0]), 14, 2),     # a sequence with more queries than keys
    (([2049], [300]), 3, 1),
    (([5000, 4100], [5, 2]), 40, 8),
]


@TYPES
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('page', [16, 32, 64, 256])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('sizes,heads,kv', CASES, ids=['x'.join(map(str, c[0][0])) for c in CASES])
def test_chunks(sizes, heads, kv, causal, page, d, dtype):
    lens, new = sizes
    cache, table, k, v = _filled(lens, page, kv, d, dtype)
    q = _queries(sum(new), heads, d)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), causal, return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens, causal))
    alone = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), causal)
    assert torch.equal(alone, got[0])


@TYPES
@pytest.mark.parametrize('n_seq', [60, 63, 64, 130, 400])
def test_many_sequences(n_seq, dtype):
    g = torch.Generator().manual_seed(n_seq)
    lens = torch.randint(0, 200, (n_seq,), generator=g).tolist()
    new = [min(n, m) for n, m in zip(lens, torch.randint(0, 9, (n_seq,), generator=g).tolist())]
    cache, table, k, v = _filled(lens, 16, 2, 64, dtype)
    q = _queries(sum(new), 6, 64)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens))


@TYPES
@pytest.mark.parametrize('d', [64, 128])
def test_long_contexts(d, dtype):
    """Over several windows of 64 steps, a table much wider than the sequences, and by norm."""
    lens, new = [9000, 20000, 130], [3, 40, 2]
    cache, table, k, v = _filled(lens, 16, 1, d, dtype, width=4096)
    q = _queries(sum(new), 4, d)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    want = pr.attend(q, k, v, new, lens)
    _check(got, want)
    assert (got[0].double() - want['out']).norm() <= pr.NORM * want['out'].norm()


@TYPES
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('rows', [15, 16, 17, 31, 32, 33, 127, 128, 129])
def test_rows_about_the_tiles_sizes(rows, d, dtype):
    """One head to a key head: as many rows as new tokens, beside a short and a long one."""
    lens, new = [900, 700, 40], [rows, 1, 40]
    cache, table, k, v = _filled(lens, 16, 2, d, dtype)
    q = _queries(sum(new), 2, d)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens))


@TYPES
@pytest.mark.parametrize('heads', [31, 33, 130, 200])
def test_many_heads_to_a_key_head(heads, dtype):
    lens, new = [300, 77], [2, 3]
    cache, table, k, v = _filled(lens, 32, 1, 64, dtype)
    q = _queries(sum(new), heads, 64)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens))


@TYPES
@pytest.mark.parametrize('n_seq', [126, 127, 140])
def test_many_sequences_with_long_ones(n_seq, dtype):
    """About as many sequences as are ordered by length, with keys that are split."""
    lens = [4000, 1500] + [20] * (n_seq - 3) + [2500]
    new = [3, 40] + [1] * (n_seq - 3) + [20]
    cache, table, k, v = _filled(lens, 16, 1, 64, dtype)
    q = _queries(sum(new), 3, 64)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens))


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('new', [[3], [60]])
@pytest.mark.parametrize('power', [-60, 0, 60])
def test_e4m3_keys_with_queries_of_every_size(power, new, d):
    """Values of a query that differ by 2^24 within its blocks of 32, rows of zeros, and rows
    and keys far from one, whose products are scores as usual."""
    lens = [400]
    cache, table, k, v = _filled(lens, 16, 1, d, E4M3, scale=2.0 ** -power)
    v = v.clone()
    q = _queries(new[0], 4, d).float()
    q = q * torch.exp2(-torch.randint(0, 24, q.shape, generator=torch.Generator().manual_seed(2))).cuda()
    q[..., ::9] = _queries(new[0], 4, d, seed=3).float()[..., ::9]
    q[0, 1] = 0
    q = (q * 2.0 ** power).to(BF16)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens))


@TYPES
def test_unsplit_long_walks(dtype):
    """Enough rows that no key is split, over many windows."""
    lens, new = [9000, 6000], [700, 1030]
    cache, table, k, v = _filled(lens, 32, 4, 64, dtype)
    q = _queries(sum(new), 40, 64)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens))


@TYPES
def test_agrees_with_one_token_and_with_the_gathered_rows(dtype):
    lens = [1, 400, 1700]
    cache, table, k, v = _filled(lens, 64, 2, 128, dtype)
    q = _queries(3, 10, 128)
    got = kernels.paged_chunk_attention(q, pr.offsets([1, 1, 1]), cache, table, _ints(lens), return_lse=True)
    want = kernels.paged_attention(q, cache, table, _ints(lens), return_lse=True)
    assert (got[0].float() - want[0].float()).abs().max() <= 2.0 ** -7 * want[0].float().abs().max()
    assert (got[1] - want[1]).abs().max() <= 1e-4
    new = [1, 40, 900]
    q = _queries(sum(new), 10, 128)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens))
    gathered = kernels.cache_gather(cache, pr.offsets(lens), table, sum(lens))
    want = kernels.packed_attention(q, *gathered, pr.offsets(new), pr.offsets(lens))
    assert (got.float() - want.float()).norm() <= 4e-3 * want.float().norm()


@TYPES
@pytest.mark.parametrize('lens,new', [([300, 90], [40, 9]), ([6000, 5000], [3, 2])])
def test_pages_outside_the_cache_draw_no_weight(lens, new, dtype):
    cache, table, k, v = _filled(lens, 16, 2, 128, dtype)
    for b, p, bad in ((0, 0, -1), (0, 5, 1 << 30), (0, 6, -(1 << 31)), (1, 5, cache.k.shape[0]), (1, 0, -7)):
        table[b, p] = bad
    q = _queries(sum(new), 4, 128)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    k, v = k.double(), v.double()
    there = torch.ones(sum(lens), dtype=torch.bool, device='cuda')
    for b, p in ((0, 0), (0, 5), (0, 6), (1, 5), (1, 0)):
        at = sum(lens[:b]) + 16 * p
        there[at:at + 16] = False
    out, lse = (torch.zeros(sum(new), 4, 128, device='cuda').double(), torch.zeros(sum(new), 4, device='cuda').double())
    i0 = j0 = 0
    for n, m in zip(lens, new):
        see = torch.ones(m, n, dtype=torch.bool, device='cuda').tril(n - m) & there[j0:j0 + n]
        for h in range(4):
            a = (q[i0:i0 + m, h].double() @ k[j0:j0 + n, h // 2].t() / math.sqrt(128)).masked_fill(~see, -math.inf)
            lse[i0:i0 + m, h] = torch.logsumexp(a, -1)
            out[i0:i0 + m, h] = torch.softmax(a, -1) @ v[j0:j0 + n, h // 2]
        i0, j0 = i0 + m, j0 + n
    assert (got[1].double() - lse).abs().max() <= 1e-4
    # out: two roundings of 2^-9 in square mean, as NORM
    assert (got[0].double() - out).norm() <= pr.NORM * out.norm()


@TYPES
def test_lengths_out_of_range_no_pages_and_rows_of_no_sequence(dtype):
    lens, new = [100, 40, 33], [5, 4, 3]
    cache, table, k, v = _filled(lens, 16, 2, 64, dtype)
    q = _queries(20, 4, 64)  # eight rows of no sequence
    cu = _ints([2, 7, 11, 14])
    got = kernels.paged_chunk_attention(q, cu, cache, table, _ints([100, -5, 0]), return_lse=True)
    want = pr.attend(q[2:7], k[:100], v[:100], [5], [100])
    _check([t[2:7] for t in got], want)
    for at in (slice(0, 2), slice(7, 20)):
        assert not got[0][at].any() and (got[1][at] == -math.inf).all()
    # a length past the table is the table's width, whose last positions have no page
    wide = torch.cat([table, torch.full((3, 2), -1, dtype=torch.int32, device='cuda')], 1)
    full = kernels.paged_chunk_attention(q[2:7], _ints([0, 5, 5, 5]), cache, table[:1].expand(3, -1),
                                         _ints([112, 0, 0]), causal=False)
    over = kernels.paged_chunk_attention(q[2:7], _ints([0, 5, 5, 5]), cache, table[:1].expand(3, -1),
                                         _ints([(1 << 31) - 1, 0, 0]), causal=False)
    assert torch.equal(torch.isnan(full), torch.isnan(over)) and wide.shape[1] == 9
    empty = kernels.paged_cache(0, 16, 2, 64, dtype)
    out, lse = kernels.paged_chunk_attention(q, cu, empty, table, _ints(lens), return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    out, lse = kernels.paged_chunk_attention(q, cu, cache, table[:, :0], _ints(lens), return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    none = kernels.paged_chunk_attention(q[:0], _ints([0]), cache, table[:0], _ints([]), return_lse=True)
    assert none[0].shape == (0, 4, 64)
    out, lse = kernels.paged_chunk_attention(q, _ints([0]), cache, table[:0], _ints([]), return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


@TYPES
@pytest.mark.parametrize('lens,new', [([200], [60]), ([5000], [3])])
def test_values_that_are_not_finite(lens, new, dtype):
    """What a row does not see does not touch it; what it sees does."""
    cache, table, k, v = _filled(lens, 16, 1, 128, dtype)
    q = _queries(new[0], 2, 128)
    # (rows that are formed key by key have their probabilities in 32 bits, the others in
    # bf16: both within the bound, not the same bits)
    clean = pr.attend(q, k, v, new, lens)
    n, m = lens[0], new[0]
    hidden = n - m + m // 2  # the rows from m / 2 on see it
    page, at = int(table[0, hidden // 16]), hidden % 16
    for t, bad in ((cache.v, [math.nan, math.inf, -math.inf]), (cache.k, [math.nan])):
        for b in bad:
            old = t[page, at].clone()
            if dtype == E4M3:
                t.view(torch.uint8)[page, at, :, 5] = 0x7f
            else:
                t[page, at, :, 5] = b
            got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens))
            rr.within(got[:m // 2], clean['out'][:m // 2], clean['out_tol'][:m // 2])
            assert not torch.isfinite(got[m // 2:, :, 5]).any()
            t.view(torch.uint8)[page, at] = old.view(torch.uint8)


@TYPES
def test_layouts(dtype):
    """Rows and heads in other strides: tokens beside each other, a wider cache, a table's
    columns, q as part of a projection."""
    lens, new = [300, 77], [9, 30]
    cache, table, k, v = _filled(lens, 32, 4, 64, dtype)
    wide = torch.randn(sum(new), 16, 64, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    q = wide[:, 3:11]
    want = kernels.paged_chunk_attention(q.contiguous(), pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    rows_first = kernels.PagedCache(*(None if t is None else t.contiguous() for t in cache))
    inside = []
    for t in cache:
        if t is not None:
            big = torch.zeros(t.shape[0], 2 * t.shape[1], t.shape[2] + 1, *t.shape[3:], dtype=t.dtype, device='cuda')
            part = big[:, 5:5 + t.shape[1], 1:]
            (part.view(torch.uint8) if dtype == E4M3 else part).copy_(t.view(torch.uint8) if dtype == E4M3 else t)
            t = part
        inside.append(t)
    columns = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device='cuda')
    columns[:, :table.shape[1]] = table
    for other in (rows_first, kernels.PagedCache(*inside)):
        got = kernels.paged_chunk_attention(q, pr.offsets(new), other, columns[:, :table.shape[1]], _ints(lens),
                                            return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Pages that lie more than 2^31 values on."""
    far = torch.zeros(3, (1 << 30) + 4096, dtype=BF16, device='cuda')
    pages = far.as_strided((3, 16, 1, 128), ((1 << 30) + 4096, 128, 2048, 1))
    cache = kernels.PagedCache(pages, far[:, 4096:].as_strided((3, 16, 1, 128), ((1 << 30) + 4096, 128, 2048, 1), 4096))
    lens, new = [40], [4]
    table = _ints([[2, 0, 1]])
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(40, 1, 128, generator=g).to(BF16).cuda() for _ in range(2))
    kernels.cache_append_(cache, k, v, pr.offsets(lens), table, _ints([0]))
    q = _queries(4, 3, 128)
    got = kernels.paged_chunk_attention(q, pr.offsets(new), cache, table, _ints(lens), return_lse=True)
    _check(got, pr.attend(q, k, v, new, lens))


@TYPES
def test_streams_and_graphs(dtype):
    """Two graphs on two streams at once, replayed for other lengths."""
    lens, new = [2000, 700, 64], [5, 3, 4]
    cases = []
    for seed in (1, 2):
        cache, table, k, v = _filled(lens, 16, 2, 128, dtype, seed=seed)
        cases.append((_queries(sum(new), 8, 128, seed), pr.offsets(new), cache, table, _ints(lens)))
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for case, stream in zip(cases, streams):
        with torch.cuda.stream(stream):
            kernels.paged_chunk_attention(*case, return_lse=True)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(kernels.paged_chunk_attention(*case, return_lse=True))
        graphs.append(graph)
    for now in (lens, [1900, 701, 5], [64, 64, 64]):
        for case in cases:
            case[-1].copy_(_ints(now))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for case, out in zip(cases, outs):
            want = kernels.paged_chunk_attention(*case, return_lse=True)
            # bits: position 700 of the second sequence, which 701 takes in, is not finite
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want))


@TYPES
def test_a_prompt_in_chunks_then_tokens(dtype):
    """The operators together: chunks and then single tokens, each normalised, rotated and
    appended, then attended, are the whole prompt at once."""
    lens, heads, kv, d = [150, 77], 8, 2, 128
    g = torch.Generator().manual_seed(3)
    x = torch.randn(sum(lens), heads + 2 * kv, d, generator=g).to(BF16).cuda()
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(BF16).cuda() for _ in range(2))
    rot = kernels.rotary([16, 24, 24])
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    at = torch.cat([torch.arange(n) for n in lens]).cuda()
    q_all, k_all = kernels.norm_rotate(q, k, at, rot, wq, wk, 1e-6)
    if dtype == E4M3:
        # as the cache holds them: the key from 32 bits, off by a code's half step from the key by way of bf16
        k_all, v_all = (pr.held(t)[0].to(BF16) for t in (k_all, v))
    else:
        v_all = v
    want = pr.attend(q_all, k_all, v_all, lens, lens)
    cache = kernels.paged_cache(30, 16, kv, d, dtype)
    table = torch.randperm(30, generator=g)[:20].to(torch.int32).view(2, 10).cuda()
    got = torch.zeros(sum(lens), heads, d, device='cuda')
    done, first = [0, 0], [0, lens[0]]
    for step in ((64, 30), (80, 46), (1, 0), (1, 1), (4, 0)):
        rows = torch.cat([torch.arange(f + a, f + a + m) for f, a, m in zip(first, done, step)]).cuda()
        now = [a + m for a, m in zip(done, step)]
        qn = kernels.cache_append_rotated_(cache, q[rows], k[rows], v[rows], pr.offsets(step), table, _ints(done),
                                           rot, None, wq, wk, 1e-6)
        got[rows] = kernels.paged_chunk_attention(qn, pr.offsets(step), cache, table, _ints(now)).float()
        if step == (1, 1):
            one = kernels.paged_attention(qn, cache, table, _ints(now))
            assert (one.float() - got[rows]).abs().max() <= 2.0 ** -7 * one.float().abs().max()
        done = now
    assert done == lens
    # a key's code by way of bf16 differs where bf16 lands on a border of e4m3 (one value in
    # 16), on the wrong side of it every other time, by a step of 2^-4 to 2^-3 of the value:
    # 0.09 sqrt(1 / 32) = 1.6e-2 by square mean, which moves a score of unit rows by as
    # much, and P and out by that share of themselves
    bound = pr.NORM if dtype == BF16 else 3e-2
    assert (got.double() - want['out']).norm() <= bound * want['out'].norm()


def test_refusals():
    lens, new = [40, 20], [4, 2]
    cache, table, k, v = _filled(lens, 16, 2, 128, BF16)
    q, cu, n = _queries(6, 4, 128), pr.offsets(new), _ints(lens)
    ok = [q, cu, cache, table, n]

    def refused(match, at, what, **kw):
        args = list(ok)
        args[at] = what
        with pytest.raises(ValueError, match=match):
            kernels.paged_chunk_attention(*args, **kw)

    refused('bfloat16', 0, q.float())
    refused('does not fit', 0, q[:, :3])
    refused('does not fit', 0, q[..., :96].contiguous())
    refused('16-byte', 0, torch.zeros(6, 4, 136, dtype=BF16, device='cuda')[..., 4:132])
    refused('cu', 1, cu.long())
    refused('cu', 1, cu[:2])
    refused('laid out alike', 2, kernels.PagedCache(cache.k, cache.v.contiguous()))
    refused('no exponents', 2, kernels.PagedCache(cache.k, cache.v, cache.k_exp, torch.zeros(1, device='cuda')))
    refused('table', 3, table.long())
    refused('lengths', 4, n[:1])
    refused('scale', 4, n, scale=0.0)
    with pytest.raises(NotImplementedError):
        kernels.paged_chunk_attention(*[t.cpu() if isinstance(t, torch.Tensor) else t for t in ok])


def _put_nan(cache, table, b, pos, head, dim):
    """A NaN in dim `dim` of the key of position `pos` of sequence b."""
    page = cache.k.shape[1]
    x = cache.k[int(table[b, pos // page]), pos % page, head]
    if x.dtype == E4M3:
        x.view(torch.uint8)[dim] = 0x7f
    else:
        x[dim] = math.nan


def _check_around(got, clean, nan):
    """NaN in out and LSE of the rows of `nan` [rows, heads], nothing else changed by it."""
    out, lse = got
    assert torch.equal(torch.isnan(lse), nan), f'{int((torch.isnan(lse) != nan).sum())} LSEs'
    assert torch.equal(torch.isnan(out), nan[..., None].expand_as(out)), f'{int((torch.isnan(out).all(-1) != nan).sum())} rows'
    rr.within(torch.where(nan[..., None], 0.0, out.double()), torch.where(nan[..., None], 0.0, clean['out']),
              clean['out_tol'])
    none = clean['lse'] == -math.inf
    assert (lse[none] == -math.inf).all()
    rr.within(torch.where(nan | none, 0.0, lse.double()), torch.where(nan | none, 0.0, clean['lse']), clean['lse_tol'])


# two query heads to a key head: up to 16 rows, up to 32 and more, keys whole and in splits
NAN_ROWS = pytest.mark.parametrize('new', [1, 5, 12, 40])
NAN_LENS = [(1, 0), (33, 32), (65, 64), (97, 96), (129, 40), (5000, 4999), (5000, 300)]


@TYPES
@NAN_ROWS
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('length,bad', NAN_LENS, ids=[f'{b}of{n}' for n, b in NAN_LENS])
def test_a_key_that_is_nan(length, bad, d, new, dtype):
    """Every row that sees it is NaN, whichever keys of the row's tiles are beside it, and no
    other row; also where the keys beside it weigh nothing."""
    lens, news = [length, 200], [new, 3]
    cache, table, k, v = _filled(lens, 16, 2, d, dtype)
    q = _queries(sum(news), 4, d)
    _put_nan(cache, table, 0, bad, 1, 5)
    got = kernels.paged_chunk_attention(q, pr.offsets(news), cache, table, _ints(lens), return_lse=True)
    sees = torch.arange(new) + length - new >= bad
    nan = torch.zeros(sum(news), 4, dtype=torch.bool)
    nan[:new, 2:] = sees[:, None]
    _check_around(got, pr.attend(q, k, v, news, lens), nan.cuda())


@TYPES
@NAN_ROWS
def test_a_nan_beside_keys_that_weigh_nothing(new, dtype):
    """The other keys of its 32 have scores some 180 below the rest: probabilities of zero in
    32 bits."""
    lens = [400]
    cache, table, k, v = _filled(lens, 16, 1, 128, dtype)
    q = torch.full((new, 2, 128), 4.0, dtype=BF16, device='cuda')
    low = torch.full((32, 1, 128), -4.0, dtype=BF16, device='cuda')  # scores of -181
    kernels.cache_append_(cache, low, v[64:96].contiguous(), pr.offsets([32]), table, _ints([64]))
    k = k.clone()
    k[64:96] = low
    _put_nan(cache, table, 0, 70, 0, 9)
    got = kernels.paged_chunk_attention(q, pr.offsets([new]), cache, table, _ints(lens), return_lse=True)
    _check_around(got, pr.attend(q, k, v, [new], lens), torch.ones(new, 2, dtype=torch.bool, device='cuda'))


@TYPES
@NAN_ROWS
@pytest.mark.parametrize('length', [1, 33, 200, 5000])
def test_a_query_that_is_nan(length, new, dtype):
    """The row is NaN where it sees a key; a row that sees none is as ever."""
    lens, news = [length, 200], [new, 3]
    cache, table, k, v = _filled(lens, 16, 2, 128, dtype)
    q = _queries(sum(news), 4, 128)
    clean = pr.attend(q, k, v, news, lens)
    nan = torch.zeros(sum(news), 4, dtype=torch.bool, device='cuda')
    for row, head in ((0, 1), (new - 1, 1), (new // 2, 3), (new, 0)):
        q[row, head, 7] = math.nan
        nan[row, head] = clean['lse'][row, head] != -math.inf
    got = kernels.paged_chunk_attention(q, pr.offsets(news), cache, table, _ints(lens), return_lse=True)
    _check_around(got, clean, nan)


@TYPES
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('new', [5, 40])
def test_lengths_past_the_table_are_its_width(new, causal, dtype):
    """All of 7 pages' 112 positions are finite, and so are those of the pages that lie
    behind them in the table's memory; two more pages are outside the cache."""
    cache, table, k, v = _filled([112, 112], 16, 2, 64, dtype)
    q = _queries(new, 4, 64)
    behind = torch.cat([table[:1], table[1:]], 1)  # 14 pages, of which 7 are given
    outside = torch.cat([table[:1], torch.full((1, 2), -1, dtype=torch.int32, device='cuda')], 1)
    for n in (113, 144, 1 << 30, (1 << 31) - 1):
        got = kernels.paged_chunk_attention(q, pr.offsets([new]), cache, behind[:, :7], _ints([n]), causal,
                                            return_lse=True)
        _check(got, pr.attend(q, k[:112], v[:112], [new], [112], causal))
        # the last query is at position min(n, 144) - 1, the keys end at 112
        got = kernels.paged_chunk_attention(q, pr.offsets([new]), cache, outside, _ints([n]), causal,
                                            return_lse=True)
        seen = [min(min(n, 144) - new + i + 1, 112) if causal else 112 for i in range(new)]
        _check(got, pr.attend(q, *(torch.cat([t[:m] for m in seen]) for t in (k, v)), [1] * new, seen))
