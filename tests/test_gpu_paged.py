"""The paged cache (kernels.cache_append_, cache_gather) and the attention of one
new token over it (kernels.paged_attention) against their definitions in 64 bits."""

import math

import pytest
import torch

from miowtion_amd import _native, kernels, ops_packed
from tests import packed_reference as pr

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
BF16 = torch.bfloat16


def _table(lens, page, pages, width=None, seed=0):
    """Every sequence its own pages, in no order; the entries behind them point
    outside the cache."""
    g = torch.Generator().manual_seed(seed)
    width = width or max(1, max(-(-n // page) for n in lens))
    table = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=g).to(torch.int32), 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order[at:at + m]
        at += m
    assert at <= pages
    return table.cuda()


def _need(lens, page):
    return sum(-(-n // page) for n in lens) + 3


def _filled(lens, page, kv, d, dtype, seed=0, width=None):
    """(cache, table, k, v): a cache of these sequences, other rows not finite,
    and the values that it stands for, packed."""
    g = torch.Generator().manual_seed(seed + 1)
    table = _table(lens, page, _need(lens, page), width, seed)
    cache = kernels.paged_cache(_need(lens, page), page, kv, d, dtype)
    for t in cache[:2]:
        (t.view(torch.uint8) if dtype == E4M3 else t).fill_(0x7f if dtype == E4M3 else math.nan)
    for t in cache[2:]:
        if t is not None:
            t.fill_(255)
    k, v = (torch.randn(sum(lens), kv, d, generator=g).to(BF16).cuda() for _ in range(2))
    zero = torch.zeros(len(lens), dtype=torch.int32, device='cuda')
    kernels.cache_append_(cache, k, v, pr.offsets(lens), table, zero)
    if dtype == E4M3:
        k, v = (pr.held(t)[0].to(BF16) for t in (k, v))
    return cache, table, k, v


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('kv', [1, 2, 3, 8])
@pytest.mark.parametrize('page', [16, 64, 256])
@pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])
def test_append_and_gather(dtype, page, kv, d):
    lens = [1, 40, 0, 257, 16]
    print(f'append and gather {dtype} {page} {kv} {d}', flush=True)
    cache, table, k, v = _filled(lens, page, kv, d, dtype)
    got_k, got_v = kernels.cache_gather(cache, pr.offsets(lens), table, sum(lens) + 5)
    assert torch.equal(got_k[:sum(lens)], k) and torch.equal(got_v[:sum(lens)], v)
    assert (got_k[sum(lens):] == 0).all() and (got_v[sum(lens):] == 0).all()
    # a second chunk behind the first: only its rows change
    more = [3, 0, 20, 1, 0]
    both = [a + b for a, b in zip(lens, more)]
    if any(-(-n // page) > table.shape[1] for n in both):
        return
    g = torch.Generator().manual_seed(9)
    spare = torch.arange(_need(lens, page), dtype=torch.int32)
    spare = spare[~torch.isin(spare, table.cpu())]
    used = 0
    for b, n in enumerate(both):  # a page for those that need one more
        for i in range(-(-lens[b] // page), -(-n // page)):
            table[b, i] = spare[used]
            used += 1
    k2, v2 = (torch.randn(sum(more) + 4, kv, d, generator=g).to(BF16).cuda() for _ in range(2))
    start = torch.tensor(lens, dtype=torch.int32, device='cuda')
    kernels.cache_append_(cache, k2, v2, pr.offsets(more), table, start)
    got_k, got_v = kernels.cache_gather(cache, pr.offsets(both), table, sum(both))
    if dtype == E4M3:
        k2, v2 = (pr.held(t)[0].to(BF16) for t in (k2, v2))
    for got, old, new in ((got_k, k, k2), (got_v, v, v2)):
        parts = [p for a, b in zip(old.split(lens), new[:sum(more)].split(more)) for p in (a, b)]
        assert torch.equal(got, torch.cat(parts))


def test_every_code_and_exponent_reads_back_exactly():
    """All 256 codes under all exponents whose values bf16 holds without rounding."""
    cache = kernels.paged_cache(256, 16, 1, 128, E4M3)
    codes = torch.arange(256, dtype=torch.uint8).reshape(2, 1, 128)
    for t in cache[:2]:
        t.view(torch.uint8)[:, :2] = codes.cuda()
    for t in cache[2:]:
        t[:, :2, 0] = torch.arange(256, dtype=torch.uint8)[:, None].cuda()
    table = torch.arange(256, dtype=torch.int32, device='cuda')[:, None]
    k, v = kernels.cache_gather(cache, pr.offsets([2] * 256), table, 512)
    values = codes.view(E4M3).double().reshape(1, 256)
    # 2^-133 is bf16's least value: codes from 2^-9 on are exact for bytes from 3 on
    byte = torch.arange(3, 247, dtype=torch.float64)[:, None]
    want = values * torch.exp2(byte - 127)
    got = k.cpu().double().reshape(256, 256)[3:247]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(v))


@pytest.mark.parametrize('d', [64, 128])
def test_quantised_rows_follow_the_definition(d):
    """Exponents and values of rows of all magnitudes, borders of the exponent's
    choice and of the codes' rounding among them, bit for bit."""
    g = torch.Generator().manual_seed(2)
    n = 600
    x = torch.randn(n, 1, d, generator=g) * torch.exp2(torch.randint(-125, 118, (n, 1, 1), generator=g).float())
    x[0] = 0.0
    x[1] = 0.0
    x[1, 0, 3] = 448.0                       # fills the range: exponent 0
    x[2, 0, :] = 0.01
    x[2, 0, 5] = 450.0                       # one step of bf16 past it
    x[3, 0, :] = torch.arange(d) * 0.25 + 16.0  # ties of the rounding
    x[3, 0, 0] = 448.0
    x[4, 0, :] = 2.0 ** -10 * torch.arange(d)   # below the normal codes
    x[4, 0, 0] = 448.0
    x[5] = -x[3]
    x[6, 0, :] = 2.0 ** -133                 # bf16's least
    x[7, 0, :] = 0.0
    x[7, 0, 7] = 2.0 ** -127
    x = x.to(BF16)
    x[8, 0, 1], x[8, 0, 2], x[8, 0, 3] = math.nan, math.inf, -math.inf
    x[9] = math.nan
    x = x.cuda()
    cache = kernels.paged_cache(n // 16 + 1, 16, 1, d, E4M3)
    table = torch.arange(n // 16 + 1, dtype=torch.int32, device='cuda')[None]
    zero = torch.zeros(1, dtype=torch.int32, device='cuda')
    kernels.cache_append_(cache, x, x.flip(0), pr.offsets([n]), table, zero)
    want, byte = pr.held(x)
    got_byte = cache.k_exp.reshape(-1, 1)[:n]
    assert torch.equal(got_byte, byte)
    k, v = kernels.cache_gather(cache, pr.offsets([n]), table, n)
    assert torch.equal(torch.isnan(k), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(want.to(BF16)))
    assert torch.equal(torch.nan_to_num(v.flip(0)), torch.nan_to_num(k))
    fine = torch.isfinite(x.double())
    unit = torch.exp2(byte.double() - 127)[..., None]
    off = (want - x.double()).abs()
    assert (off[fine] <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * unit)[fine]).all()


@pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])
def test_places_that_are_no_rows_are_left_alone(dtype):
    page, kv, d = 16, 2, 64
    cache = kernels.paged_cache(4, page, kv, d, dtype)
    for t in cache[:2]:
        t.view(torch.uint8).fill_(3) if dtype == E4M3 else t.fill_(3.0)
    before = [t.clone() for t in cache if t is not None]
    k = torch.randn(40, kv, d).to(BF16).cuda()
    table = torch.tensor([[1, -1], [4, 1 << 30], [-2 ** 31, 0]], dtype=torch.int32, device='cuda')
    for cu, start in (([0, 20, 30, 40], [16, 0, 0]),   # bad pages
                      ([0, 20, 30, 40], [32, 1 << 30, 2 ** 31 - 1]),  # past the table
                      ([0, 20, 30, 40], [-20, -10, -2 ** 31]),  # before it
                      ([40, 40, 40, 40], [0, 0, 16]), ([0, 0, 0, 0], [0, 0, 16])):  # rows of no sequence
        print(f'no rows: {cu} {start}', flush=True)
        kernels.cache_append_(cache, k, k, torch.tensor(cu, dtype=torch.int32, device='cuda'), table,
                              torch.tensor(start, dtype=torch.int32, device='cuda'))
        for t, old in zip([t for t in cache if t is not None], before):
            assert torch.equal(t.view(torch.uint8) if t.dtype == E4M3 else t,
                               old.view(torch.uint8) if old.dtype == E4M3 else old)
    got, _ = kernels.cache_gather(cache, pr.offsets([33, 3, 2]), table, 38)
    # what the page holds: 3.0, or code 3 = 3 2^-9 under exponent byte 0, 2^-127,
    # which is below half of bf16's least 2^-133 and reads 0
    held = torch.tensor(3.0 if dtype == BF16 else 3 * 2.0 ** -136, dtype=torch.float64).to(BF16)
    assert (got[:16] == held.cuda()).all() and (got[16:36] == 0).all() and (got[36:] == 0).all()
    # a sequence that has one row in the cache and others outside it
    kernels.cache_append_(cache, k, k, pr.offsets([0, 0, 40]), table,
                          torch.tensor([0, 0, 1], dtype=torch.int32, device='cuda'))
    want = pr.held(k)[0].to(BF16) if dtype == E4M3 else k
    got, _ = kernels.cache_gather(cache, pr.offsets([0, 0, 40]), table, 40)
    assert (got[:16] == 0).all() and torch.equal(got[16:32], want[15:31]) and (got[32:] == 0).all()


TOKENS = [
    # lens, heads, kv, d, page, width
    ([1], 1, 1, 128, 16, None),
    ([1500], 24, 8, 64, 16, None),
    ([1, 15, 16, 17, 31, 32, 33, 500], 4, 2, 128, 16, None),
    ([1, 15, 16, 17, 31, 32, 33, 500], 4, 2, 64, 32, None),
    ([0, 3, 0, 130], 5, 1, 128, 64, None),
    ([2049, 100, 1], 7, 1, 64, 128, None),
    ([2049, 100, 1], 56, 8, 128, 256, None),
    ([700, 0, 90], 40, 2, 128, 16, None),      # twenty heads to a group: two workgroups
    ([77, 20], 8, 8, 128, 16, 200),            # a table far wider than the sequences
    ([129], 16, 1, 128, 16, 9),
]


@pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])
@pytest.mark.parametrize('case', TOKENS, ids=lambda c: f'{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-{c[3]}-{c[4]}')
def test_one_token(case, dtype):
    lens, heads, kv, d, page, width = case
    print(f'one token {case} {dtype}', flush=True)
    cache, table, k, v = _filled(lens, page, kv, d, dtype, width=width)
    q = torch.randn(len(lens), heads, d, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    out, lse = kernels.paged_attention(q, cache, table, lengths, return_lse=True)
    ref = pr.attend(q, k, v, [1] * len(lens), lens)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')
    assert torch.equal(out, kernels.paged_attention(q, cache, table, lengths))


def _near_by_norm(out, ref):
    """Each sequence's out by norm: thousands of keys of like weight leave an out of
    some hundredths, and the bound of a value, of the size of v, lets a part go."""
    off = (out.double() - ref['out']).norm(dim=(1, 2))
    assert (off <= pr.NORM * ref['out'].norm(dim=(1, 2))).all(), off


PARTS = [
    # lens, heads, kv, d, page, width: more than 64 parts, joined by eight waves: some
    # of them without a part, parts that do not divide by eight, more than 512
    ([1, 16500, 0, 9000], 5, 1, 128, 16, 1100),
    ([1, 16500, 0, 9000], 5, 1, 64, 16, 1300),
    ([17000, 30], 17, 1, 64, 64, 300),
    ([33000, 16640], 3, 3, 128, 256, None),
    ([600001, 70000], 3, 1, 64, 32, None),
]


@pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])
@pytest.mark.parametrize('case', PARTS, ids=lambda c: f'{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-{c[3]}-{c[4]}')
def test_one_token_of_many_parts(case, dtype):
    lens, heads, kv, d, page, width = case
    cache, table, k, v = _filled(lens, page, kv, d, dtype, width=width)
    capacity = table.shape[1] * page
    parts = -(-capacity // ops_packed._chunk(len(lens), kv, heads // kv, capacity, page))
    print(f'one token of many parts {case} {dtype}: {parts}', flush=True)
    assert parts > (512 if max(lens) > 500000 else 64)
    q = torch.randn(len(lens), heads, d, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    out, lse = kernels.paged_attention(q, cache, table, lengths, return_lse=True)
    ref = pr.attend(q, k, v, [1] * len(lens), lens)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')
    _near_by_norm(out, ref)
    assert torch.equal(out, kernels.paged_attention(q, cache, table, lengths))
    # a page of the longest sequence outside the cache
    b = lens.index(max(lens))
    first = sum(lens[:b])
    at = 300 // page
    table[b, at] = -1
    seen = torch.ones(lens[b], dtype=torch.bool)
    seen[at * page:(at + 1) * page] = False
    rows = slice(first, first + lens[b])
    ref = pr.attend(q[b:b + 1], k[rows][seen], v[rows][seen], [1], [int(seen.sum())])
    out, lse = kernels.paged_attention(q, cache, table, lengths, return_lse=True)
    pr.check(out[b:b + 1], ref, 'out')
    pr.check(lse[b:b + 1], ref, 'lse')


@pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])
@pytest.mark.parametrize('pages', [66, 128])
def test_chunks_of_more_pages_than_a_wave_has_lanes(pages, dtype):
    """Through the library's entry point: the ops ask for 64 pages to a chunk at most."""
    lens, heads, kv, d, page, width = [3000, 1, 0, 4999], 4, 2, 128, 16, 320
    cache, table, k, v = _filled(lens, page, kv, d, dtype, width=width)
    q = torch.randn(len(lens), heads, d, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    out, lse = torch.empty_like(q), torch.empty(len(lens), heads, device='cuda')
    chunk = pages * page
    work = torch.empty(len(lens) * heads * -(-width * page // chunk) * (d + 4), device='cuda')
    args, sizes = ops_packed._check_cache(*cache, table, kv, d, 0)
    print(f'chunks of {pages} pages {dtype}', flush=True)
    _native.call('veda_paged_fwd', q.data_ptr(), heads * d, d, len(lens), heads, kv, d, *args, *sizes,
                 lengths.data_ptr(), d ** -0.5, chunk, out.data_ptr(), heads * d, d, lse.data_ptr(),
                 work.data_ptr(), 4 * work.numel(), torch.cuda.current_stream().cuda_stream)
    ref = pr.attend(q, k, v, [1] * len(lens), lens)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')
    _near_by_norm(out, ref)


def test_lengths_and_pages_out_of_range():
    lens = [100, 60]
    cache, table, k, v = _filled(lens, 16, 2, 128, BF16, width=7)
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    table[1, 4:] = table[0, 0]  # sequence 1 runs on into a page of sequence 0
    long = torch.tensor([-3, 1 << 30], dtype=torch.int32, device='cuda')
    out, lse = kernels.paged_attention(q, cache, table, long, return_lse=True)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    assert torch.isnan(out[1]).all()  # rows 60 .. 63 hold NaN and are seen
    # a page outside the cache: its positions draw no weight
    table[0, 2], table[0, 5] = -1, 99
    out, lse = kernels.paged_attention(q, cache, table, torch.tensor(lens, dtype=torch.int32, device='cuda'),
                                       return_lse=True)
    seen = torch.ones(100, dtype=torch.bool)
    seen[32:48] = seen[80:96] = False
    ref = pr.attend(q[:1], k[:100][seen], v[:100][seen], [1], [int(seen.sum())])
    pr.check(out[:1], ref, 'out')
    pr.check(lse[:1], ref, 'lse')


def test_other_layouts_of_the_cache():
    lens, page, kv, d = [70, 33], 16, 2, 128
    q = torch.randn(2, 6, d, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    for dtype in (BF16, E4M3):
        cache, table, k, v = _filled(lens, page, kv, d, dtype)
        # rows of all heads side by side, K and V in one tensor of all layers
        n = cache.k.shape[0]
        both = torch.zeros(n, 3, 2, page, kv, d, dtype=BF16).to(dtype).cuda()
        flat = kernels.PagedCache(both[:, 1, 0], both[:, 1, 1],
                                  *(() if dtype == BF16 else
                                    torch.zeros(2, n, page, kv, dtype=torch.uint8, device='cuda').unbind(0)))
        zero = torch.zeros(2, dtype=torch.int32, device='cuda')
        g = torch.Generator().manual_seed(1)
        kk, vv = (torch.randn(sum(lens), kv, d, generator=g).to(BF16).cuda() for _ in range(2))
        kernels.cache_append_(flat, kk, vv, pr.offsets(lens), table, zero)
        for a, b in zip(kernels.cache_gather(flat, pr.offsets(lens), table, sum(lens)), (k, v)):
            assert torch.equal(a, b)
        assert (both[:, ::2].float() == 0).all()  # the other layers
        out = kernels.paged_attention(q, flat, table, torch.tensor(lens, dtype=torch.int32, device='cuda'))
        pr.check(out, pr.attend(q, k, v, [1, 1], lens), 'out')


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: its last page is written, read and seen."""
    page, kv, d = 256, 8, 128
    pages = (1 << 31) // (page * kv * d) + 40
    k = torch.empty(pages, kv, page, d, dtype=BF16, device='cuda').transpose(1, 2)
    cache = kernels.PagedCache(k, torch.empty_like(k))
    lens = [300]
    table = torch.tensor([[pages - 1, pages - 7]], dtype=torch.int32, device='cuda')
    g = torch.Generator().manual_seed(1)
    kk, vv = (torch.randn(300, kv, d, generator=g).to(BF16).cuda() for _ in range(2))
    cu = pr.offsets(lens)
    kernels.cache_append_(cache, kk, vv, cu, table, torch.zeros(1, dtype=torch.int32, device='cuda'))
    got = kernels.cache_gather(cache, cu, table, 300)
    assert torch.equal(got[0], kk) and torch.equal(got[1], vv)
    assert torch.equal(cache.k[pages - 1], kk[:256])
    q = torch.randn(1, 16, d, generator=g).to(BF16).cuda()
    out = kernels.paged_attention(q, cache, table, torch.tensor(lens, dtype=torch.int32, device='cuda'))
    pr.check(out, pr.attend(q, kk, vv, [1], lens), 'out')


def test_prompt_then_tokens():
    """The operators as a program runs them: a prompt's first chunk, its second
    chunk against the cache, then token by token in a captured graph; every
    output is that of one packed attention over what the cache holds."""
    heads, kv, d, page = 6, 2, 64, 16
    lens, first, steps = [50, 90, 33], [20, 64, 32], 5
    full = [n + steps for n in lens]
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(sum(full), h, d, generator=g).to(BF16).cuda() for h in (heads, kv, kv))
    rows = torch.arange(sum(full), device='cuda').split(full)

    def part(x, begin, end):
        return torch.cat([x[r[a:b]] for r, a, b in zip(rows, begin, end)])

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device='cuda')

    for dtype in (BF16, E4M3):
        held_k, held_v = (pr.held(t)[0].to(BF16) if dtype == E4M3 else t for t in (k, v))
        ref = pr.attend(q, held_k, held_v, full, full)
        table = _table(full, page, 64)
        cache = kernels.paged_cache(64, page, kv, d, dtype)
        done = [0, 0, 0]
        for upto in (first, lens):  # the chunks
            new = [a - b for a, b in zip(upto, done)]
            kernels.cache_append_(cache, part(k, done, upto), part(v, done, upto), pr.offsets(new), table,
                                  ints(done))
            ck, cv = kernels.cache_gather(cache, pr.offsets(upto), table, sum(upto))
            out = kernels.packed_attention(part(q, done, upto), ck, cv, pr.offsets(new), pr.offsets(upto))
            pr.check(out, {n: part(t, done, upto) for n, t in ref.items()}, 'out')
            done = upto
        # a token: the static tensors of a captured graph
        sq, sk, sv = (torch.empty(3, h, d, dtype=BF16, device='cuda') for h in (heads, kv, kv))
        lengths, at, one = ints(done), ints(done), pr.offsets([1, 1, 1])

        def token():
            kernels.cache_append_(cache, sk, sv, one, table, at)
            lengths.copy_(at + 1)
            res = kernels.paged_attention(sq, cache, table, lengths, return_lse=True)
            at.add_(1)
            return res

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = token()
        at.copy_(ints(done))
        for step in range(steps):
            here, there = [n + step for n in lens], [n + step + 1 for n in lens]
            for static, x in ((sq, q), (sk, k), (sv, v)):
                static.copy_(part(x, here, there))
            graph.replay()
            torch.cuda.synchronize()
            mine = {n: part(t, here, there) for n, t in ref.items()}
            pr.check(out, mine, 'out')
            pr.check(lse, mine, 'lse')
            eager, _ = kernels.paged_attention(sq, cache, table, lengths, return_lse=True)
            assert torch.equal(out, eager)


def test_two_graphs_do_not_share_partial_sums():
    lens = [3000, 2000]
    cache, table, k, v = _filled(lens, 16, 2, 128, BF16)
    g = torch.Generator().manual_seed(4)
    qs = [torch.randn(2, 8, 128, generator=g).to(BF16).cuda() for _ in range(2)]
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    want = [kernels.paged_attention(q, cache, table, lengths) for q in qs]
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kernels.paged_attention(q, cache, table, lengths))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_refusals():
    cache = kernels.paged_cache(4, 16, 2, 128)
    c8 = kernels.paged_cache(4, 16, 2, 128, E4M3)
    table = torch.zeros(1, 2, dtype=torch.int32, device='cuda')
    one = torch.ones(1, dtype=torch.int32, device='cuda')
    cu = pr.offsets([1])
    q = torch.zeros(1, 4, 128, dtype=BF16, device='cuda')
    x = torch.zeros(1, 2, 128, dtype=BF16, device='cuda')
    att, app, gat = kernels.paged_attention, kernels.cache_append_, kernels.cache_gather
    for bad, match in [
            (lambda: att(q.half(), cache, table, one), 'bfloat16'),
            (lambda: att(q[:, :3], cache, table, one), 'multiple'),
            (lambda: att(q[..., :64], cache, table, one), 'wanted'),
            (lambda: att(q, cache, table.long(), one), 'int32'),
            (lambda: att(q, cache, table.expand(2, -1), one), 'sequences'),
            (lambda: att(q, cache, table, one.long()), 'int32'),
            (lambda: att(q, cache, table, one, scale=0.0), 'scale'),
            (lambda: att(q, cache._replace(v=cache.v[:3]), table, one), 'alike'),
            (lambda: att(q, cache._replace(v=cache.v.contiguous()), table, one), 'alike'),
            (lambda: att(q, cache._replace(k_exp=c8.k_exp), table, one), 'no exponents'),
            (lambda: att(q, c8._replace(k_exp=None), table, one), 'k_exp'),
            (lambda: att(q, c8._replace(v_exp=c8.v_exp[:2]), table, one), 'v_exp'),
            (lambda: att(q, kernels.PagedCache(cache.k.float(), cache.v.float()), table, one), 'bfloat16 or'),
            (lambda: att(q, kernels.PagedCache(cache.k[:, :8], cache.v[:, :8]), table, one), '16 | 32'),
            (lambda: app(cache, x.float(), x, cu, table, one), 'bfloat16'),
            (lambda: app(cache, x[:, :1], x[:, :1], cu, table, one), 'wanted'),
            (lambda: app(cache, x, x[:0], cu, table, one), 'alike'),
            (lambda: app(cache, x, x, cu[:1], table, one), 'int32'),
            (lambda: app(cache, x, x, cu, table, cu), 'int32'),
            (lambda: gat(cache, cu, table, -1), 'rows'),
            (lambda: gat(cache, cu[:1], table, 1), 'int32'),
            (lambda: kernels.paged_cache(4, 24, 2, 128), 'pages of'),
            (lambda: kernels.paged_cache(4, 16, 2, 96), 'pages of'),
            (lambda: kernels.paged_cache(4, 16, 2, 128, torch.float16), 'bfloat16 or')]:
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises((ValueError, NotImplementedError)):
        att(q.cpu(), cache, table, one)
