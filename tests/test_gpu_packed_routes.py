"""How the ops of packed sequences and the paged cache are reached: through the
dispatcher as directly, in place with their versions raised, from views and on
streams, at sizes past 32 bits; and what they refuse on the GPU."""

import pytest
import torch

from miowtion_amd import kernels, ops_packed
from tests import packed_reference as pr
from tests.test_gpu_packed import _inputs

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _cache(dtype=BF16, kv=2, d=64):
    cache = kernels.paged_cache(8, 16, kv, d, dtype)
    table = torch.tensor([[3, 1, 7], [0, 5, 2]], dtype=torch.int32, device='cuda')
    lengths = torch.tensor([40, 17], dtype=torch.int32, device='cuda')
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(57, kv, d, generator=g).to(BF16).cuda() for _ in range(2))
    start = torch.zeros(2, dtype=torch.int32, device='cuda')
    return cache, table, lengths, k, v, start, pr.offsets([40, 17])


@pytest.mark.parametrize('dtype', [BF16, torch.float8_e4m3fn], ids=['bf16', 'e4m3'])
def test_dispatcher_and_direct_calls_agree(dtype):
    cache, table, lengths, k, v, start, cu = _cache(dtype)
    veda = torch.ops.veda
    before = [t._version for t in cache if t is not None]
    kernels.cache_append_(cache, k, v, cu, table, start)
    assert [t._version for t in cache if t is not None] == [n + 1 for n in before]
    other = kernels.PagedCache(*(None if t is None else t.clone() for t in cache))
    veda.cache_append_(*other, v, k, cu, table, start)
    veda.cache_append_(*other, k, v, cu, table, start)
    for a, b in zip(cache, other):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in zip(kernels.cache_gather(cache, cu, table, 60), veda.cache_gather(*cache, cu, table, 60)):
        assert torch.equal(a, b)
    q = torch.randn(2, 6, 64, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    for a, b in zip(kernels.paged_attention(q, cache, table, lengths, return_lse=True),
                    veda.paged_fwd(q, *cache, table, lengths, 0.125, True)):
        assert torch.equal(a, b)
    qq = torch.randn(57, 6, 64, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    out, lse = kernels.packed_attention(qq, k, v, cu, return_lse=True)
    for a, b in zip((out, lse), veda.packed_fwd(qq, k, v, cu, cu, True, 0.125, True)):
        assert torch.equal(a, b)
    grads = ops_packed.packed_bwd(qq, k, v, out, qq, lse, None, cu, cu, True, 0.125)
    for a, b in zip(grads, veda.packed_bwd(qq, k, v, out, qq, lse, None, cu, cu, True, 0.125)):
        assert torch.equal(a, b)


def test_schemas_and_fakes():
    cache, table, lengths, k, v, start, cu = _cache()
    q = torch.randn(57, 6, 64).to(BF16).cuda()
    check = dict(test_utils=('test_schema', 'test_faketensor'))
    torch.library.opcheck(torch.ops.veda.packed_fwd.default, (q, k, v, cu, cu, True, 0.1, True), **check)
    out, lse = torch.ops.veda.packed_fwd(q, k, v, cu, cu, True, 0.1, True)
    torch.library.opcheck(torch.ops.veda.packed_bwd.default, (q, k, v, out, q, lse, None, cu, cu, True, 0.1), **check)
    torch.library.opcheck(torch.ops.veda.cache_append_.default, (*cache, k, v, cu, table, start), **check)
    torch.library.opcheck(torch.ops.veda.cache_gather.default, (*cache, cu, table, 60), **check)
    torch.library.opcheck(torch.ops.veda.paged_fwd.default, (q[:2], *cache, table, lengths, 0.1, True), **check)


def test_a_cache_written_in_place_is_not_used_by_an_older_graph():
    """autograd sees the write: a graph that saved the rows refuses."""
    cache, table, lengths, k, v, start, cu = _cache()
    w = torch.ones((), device='cuda', requires_grad=True)
    y = (cache.k.float() * w).sum() + (cache.k.to(torch.float64) ** 2 * w).sum()
    x = cache.k * w.to(BF16)
    kernels.cache_append_(cache, k, v, cu, table, start)
    del y
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        x.sum().backward()


def test_gradients_through_the_token_form_are_refused():
    cache, table, lengths, *_ = _cache()
    q = torch.zeros(2, 4, 64, dtype=BF16, device='cuda', requires_grad=True)
    out = kernels.paged_attention(q, cache, table, lengths)
    with pytest.raises(RuntimeError):
        out.sum().backward()


def test_rows_that_share_memory_are_not_written():
    cache, table, lengths, k, v, start, cu = _cache()
    flat = kernels.PagedCache(*(t[:, :, :1].expand(-1, -1, 2, -1) for t in cache[:2]))
    with pytest.raises(ValueError, match='share memory'):
        kernels.cache_append_(flat, k, v, cu, table, start)
    # reading them is fine
    got, _ = kernels.cache_gather(flat, cu, table, 57)
    assert torch.equal(got[:, 0], got[:, 1])


def test_exponents_that_share_memory_are_not_written():
    cache, table, lengths, k, v, start, cu = _cache(torch.float8_e4m3fn)
    flat = [t[:, :, :1].expand(-1, -1, 2) for t in cache[2:]]
    for bad in (cache._replace(k_exp=flat[0], v_exp=flat[1]), cache._replace(v_exp=cache.k_exp),
                cache._replace(v=cache.k)):
        with pytest.raises(ValueError, match='share memory'):
            kernels.cache_append_(bad, k, v, cu, table, start)
    # reading them is fine
    kernels.cache_append_(cache, k, v, cu, table, start)
    got, _ = kernels.cache_gather(cache._replace(k_exp=flat[0], v_exp=flat[1]), cu, table, 57)
    want, _ = kernels.cache_gather(cache, cu, table, 57)
    assert torch.equal(got[:, 0], want[:, 0])


@pytest.mark.parametrize('dtype', [BF16, torch.float8_e4m3fn], ids=['bf16', 'e4m3'])
def test_one_cache_for_keys_and_values(dtype):
    """Rows that are both: written where k and v are one tensor too."""
    cache, table, lengths, k, v, start, cu = _cache(dtype)
    kernels.cache_append_(cache, k, k, cu, table, start)
    other = kernels.paged_cache(8, 16, 2, 64, dtype)
    one = other._replace(v=other.k, v_exp=other.k_exp)
    kernels.cache_append_(one, k, k, cu, table, start)
    for a, b in zip(one, cache):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with pytest.raises(ValueError, match='share memory'):
        kernels.cache_append_(one, k, v, cu, table, start)


def test_calls_on_two_streams_at_once():
    lens = [700, 300]
    cases = [_inputs(lens, lens, 8, 2, 128, seed=s) for s in range(4)]
    cu = pr.offsets(lens)
    want = [kernels.packed_attention(*c, cu) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, c in enumerate(cases * 3):
        with torch.cuda.stream(streams[i % 2]):
            got.append(kernels.packed_attention(*c, cu))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 4])


def test_queries_past_32_bits():
    """More than 2^31 elements of q, out and dq: the last sequences are right."""
    heads, n, d = 64, 64, 128
    seqs = (1 << 31) // (heads * n * d) + 3
    rows = seqs * n
    lens = [n] * seqs
    cu = torch.arange(seqs + 1, dtype=torch.int32, device='cuda') * n
    g = torch.Generator(device='cuda').manual_seed(0)
    q = torch.empty(rows, heads, d, dtype=BF16, device='cuda')
    for part in q.split(1 << 14):
        part.copy_(torch.randn(part.shape, generator=g, device='cuda'))
    k, v = (torch.randn(rows, 1, d, generator=g, device='cuda').to(BF16) for _ in range(2))
    print(f'{q.numel()} elements of q', flush=True)
    out, lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
    dq, dk, dv = ops_packed.packed_bwd(q, k, v, out, q, lse, None, cu, cu, True, d ** -0.5)
    for at in (slice(0, n), slice(rows - 2 * n, rows)):
        some = [n] * ((at.stop - at.start) // n)
        ref = pr.attend(q[at], k[at], v[at], some, some, dout=q[at])
        for name, x in (('out', out), ('lse', lse), ('dq', dq), ('dk', dk), ('dv', dv)):
            pr.check(x[at], ref, name)
    assert len(lens) == seqs


@pytest.mark.parametrize('d', [64, 128])
def test_long_sequences(d):
    """Several thousand keys: forward and gradients, with a short neighbour."""
    lens = [5003, 70]
    q, k, v = _inputs(lens, lens, 2, 1, d, seed=7)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    cu = pr.offsets(lens)
    ts = [t.requires_grad_(True) for t in (q, k, v)]
    out = kernels.packed_attention(*ts, cu)
    ref = pr.attend(q, k, v, lens, lens, dout=dout)
    for name, x in zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *torch.autograd.grad(out, ts, dout))):
        pr.check(x, ref, name)


MANY = [
    # sequences, longest, heads, kv, d, causal, chunk: several workgroups to each
    # place on the device, their walks of very different lengths
    (40, 700, 16, 4, 128, True, False),
    (40, 700, 16, 4, 64, False, False),
    (120, 300, 14, 2, 64, True, False),
    (9, 1500, 24, 8, 64, True, True),
    (24, 1500, 24, 8, 64, True, True),
    (126, 200, 20, 20, 64, True, True),
    (127, 200, 20, 20, 64, True, False),
]


@pytest.mark.parametrize('case', MANY, ids=lambda c: '-'.join(map(str, c)))
def test_many_tiles_of_different_lengths(case):
    n, longest, heads, kv, d, causal, chunk = case
    g = torch.Generator().manual_seed(n)
    lens_k = torch.randint(0, longest, (n,), generator=g).tolist()
    lens_q = [min(m, int(torch.randint(0, 500, (1,), generator=g))) for m in lens_k] if chunk else lens_k
    lens_k[n // 2] = lens_q[n // 2] = 0
    print(f'{case}: {sum(lens_q) * heads // 128} query tiles', flush=True)
    q, k, v = _inputs(lens_q, lens_k, heads, kv, d, seed=n, pad_q=130, pad_k=3)
    dout = torch.randn(q.shape, generator=g).to(BF16).cuda()
    ts = [t.requires_grad_(True) for t in (q, k, v)]
    out, lse = kernels.packed_attention(*ts, pr.offsets(lens_q), pr.offsets(lens_k), causal=causal,
                                        return_lse=True)
    ref = pr.attend(q, k, v, lens_q, lens_k, causal, dout=dout)
    pr.check(lse.detach(), ref, 'lse')
    for name, x in zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *torch.autograd.grad(out, ts, dout))):
        pr.check(x, ref, name)


@pytest.mark.parametrize('n,length', [(40, 130), (126, 64), (17, 300)])
def test_many_sequences_of_one_length(n, length):
    """Equal lengths: every tile of every sequence is met once."""
    lens = [length] * n
    q, k, v = _inputs(lens, lens, 32, 4, 64, seed=n)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(n)).to(BF16).cuda()
    ts = [t.requires_grad_(True) for t in (q, k, v)]
    out = kernels.packed_attention(*ts, pr.offsets(lens))
    ref = pr.attend(q, k, v, lens, lens, dout=dout)
    for name, x in zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *torch.autograd.grad(out, ts, dout))):
        pr.check(x, ref, name)


@pytest.mark.parametrize('d', [64, 128])
def test_chunks_of_different_lengths_share_their_keys(d):
    """A few queries onto many keys: split over the keys, the sequences ordered by
    their length."""
    lens_q, lens_k = [64, 1, 70, 50], [1000, 4096, 3001, 3900]
    heads, kv = 32, 8
    splits = ops_packed._key_splits(sum(lens_q), sum(lens_k), 4, heads, kv)
    assert splits > 1 and sum(lens_q) * heads // 128 * splits >= 256
    q, k, v = _inputs(lens_q, lens_k, heads, kv, d, seed=4, pad_q=2, pad_k=9)
    out, lse = kernels.packed_attention(q, k, v, pr.offsets(lens_q), pr.offsets(lens_k), return_lse=True)
    ref = pr.attend(q, k, v, lens_q, lens_k)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')


def test_graph_of_many_sequences_serves_new_lengths():
    """Forward and gradients captured once, replayed for lists whose longest
    sequence lies elsewhere, with rows behind the last one."""
    n, heads, kv, d, rows = 30, 16, 4, 64, 4096
    g = torch.Generator().manual_seed(11)
    q, k, v, dout = (torch.randn(rows, h, d, generator=g).to(BF16).cuda() for h in (heads, kv, kv, heads))
    cu = pr.offsets([rows // n] * n)

    def step():
        out, lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
        return [out, lse, *ops_packed.packed_bwd(q, k, v, out, dout, lse, None, cu, cu, True, d ** -0.5)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(4):
        lens = [int(x) for x in torch.randint(0, 90, (n,), generator=g)]
        lens[7 * seed] = 1200 + seed
        cu.copy_(pr.offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        ref = pr.attend(q, k, v, lens, lens, dout=dout)
        for name, x in zip(('out', 'lse', 'dq', 'dk', 'dv'), got):
            pr.check(x, ref, name)
        for x, y in zip(got, step()):  # the same bits as the eager call
            assert torch.equal(x, y)


def test_offsets_out_of_order():
    """Offsets that do not ascend name no sequences: what they give is not said,
    but the calls end, and their inputs stay."""
    g = torch.Generator().manual_seed(3)
    for n, heads in ((2, 6), (5, 6), (61, 6), (62, 6), (63, 6), (200, 6), (5, 64), (100, 64), (126, 128)):
        kv, d = 2, 64
        cu_q, cu_k = (torch.randint(-50, 1000, (n + 1,), generator=g).int().cuda() for _ in range(2))
        q, k, v = (torch.full((rows, h, d), 3.0, dtype=BF16, device='cuda')
                   for rows, h in ((700, heads), (600, kv), (600, kv)))
        out, lse = kernels.packed_attention(q, k, v, cu_q, cu_k, return_lse=True)
        grads = ops_packed.packed_bwd(q, k, v, out, q, lse, None, cu_q, cu_k, True, d ** -0.5)
        torch.cuda.synchronize()
        print(f'{n} sequences', flush=True)
        assert all((x == 3.0).all() for x in (q, k, v))
        assert [x.shape for x in grads] == [q.shape, k.shape, v.shape]
