"""How norms with rotation, appends with both and chunks over a paged cache are reached:
through the dispatcher as directly, compiled, in inference mode, with versions raised,
on streams at once; and rows enough to be moved past the caches."""

import pytest
import torch

from miowtion_amd import kernels, ops_packed, ops_rotary
from tests import packed_reference as pr
from tests import rotary_reference as rr

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _case(dtype=BF16, rows=21, heads=6, kv=2, d=64):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(rows, h, d, generator=g).to(BF16).cuda() for h in (heads, kv, kv))
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).cuda() for _ in range(2))
    cache = kernels.paged_cache(8, 16, kv, d, dtype)
    table = torch.tensor([[3, 1, 7], [0, 5, 2]], dtype=torch.int32, device='cuda')
    start = torch.tensor([0, 4], dtype=torch.int32, device='cuda')
    lengths = torch.tensor([14, 11], dtype=torch.int32, device='cuda')
    pos = torch.randint(0, 999, (rows, 2), generator=g).cuda()
    return q, k, v, wq, wk, cache, table, start, lengths, pos, kernels.rotary([8, 8]), pr.offsets([14, 7])


@pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])
def test_dispatcher_and_direct_calls_agree(dtype):
    q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu = _case(dtype)
    veda = torch.ops.veda
    got = kernels.norm_rotate(q, k, pos, rot, wq, wk, 1e-6)
    for a, b in zip(got, veda.norm_rotate(q, k, pos, *rot, wq, wk, 1e-6)):
        assert torch.equal(a, b)
    for a, b in zip(ops_rotary.norm_rotate_bwd(q, q, k, k, pos, *rot, wq, wk, 1e-6, True, True),
                    veda.norm_rotate_bwd(q, q, k, k, pos, *rot, wq, wk, 1e-6, True, True)):
        assert torch.equal(a, b)
    before = [t._version for t in cache if t is not None]
    y = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, pos, wq, wk, 1e-6)
    assert [t._version for t in cache if t is not None] == [n + 1 for n in before]
    other = kernels.paged_cache(8, 16, 2, 64, dtype)
    assert torch.equal(y, veda.cache_append_rotated_(*other, q, k, v, cu, table, start, pos, *rot, wq, wk, 1e-6))
    for a, b in zip(cache, other):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in zip(kernels.paged_chunk_attention(q, cu, cache, table, lengths, return_lse=True),
                    veda.chunk_fwd(q, cu, *cache, table, lengths, True, 0.125, True)):
        assert torch.equal(a, b)


def test_schemas_and_fakes():
    q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu = _case()
    check = dict(test_utils=('test_schema', 'test_faketensor'))
    ops = torch.ops.veda
    torch.library.opcheck(ops.norm_rotate.default, (q, k, pos, *rot, wq, wk, 1e-6), **check)
    torch.library.opcheck(ops.norm_rotate.default, (q, None, None, None, None, 0, False, None, None, None), **check)
    torch.library.opcheck(ops.norm_rotate_bwd.default, (q, q, k, k, pos, *rot, wq, wk, 1e-6, True, True), **check)
    torch.library.opcheck(ops.cache_append_rotated_.default,
                          (*cache, q, k, v, cu, table, start, pos, *rot, wq, wk, 1e-6), **check)
    torch.library.opcheck(ops.chunk_fwd.default, (q, cu, *cache, table, lengths, True, 0.1, True), **check)


def test_inference_mode_and_no_grad():
    q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu = _case()
    want = kernels.norm_rotate(q, k, pos, rot, wq, wk, 1e-6)
    leaf = wq.clone().requires_grad_(True)
    with torch.inference_mode():
        got = kernels.norm_rotate(q, k, pos, rot, leaf, wk, 1e-6)
        assert all(t.is_inference() for t in got)
    with torch.no_grad():
        more = kernels.norm_rotate(q, k, pos, rot, leaf, wk, 1e-6)
    for a, b, c in zip(want, got, more):
        assert torch.equal(a, b) and torch.equal(a, c) and not c.requires_grad


def test_a_projection_and_its_norms_train_together():
    """Gradients reach a projection through views of it, accumulated over two passes."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(70, 96, generator=g).cuda().to(BF16)
    w = (torch.randn(96, 10 * 64, generator=g) / 10).cuda().to(BF16).requires_grad_(True)
    wq, wk = (torch.ones(64, device='cuda').requires_grad_(True) for _ in range(2))
    pos, rot = torch.arange(70, device='cuda'), kernels.rotary(32)
    cu = pr.offsets([50, 20])
    for _ in range(2):
        qkv = (x @ w).view(70, 10, 64)
        q, k = kernels.norm_rotate(qkv[:, :6], qkv[:, 6:8], pos, rot, wq, wk, 1e-6)
        kernels.packed_attention(q, k, qkv[:, 8:], cu).float().square().sum().backward()
        if _ == 0:
            once = [t.grad.clone() for t in (w, wq, wk)]
    for t, a in zip((w, wq, wk), once):
        assert torch.isfinite(a).all() and a.abs().max() > 0 and torch.equal(t.grad, 2 * a)


def test_gradients_through_the_serving_forms_are_refused():
    q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu = _case()
    leaf = q.clone().requires_grad_(True)
    for call in (lambda: kernels.paged_chunk_attention(leaf, cu, cache, table, lengths),
                 lambda: kernels.cache_append_rotated_(cache, leaf, k, v, cu, table, start, rot, pos)):
        with pytest.raises(RuntimeError):
            call().sum().backward()


def test_calls_on_two_streams_at_once():
    cases = [_case(rows=21), _case(rows=21)]
    streams = [torch.cuda.Stream() for _ in cases]
    want = []
    for q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu in cases:
        y = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, pos, wq, wk, 1e-6)
        want.append(kernels.paged_chunk_attention(y, cu, cache, table, lengths))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (case, stream) in enumerate(zip(cases, streams)):
            q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu = case
            with torch.cuda.stream(stream):
                y = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, pos, wq, wk, 1e-6)
                got[i].append(kernels.paged_chunk_attention(y, cu, cache, table, lengths))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


@pytest.mark.parametrize('rows', [2000, 9000])  # 65 MB and 295 MB of q and k
@pytest.mark.parametrize('interleaved', [False, True])
def test_rows_that_are_moved_past_the_caches(rows, interleaved):
    """The same bits as in pieces that are not; the weights' gradients within the bound."""
    g = torch.Generator(device='cuda').manual_seed(1)
    q, k, dq, dk = (torch.randn(rows, h, 128, generator=g, device='cuda').to(BF16) for h in (96, 32, 96, 32))
    wq, wk = (1 + 0.2 * torch.randn(128, generator=g, device='cuda') for _ in range(2))
    rot, pos = kernels.rotary([16, 24, 24], interleaved=interleaved), torch.randint(0, 5000, (rows, 3), device='cuda')

    def step(at):
        leaves = [t[at].detach().requires_grad_(True) for t in (q, k)] + [t.clone().requires_grad_(True) for t in (wq, wk)]
        out = kernels.norm_rotate(*leaves[:2], pos[at], rot, *leaves[2:], 1e-6)
        return (*[t.detach() for t in out], *torch.autograd.grad(out, leaves, (dq[at], dk[at])))

    whole = step(slice(0, rows))
    sums = [0, 0]
    for i in range(0, rows, 500):
        part = step(slice(i, i + 500))
        for a, b in zip(whole[:4], part[:4]):
            assert torch.equal(a[i:i + 500], b)
        sums = [s + t.double() for s, t in zip(sums, part[4:])]
    for s, t, dy, x in zip(sums, whole[4:], (dq, dk), (q, k)):
        # of two pairs' |dy| |x r|, below 4 by square mean each: both sides' sums in 32 bits
        most = 2 * dy.float().abs().mean() * 1.2 * x.shape[0] * x.shape[1]
        assert (s - t.double()).abs().max() <= 2 * (rr.S + rr.LONG) * most


def test_different_calls_on_two_streams_at_once():
    """Every operator of the path, each stream with values and lengths of its own in the same
    shapes, keys in several splits and weights with gradients: what one call keeps in
    buffers is no other's."""
    heads, kv, d, new = 8, 2, 128, [40, 3]
    rot = kernels.rotary(64)
    cases = []
    for seed, lens in ((1, [1500, 2000]), (2, [900, 700])):
        g = torch.Generator().manual_seed(seed)
        q, k, v, dq, dk = (torch.randn(sum(new), h, d, generator=g).to(BF16).cuda() for h in (heads, kv, kv, heads, kv))
        wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).cuda() for _ in range(2))
        cache = kernels.paged_cache(256, 16, kv, d)
        for t in cache[:2]:
            t.copy_(torch.randn(t.shape, generator=g))
        table = torch.randperm(256, generator=g).to(torch.int32).view(2, 128).cuda()
        lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
        start = lengths - torch.tensor(new, dtype=torch.int32, device='cuda')
        pos = torch.randint(0, 9999, (sum(new),), generator=g).cuda()
        cases.append((q, k, v, dq, dk, wq, wk, cache, table, start, lengths, pos))
    assert ops_packed._chunk_splits(sum(new), heads, kv, d, 2, 128 * 16)[0] > 1
    cu = pr.offsets(new)

    def step(case):
        q, k, v, dq, dk, wq, wk, cache, table, start, lengths, pos = case
        leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        out = kernels.norm_rotate(*leaves[:2], pos, rot, *leaves[2:], 1e-6)
        grads = torch.autograd.grad(out, leaves, (dq, dk))
        y = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, None, wq, wk, 1e-6)
        return (*[t.detach() for t in out], *grads, y,
                *kernels.paged_chunk_attention(y, cu, cache, table, lengths, return_lse=True))

    want = [step(case) for case in cases]
    assert not any(torch.equal(a, b) for a, b in zip(*want))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for mine, case, stream in zip(got, cases, streams):
            with torch.cuda.stream(stream):
                mine.append(step(case))
    torch.cuda.synchronize()
    for mine, w in zip(got, want):
        for found in mine:
            assert all(torch.equal(a, b) for a, b in zip(found, w))


@pytest.mark.parametrize('dtype', [BF16, E4M3], ids=['bf16', 'e4m3'])
def test_compiled(dtype):
    """The public functions within torch.compile: the same bits, the ops in its graph."""
    q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu = _case(dtype)
    seen = []

    def backend(graph, _):
        seen.extend(str(n.target) for n in graph.graph.nodes)
        return graph.forward

    def serve(q, k, v, lengths):
        y, z = kernels.norm_rotate(q, k, pos, rot, wq, wk, 1e-6)
        x = kernels.cache_append_rotated_(cache, q, k, v, cu, table, start, rot, pos, wq, wk, 1e-6)
        return y, z, x, *kernels.paged_chunk_attention(x, cu, cache, table, lengths, return_lse=True)

    want = serve(q, k, v, lengths)
    held = [None if t is None else t.view(torch.uint8).clone() for t in cache]
    for t in cache:
        if t is not None:
            t.view(torch.uint8).zero_()
    got = torch.compile(serve, backend=backend, fullgraph=True)(q, k, v, lengths)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(a is None or torch.equal(a.view(torch.uint8), b) for a, b in zip(cache, held))
    for name in ('norm_rotate', 'cache_append_rotated_', 'chunk_fwd'):
        assert any(name in s for s in seen)


def test_compiled_with_gradients():
    q, k, v, wq, wk, cache, table, start, lengths, pos, rot, cu = _case()
    dq, dk = (torch.randn_like(t) for t in (q, k))

    def train(q, k, wq, wk):
        y, z = kernels.norm_rotate(q * 2, k * 2, pos, rot, wq, wk, 1e-6)
        return y + 1, z + 1

    def step(fn):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
        out = fn(*leaves)
        return (*[t.detach() for t in out], *torch.autograd.grad(out, leaves, (dq, dk)))

    got, want = step(torch.compile(train, backend='eager')), step(train)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
