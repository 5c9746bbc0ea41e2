"""Attention of packed sequences (kernels.packed_attention) against its
definition in 64 bits: grouped heads, both head dims, causal and not, lengths
from none to several tiles, rows that see nothing, strides, non-finite values
where no row looks, and captured graphs."""

import math

import pytest
import torch

from miowtion_amd import kernels, ops_packed
from tests import packed_reference as pr

pytestmark = pytest.mark.gpu


def _inputs(lens_q, lens_k, heads, kv, d, seed=0, pad_q=0, pad_k=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(lens_q) + pad_q, heads, d, generator=g)
    k = torch.randn(sum(lens_k) + pad_k, kv, d, generator=g)
    v = torch.randn(sum(lens_k) + pad_k, kv, d, generator=g)
    return [t.to(torch.bfloat16).cuda() for t in (q, k, v)]


CASES = [
    # lens_q, lens_k (None: lens_q), heads, kv, d, causal
    ([1], None, 1, 1, 128, True),
    ([77], None, 40, 8, 128, True),
    ([1, 2, 3, 64, 65, 127, 128, 129], None, 4, 2, 128, True),
    ([1, 2, 3, 64, 65, 127, 128, 129], None, 4, 2, 64, True),
    ([300, 0, 45, 513], None, 6, 2, 128, True),
    ([300, 0, 45, 513], None, 6, 2, 64, False),
    ([257, 130], None, 5, 1, 128, False),
    ([257, 130], None, 7, 7, 64, True),
    ([1, 17, 128], [700, 17, 1025], 8, 2, 128, True),
    ([1, 17, 128], [700, 17, 1025], 8, 8, 64, False),
    ([40, 5, 200], [7, 0, 199], 3, 1, 128, True),    # rows that see nothing
    ([40, 5, 200], [7, 0, 199], 14, 2, 64, True),
    ([40, 5, 200], [7, 0, 199], 4, 4, 128, False),
    ([1100], None, 2, 1, 128, True),
    ([1500, 9], None, 1, 1, 64, True),
    ([3] * 150 + [70], None, 4, 2, 64, True),        # more sequences than a wave has lanes
    ([20], None, 34, 2, 128, True),                   # seventeen heads to a group
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}')
def test_forward(case):
    lens_q, lens_k, heads, kv, d, causal = case
    lens_k = lens_k or lens_q
    print(f'packed forward {case}', flush=True)
    q, k, v = _inputs(lens_q, lens_k, heads, kv, d)
    cu_q, cu_k = pr.offsets(lens_q), pr.offsets(lens_k)
    out, lse = kernels.packed_attention(q, k, v, cu_q, cu_k, causal=causal, return_lse=True)
    ref = pr.attend(q, k, v, lens_q, lens_k, causal)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')
    again = kernels.packed_attention(q, k, v, cu_q, None if lens_k == lens_q else cu_k, causal=causal)
    assert torch.equal(out, again)


SPLIT = [
    # few rows against many keys: several workgroups share a row's keys
    ([5, 0, 130], [4000, 2100, 3001], 8, 2, 128, True),
    ([5, 0, 130], [4000, 2100, 3001], 4, 4, 64, False),
    ([1], [5000], 6, 1, 64, True),
    ([2500], None, 2, 1, 128, True),
    ([700, 40, 1], [700, 6000, 30], 2, 2, 64, True),
    ([3000, 2], [2000, 1], 1, 1, 128, True),         # rows that see nothing
]


@pytest.mark.parametrize('case', SPLIT, ids=lambda c: f'{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}')
def test_keys_shared_by_workgroups(case):
    lens_q, lens_k, heads, kv, d, causal = case
    lens_k = lens_k or lens_q
    print(f'packed forward, keys split {case}', flush=True)
    assert ops_packed._key_splits(sum(lens_q), sum(lens_k), len(lens_q), heads, kv) > 1
    q, k, v = _inputs(lens_q, lens_k, heads, kv, d, seed=2)
    cu_q, cu_k = pr.offsets(lens_q), pr.offsets(lens_k)
    out, lse = kernels.packed_attention(q, k, v, cu_q, cu_k, causal=causal, return_lse=True)
    ref = pr.attend(q, k, v, lens_q, lens_k, causal)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')
    assert torch.equal(out, kernels.packed_attention(q, k, v, cu_q, cu_k, causal=causal))
    # a value that is not finite in the middle of the first sequence's keys
    at = lens_k[0] // 2
    v[at, 0, 3] = math.nan
    got = kernels.packed_attention(q, k, v, cu_q, cu_k, causal=causal)
    sees = torch.zeros(sum(lens_q), dtype=torch.bool)
    first = lens_q[0]
    i = torch.arange(first)
    sees[:first] = (i + lens_k[0] - lens_q[0] >= at) if causal else True
    group = heads // kv
    assert torch.isnan(got[sees][:, :group, 3]).all()
    rest = got.clone()
    rest[:, :group, 3] = torch.where(sees[:, None].cuda(), ref['out'][:, :group, 3].to(got.dtype), got[:, :group, 3])
    pr.check(rest, ref, 'out')


@pytest.mark.parametrize('case', SPLIT + [([3000, 1000], None, 4, 2, 64, True), ([3000, 1000], None, 4, 2, 128, False)],
                         ids=lambda c: f'{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}')
def test_distance_by_norm(case):
    """Thousands of keys of like weight leave an out of some hundredths: the bound of a
    value, of the size of v, would let a split's sums go."""
    lens_q, lens_k, heads, kv, d, causal = case
    lens_k = lens_k or lens_q
    print(f'packed forward by norm {case}', flush=True)
    q, k, v = _inputs(lens_q, lens_k, heads, kv, d, seed=2)
    out = kernels.packed_attention(q, k, v, pr.offsets(lens_q), pr.offsets(lens_k), causal=causal)
    ref = pr.attend(q, k, v, lens_q, lens_k, causal)['out']
    first = 0
    for n in lens_q:
        rows, first = slice(first, first + n), first + n
        off = (out[rows].double() - ref[rows]).norm(dim=(0, 2))
        assert (off <= pr.NORM * ref[rows].norm(dim=(0, 2))).all(), off


def test_scale_and_large_scores():
    lens = [200, 33]
    q, k, v = _inputs(lens, lens, 4, 2, 128, seed=3)
    for scale, grow in ((0.3, 1.0), (1.0, 2.0), (1e-4, 1.0)):
        out, lse = kernels.packed_attention(q * grow, k, v, pr.offsets(lens), scale=scale, return_lse=True)
        ref = pr.attend(q * grow, k, v, lens, lens, True, scale)
        # scores up to 300: a score's error (128 2^-24 of sum |q k| scale, up to
        # 2,000) is past the bound's share for FP32 work, so it is added here
        reach = float((q.abs().double().amax() * grow * k.abs().double().amax() * scale) * 128)
        more = math.expm1(min(reach * 2.0 ** -17, 0.1))
        ref['out_tol'] = ref['out_tol'] + 2 * more * v.double().abs().amax()
        pr.check(out, ref, 'out')
        pr.check(lse, ref, 'lse')


def test_rows_of_no_sequence():
    lens = [50, 200]
    q, k, v = _inputs(lens, lens, 4, 2, 128, pad_q=150, pad_k=9)
    k[250:], v[250:] = math.nan, math.inf  # read by nobody
    q[250:] = math.nan
    out, lse = kernels.packed_attention(q, k, v, pr.offsets(lens), return_lse=True)
    ref = pr.attend(q, k, v, lens, lens)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')
    assert (out[250:] == 0).all() and (lse[250:] == -math.inf).all()
    # offsets that do not begin at row 0
    cu = pr.offsets(lens) + 7
    out, lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
    assert (out[:7] == 0).all() and (lse[:7] == -math.inf).all()
    assert (out[257:] == 0).all()
    ref = pr.attend(q[7:250], k[7:250], v[7:250], [50, 193], [50, 193])
    pr.check(out[7:57], {n: t[:50] for n, t in ref.items()}, 'out')


@pytest.mark.parametrize('d', [64, 128])
def test_values_behind_the_mask_do_not_reach_a_row(d):
    """A later token that is not finite changes no earlier row, and one sequence
    none of its neighbours."""
    lens = [90, 200, 70]
    q, k, v = _inputs(lens, lens, 4, 2, d, seed=5)
    cu = pr.offsets(lens)
    clean, clean_lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
    bad_v, bad_k = v.clone(), k.clone()
    bad_v[90 + 130, 0, 5] = math.nan
    bad_v[90 + 140, 1] = math.inf
    bad_k[90 + 150, 0, :3] = math.nan
    out, lse = kernels.packed_attention(q, bad_k, bad_v, cu, return_lse=True)
    before = torch.ones(360, dtype=torch.bool)
    before[90 + 130:290] = False
    # those rows are formed another way where they shared a tile with the rest
    ref = pr.attend(q, k, v, lens, lens)
    ref = {n: t[before] for n, t in ref.items()}
    pr.check(out[before], ref, 'out')
    assert torch.equal(lse[before], clean_lse[before])
    assert torch.isnan(out[90 + 130:290, :2, 5]).all()  # the heads of key head 0 from then on
    assert torch.isfinite(out[90 + 130:90 + 150, :2, 6]).all()
    assert (out[90 + 140:290, 2:] == math.inf).all()
    assert torch.isnan(lse[90 + 150:290, :2]).all()
    assert torch.equal(out[290:], clean[290:]) and torch.equal(out[:90], clean[:90])


def _time(fn, *args):
    """The least of five times, in us."""
    fn(*args)
    times = []
    for _ in range(5):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        fn(*args)
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end) * 1e3)
    return min(times)


@pytest.mark.parametrize('d', [64, 128])
def test_what_every_row_sees_takes_no_longer(d):
    """A key or a value that is not finite where every row sees it: not a case for
    the way that forms a row key by key, which takes 200 times as long."""
    lens = [4096, 300]
    q, k, v = _inputs(lens, lens, 8, 2, d, seed=8)
    cu = pr.offsets(lens)

    def attend(k, v):
        return kernels.packed_attention(q, k, v, cu, return_lse=True)

    clean, clean_lse = attend(k, v)
    plain = _time(attend, k, v)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[0, 0] = math.nan
    bad_v[0, 1, 3] = -math.inf
    out, lse = attend(bad_k, v)
    assert torch.isnan(out[:4096, :4]).all() and torch.isnan(lse[:4096, :4]).all()
    assert torch.equal(out[4096:], clean[4096:]) and torch.equal(lse[4096:], clean_lse[4096:])
    assert torch.equal(out[:, 4:], clean[:, 4:]) and torch.equal(lse[:, 4:], clean_lse[:, 4:])
    took = _time(attend, bad_k, v)
    print(f'{plain:.0f} us, with a key that is NaN {took:.0f}', flush=True)
    assert took < 10 * plain
    out, lse = attend(k, bad_v)
    assert (out[:4096, 4:, 3] == -math.inf).all() and torch.equal(lse, clean_lse)
    out[:4096, 4:, 3] = clean[:4096, 4:, 3]
    assert torch.equal(out, clean)
    took = _time(attend, k, bad_v)
    print(f'{plain:.0f} us, with a value that is infinite {took:.0f}', flush=True)
    assert took < 10 * plain


@pytest.mark.parametrize('d', [64, 128])
def test_a_score_that_is_not_a_number_in_some_splits(d):
    """Keys shared by workgroups: the NaN of one split's sum of weights reaches every
    column, and where another's V is behind the mask as well."""
    lens_q, lens_k = [130, 3], [6000, 4000]
    assert ops_packed._key_splits(133, 10000, 2, 4, 2) > 1
    q, k, v = _inputs(lens_q, lens_k, 4, 2, d, seed=12)
    cu_q, cu_k = pr.offsets(lens_q), pr.offsets(lens_k)
    ref = pr.attend(q, k, v, lens_q, lens_k)
    k[40, 0, 1] = math.nan
    v[5950, 0, 2] = math.inf   # seen by the rows from 80 on
    v[5950, 1, 2] = math.inf
    out, lse = kernels.packed_attention(q, k, v, cu_q, cu_k, return_lse=True)
    assert torch.isnan(out[:130, :2]).all() and torch.isnan(lse[:130, :2]).all()
    assert (out[80:130, 2:, 2] == math.inf).all()
    out[:130, :2], lse[:130, :2] = ref['out'][:130, :2].to(out.dtype), ref['lse'][:130, :2].float()
    out[80:130, 2:, 2] = ref['out'][80:130, 2:, 2].to(out.dtype)
    pr.check(out, ref, 'out')
    pr.check(lse, ref, 'lse')


def test_strides_and_shared_storage():
    lens = [130, 61]
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(sum(lens), 8 + 2 + 2, 128, generator=g).to(torch.bfloat16).cuda()
    q, k, v = qkv.split([8, 2, 2], 1)  # one projection's rows
    ref = pr.attend(q, k, v, lens, lens)
    pr.check(kernels.packed_attention(q, k, v, pr.offsets(lens)), ref, 'out')
    # heads first, and one key head for all by a stride of 0
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    ke, ve = (t[:, :1].expand(-1, 4, -1) for t in (k, v))
    ref = pr.attend(qt, ke, ve, lens, lens)
    pr.check(kernels.packed_attention(qt, ke, ve, pr.offsets(lens)), ref, 'out')
    # every second row
    q2, k2, v2 = (t[::2] for t in (q, k, v))
    lens2 = [65, 31]
    ref = pr.attend(q2, k2, v2, lens2, lens2)
    pr.check(kernels.packed_attention(q2, k2, v2, pr.offsets(lens2)), ref, 'out')


def test_nothing_to_do():
    q, k, v = _inputs([4], [4], 4, 2, 64)
    none = torch.zeros(1, dtype=torch.int32, device='cuda')
    out, lse = kernels.packed_attention(q, k, v, none, return_lse=True)  # no sequence
    assert (out == 0).all() and (lse == -math.inf).all()
    assert kernels.packed_attention(q[:0], k, v, torch.zeros(2, dtype=torch.int32, device='cuda')).shape == (0, 4, 64)
    out = kernels.packed_attention(q, k[:0], v[:0], pr.offsets([4]), torch.zeros(2, dtype=torch.int32, device='cuda'))
    assert (out == 0).all()


def test_offsets_that_make_no_sense_stay_within_the_tensors():
    q, k, v = _inputs([300], [300], 4, 2, 128)
    guard = torch.full((64, 4, 128), 7.0, dtype=torch.bfloat16, device='cuda')
    for cu in ([0, 500], [-5, 10, 100000], [200, 100, 300], [300, 0], [5, 5, 5]):
        print(f'offsets {cu}', flush=True)
        out = kernels.packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device='cuda'))
        assert out.shape == q.shape
    assert (guard == 7.0).all()
    out = kernels.packed_attention(q, k, v, torch.tensor([0, 500], dtype=torch.int32, device='cuda'))
    pr.check(out, pr.attend(q, k, v, [300], [300]), 'out')


def test_graph_serves_new_lengths():
    q, k, v = _inputs([300], [300], 4, 2, 128)
    cu = pr.offsets([100, 200])
    kernels.packed_attention(q, k, v, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
    for lens in ([100, 200], [1, 299], [300, 0], [17, 100]):
        cu.copy_(pr.offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse = kernels.packed_attention(q, k, v, cu, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        pr.check(out, pr.attend(q, k, v, lens, lens), 'out')


def test_side_stream_and_inference_mode():
    lens = [200]
    q, k, v = _inputs(lens, lens, 4, 2, 128)
    cu = pr.offsets(lens)
    want = kernels.packed_attention(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.inference_mode():
        out = kernels.packed_attention(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


def test_refusals():
    q, k, v = _inputs([16], [16], 4, 2, 128)
    cu = pr.offsets([16])
    f = kernels.packed_attention
    for bad, match in [
            (lambda: f(q.float(), k, v, cu), 'bfloat16'),
            (lambda: f(q[0], k, v, cu), 'rows, heads'),
            (lambda: f(q, k[..., :64], v[..., :64], cu), 'head_dim'),
            (lambda: f(q[..., :96], k[..., :96], v[..., :96], cu), 'head_dim'),
            (lambda: f(q[:, :3], k, v, cu), 'multiple'),
            (lambda: f(q, k, v[:8], cu), 'equal shapes'),
            (lambda: f(q, k, v, cu.long()), 'int32'),
            (lambda: f(q, k, v, cu, cu[:1]), 'int32'),
            (lambda: f(q, k, v, cu, scale=0.0), 'scale'),
            (lambda: f(q, k, v, cu, scale=-1.0), 'scale'),
            (lambda: f(q, k, v, cu, scale=math.nan), 'scale'),
            (lambda: f(q.new_empty(16 * 4 * 128 + 8)[4:-4].view(16, 4, 128), k, v, cu), '16-byte')]:
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises((ValueError, NotImplementedError)):
        f(q, k, v, cu.cpu())
