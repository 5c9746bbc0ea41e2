"""Attention over packed prompts and over a paged cache, as measurable cases.

What is measured are the operators that a text side needs beside this package's
video attention: prompts of different lengths packed one behind the other, in
inference and in training, a paged key-value cache that is written in bf16 or in
eight bits and read back, and the attention of one new token over it.

Kinds of case:
  prompt  packed attention, causal or not, grouped heads: out and LSE
  train   the same with the gradients of q, k and v
  cache   new tokens appended to a paged cache, and the whole context read back
          from it (what the next chunk of a long prompt attends to)
  token   one new token of every sequence over the paged cache: out and LSE

Fields of a case: `lens` are the key lengths of the sequences, a text of numbers,
or `seqs` lengths spread over `shortest` .. `longest` by their logarithm (`spread`
is their seed); `new` is how many of a sequence's last tokens are queries or are appended
(0: all of them), `pad` how many rows stand behind the last sequence.
"""

from __future__ import annotations

import math
import random

import torch

own = False

# what an optional field of a case is when it is absent
DEFAULTS = dict(lens='', seqs=0, shortest=1, longest=0, spread=0, new=0, pad=0, causal=True, bits=16, page=16)
BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn


def listed() -> list[dict]:
    return [
        # one short caption through a text encoder: launches are all that counts
        dict(name='prompt_caption', kind='prompt', lens='77', heads=40, kv=8, dim=128),
        # a batch of ragged prompts packed without padding, behind them the rows
        # that align the buffer
        dict(name='prompt_ragged', kind='prompt', seqs=16, longest=2048, spread=3, heads=40, kv=8,
             dim=128, pad=29),
        # the next chunk of four long prompts against what the cache held, narrow heads
        dict(name='prompt_chunk', kind='prompt', lens='8192,5003,7168,1025', new=512, heads=32, kv=8,
             dim=64),
        # one long document: the whole prompt at once
        dict(name='prompt_long', kind='prompt', lens='16384', heads=16, kv=4, dim=128),
        # a small fine-tuning step: three captions, two key heads
        dict(name='train_captions', kind='train', lens='333,77,201', heads=8, kv=2, dim=64),
        # a packed training batch of ragged prompts
        dict(name='train_ragged', kind='train', seqs=12, longest=2048, spread=5, heads=32, kv=8,
             dim=128, pad=13),
        # training on long documents
        dict(name='train_long', kind='train', lens='8192', heads=28, kv=4, dim=128),
        # one token of each of 32 sequences into an eight-bit cache, and the contexts back
        dict(name='cache_e4m3', kind='cache', seqs=32, longest=4096, spread=7, new=1, bits=8, page=16,
             kv=8, dim=128),
        # a chunk of long prompts into a bf16 cache with large pages, and the contexts back
        dict(name='cache_chunk', kind='cache', lens='32768,20001', new=2048, bits=16, page=64, kv=8,
             dim=128),
        # one sequence being written, a token at a time
        dict(name='token_one', kind='token', lens='1500', heads=32, kv=8, dim=128, page=16),
        # a batch of sequences of all lengths over an eight-bit cache
        dict(name='token_ragged', kind='token', seqs=64, longest=8192, spread=11, bits=8, page=16,
             heads=40, kv=8, dim=128),
        # few sequences with long contexts
        dict(name='token_long', kind='token', lens='131072,65537,100003,90001', heads=56, kv=8, dim=128,
             page=64),
    ]


def draw(rng) -> dict:
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    tops = {}
    for c in listed():
        c = _full(c)
        tops[c['kind']] = max(tops.get(c['kind'], 0), _cost(c))
    while True:
        kind = rng.choice(['prompt', 'prompt', 'train', 'train', 'cache', 'token', 'token'])
        kv = rng.choice([1, 2, 3, 4, 8])
        case = dict(kind=kind, kv=kv, dim=rng.choice([64, 128, 128]), seqs=log(1, 64),
                    longest=log(2, 131072 if kind == 'token' else 32768), spread=rng.randrange(10 ** 6))
        if rng.random() < 0.5:
            case['shortest'] = case['longest'] // 2 + 1
        if kind != 'cache':
            case['heads'] = kv * rng.choice([1, 2, 3, 4, 5, 7, 8])
        if kind in ('prompt', 'train'):
            case['causal'] = rng.random() < 0.8
            case['pad'] = rng.choice([0, 0, rng.randint(1, 200)])
        if kind == 'prompt':
            case['new'] = rng.choice([0, 0, 0, log(1, 2048)])
        if kind in ('cache', 'token'):
            case['bits'] = rng.choice([8, 16])
            case['page'] = rng.choice([16, 32, 64, 128])
        if kind == 'cache':
            case['new'] = rng.choice([0, 1, log(1, 4096)])
            case['pad'] = rng.choice([0, 0, rng.randint(1, 200)])
        if _cost(_full(case)) <= tops[kind]:
            return case


# ---------------------------------------------------------------------------
# Sizes


def _full(case: dict) -> dict:
    return {**DEFAULTS, **case}


def _lens(case: dict) -> list[int]:
    """Key lengths of the sequences."""
    if case['lens']:
        return [int(n) for n in case['lens'].split(',')]
    rng = random.Random(case['spread'])
    return [int(round(math.exp(rng.uniform(math.log(case['shortest']), math.log(case['longest']))))) for _ in range(case['seqs'])]


def _new(case: dict) -> list[int]:
    """Queries (or appended tokens) of the sequences: their last ones."""
    return [min(n, case['new']) if case['new'] else n for n in _lens(case)]


def _cost(case: dict) -> float:
    """What a case may cost at most: its padded products or rows, which bound the
    plain form's memory and time."""
    lens, new = _lens(case), _new(case)
    rows = len(lens) * max(lens)
    if case['kind'] in ('prompt', 'train'):
        return rows * max(new) * case['heads'] * case['dim']
    return rows * case['kv'] * case['dim']


def _pairs(case: dict) -> int:
    """(query, key) pairs of one head that are not masked."""
    total = 0
    for n, m in zip(_lens(case), _new(case)):
        total += m * n - (m * (m - 1) // 2 if case['causal'] else 0)
    return total


def work(case: dict) -> dict:
    c = _full(case)
    lens, new = _lens(c), _new(c)
    nk, nq, d = sum(lens), sum(new), c['dim']
    if c['kind'] == 'prompt':
        pad = c['pad']
        return dict(bytes=2 * d * (2 * (nq + pad) * c['heads'] + 2 * nk * c['kv']) + 4 * nq * c['heads'],
                    flops=4 * d * c['heads'] * _pairs(c))
    if c['kind'] == 'train':
        # q, k, v and the output's gradient read, out and three gradients written
        return dict(bytes=2 * d * (4 * nq * c['heads'] + 4 * nk * c['kv']),
                    flops=14 * d * c['heads'] * _pairs(c))
    row = d * c['bits'] // 8 + (1 if c['bits'] == 8 else 0)  # a cached row and its exponent
    if c['kind'] == 'cache':
        # new rows read and written, the contexts read and written as bf16
        return dict(bytes=2 * c['kv'] * (nq * (2 * d + row) + nk * (row + 2 * d)), flops=0)
    return dict(bytes=2 * c['kv'] * nk * row + 4 * len(lens) * c['heads'] * d,
                flops=4 * d * c['heads'] * nk)


# ---------------------------------------------------------------------------
# Inputs


def _offsets(lens: list[int]) -> list[int]:
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def prepare(case: dict, seed: int) -> dict:
    c = _full(case)
    lens, new = _lens(c), _new(c)
    d, kv = c['dim'], c['kv']
    g = torch.Generator(device='cuda').manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device='cuda')

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device='cuda')

    s = dict(c, longest_k=max(lens), longest_q=max(new))
    if c['kind'] in ('prompt', 'train'):
        # queries and keys after normalisation: unit noise, and a direction that
        # all share, so that some keys draw more weight than others
        heads, nk, nq, pad = c['heads'], sum(lens), sum(new), c['pad']
        s['cu_k'], s['cu_q'] = ints(_offsets(lens)), ints(_offsets(new))
        shared = rand(1, 1, d)
        s['q'] = (rand(nq + pad, heads, d) + 0.7 * shared).to(BF16)
        s['k'] = (rand(nk + pad, kv, d) + 0.7 * rand(nk + pad, kv, 1) * shared).to(BF16)
        s['v'] = rand(nk + pad, kv, d).to(BF16)
        if c['kind'] == 'train':
            s['dout'] = rand(nq + pad, heads, d).to(BF16)
            for t in ('q', 'k', 'v'):
                s[t].requires_grad_(True)
        return s

    # a paged cache that has been in use: a sequence's pages lie anywhere
    page = c['page']
    width = -(-max(lens) // page)
    need = sum(-(-n // page) for n in lens)
    pages = need + need // 8 + 1
    order = torch.randperm(pages, generator=g, device='cuda').to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device='cuda')
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order[at:at + m]
        at += m
    s['table'] = table
    for t in ('k', 'v'):
        # a head's rows of a page lie together; rows of different tokens differ in size
        rows = rand(pages, kv, page, d)
        if t == 'k':
            rows = rows * torch.exp(0.3 * rand(pages, kv, page, 1))
        if c['bits'] == 8:
            power = _power(rows)
            s[t + '_pages'] = torch.ldexp(rows, -power).to(E4M3).transpose(1, 2)
            s[t + '_exp'] = (power[..., 0] + 127).to(torch.uint8).transpose(1, 2)
        else:
            s[t + '_pages'] = rows.to(BF16).transpose(1, 2)
            s[t + '_exp'] = None
        del rows
    if c['kind'] == 'cache':
        s['cu_new'], s['cu'] = ints(_offsets(new)), ints(_offsets(lens))
        s['start'] = ints([n - m for n, m in zip(lens, new)])
        s['rows'] = sum(lens)
        s['k_new'] = (rand(sum(new) + c['pad'], kv, d) * 1.5).to(BF16)
        s['v_new'] = rand(sum(new) + c['pad'], kv, d).to(BF16)
    else:
        s['lengths'] = ints(lens)
        s['q'] = rand(len(lens), c['heads'], d).to(BF16)
    return s


# ---------------------------------------------------------------------------
# One pass


def run(s: dict):
    if own:
        from miowtion_amd import kernels
        if s['kind'] == 'prompt':
            return kernels.packed_attention(s['q'], s['k'], s['v'], s['cu_q'], s['cu_k'],
                                            causal=s['causal'], return_lse=True)
        if s['kind'] == 'train':
            out = kernels.packed_attention(s['q'], s['k'], s['v'], s['cu_q'], s['cu_k'],
                                           causal=s['causal'])
            return (out.detach(), *torch.autograd.grad(out, (s['q'], s['k'], s['v']), s['dout']))
        cache = kernels.PagedCache(s['k_pages'], s['v_pages'], s['k_exp'], s['v_exp'])
        if s['kind'] == 'cache':
            kernels.cache_append_(cache, s['k_new'], s['v_new'], s['cu_new'], s['table'], s['start'])
            return kernels.cache_gather(cache, s['cu'], s['table'], s['rows'])
        return kernels.paged_attention(s['q'], cache, s['table'], s['lengths'], return_lse=True)
    if s['kind'] == 'prompt':
        out, lse, _ = _attend(s)
        return out.to(BF16), lse
    if s['kind'] == 'train':
        return _train(s)
    if s['kind'] == 'cache':
        return _append_and_read(s)
    return _token(s)


def _padded(x, cu, longest):
    """Packed rows [T, H, D] as [B, H, longest, D] in 32 bits, and which of them are rows."""
    at = torch.arange(longest, device=x.device)
    there = at < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + at).clamp(max=max(x.shape[0] - 1, 0))
    return (x[rows].float() * there[..., None, None]).permute(0, 2, 1, 3), there


def _packed(x, cu, total):
    """The rows of [B, H, longest, D] back in their places, zero elsewhere."""
    row = torch.arange(total, device=x.device, dtype=torch.int32)
    seq = torch.searchsorted(cu, row, right=True) - 1
    there = (seq >= 0) & (row < cu[-1])
    seq = seq.clamp(0, x.shape[0] - 1)
    at = (row - cu[seq]).clamp(0, x.shape[2] - 1)
    return x[seq, :, at] * there[:, None, None]


def _attend(s):
    cu_q, cu_k = s['cu_q'], s['cu_k']
    q, q_ok = _padded(s['q'].detach(), cu_q, s['longest_q'])
    k, k_ok = _padded(s['k'].detach(), cu_k, s['longest_k'])
    v, _ = _padded(s['v'].detach(), cu_k, s['longest_k'])
    b, heads, m, d = q.shape
    kv, n = k.shape[1], k.shape[2]
    q = q.reshape(b, kv, heads // kv * m, d)  # the heads of a group beside each other
    see = k_ok[:, None, :] & q_ok[:, :, None]
    if s['causal']:
        nq, nk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
        i = torch.arange(m, device=q.device)[:, None]
        see = see & (torch.arange(n, device=q.device) <= i + (nk - nq)[:, None, None])
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).reshape(b, heads, m, n)
    p.masked_fill_(~see[:, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(p.reshape(b, kv, heads // kv * m, n), v).reshape(b, heads, m, d)
    lse = top + torch.log(total)
    rows = s['q'].shape[0]
    lse = _packed(torch.where(lse == -math.inf, 0.0, lse), cu_q, rows)[..., 0]
    sees = _packed((total > 0).float(), cu_q, rows)[..., 0]
    lse = torch.where(sees > 0, lse, -math.inf)
    return _packed(out, cu_q, rows), lse, (q, k, v, p, out)


def _train(s):
    packed, _, (q, k, v, p, out) = _attend(s)
    dout, _ = _padded(s['dout'], s['cu_q'], s['longest_q'])
    b, heads, m, d = out.shape
    kv, n = k.shape[1], k.shape[2]
    group = (b, kv, heads // kv * m)
    dout_g, p = dout.reshape(*group, d), p.reshape(*group, n)
    dv = torch.matmul(p.transpose(-1, -2), dout_g)
    ds = torch.matmul(dout_g, v.transpose(-1, -2))
    ds.sub_((dout * out).sum(-1).reshape(*group, 1)).mul_(p).mul_(d ** -0.5)
    dq = torch.matmul(ds, k).reshape(b, heads, m, d)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    rows, keys = s['q'].shape[0], s['k'].shape[0]
    return (packed.to(BF16), _packed(dq, s['cu_q'], rows).to(BF16), _packed(dk, s['cu_k'], keys).to(BF16),
            _packed(dv, s['cu_k'], keys).to(BF16))


def _power(rows):
    """The least power of two that brings a row's largest magnitude to 448 or less."""
    m, e = torch.frexp(rows.abs().amax(-1, keepdim=True).float())
    return (e - 9 + (m > 0.875)).clamp(min=-127)


def _context(s, t, longest):
    """Every sequence's cached rows in 32 bits, [B, longest, kv, d]."""
    pages, page = s[t + '_pages'], s['page']
    at = torch.arange(longest, device=pages.device)
    where = s['table'][:, at // page]
    rows = pages[where, at % page].float()
    if s[t + '_exp'] is None:
        return rows
    return torch.ldexp(rows, s[t + '_exp'][where, at % page, :, None].int() - 127)


def _append_and_read(s):
    cu_new, cu, page = s['cu_new'], s['cu'], s['page']
    row = torch.arange(s['longest_q'], device=cu.device)
    count = (cu_new[1:] - cu_new[:-1])[:, None]
    # every sequence's slot of the grid; those past its end repeat its last row
    i = torch.minimum(row, count - 1)
    src = (cu_new[:-1, None] + i).reshape(-1)
    pos = (s['start'][:, None] + i).long()
    where = s['table'].gather(1, pos // page).reshape(-1)
    at = pos.reshape(-1) % page
    out = []
    for t in ('k', 'v'):
        rows, pages = s[t + '_new'][src], s[t + '_pages']
        if s[t + '_exp'] is None:
            pages[where, at] = rows
        else:
            power = _power(rows)
            codes = torch.ldexp(rows.float(), -power).to(E4M3)
            pages.view(torch.uint8)[where, at] = codes.view(torch.uint8)
            s[t + '_exp'][where, at] = (power[..., 0] + 127).to(torch.uint8)
        context = _context(s, t, s['longest_k']).permute(0, 2, 1, 3)
        out.append(_packed(context, cu, s['rows']).to(BF16))
    return tuple(out)


def _token(s):
    b, heads, d = s['q'].shape
    kv, n = s['kv'], s['longest_k']
    q = s['q'].float().reshape(b, kv, heads // kv, d)
    k = _context(s, 'k', n).permute(0, 2, 1, 3)
    there = torch.arange(n, device=q.device) < s['lengths'][:, None]
    p = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    p = p.masked_fill(~there[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - top)
    total = p.sum(-1, keepdim=True)
    p, lse = p / total, top + torch.log(total)
    v = _context(s, 'v', n).permute(0, 2, 1, 3)
    return torch.matmul(p, v).reshape(b, heads, d).to(BF16), lse.reshape(b, heads)


# ---------------------------------------------------------------------------
# The definition in 64 bits, a sequence and a head at a time


def exact(case: dict, seed: int):
    c = _full(case)
    lens, new = _lens(c), _new(c)
    if c['kind'] in ('prompt', 'train') and sum(n * m for n, m in zip(lens, new)) * c['heads'] > 1.5e10:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        if c['kind'] in ('prompt', 'train'):
            return _exact_packed(s, lens, new)
        if c['kind'] == 'cache':
            return _exact_cache(s, lens, new)
        return _exact_token(s, lens)


def _exact_packed(s, lens, new):
    q, k, v = (s[t].detach() for t in ('q', 'k', 'v'))
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v))
    i0 = j0 = 0
    for n, m in zip(lens, new):
        hidden = None
        if s['causal']:
            hidden = torch.ones(m, n, dtype=torch.bool, device=q.device).triu(n - m + 1)
        for h in range(q.shape[1]):
            qh, kh, vh = q[i0:i0 + m, h].double(), k[j0:j0 + n, h // group].double(), \
                v[j0:j0 + n, h // group].double()
            a = qh @ kh.t() / math.sqrt(d)
            if hidden is not None:
                a[hidden] = -math.inf
            lse[i0:i0 + m, h] = torch.logsumexp(a, -1)
            a = torch.softmax(a, -1)
            out[i0:i0 + m, h] = a @ vh
            if s['kind'] == 'train':
                go = s['dout'][i0:i0 + m, h].double()
                dv[j0:j0 + n, h // group] += a.t() @ go
                ga = go @ vh.t()
                ga = a * (ga - (a * ga).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[i0:i0 + m, h] = ga @ kh
                dk[j0:j0 + n, h // group] += ga.t() @ qh
        i0, j0 = i0 + m, j0 + n
    return (out, dq, dk, dv) if s['kind'] == 'train' else (out, lse)


def _exact_rows(s, t, b, n):
    used = s['table'][b, :-(-n // s['page'])].long()
    x = s[t + '_pages'][used].double()
    if s[t + '_exp'] is not None:
        x = x * torch.exp2(s[t + '_exp'][used].double() - 127)[..., None]
    return x.flatten(0, 1)[:n]


def _exact_cache(s, lens, new):
    found = []
    for t in ('k', 'v'):
        parts, i0 = [], 0
        for b, (n, m) in enumerate(zip(lens, new)):
            rows = s[t + '_new'][i0:i0 + m].double()
            if s[t + '_exp'] is not None:
                # steps of an eighth of the value's own power of two, no finer than
                # that of 2^-6, in units that bring the row's largest to 448 or less
                unit = torch.exp2(torch.ceil(torch.log2(rows.abs().amax(-1, keepdim=True) / 448)))
                x = rows / unit
                step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
                rows = torch.round(x / step) * step * unit
            parts += [_exact_rows(s, t, b, n)[:n - m], rows]
            i0 += m
        found.append(torch.cat(parts))
    return tuple(found)


def _exact_token(s, lens):
    q = s['q']
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    group = q.shape[1] // s['kv']
    for b, n in enumerate(lens):
        keys, values = (_exact_rows(s, t, b, n).transpose(0, 1).contiguous() for t in ('k', 'v'))
        for h in range(s['kv']):
            mine = slice(h * group, (h + 1) * group)
            a = q[b, mine].double() @ keys[h].t() / math.sqrt(q.shape[2])
            lse[b, mine] = torch.logsumexp(a, -1)
            out[b, mine] = torch.softmax(a, -1) @ values[h]
    return out, lse
