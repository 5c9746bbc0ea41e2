"""The way from projections to attention, as measurable cases.

What is measured are the operators before and behind the cache of new keys: norms
of the query and key heads with the rotation by position (one axis for text, three
for the tokens of a clip), in inference and in training; the same on the way into
a paged cache; and attention of a chunk of new tokens, from a few that are to be
verified to the next part of a long prompt, over the cache's pages as they lie.

Kinds of case:
  rotate  q and k normalised by head and rotated
  train   the same with the gradients of q, k and both weights
  append  new rows normalised and rotated, q returned, k and v written to the cache
  chunk   attention of every sequence's last tokens over the cache: out and LSE

Fields of a case: tokens are the rows of a clip's `grid` (frames, rows, columns)
or of sequences, `lens` a text of their lengths or `seqs` lengths spread over
`shortest` .. `longest` by their logarithm (`spread` is their seed); `new` is how
many of a sequence's last tokens are queries or are appended (0: all of them).
`sections` are the pairs of dims that turn with each axis of the positions,
`adjacent` whether a pair is two dims side by side, `fps` a factor of the first
axis (0: positions are whole numbers), `eps` the norm's (0: no norm), `wbits` the
bits of its weights.
"""

from __future__ import annotations

import math
import random

import torch

own = False

# what an optional field of a case is when it is absent
DEFAULTS = dict(grid='', lens='', seqs=0, shortest=1, longest=0, spread=0, new=0, causal=True, bits=16, page=16,
                sections='', adjacent=False, fps=0.0, base=10000.0, eps=1e-6, wbits=16)
BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn


def listed() -> list[dict]:
    return [
        # one short caption through a layer of a text encoder: launches are all that counts
        dict(name='rotate_caption', kind='rotate', lens='77', heads=40, kv=8, dim=128, sections='64'),
        # a four-frame preview with narrow heads, frames at their time in seconds
        dict(name='rotate_preview', kind='rotate', grid='4,30,52', heads=40, kv=8, dim=64, sections='8,12,12',
             adjacent=True, fps=0.6875),
        # a layer of a whole clip
        dict(name='rotate_clip', kind='rotate', grid='37,30,52', heads=48, kv=48, dim=128, sections='16,24,24'),
        # a small fine-tuning step: three captions, two key heads
        dict(name='train_captions', kind='train', lens='333,77,201', heads=8, kv=2, dim=64, sections='32'),
        # training on a clip of sixteen frames, weights in 32 bits
        dict(name='train_clip', kind='train', grid='16,30,52', heads=48, kv=48, dim=128, sections='16,24,24',
             wbits=32),
        # one token of each of 32 sequences that are being written
        dict(name='append_token', kind='append', seqs=32, longest=4096, spread=7, new=1, heads=40, kv=8, dim=128,
             sections='64'),
        # ragged prompts into an eight-bit cache, and its contexts back
        dict(name='append_e4m3', kind='append', seqs=12, longest=2048, spread=5, bits=8, heads=40, kv=8, dim=128,
             sections='64', base=1e6),
        # the next chunk of long prompts with clips in them, into large pages
        dict(name='append_chunk', kind='append', lens='32768,20001', new=2048, page=64, heads=32, kv=8, dim=128,
             sections='16,24,24'),
        # four proposed tokens of eight sequences to be verified
        dict(name='chunk_verify', kind='chunk', seqs=8, shortest=2000, longest=8192, spread=2, new=4, heads=32,
             kv=8, dim=128),
        # a batch of sequences of all lengths over an eight-bit cache, sixteen tokens each
        dict(name='chunk_ragged', kind='chunk', seqs=48, longest=8192, spread=11, new=16, bits=8, heads=40, kv=8,
             dim=128),
        # the next chunk of four prompts, narrow heads, eight bits
        dict(name='chunk_narrow', kind='chunk', lens='8192,5003,7168,1025', new=512, bits=8, page=32, heads=32,
             kv=8, dim=64),
        # the next chunk of two long prompts
        dict(name='chunk_prompt', kind='chunk', lens='32768,20001', new=2048, page=64, heads=32, kv=8, dim=128),
    ]


def draw(rng) -> dict:
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    tops = {}
    for c in listed():
        c = _full(c)
        tops[c['kind']] = max(tops.get(c['kind'], 0), _cost(c))
    while True:
        kind = rng.choice(['rotate', 'train', 'append', 'append', 'chunk', 'chunk', 'chunk'])
        kv = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 128, 128])
        case = dict(kind=kind, kv=kv, heads=kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), dim=dim)
        if kind != 'chunk':
            quarter = dim // 8  # of the pairs that the head has
            case['sections'] = ','.join(map(str, rng.choice([
                [4 * quarter], [2 * quarter], [quarter, quarter, 2 * quarter], [2 * quarter, quarter, quarter],
                [quarter, quarter]])))
            case['adjacent'] = rng.random() < 0.4
            case['base'] = rng.choice([1e4, 1e6])
            case['wbits'] = rng.choice([16, 32])
            if kind != 'train' and rng.random() < 0.2:
                case['eps'] = 0.0
            if kind == 'rotate' and rng.random() < 0.3:
                case['fps'] = round(rng.uniform(0.1, 2.0), 3)
        if kind in ('rotate', 'train') and rng.random() < 0.5:
            case['kv'] = case['heads'] = rng.choice([5, 16, 28, 40])
            case['grid'] = f'{log(1, 102)},{rng.randint(5, 60)},{rng.randint(5, 60)}'
        else:
            case['seqs'], case['spread'] = log(1, 64), rng.randrange(10 ** 6)
            case['longest'] = log(2, 32768)
            if rng.random() < 0.5:
                case['shortest'] = case['longest'] // 2 + 1
        if kind in ('append', 'chunk'):
            case['bits'] = rng.choice([8, 16])
            case['page'] = rng.choice([16, 32, 64, 128])
            case['new'] = rng.choice([log(1, 16), log(1, 4096), 0]) if kind == 'append' else \
                rng.choice([log(2, 16), log(2, 2048)])
        if kind == 'chunk':
            case['causal'] = rng.random() < 0.8
        if _cost(_full(case)) <= tops[kind]:
            return case


# ---------------------------------------------------------------------------
# Sizes


def _full(case: dict) -> dict:
    return {**DEFAULTS, **case}


def _grid(case: dict) -> list[int]:
    return [int(n) for n in case['grid'].split(',')]


def _sections(case: dict) -> list[int]:
    return [int(n) for n in case['sections'].split(',')]


def _lens(case: dict) -> list[int]:
    """Lengths of the sequences, new tokens included."""
    if case['grid']:
        return [math.prod(_grid(case))]
    if case['lens']:
        return [int(n) for n in case['lens'].split(',')]
    rng = random.Random(case['spread'])
    return [int(round(math.exp(rng.uniform(math.log(case['shortest']), math.log(case['longest']))))) for _ in range(case['seqs'])]


def _new(case: dict) -> list[int]:
    """Queries (or appended tokens) of the sequences: their last ones."""
    return [min(n, case['new']) if case['new'] else n for n in _lens(case)]


def _cost(case: dict) -> float:
    """What a case may cost at most, by rows and padded products, which bound the
    plain form's memory and time."""
    lens, new = _lens(case), _new(case)
    if case['kind'] == 'chunk':
        return len(lens) * max(lens) * max(new) * case['heads'] * case['dim']
    rows = sum(new) * (case['heads'] + case['kv']) * case['dim']
    if case['kind'] == 'append':
        rows += sum(lens) * case['kv'] * case['dim']  # the cache that is returned
    return rows


def work(case: dict) -> dict:
    c = _full(case)
    lens, new = _lens(c), _new(c)
    nk, nq, d = sum(lens), sum(new), c['dim']
    values = nq * (c['heads'] + c['kv']) * d
    if c['kind'] == 'rotate':
        return dict(bytes=4 * values, flops=10 * values)
    if c['kind'] == 'train':
        # q, k and the gradients read, the rotated and two gradients written
        return dict(bytes=8 * values, flops=30 * values)
    row = d * c['bits'] // 8 + (1 if c['bits'] == 8 else 0)  # a cached row and its exponent
    if c['kind'] == 'append':
        # new rows read and written; an eight-bit cache's contexts read and written as bf16
        back = 2 * c['kv'] * nk * (row + 2 * d) if c['bits'] == 8 else 0
        return dict(bytes=4 * nq * c['heads'] * d + 2 * c['kv'] * nq * (2 * d + row) + back, flops=10 * values)
    pairs = sum(m * n - (m * (m - 1) // 2 if c['causal'] else 0) for n, m in zip(lens, new))
    return dict(bytes=2 * c['kv'] * nk * row + nq * c['heads'] * (4 * d + 4), flops=4 * d * c['heads'] * pairs)


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
    d, heads, kv = c['dim'], c['heads'], c['kv']
    g = torch.Generator(device='cuda').manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device='cuda')

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device='cuda')

    s = dict(c, longest_k=max(lens), longest_q=max(new))
    rows = sum(new)
    if c['kind'] != 'chunk':
        # projections as they come: heads of different size, and a direction in common
        shared = rand(1, 1, d)
        s['q'] = ((rand(rows, heads, d) + 0.7 * shared) * torch.exp(0.5 * rand(1, heads, 1))).to(BF16)
        s['k'] = ((rand(rows, kv, d) + 0.7 * shared) * torch.exp(0.5 * rand(1, kv, 1))).to(BF16)
        for t in ('q', 'k'):
            s[t + '_weight'] = None
            if c['eps'] > 0:
                s[t + '_weight'] = (1 + 0.2 * rand(d)).to(BF16 if c['wbits'] == 16 else torch.float32)
        s['positions'] = _positions(c, lens, new, g)
        if own:
            from miowtion_amd import kernels
            s['rotary'] = kernels.rotary(_sections(c), base=c['base'], interleaved=c['adjacent'], device='cuda')
        if c['kind'] == 'train':
            s['dq'], s['dk'] = rand(rows, heads, d).to(BF16), rand(rows, kv, d).to(BF16)
            for t in ('q', 'k', 'q_weight', 'k_weight'):
                s[t].requires_grad_(True)
    if c['kind'] in ('rotate', 'train'):
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
        x = rand(pages, kv, page, d)
        if t == 'k':
            x = x * torch.exp(0.3 * rand(pages, kv, page, 1))
        if c['bits'] == 8:
            power = _power(x)
            s[t + '_pages'] = torch.ldexp(x, -power).to(E4M3).transpose(1, 2)
            s[t + '_exp'] = (power[..., 0] + 127).to(torch.uint8).transpose(1, 2)
        else:
            s[t + '_pages'] = x.to(BF16).transpose(1, 2)
            s[t + '_exp'] = None
        del x
    s['cu_new'], s['cu'] = ints(_offsets(new)), ints(_offsets(lens))
    if c['kind'] == 'append':
        s['start'] = ints([n - m for n, m in zip(lens, new)])
        s['rows'] = sum(lens)
        s['v'] = rand(rows, kv, d).to(BF16)
    else:
        s['lengths'] = ints(lens)
        s['q'] = (rand(rows, heads, d) * 1.2).to(BF16)
    return s


def _positions(c, lens, new, g):
    """Positions of the rows: of a clip's tokens by frame, row and column, of a
    sequence's by their place in it; on several axes text goes along on all, and
    stretches of it that stand for images leave the diagonal."""
    axes = len(_sections(c))
    if c['grid']:
        parts = torch.meshgrid(*(torch.arange(n, device='cuda') for n in _grid(c)), indexing='ij')
        at = torch.stack([p.reshape(-1) for p in parts], 1)
        at = at[:, :axes] if axes > 1 else torch.arange(at.shape[0], device='cuda')[:, None]
    else:
        at = torch.cat([torch.arange(n - m, n, device='cuda') for n, m in zip(lens, new)])[:, None]
        at = at.expand(-1, axes).clone()
        if axes > 1:
            drift = torch.randint(0, 40, (at.shape[0], axes), generator=g, device='cuda')
            picture = (at[:, :1] // 64) % 2 == 1
            at = torch.where(picture, at // 64 * 64 + drift, at)
    if c['fps']:
        at = at.float()
        at[:, 0] *= c['fps']
        return at
    return at.to(torch.int32)


# ---------------------------------------------------------------------------
# One pass


def run(s: dict):
    if own:
        from miowtion_amd import kernels
        eps = s['eps'] if s['eps'] > 0 else None
        if s['kind'] in ('rotate', 'train'):
            q, k = kernels.norm_rotate(s['q'], s['k'], s['positions'], s['rotary'], s['q_weight'], s['k_weight'],
                                       eps=eps)
            if s['kind'] == 'rotate':
                return q, k
            grads = torch.autograd.grad((q, k), (s['q'], s['k'], s['q_weight'], s['k_weight']), (s['dq'], s['dk']))
            return (q.detach(), k.detach(), *grads)
        cache = kernels.PagedCache(s['k_pages'], s['v_pages'], s['k_exp'], s['v_exp'])
        if s['kind'] == 'append':
            # (positions of text are those of the cache)
            q = kernels.cache_append_rotated_(cache, s['q'], s['k'], s['v'], s['cu_new'], s['table'], s['start'],
                                              s['rotary'], s['positions'] if s['positions'].shape[1] > 1 else None,
                                              s['q_weight'], s['k_weight'], eps=eps)
            if s['bits'] == 16:
                return q, s['k_pages'], s['v_pages']
            return (q, *kernels.cache_gather(cache, s['cu'], s['table'], s['rows']))
        return kernels.paged_chunk_attention(s['q'], s['cu_new'], cache, s['table'], s['lengths'],
                                             causal=s['causal'], return_lse=True)
    if s['kind'] == 'rotate':
        turn = _turn(s)
        return tuple(_rotate(s, t, turn)[0].to(BF16) for t in ('q', 'k'))
    if s['kind'] == 'train':
        return _train(s)
    if s['kind'] == 'append':
        return _append(s)
    return _chunk(s)


def _turn(s):
    """(cos, sin) [rows, 1, pairs] in 32 bits, the angles in 64."""
    angle = []
    for axis, n in enumerate(_sections(s)):
        rate = s['base'] ** (-torch.arange(n, dtype=torch.float64, device='cuda') / n)
        angle.append(s['positions'][:, axis, None].double() * rate)
    angle = torch.cat(angle, 1)[:, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _halves(s, x):
    """The first and the second dims of the pairs, and the dims that do not turn."""
    pairs = sum(_sections(s))
    rest = x[..., 2 * pairs:]
    if s['adjacent']:
        return x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2], rest
    return x[..., :pairs], x[..., pairs:2 * pairs], rest


def _joined(s, a, b, rest):
    turned = torch.stack((a, b), -1).flatten(-2) if s['adjacent'] else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1)


def _rotate(s, t, turn):
    """(rotated, normalised by r alone, r) in 32 bits."""
    x, r = s[t].detach().float(), None
    normal = x
    if s['eps'] > 0:
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + s['eps'])
        normal = x * r
        x = normal * s[t + '_weight'].detach().float()
    a, b, rest = _halves(s, x)
    cos, sin = turn
    return _joined(s, a * cos - b * sin, b * cos + a * sin, rest), normal, r


def _train(s):
    turn = _turn(s)
    cos, sin = turn
    out, grads, weights = [], [], []
    for t in ('q', 'k'):
        y, normal, r = _rotate(s, t, turn)
        out.append(y.to(BF16))
        a, b, rest = _halves(s, s['d' + t].float())
        dz = _joined(s, a * cos + b * sin, b * cos - a * sin, rest)
        w = s[t + '_weight'].detach()
        weights.append((dz * normal).sum((0, 1)).to(w.dtype))
        dz = dz * w.float()
        grads.append((r * (dz - normal * (dz * normal).mean(-1, keepdim=True))).to(BF16))
    return (*out, *grads, *weights)


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


def _append(s):
    turn, page, cu = _turn(s), s['page'], s['cu_new']
    q, k = (_rotate(s, t, turn)[0] for t in ('q', 'k'))
    row = torch.arange(s['k'].shape[0], device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu, row, right=True) - 1
    pos = (s['start'][seq] + row - cu[seq]).long()
    where, at = s['table'][seq, pos // page], pos % page
    for t, rows in (('k', k), ('v', s['v'])):
        pages = s[t + '_pages']
        if s[t + '_exp'] is None:
            pages[where, at] = rows.to(BF16)
        else:
            power = _power(rows)
            codes = torch.ldexp(rows.float(), -power).to(E4M3)
            pages.view(torch.uint8)[where, at] = codes.view(torch.uint8)
            s[t + '_exp'][where, at] = (power[..., 0] + 127).to(torch.uint8)
    if s['bits'] == 16:
        return q.to(BF16), s['k_pages'], s['v_pages']
    row = torch.arange(s['rows'], device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(s['cu'], row, right=True) - 1
    at = row - s['cu'][seq]
    return (q.to(BF16), *(_context(s, t, s['longest_k'])[seq, at].to(BF16) for t in ('k', 'v')))


def _chunk(s):
    cu, lengths, n, m = s['cu_new'], s['lengths'], s['longest_k'], s['longest_q']
    heads, d = s['q'].shape[1:]
    b, kv = lengths.shape[0], s['kv']
    new = cu[1:] - cu[:-1]
    i = torch.arange(m, device=cu.device)
    rows = (cu[:-1, None] + i).clamp(max=s['q'].shape[0] - 1)
    q = s['q'][rows].float().permute(0, 2, 1, 3).reshape(b, kv, heads // kv * m, d)
    k = _context(s, 'k', n).permute(0, 2, 1, 3)
    j = torch.arange(n, device=cu.device)
    hidden = (j >= lengths[:, None])[:, None].expand(b, m, n)
    if s['causal']:
        hidden = hidden | (j > i[:, None] + (lengths - new)[:, None, None])
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).reshape(b, heads, m, n)
    p.masked_fill_(hidden[:, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total)
    v = _context(s, 'v', n).permute(0, 2, 1, 3)
    out = torch.matmul(p.reshape(b, kv, heads // kv * m, n), v).reshape(b, heads, m, d)
    lse = (top + torch.log(total))[..., 0]
    real = i < new[:, None]
    return out.transpose(1, 2)[real].to(BF16), lse.transpose(1, 2)[real]


# ---------------------------------------------------------------------------
# The definition in 64 bits: rotations as complex numbers, gradients by autograd,
# attention a sequence and a head at a time


def exact(case: dict, seed: int):
    c = _full(case)
    lens, new = _lens(c), _new(c)
    if c['kind'] == 'chunk' and sum(n * m for n, m in zip(lens, new)) * c['heads'] > 1.5e10:
        return None
    s = prepare(case, seed)
    if c['kind'] == 'chunk':
        return _exact_chunk(s, lens, new)
    found = [_exact_rotated(s, t) for t in ('q', 'k')]
    if c['kind'] == 'rotate':
        return tuple(y for y, *_ in found)
    if c['kind'] == 'train':
        return (*(y for y, *_ in found), *(x for _, x, _ in found), *(w for _, _, w in found))
    return _exact_append(s, found[0][0], found[1][0], lens, new)


def _exact_rotated(s, t):
    """(rotated, gradient of x, gradient of the weight), some heads at a time."""
    train = s['kind'] == 'train'
    place, parts = 0, []
    for axis, n in enumerate(_sections(s)):
        rate = torch.exp(-math.log(s['base']) * torch.arange(n, dtype=torch.float64, device='cuda') / n)
        parts.append(torch.outer(s['positions'][:, axis].double(), rate))
        place += n
    turn = torch.polar(torch.ones_like(torch.cat(parts, 1)), torch.cat(parts, 1))[:, None]
    a = torch.arange(place, device='cuda')
    first, second = (2 * a, 2 * a + 1) if s['adjacent'] else (a, a + place)
    ys, gxs, gw = [], [], None
    weight = None if s[t + '_weight'] is None else s[t + '_weight'].detach().double().requires_grad_(train)
    for h in range(0, s[t].shape[1], 8):
        x = s[t].detach()[:, h:h + 8].double().requires_grad_(train)
        with torch.set_grad_enabled(train):
            z = x
            if weight is not None:
                z = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s['eps']) * weight
            pair = torch.complex(z[..., first], z[..., second]) * turn
            y = z.index_copy(2, first, pair.real).index_copy(2, second, pair.imag)
        if train:
            gx, g = torch.autograd.grad(y, (x, weight), s['d' + t][:, h:h + 8].double())
            gxs.append(gx)
            gw = g if gw is None else gw + g
        ys.append(y.detach())
    return torch.cat(ys, 1), torch.cat(gxs, 1) if train else None, gw


def _exact_row(rows):
    """Rows as an eight-bit cache holds them: steps of an eighth of the value's own
    power of two, no finer than that of 2^-6, in units that bring the row's largest
    to 448 or less."""
    unit = torch.exp2(torch.ceil(torch.log2(rows.abs().amax(-1, keepdim=True) / 448)))
    x = rows / unit
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step * unit


def _exact_rows(s, t, b, n):
    used = s['table'][b, :-(-n // s['page'])].long()
    x = s[t + '_pages'][used].double()
    if s[t + '_exp'] is not None:
        x = x * torch.exp2(s[t + '_exp'][used].double() - 127)[..., None]
    return x.flatten(0, 1)[:n]


def _exact_append(s, q, k, lens, new):
    found = [q]
    for t, rows in (('k', k), ('v', s['v'].double())):
        if s['bits'] == 16:
            pages, i0 = s[t + '_pages'].double(), 0
            for b, (n, m) in enumerate(zip(lens, new)):
                for p in range((n - m) // s['page'], -(-n // s['page'])):
                    lo, hi = max(p * s['page'], n - m), min((p + 1) * s['page'], n)
                    pages[s['table'][b, p].long(), lo - p * s['page']:hi - p * s['page']] = \
                        rows[i0 + lo - (n - m):i0 + hi - (n - m)]
                i0 += m
            found.append(pages)
        else:
            parts, i0 = [], 0
            for b, (n, m) in enumerate(zip(lens, new)):
                parts += [_exact_rows(s, t, b, n)[:n - m], _exact_row(rows[i0:i0 + m])]
                i0 += m
            found.append(torch.cat(parts))
    return tuple(found)


def _exact_chunk(s, lens, new):
    q = s['q']
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    group, i0 = q.shape[1] // s['kv'], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        keys, values = (_exact_rows(s, t, b, n).transpose(0, 1).contiguous() for t in ('k', 'v'))
        hidden = torch.ones(m, n, dtype=torch.bool, device=q.device).triu(n - m + 1) if s['causal'] else None
        for h in range(q.shape[1]):
            a = q[i0:i0 + m, h].double() @ keys[h // group].t() / math.sqrt(q.shape[2])
            if hidden is not None:
                a[hidden] = -math.inf
            lse[i0:i0 + m, h] = torch.logsumexp(a, -1)
            out[i0:i0 + m, h] = torch.softmax(a, -1) @ values[h // group]
        i0 += m
    return out, lse
