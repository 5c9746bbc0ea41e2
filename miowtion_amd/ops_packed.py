"""PyTorch-ROCm custom ops (`torch.ops.veda.*`) of packed sequences and the
paged cache, as `miowtion_amd.ops` has the tile kernels': shapes and devices
checked on the host, outputs and workspaces from torch, kernels on the current
stream of the tensors' device. `miowtion_amd.packed` wraps them.

A call at a caption's or a single token's size is bound by its host work, so the
checks are written for few Python calls: a tensor's device is compared by its
index, and row alignment and negative sizes are left to the library, which
refuses them with the same ValueError.
"""

from __future__ import annotations

import torch

from miowtion_amd import _native
from miowtion_amd.ops import TILE, _custom_op, _p, _raw_stream

HEAD_DIMS = (64, 128)
PAGES = (16, 32, 64, 128, 256)
_BF16, _F32, _I32, _E4M3 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn
# absent from a torch built without a GPU, where no op gets as far as a launch
_current_device = getattr(torch._C, '_cuda_getDevice', None)


def _launch(name: str, device: int, *args) -> None:
    """One entry point on the current stream of `device`, with it as the current
    device."""
    if _current_device() == device:
        _native.call(name, *args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            _native.call(name, *args, _raw_stream(device))


def _rows(name: str, t: torch.Tensor, device: int):
    """(shape, pointer, row stride, head stride) of bf16 rows [rows, heads, D]; the
    stride of a dim of one is 0, as it makes none."""
    shape = t.shape
    if len(shape) != 3 or t.dtype is not _BF16:
        raise ValueError(f'{name} must be bfloat16 [rows, heads, head_dim], got {t.dtype} {list(shape)}')
    s, h, one = t.stride()
    if one != 1:
        raise ValueError(f'{name} must have a contiguous last dim')
    if t.get_device() != device:
        raise ValueError(f'{name} must be on GPU {device}, got {t.device}')
    return shape, t.data_ptr(), s if shape[0] > 1 else 0, h if shape[1] > 1 else 0


def _ints(name: str, t: torch.Tensor, n: int, device: int) -> int:
    """The pointer of a contiguous int32 [n]."""
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f'{name} must be contiguous int32 [{n}]')
    if t.get_device() != device:
        raise ValueError(f'{name} must be on GPU {device}, got {t.device}')
    return t.data_ptr()


def _check_packed(q, k, v, cu_q, cu_k, scale):
    """What both entry points take first: (device, shape of q, [q, k, v pointers and
    strides], [sizes, offsets])."""
    dev = q.get_device()
    (rows, heads, d), *qa = _rows('q', q, dev)
    kshape, *ka = _rows('k', k, dev)
    vshape, *va = _rows('v', v, dev)
    k_rows, kv, kd = kshape
    if d not in HEAD_DIMS or kd != d:
        raise ValueError(f'q and k need head_dim 64 or 128 alike, got {d} and {kd}')
    if vshape != kshape:
        raise ValueError(f'k {list(kshape)} and v {list(vshape)} must have equal shapes')
    if kv == 0 or heads == 0 or heads % kv:
        raise ValueError(f'{heads} query heads are no multiple of {kv} key heads')
    n = cu_q.shape[0] if cu_q.dim() == 1 else 0
    if n < 1:
        raise ValueError('cu_q must be int32 [sequences + 1]')
    return dev, (rows, heads, d), [*qa, *ka, *va], [
        rows, k_rows, heads, kv, d, _ints('cu_q', cu_q, n, dev),
        _ints('cu_k', cu_k, n, dev), n - 1]


def _key_splits(q_rows: int, k_rows: int, n_seq: int, heads: int, kv_heads: int) -> int:
    """Workgroups that share the keys of 128 query rows: enough to fill the GPU
    (512 are resident), of fifteen steps of 64 keys at least where half of the
    sequences hold all of the keys. A split's sums cost 8 bytes of traffic for each
    of its 32-bit values, so splits past that cost more than they give. Times in us
    with 1, 2, 4, 8 and 16 splits: 2 x 16 queries of 16 heads over 52,768 keys 419,
    222, 119, 67, 43; 512 of 32 over 8,192: 115, 81, 79, 90, 113; 4 x 512 of 32
    (head_dim 64) over 21,388: 107, 107, 119, 144, 202; whole prompts of 1,024, 1,000,
    900 and 800 tokens, 8 heads: 25, 34, 44, 69, 129."""
    tiles = max(q_rows * heads // TILE, min(n_seq, q_rows) * kv_heads, 1)
    if tiles >= 512 or n_seq == 0:
        return 1
    return max(min(-(-512 // tiles), k_rows // -(-n_seq // 2) // 960, 32), 1)


@_custom_op('veda::packed_fwd', mutates_args=())
def packed_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
               cu_k: torch.Tensor, causal: bool, scale: float, return_lse: bool) -> list[torch.Tensor]:
    """[out] or [out, lse]: out [Tq, H, D] bf16, lse [Tq, H] fp32."""
    dev, (rows, heads, d), tensors, sizes = _check_packed(q, k, v, cu_q, cu_k, scale)
    out = q.new_empty((rows, heads, d))
    lse = q.new_empty((rows, heads), dtype=_F32) if return_lse else None
    n_split = _key_splits(rows, sizes[1], sizes[-1], heads, sizes[3])
    work, nbytes = None, 0
    if n_split > 1:
        nbytes = 4 * n_split * rows * heads * (d + 2)
        work = q.new_empty(nbytes // 4, dtype=_F32)
    _launch('veda_packed_fwd', dev, *tensors, *sizes, causal, scale, n_split, out.data_ptr(),
            heads * d, d, lse.data_ptr() if return_lse else None,
            None if work is None else work.data_ptr(), nbytes)
    return [out, lse] if return_lse else [out]


@packed_fwd.register_fake
def _(q, k, v, cu_q, cu_k, causal, scale, return_lse):
    out = q.new_empty(q.shape)
    return [out, q.new_empty(q.shape[:2], dtype=torch.float32)] if return_lse else [out]


def _splits(k_rows: int, kv_heads: int, walk: int = 1 << 14) -> int:
    """Workgroups that share the query rows of a key tile: 512 in all at least, as
    many as are resident, of four steps of 64 rows at least (`walk`: the rows of a
    sequence for each key head, if half of the sequences hold all); half as many
    again where walks are long, for under a causal mask the first keys have most of
    the rows, and few sequences leave no others to fill in. A split's sums cost 16
    bytes of traffic for each value of dk. Forward and backward in us with 1, 2, 3
    and 4 splits: 8,192 tokens, 28 heads on 4 (256 tiles) 2,961, 2,298, 2,144, 2,152;
    twelve prompts, 32 on 8 (378) 378, 335, 347, 365; 32 x 512, 16 on 4 (512) 299, 324,
    340, 364; forty of up to 600, 32 on 8, head_dim 64 (764) 184, 204, 221, 242; 2,000
    and fifteen of up to 100, 16 on 4 349, 248, 212, 197."""
    tiles = max(-(-k_rows // TILE), 1) * kv_heads
    want = 768 if walk >= 1 << 14 else 512
    return max(min(-(-want // tiles), walk // 256, 16), 1)


def _near(t: torch.Tensor, at: list, group: int, device: int):
    """`at` ([pointer, row stride, head stride] of t) if the dk and dv kernel can load
    rows in these strides, which it addresses by 32-bit offsets within a step of 64;
    else a contiguous copy and its own, which it can below 2^24 values a row."""
    _, s, h = at
    if s < 1 << 24 and (group == 1 or h < 1 << 24) and (group <= 64 or h * group < 1 << 30):
        return t, at
    t = t.contiguous()
    return t, list(_rows('q', t, device)[1:])


@_custom_op('veda::packed_bwd', mutates_args=())
def packed_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
               dout: torch.Tensor, lse: torch.Tensor, dlse: torch.Tensor | None,
               cu_q: torch.Tensor, cu_k: torch.Tensor, causal: bool,
               scale: float) -> list[torch.Tensor]:
    """[dq, dk, dv] of packed_fwd, from its out and lse."""
    dev, shape, tensors, sizes = _check_packed(q, k, v, cu_q, cu_k, scale)
    rows, heads, d = shape
    group = heads // k.shape[1]
    q, tensors[:3] = _near(q, tensors[:3], group, dev)
    for name, t in (('out', out), ('dout', dout)):
        got, *more = _rows(name, t, dev)
        if got != shape:
            raise ValueError(f'{name} {list(got)} must be as q {list(shape)}')
        tensors += more
    dout, tensors[-3:] = _near(dout, tensors[-3:], group, dev)
    for name, t in (('lse', lse), ('dlse', dlse)):
        if t is not None and (t.dtype is not _F32 or t.shape != (rows, heads)
                              or not t.is_contiguous() or t.get_device() != dev):
            raise ValueError(f'{name} must be contiguous fp32 {[rows, heads]} on GPU {dev}')
    k_rows, kv, n_seq = k.shape[0], k.shape[1], cu_q.shape[0] - 1
    dq, dk, dv = q.new_empty(shape), k.new_empty(k.shape), k.new_empty(k.shape)
    n_split = _splits(k_rows, kv, rows * (heads // kv) // -(-max(n_seq, 1) // 2))
    work = q.new_empty(kv * (rows * (heads // kv) // TILE + n_seq + 2) * 256
                       + (2 * n_split * k_rows * kv * d if n_split > 1 else 0), dtype=_F32)
    _launch('veda_packed_bwd', dev, *tensors, lse.data_ptr(), _p(dlse), *sizes, causal, scale, n_split,
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), work.data_ptr(), 4 * work.numel())
    return [dq, dk, dv]


@packed_bwd.register_fake
def _(q, k, v, out, dout, lse, dlse, cu_q, cu_k, causal, scale):
    return [t.new_empty(t.shape) for t in (q, k, v)]


# --------------------------------------------------------------------------
# the paged cache


def _check_cache(k_pages, v_pages, k_exp, v_exp, table, heads, d, dev):
    """The cache and table arguments of the entry points: [pointers, strides and
    format], [sizes, table]."""
    shape, strides = k_pages.shape, k_pages.stride()
    e4m3 = k_pages.dtype is _E4M3
    if not e4m3 and k_pages.dtype is not _BF16:
        raise ValueError(f'the cache must be bfloat16 or float8_e4m3fn, got {k_pages.dtype}')
    if len(shape) != 4 or strides[3] != 1 or shape[1] not in PAGES:
        raise ValueError('cache tensors must be [pages, 16 | 32 | 64 | 128 | 256, key heads, '
                         f'head_dim] with a contiguous last dim, got {list(shape)}')
    if v_pages.dtype is not k_pages.dtype or v_pages.shape != shape or v_pages.stride() != strides:
        raise ValueError('the K and V pages must be laid out alike')
    if shape[2] != heads or shape[3] != d:
        raise ValueError(f'the cache has {shape[2]} key heads of {shape[3]}, wanted {heads} of {d}')
    if e4m3:
        for name, t in (('k_exp', k_exp), ('v_exp', v_exp)):
            if t is None or t.dtype is not torch.uint8 or t.shape != shape[:3]:
                raise ValueError(f'an e4m3 cache needs {name} uint8 {list(shape[:3])}')
        exp_strides = k_exp.stride()
        if v_exp.stride() != exp_strides:
            raise ValueError('k_exp and v_exp must be laid out alike')
        exps = [k_exp.data_ptr(), v_exp.data_ptr(), *exp_strides]
        away = k_exp.get_device() != dev or v_exp.get_device() != dev
    else:
        if k_exp is not None or v_exp is not None:
            raise ValueError('a bfloat16 cache has no exponents')
        exps, away = [None, None, 0, 0, 0], False
    if table.dtype is not _I32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError('table must be int32 [sequences, pages] with contiguous rows')
    if (away or k_pages.get_device() != dev or v_pages.get_device() != dev
            or table.get_device() != dev):
        raise ValueError(f'the cache and its table must be on GPU {dev}')
    return ([k_pages.data_ptr(), v_pages.data_ptr(), strides[0] if shape[0] > 1 else 0, strides[1],
             strides[2] if heads > 1 else 0, e4m3, *exps],
            [shape[0], shape[1], table.data_ptr(), table.stride(0), table.shape[1]])


def _folded(t: torch.Tensor) -> bool:
    """Whether a stride of 0 holds several of t's values in one place."""
    strides = t.stride()
    return 0 in strides and any(n > 1 and s == 0 for n, s in zip(t.shape, strides))


@_custom_op('veda::cache_append_', mutates_args=('k_pages', 'v_pages', 'k_exp', 'v_exp'))
def cache_append_(k_pages: torch.Tensor, v_pages: torch.Tensor, k_exp: torch.Tensor | None,
                  v_exp: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor,
                  table: torch.Tensor, start: torch.Tensor) -> None:
    dev = k.get_device()
    (rows, heads, d), *ka = _rows('k', k, dev)
    vshape, *va = _rows('v', v, dev)
    if vshape != (rows, heads, d) or d not in HEAD_DIMS or heads == 0:
        raise ValueError(f'k {[rows, heads, d]} and v {list(vshape)} must be [rows, key heads, '
                         '64 or 128] alike')
    cache, sizes = _check_cache(k_pages, v_pages, k_exp, v_exp, table, heads, d, dev)
    # (V and its exponents have K's strides; K may be V where their new rows are one too)
    shared = _folded(k_pages) or (k_exp is not None and _folded(k_exp))
    if cache[0] == cache[1] or (k_exp is not None and cache[6] == cache[7]):
        shared |= ka != va and k_pages.shape[0] > 0
    if shared:
        raise ValueError('cache_append_ needs a cache whose rows and exponents do not share memory')
    n = table.shape[0]
    _launch('veda_cache_append', dev, *ka, *va, rows, heads, d, _ints('cu', cu, n + 1, dev),
            _ints('start', start, n, dev), n, *cache, *sizes)


@_custom_op('veda::cache_gather', mutates_args=())
def cache_gather(k_pages: torch.Tensor, v_pages: torch.Tensor, k_exp: torch.Tensor | None,
                 v_exp: torch.Tensor | None, cu: torch.Tensor, table: torch.Tensor,
                 rows: int) -> list[torch.Tensor]:
    """[k, v] [rows, key heads, D] bf16."""
    if k_pages.dim() != 4 or k_pages.shape[2] == 0 or k_pages.shape[3] not in HEAD_DIMS:
        raise ValueError('cache tensors must be [pages, page, key heads, 64 or 128]')
    if rows < 0:
        raise ValueError(f'rows must not be negative, got {rows}')
    dev, (heads, d), n = k_pages.get_device(), k_pages.shape[2:], table.shape[0]
    cache, sizes = _check_cache(k_pages, v_pages, k_exp, v_exp, table, heads, d, dev)
    shape = (rows, heads, d)
    k, v = k_pages.new_empty(shape, dtype=_BF16), k_pages.new_empty(shape, dtype=_BF16)
    _launch('veda_cache_gather', dev, *cache, *sizes, _ints('cu', cu, n + 1, dev), n, rows, heads, d,
            k.data_ptr(), v.data_ptr())
    return [k, v]


@cache_gather.register_fake
def _(k_pages, v_pages, k_exp, v_exp, cu, table, rows):
    return [k_pages.new_empty(rows, *k_pages.shape[2:], dtype=torch.bfloat16) for _ in range(2)]


def _chunk(n_seq: int, kv_heads: int, group: int, capacity: int, page: int) -> int:
    """Keys of a workgroup of paged_fwd, from how far the table reaches (the
    lengths are on the GPU): short enough for ragged lengths to even out over the
    768 workgroups that are resident, long enough to hide their start and end.
    Times in us with chunks of 128, 256, 384, 512 and 1,024: 64 sequences of up to
    8,021 (8 key heads, e4m3) 56, 49, 41, 45, 49; four of about 100,000 349, 326,
    314, 306, 289; eight of 4,096 29, 28, 27, 27, 27. Short sequences, or not so
    short ones in many workgroups, are not split: in a captured graph, whole and
    in chunks of 128, bf16, 8 key heads: one of 300 7.4 and 7.2, of 600 9.8 and 7.4,
    of 1,500 18.4 and 7.8; sixteen of 300 7.5 and 9.1, of 600 11.2 and 13.0, of
    1,000 15.8 and 17.5 (a call by itself is 4 us of host work less)."""
    groups = n_seq * kv_heads * -(-group // 16)
    if capacity <= 512 or (capacity <= 1024 and groups >= 128):
        chunk = capacity
    else:
        chunk = min(max(capacity // 24, 256), 1024)
        if groups * -(-capacity // chunk) < 512:  # few workgroups: smaller ones, to a point
            chunk = max(capacity * groups // 512, 128 if capacity <= 4096 else 256)
    unit = max(page, 128)
    return min(max(-(-chunk // unit), 1) * unit, 128 * page)


@_custom_op('veda::paged_fwd', mutates_args=())
def paged_fwd(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              k_exp: torch.Tensor | None, v_exp: torch.Tensor | None, table: torch.Tensor,
              lengths: torch.Tensor, scale: float, return_lse: bool) -> list[torch.Tensor]:
    """[out] or [out, lse]: out [B, H, D] bf16, lse [B, H] fp32."""
    dev = q.get_device()
    (n, heads, d), *qa = _rows('q', q, dev)
    kv = k_pages.shape[2] if k_pages.dim() == 4 else 0
    if d not in HEAD_DIMS or kv == 0 or heads == 0 or heads % kv:
        raise ValueError(f'q {[n, heads, d]} does not fit a cache of {kv} key heads: head_dim 64 or '
                         '128, query heads a multiple of the key heads')
    cache, sizes = _check_cache(k_pages, v_pages, k_exp, v_exp, table, kv, d, dev)
    if table.shape[0] != n:
        raise ValueError(f'table has {table.shape[0]} sequences, q {n}')
    capacity = table.shape[1] * k_pages.shape[1]
    chunk = _chunk(n, kv, heads // kv, capacity, k_pages.shape[1])
    n_split = -(-capacity // chunk)
    out = q.new_empty((n, heads, d))
    lse = q.new_empty((n, heads), dtype=_F32) if return_lse else None
    work, nbytes = None, 0
    if n_split > 1:
        nbytes = 4 * n * heads * n_split * (d + 4)
        work = q.new_empty(nbytes // 4, dtype=_F32)
    _launch('veda_paged_fwd', dev, *qa, n, heads, kv, d, *cache, *sizes,
            _ints('lengths', lengths, n, dev), scale, chunk, out.data_ptr(), heads * d, d,
            lse.data_ptr() if return_lse else None, None if work is None else work.data_ptr(), nbytes)
    return [out, lse] if return_lse else [out]


@paged_fwd.register_fake
def _(q, k_pages, v_pages, k_exp, v_exp, table, lengths, scale, return_lse):
    out = q.new_empty(q.shape)
    return [out, q.new_empty(q.shape[:2], dtype=torch.float32)] if return_lse else [out]
