"""PyTorch-ROCm custom ops (`torch.ops.veda.*`) of packed sequences and the
paged cache, as `miowtion_amd.ops` has the tile kernels': shapes and devices
checked on the host, outputs and workspaces from torch, kernels on the current
stream of the tensors' device. `miowtion_amd.packed` wraps them.
"""

from __future__ import annotations

import contextlib

import torch

from miowtion_amd import _native
from miowtion_amd.ops import TILE, _check_rows, _custom_op, _p, _stream

HEAD_DIMS = (64, 128)
PAGES = (16, 32, 64, 128, 256)
_NO_GUARD = contextlib.nullcontext()


def _on(t: torch.Tensor):
    """A guard that makes t's device the current one, where it is not."""
    return _NO_GUARD if torch.cuda.current_device() == t.device.index else torch.cuda.device(t.device)


def _check_aligned(name: str, t: torch.Tensor, size: int = 8) -> None:
    """Every row of t [.., D] starts on a 16-byte boundary (size elements)."""
    if t.data_ptr() % 16 or any(s % size for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        raise ValueError(f'{name}: every row must start on a 16-byte boundary')


def _strides(t: torch.Tensor) -> list[int]:
    """Strides of all but the last dim, 0 where a dim of one makes none."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape[:-1])]


def _check_ints(name: str, t: torch.Tensor, n: int, like: torch.Tensor) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f'{name} must be contiguous int32 [{n}]')
    if t.device != like.device:
        raise ValueError(f'{name} must be on {like.device}, got {t.device}')


def _check_packed(q, k, v, cu_q, cu_k, scale):
    for name, t in (('q', q), ('k', k), ('v', v)):
        _check_rows(name, t)
        _check_aligned(name, t)
        if t.device != q.device:
            raise ValueError(f'{name} must be on {q.device}, got {t.device}')
    d = q.shape[2]
    if d not in HEAD_DIMS or k.shape[2] != d:
        raise ValueError(f'q and k need head_dim 64 or 128 alike, got {d} and {k.shape[2]}')
    if v.shape != k.shape:
        raise ValueError(f'k {tuple(k.shape)} and v {tuple(v.shape)} must have equal shapes')
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f'{q.shape[1]} query heads are no multiple of {k.shape[1]} key heads')
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError('cu_q must be int32 [sequences + 1]')
    _check_ints('cu_q', cu_q, cu_q.shape[0], q)
    _check_ints('cu_k', cu_k, cu_q.shape[0], q)
    if not 0.0 < scale < float('inf'):
        raise ValueError(f'scale must be positive and finite, got {scale}')


@_custom_op('veda::packed_fwd', mutates_args=())
def packed_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
               cu_k: torch.Tensor, causal: bool, scale: float, return_lse: bool) -> list[torch.Tensor]:
    """[out] or [out, lse]: out [Tq, H, D] bf16, lse [Tq, H] fp32."""
    _check_packed(q, k, v, cu_q, cu_k, scale)
    rows, heads, d = q.shape
    out = torch.empty(rows, heads, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(rows, heads, dtype=torch.float32, device=q.device) if return_lse else None
    with _on(q):
        _native.call('veda_packed_fwd', q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k),
                     v.data_ptr(), *_strides(v), rows,
                     k.shape[0], heads, k.shape[1], d, cu_q.data_ptr(), cu_k.data_ptr(),
                     cu_q.shape[0] - 1, int(causal), scale, out.data_ptr(), out.stride(0),
                     out.stride(1), _p(lse), _stream(q))
    return [out, lse] if return_lse else [out]


@packed_fwd.register_fake
def _(q, k, v, cu_q, cu_k, causal, scale, return_lse):
    out = q.new_empty(q.shape)
    return [out, q.new_empty(q.shape[:2], dtype=torch.float32)] if return_lse else [out]


@_custom_op('veda::packed_bwd', mutates_args=())
def packed_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
               dout: torch.Tensor, lse: torch.Tensor, dlse: torch.Tensor | None,
               cu_q: torch.Tensor, cu_k: torch.Tensor, causal: bool,
               scale: float) -> list[torch.Tensor]:
    """[dq, dk, dv] of packed_fwd, from its out and lse."""
    _check_packed(q, k, v, cu_q, cu_k, scale)
    for name, t in (('out', out), ('dout', dout)):
        _check_rows(name, t)
        _check_aligned(name, t)
        if t.shape != q.shape or t.device != q.device:
            raise ValueError(f'{name} {tuple(t.shape)} must be as q {tuple(q.shape)}')
    for name, t in (('lse', lse), ('dlse', dlse)):
        if t is not None and (t.dtype != torch.float32 or t.shape != q.shape[:2]
                              or not t.is_contiguous() or t.device != q.device):
            raise ValueError(f'{name} must be contiguous fp32 {list(q.shape[:2])}')
    rows, heads, d = q.shape
    kv, n_seq = k.shape[1], cu_q.shape[0] - 1
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    work = torch.empty(kv * (rows * (heads // kv) // TILE + n_seq + 2) * 256, dtype=torch.float32,
                       device=q.device)
    with _on(q):
        _native.call('veda_packed_bwd', q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k),
                     v.data_ptr(), *_strides(v), out.data_ptr(), *_strides(out), dout.data_ptr(),
                     *_strides(dout), lse.data_ptr(), _p(dlse), rows, k.shape[0], heads, kv, d,
                     cu_q.data_ptr(), cu_k.data_ptr(), n_seq, int(causal), scale, dq.data_ptr(),
                     dk.data_ptr(), dv.data_ptr(), work.data_ptr(), 4 * work.numel(), _stream(q))
    return [dq, dk, dv]


@packed_bwd.register_fake
def _(q, k, v, out, dout, lse, dlse, cu_q, cu_k, causal, scale):
    return [t.new_empty(t.shape) for t in (q, k, v)]


# --------------------------------------------------------------------------
# the paged cache


def _check_cache(k_pages, v_pages, k_exp, v_exp, table, heads, d, like) -> bool:
    """Checks the cache's tensors; whether they hold e4m3."""
    e4m3 = k_pages.dtype == torch.float8_e4m3fn
    if not e4m3 and k_pages.dtype != torch.bfloat16:
        raise ValueError(f'the cache must be bfloat16 or float8_e4m3fn, got {k_pages.dtype}')
    if k_pages.dim() != 4 or k_pages.stride(-1) != 1 or k_pages.shape[1] not in PAGES:
        raise ValueError('cache tensors must be [pages, 16 | 32 | 64 | 128 | 256, key heads, '
                         f'head_dim] with a contiguous last dim, got {tuple(k_pages.shape)}')
    if (v_pages.dtype != k_pages.dtype or v_pages.shape != k_pages.shape
            or v_pages.stride() != k_pages.stride()):
        raise ValueError('the K and V pages must be laid out alike')
    if k_pages.shape[2] != heads or k_pages.shape[3] != d:
        raise ValueError(f'the cache has {k_pages.shape[2]} key heads of {k_pages.shape[3]}, '
                         f'wanted {heads} of {d}')
    _check_aligned('k_pages', k_pages, 16 if e4m3 else 8)
    _check_aligned('v_pages', v_pages, 16 if e4m3 else 8)
    if e4m3:
        for name, t in (('k_exp', k_exp), ('v_exp', v_exp)):
            if t is None or t.dtype != torch.uint8 or t.shape != k_pages.shape[:3]:
                raise ValueError(f'an e4m3 cache needs {name} uint8 {list(k_pages.shape[:3])}')
        if v_exp.stride() != k_exp.stride():
            raise ValueError('k_exp and v_exp must be laid out alike')
    elif k_exp is not None or v_exp is not None:
        raise ValueError('a bfloat16 cache has no exponents')
    if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError('table must be int32 [sequences, pages] with contiguous rows')
    for t in (k_pages, v_pages, k_exp, v_exp, table):
        if t is not None and t.device != like.device:
            raise ValueError(f'the cache and its table must be on {like.device}, got {t.device}')
    return e4m3


def _exp_strides(e):
    return (0, 0, 0) if e is None else [s if n > 1 else 0 for s, n in zip(e.stride(), e.shape)]


@_custom_op('veda::cache_append_', mutates_args=('k_pages', 'v_pages', 'k_exp', 'v_exp'))
def cache_append_(k_pages: torch.Tensor, v_pages: torch.Tensor, k_exp: torch.Tensor | None,
                  v_exp: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor,
                  table: torch.Tensor, start: torch.Tensor) -> None:
    for name, t in (('k', k), ('v', v)):
        _check_rows(name, t)
        _check_aligned(name, t)
    rows, heads, d = k.shape
    if v.shape != k.shape or d not in HEAD_DIMS or heads == 0 or v.device != k.device:
        raise ValueError(f'k {tuple(k.shape)} and v {tuple(v.shape)} must be [rows, key heads, '
                         '64 or 128] alike')
    e4m3 = _check_cache(k_pages, v_pages, k_exp, v_exp, table, heads, d, k)
    _check_ints('cu', cu, table.shape[0] + 1, k)
    _check_ints('start', start, table.shape[0], k)
    with _on(k):
        _native.call('veda_cache_append', k.data_ptr(), *_strides(k), v.data_ptr(),
                     *_strides(v), rows, heads, d, cu.data_ptr(), start.data_ptr(),
                     table.shape[0], k_pages.data_ptr(), v_pages.data_ptr(), *_strides(k_pages),
                     int(e4m3), _p(k_exp), _p(v_exp), *_exp_strides(k_exp), k_pages.shape[0],
                     k_pages.shape[1], table.data_ptr(), table.stride(0), table.shape[1], _stream(k))


@_custom_op('veda::cache_gather', mutates_args=())
def cache_gather(k_pages: torch.Tensor, v_pages: torch.Tensor, k_exp: torch.Tensor | None,
                 v_exp: torch.Tensor | None, cu: torch.Tensor, table: torch.Tensor,
                 rows: int) -> list[torch.Tensor]:
    """[k, v] [rows, key heads, D] bf16."""
    if k_pages.dim() != 4 or k_pages.shape[2] == 0 or k_pages.shape[3] not in HEAD_DIMS:
        raise ValueError('cache tensors must be [pages, page, key heads, 64 or 128]')
    heads, d = k_pages.shape[2:]
    e4m3 = _check_cache(k_pages, v_pages, k_exp, v_exp, table, heads, d, k_pages)
    _check_ints('cu', cu, table.shape[0] + 1, k_pages)
    if rows < 0:
        raise ValueError(f'rows must not be negative, got {rows}')
    k, v = (torch.empty(rows, heads, d, dtype=torch.bfloat16, device=k_pages.device) for _ in range(2))
    with _on(k):
        _native.call('veda_cache_gather', k_pages.data_ptr(), v_pages.data_ptr(), *_strides(k_pages),
                     int(e4m3), _p(k_exp), _p(v_exp), *_exp_strides(k_exp), k_pages.shape[0],
                     k_pages.shape[1], table.data_ptr(), table.stride(0), table.shape[1],
                     cu.data_ptr(), table.shape[0], rows, heads, d, k.data_ptr(), v.data_ptr(),
                     _stream(k))
    return [k, v]


@cache_gather.register_fake
def _(k_pages, v_pages, k_exp, v_exp, cu, table, rows):
    return [k_pages.new_empty(rows, *k_pages.shape[2:], dtype=torch.bfloat16) for _ in range(2)]


def _chunk(n_seq: int, kv_heads: int, group: int, capacity: int) -> int:
    """Keys of a workgroup of paged_fwd."""
    groups = n_seq * kv_heads * -(-group // 16)
    even = -(-(capacity * groups // 1024) // 128) * 128
    return min(max(even, 128), 1024)


@_custom_op('veda::paged_fwd', mutates_args=())
def paged_fwd(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              k_exp: torch.Tensor | None, v_exp: torch.Tensor | None, table: torch.Tensor,
              lengths: torch.Tensor, scale: float, return_lse: bool) -> list[torch.Tensor]:
    """[out] or [out, lse]: out [B, H, D] bf16, lse [B, H] fp32."""
    _check_rows('q', q)
    _check_aligned('q', q)
    n, heads, d = q.shape
    kv = k_pages.shape[2] if k_pages.dim() == 4 else 0
    if d not in HEAD_DIMS or kv == 0 or heads == 0 or heads % kv:
        raise ValueError(f'q {tuple(q.shape)} does not fit a cache of {kv} key heads: head_dim 64 '
                         'or 128, query heads a multiple of the key heads')
    e4m3 = _check_cache(k_pages, v_pages, k_exp, v_exp, table, kv, d, q)
    if table.shape[0] != n:
        raise ValueError(f'table has {table.shape[0]} sequences, q {n}')
    _check_ints('lengths', lengths, n, q)
    if not 0.0 < scale < float('inf'):
        raise ValueError(f'scale must be positive and finite, got {scale}')
    capacity = table.shape[1] * k_pages.shape[1]
    chunk = _chunk(n, kv, heads // kv, capacity)
    n_split = -(-capacity // chunk)
    out = torch.empty(n, heads, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(n, heads, dtype=torch.float32, device=q.device) if return_lse else None
    work = (torch.empty(n * heads * n_split * (d + 4), dtype=torch.float32, device=q.device)
            if n_split > 1 else None)
    with _on(q):
        _native.call('veda_paged_fwd', q.data_ptr(), *_strides(q), n, heads, kv, d,
                     k_pages.data_ptr(), v_pages.data_ptr(), *_strides(k_pages), int(e4m3),
                     _p(k_exp), _p(v_exp), *_exp_strides(k_exp), k_pages.shape[0], k_pages.shape[1],
                     table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(), scale,
                     chunk, out.data_ptr(), out.stride(0), out.stride(1), _p(lse), _p(work),
                     0 if work is None else 4 * work.numel(), _stream(q))
    return [out, lse] if return_lse else [out]


@paged_fwd.register_fake
def _(q, k_pages, v_pages, k_exp, v_exp, table, lengths, scale, return_lse):
    out = q.new_empty(q.shape)
    return [out, q.new_empty(q.shape[:2], dtype=torch.float32)] if return_lse else [out]
