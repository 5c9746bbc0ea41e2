"""PyTorch-ROCm custom ops (`torch.ops.veda.*`) of norms with rotation, in the
manner of `miowtion_amd.ops_packed`: shapes and devices checked on the host,
outputs and workspaces from torch, kernels on the current stream of the tensors'
device, row alignment and sizes left to the library, which refuses them with a
ValueError. `miowtion_amd.rotary` wraps them.
"""

from __future__ import annotations

import torch

from miowtion_amd.ops import _custom_op
from miowtion_amd.ops_packed import HEAD_DIMS, _BF16, _F32, _I32, _check_cache, _folded, _ints, _launch, _rows

_KINDS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
# workgroups of the backward at most, each with sums of its own for the weights
_BWD_BLOCKS = 768


def _like(x: torch.Tensor) -> torch.Tensor:
    """Room for a result as x, contiguous (0.6 us of host time less than new_empty)."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _rotation(rows: int, positions, turns, axes, n_axes: int, interleaved: bool, own: bool, dev: int) -> list:
    """[positions, kind, strides, rates, axes, pairs, axes' count, adjacent] of the entry
    points. `own`: without positions, rows have those of the cache."""
    if turns is None:
        if positions is not None:
            raise ValueError('positions without a rotary have no use')
        return [None, 0, 0, 0, None, None, 0, 0, False]
    if (turns.dtype is not torch.float64 or axes is None or axes.dtype is not _I32 or turns.dim() != 1
            or axes.shape != turns.shape or not turns.is_contiguous() or not axes.is_contiguous()):
        raise ValueError('a rotary has contiguous float64 turns and int32 axes of every pair')
    if turns.get_device() != dev or axes.get_device() != dev:
        raise ValueError(f'the rotary must be on GPU {dev}, got {turns.device} and {axes.device}')
    more = [turns.data_ptr(), axes.data_ptr(), turns.shape[0], n_axes, interleaved]
    if positions is None:
        if not own:
            raise ValueError('a rotary needs positions')
        return [None, 0, 0, 0, *more]
    kind = _KINDS.get(positions.dtype)
    shape = positions.shape
    if kind is None or (shape != (rows,) and shape != (rows, n_axes)):
        raise ValueError(f'positions must be int32, int64 or float32 [{rows}] or [{rows}, {n_axes}], got '
                         f'{positions.dtype} {list(shape)}')
    if positions.get_device() != dev:
        raise ValueError(f'positions must be on GPU {dev}, got {positions.device}')
    strides = positions.stride()
    return [positions.data_ptr(), kind, strides[0], strides[1] if len(shape) > 1 else 0, *more]


def _weight(name: str, w, d: int, normed: bool, dev: int) -> list:
    """[pointer, whether bf16] of a weight."""
    if w is None:
        return [None, False]
    if not normed:
        raise ValueError(f'{name} without eps: there is no norm to weigh')
    if w.shape != (d,) or w.dtype not in (_BF16, _F32) or not w.is_contiguous():
        raise ValueError(f'{name} must be contiguous bfloat16 or float32 [{d}], got {w.dtype} {list(w.shape)}')
    if w.get_device() != dev:
        raise ValueError(f'{name} must be on GPU {dev}, got {w.device}')
    return [w.data_ptr(), w.dtype is _BF16]


def _eps(eps: float | None) -> float:
    """The entry points' eps: negative without a norm."""
    if eps is None:
        return -1.0
    if not eps > 0.0:
        raise ValueError(f'eps must be positive, got {eps}')
    return eps


def _check_heads(q, k, dev: int):
    """(rows, head_dim, [pointer, strides, heads] of q, of k): k may be None."""
    (rows, heads, d), *qa = _rows('q', q, dev)
    if k is None:
        return rows, d, [*qa, heads], [None, 0, 0, 0]
    kshape, *ka = _rows('k', k, dev)
    if kshape[0] != rows or kshape[2] != d:
        raise ValueError(f'q {[rows, heads, d]} and k {list(kshape)} must have equal rows and head_dim')
    return rows, d, [*qa, heads], [*ka, kshape[1]]


@_custom_op('veda::norm_rotate', mutates_args=())
def norm_rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None,
                turns: torch.Tensor | None, axes: torch.Tensor | None, n_axes: int, interleaved: bool,
                q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                eps: float | None) -> list[torch.Tensor]:
    """[q] or [q, k], normalised and rotated, contiguous."""
    dev = q.get_device()
    rows, d, qa, ka = _check_heads(q, k, dev)
    turn = _rotation(rows, positions, turns, axes, n_axes, interleaved, False, dev)
    normed = eps is not None
    weights = _weight('q_weight', q_weight, d, normed, dev) + _weight('k_weight', k_weight, d, normed, dev)
    out = [_like(q)] if k is None else [_like(q), _like(k)]
    _launch('veda_norm_rotate', dev, *qa, *ka, rows, d, *turn, *weights, _eps(eps), out[0].data_ptr(),
            None if k is None else out[1].data_ptr())
    return out


@norm_rotate.register_fake
def _(q, k, positions, turns, axes, n_axes, interleaved, q_weight, k_weight, eps):
    return [t.new_empty(t.shape) for t in (q, k) if t is not None]


@_custom_op('veda::norm_rotate_bwd', mutates_args=())
def norm_rotate_bwd(q: torch.Tensor | None, dq: torch.Tensor | None, k: torch.Tensor | None,
                    dk: torch.Tensor | None, positions: torch.Tensor | None, turns: torch.Tensor | None,
                    axes: torch.Tensor | None, n_axes: int, interleaved: bool, q_weight: torch.Tensor | None,
                    k_weight: torch.Tensor | None, eps: float | None, of_q_weight: bool,
                    of_k_weight: bool) -> list[torch.Tensor]:
    """From the gradients dq and dk of norm_rotate's results those of q, k, q_weight and
    k_weight: of q and k where they are given, of the weights where asked for."""
    one = k if q is None else q
    dev, rows, d = one.get_device(), one.shape[0], one.shape[-1]
    tensors, out = [], []
    for name, x, g in (('q', q, dq), ('k', k, dk)):
        if x is None:
            tensors += [None, 0, 0, None, 0, 0, 0]
            continue
        shape, *xa = _rows(name, x, dev)
        gshape, *ga = _rows(f"{name}'s gradient", g, dev)
        if gshape != shape or shape[0] != rows or shape[2] != d:
            raise ValueError(f"{name} {list(shape)} and its gradient {list(gshape)} must be alike, of {rows} rows "
                             f'of {d}')
        tensors += [*xa, *ga, shape[1]]
        out.append(_like(x))
    turn = _rotation(rows, positions, turns, axes, n_axes, interleaved, False, dev)
    normed = eps is not None
    weights = _weight('q_weight', q_weight, d, normed, dev) + _weight('k_weight', k_weight, d, normed, dev)
    dx = [None if q is None else out[0].data_ptr(), None if k is None else out[-1].data_ptr()]
    dw, work = [None, None], None
    for i, (w, asked) in enumerate(((q_weight, of_q_weight), (k_weight, of_k_weight))):
        if asked:
            out.append(_like(w))
            dw[i] = out[-1].data_ptr()
    if of_q_weight or of_k_weight:
        work = one.new_empty(_BWD_BLOCKS * 2 * d, dtype=_F32)
    _launch('veda_norm_rotate_bwd', dev, *tensors, rows, d, *turn, *weights, _eps(eps), *dx, *dw,
            None if work is None else work.data_ptr(), 0 if work is None else 4 * work.numel())
    return out


@norm_rotate_bwd.register_fake
def _(q, dq, k, dk, positions, turns, axes, n_axes, interleaved, q_weight, k_weight, eps, of_q_weight,
      of_k_weight):
    given = [q, k, q_weight if of_q_weight else None, k_weight if of_k_weight else None]
    return [t.new_empty(t.shape) for t in given if t is not None]


@_custom_op('veda::cache_append_rotated_', mutates_args=('k_pages', 'v_pages', 'k_exp', 'v_exp'))
def cache_append_rotated_(k_pages: torch.Tensor, v_pages: torch.Tensor, k_exp: torch.Tensor | None,
                          v_exp: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          cu: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
                          positions: torch.Tensor | None, turns: torch.Tensor | None,
                          axes: torch.Tensor | None, n_axes: int, interleaved: bool,
                          q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                          eps: float | None) -> torch.Tensor:
    """q, normalised and rotated, contiguous; k as well into the cache, and v."""
    dev = q.get_device()
    rows, d, qa, ka = _check_heads(q, k, dev)
    vshape, *va = _rows('v', v, dev)
    heads = k.shape[1]
    if vshape != k.shape or d not in HEAD_DIMS or heads == 0:
        raise ValueError(f'k {list(k.shape)} and v {list(vshape)} must be [rows, key heads, 64 or 128] alike')
    cache, sizes = _check_cache(k_pages, v_pages, k_exp, v_exp, table, heads, d, dev)
    if _folded(k_pages) or (k_exp is not None and _folded(k_exp)) or (k_pages.shape[0] > 0 and (
            cache[0] == cache[1] or (k_exp is not None and cache[6] == cache[7]))):
        raise ValueError('cache_append_rotated_ needs a cache whose rows and exponents do not share memory')
    n = table.shape[0]
    turn = _rotation(rows, positions, turns, axes, n_axes, interleaved, True, dev)
    normed = eps is not None
    weights = _weight('q_weight', q_weight, d, normed, dev) + _weight('k_weight', k_weight, d, normed, dev)
    out = _like(q)
    _launch('veda_cache_append_rotated', dev, *qa, *ka[:3], *va, rows, heads, d, _ints('cu', cu, n + 1, dev),
            _ints('start', start, n, dev), n, *cache, *sizes, *turn, *weights, _eps(eps), out.data_ptr())
    return out


@cache_append_rotated_.register_fake
def _(k_pages, v_pages, k_exp, v_exp, q, k, v, cu, table, start, positions, turns, axes, n_axes, interleaved,
      q_weight, k_weight, eps):
    return q.new_empty(q.shape)
