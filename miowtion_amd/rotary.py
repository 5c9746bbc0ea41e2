"""Norms of query and key heads and their rotation by position: the step between
a layer's projections and its attention.

The attention of this package takes q and k after both. `norm_rotate` does them in
one pass over q and k, with gradients; `cache_append_rotated_` does them on the way
into a paged cache. Positions have one axis (text) or several (frame, row and
column of a clip's tokens); `rotary` says which pairs of a head's dims turn with
which axis, and how fast. All are reached through `miowtion_amd.kernels`.
"""

from __future__ import annotations

import math
import typing

import torch

from miowtion_amd import ops_rotary
from miowtion_amd.packed import PagedCache


class Rotary(typing.NamedTuple):
    """The rotation of a head. Pair j of P turns by `turns[j]` whole turns for a step of
    positions[:, axes[j]]; it is dims j and j + P of the head, or 2 j and 2 j + 1
    where `interleaved`. Dims from 2 P on stay as they are. turns float64 [P], axes
    int32 [P] below n_axes, both on the GPU; P at most half the head, and a multiple
    of 8 unless `interleaved`."""
    turns: torch.Tensor
    axes: torch.Tensor
    n_axes: int
    interleaved: bool = False


def rotary(sections: int | typing.Sequence[int], base: float = 10000.0, interleaved: bool = False,
           device='cuda') -> Rotary:
    """The usual rates: pair j of the n of an axis turns by base ** (-j / n) radians a step.

    sections: the pairs of each axis, one behind the other: 64 (or [64]) for text in a
        head of 128, [16, 24, 24] for frame, row and column.
    Other rates (through all axes' pairs, or scaled for long contexts) make a `Rotary`
    of their own. Build it once: it copies to the GPU.
    """
    sections = [sections] if isinstance(sections, int) else list(sections)
    pairs = sum(sections)
    if not sections or min(sections) < 1 or pairs > 64:
        raise ValueError(f'every axis needs a pair, all together at most 64: {sections}')
    if not interleaved and pairs % 8:
        raise ValueError(f'pairs of dims apart must be a multiple of 8, got {pairs}')
    if not 0 < base < math.inf:
        raise ValueError(f'base must be positive and finite, got {base}')
    rates = [base ** (-j / n) / (2 * math.pi) for n in sections for j in range(n)]
    axes = [axis for axis, n in enumerate(sections) for _ in range(n)]
    return Rotary(torch.tensor(rates, dtype=torch.float64, device=device),
                  torch.tensor(axes, dtype=torch.int32, device=device), len(sections), interleaved)


def _parts(rotary: Rotary | None) -> tuple:
    return (None, None, 0, False) if rotary is None else tuple(rotary)


def _row_grad(g: torch.Tensor) -> torch.Tensor:
    """A gradient whose rows the kernel can load as they lie: as it is, or a copy."""
    s, h, one = g.stride()
    return g if one == 1 and g.data_ptr() % 16 == 0 and s % 8 == 0 and h % 8 == 0 else g.clone(
        memory_format=torch.contiguous_format)


class _NormRotate(torch.autograd.Function):
    """norm_rotate with gradients of q, k and the weights."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, turns, axes, n_axes, interleaved, eps):
        out = ops_rotary.norm_rotate(q, k, positions, turns, axes, n_axes, interleaved, q_weight, k_weight, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, turns, axes)
        ctx.plan = n_axes, interleaved, eps
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        q, k, q_weight, k_weight, positions, turns, axes = ctx.saved_tensors
        need = ctx.needs_input_grad
        of_q = dq is not None and (need[0] or need[2])
        of_k = dk is not None and (need[1] or need[3])
        grads = [None] * 10
        if not (of_q or of_k):
            return tuple(grads)
        n_axes, interleaved, eps = ctx.plan
        found = iter(ops_rotary.norm_rotate_bwd(
            q if of_q else None, _row_grad(dq) if of_q else None, k if of_k else None,
            _row_grad(dk) if of_k else None, positions, turns, axes, n_axes, interleaved, q_weight, k_weight, eps,
            of_q and need[2], of_k and need[3]))
        for i, there in enumerate((of_q, of_k, of_q and need[2], of_k and need[3])):
            if there:
                grads[i] = next(found)
        return tuple(grads)


def norm_rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None = None,
                rotary: Rotary | None = None, q_weight: torch.Tensor | None = None,
                k_weight: torch.Tensor | None = None, eps: float | None = None):
    """Query and key heads normalised and rotated, in one pass over each.

    Args:
        q: [T, H, D] bf16, D 64 or 128; rows in any strides on 16-byte boundaries (a
            projection's view as it is).
        k: [T, Hkv, D] bf16, or None.
        positions: int32, int64 or float32 [T, axes], or [T] for the same on every axis;
            any strides. Angles are formed in 64 bits, so far positions lose nothing.
        rotary: which dims turn with which axis (`rotary`); None: no rotation.
        q_weight, k_weight: [D] bf16 or fp32, the norm's weights; None: ones.
        eps: a head's row x becomes x / sqrt(mean(x^2) + eps) times its weight; at
            least 1e-30. None: no norm.

    Returns:
        (q, k) bf16, contiguous, k None where it was. Differentiable in q, k and the
        weights, once; gradients are the same bits on every call.

    Values are held in 32 bits from the load on and rounded once, so a norm followed by
    a rotation is not rounded between them. A row with an infinity or a NaN has NaNs
    where the formula has them; no other row is touched by it.
    """
    turns, axes, n_axes, interleaved = _parts(rotary)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)
                                    or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        out = _NormRotate.apply(q, k, q_weight, k_weight, positions, turns, axes, n_axes, interleaved, eps)
    else:
        out = ops_rotary.norm_rotate(q, k, positions, turns, axes, n_axes, interleaved, q_weight, k_weight, eps)
    return (out[0], None) if k is None else (out[0], out[1])


def cache_append_rotated_(cache: PagedCache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor,
                          table: torch.Tensor, start: torch.Tensor, rotary: Rotary | None,
                          positions: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                          k_weight: torch.Tensor | None = None, eps: float | None = None) -> torch.Tensor:
    """norm_rotate of q and k and cache_append_ of that k and of v, in one launch.

    Args:
        cache, cu, table, start: as of cache_append_: row cu[b] + i of k and v goes to
            position start[b] + i of sequence b.
        q: [T, H, D] bf16; k, v: [T, Hkv, D] bf16.
        rotary: None: no rotation.
        positions: as of norm_rotate. None: of every row its position in the cache, on
            every axis.
        q_weight, k_weight, eps: as of norm_rotate.

    Returns:
        q [T, H, D] bf16, contiguous, for packed_attention, paged_attention or
        paged_chunk_attention; zeros for rows of no sequence. A row that the cache has no
        page for still has its q.

    In a bf16 cache the rows are those that norm_rotate gives, bit for bit; an e4m3
    cache has the key's value in 32 bits rounded once. What cache_append_ leaves out
    and refuses is left out and refused here, and so is any cache that holds K where it
    holds V.
    """
    return ops_rotary.cache_append_rotated_(cache.k, cache.v, cache.k_exp, cache.v_exp, q, k, v, cu, table, start,
                                            positions, *_parts(rotary), q_weight, k_weight, eps)
