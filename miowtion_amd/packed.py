"""Attention of packed sequences, and a paged key-value cache.

`kernels.dense_attention` attends within one sequence, every row to every row,
with as many key heads as query heads. These are the operators beside it for
sequences of different lengths, grouped heads and a causal mask: whole prompts
(`packed_attention`, with its gradients), and one token at a time over a cache
(`paged_attention`) that is written as tokens come (`cache_append_`), in bf16 or
in eight bits, and read back for the next chunk of a long prompt
(`cache_gather`). All are reached through `miowtion_amd.kernels`.

No length is needed on the host: the sequences' offsets and lengths stay on the
GPU, so a captured graph serves any lengths that fit its tensors.
"""

from __future__ import annotations

import math
import typing

import torch

from miowtion_amd import ops_packed


class PagedCache(typing.NamedTuple):
    """K and V pages [pages, page, key heads, head_dim], bf16 or e4m3; e4m3 pages
    with an exponent byte of every row [pages, page, key heads] (the row is its
    codes times 2^(byte - 127)). K and V are laid out alike, in any strides with
    a contiguous last dim and rows on 16-byte boundaries; `paged_cache` lays a
    head's rows of a page side by side."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor | None = None
    v_exp: torch.Tensor | None = None


def paged_cache(pages: int, page: int, kv_heads: int, head_dim: int,
                dtype: torch.dtype = torch.bfloat16, device='cuda') -> PagedCache:
    """A cache of `pages` pages of `page` rows (16, 32, 64, 128 or 256), zeros."""
    if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
        raise ValueError(f'the cache must be bfloat16 or float8_e4m3fn, got {dtype}')
    if page not in ops_packed.PAGES or head_dim not in ops_packed.HEAD_DIMS:
        raise ValueError(f'pages of {ops_packed.PAGES} rows and head_dim 64 or 128, got {page} and '
                         f'{head_dim}')
    shape = (pages, kv_heads, page, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
    if dtype == torch.bfloat16:
        return PagedCache(k, v)
    exps = (torch.zeros(shape[:3], dtype=torch.uint8, device=device).transpose(1, 2)
            for _ in range(2))
    return PagedCache(k, v, *exps)


def _scale(scale: float | None, head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim) if scale is None else float(scale)


class _PackedAttention(torch.autograd.Function):
    """packed_attention with gradients of q, k and v, through out and the LSE."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, causal, scale):
        if q.shape[0] > 1 and math.prod(q.shape[1:]) >= 1 << 24:  # refused here, not by the backward
            raise ValueError(f'gradients need fewer than 2^24 values in a row of q, got {list(q.shape)}')
        out, lse = ops_packed.packed_fwd(q, k, v, cu_q, cu_k, causal, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k)
        ctx.causal, ctx.scale = causal, scale
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v, out, lse, cu_q, cu_k = ctx.saved_tensors
        dout = torch.zeros_like(out) if dout is None else dout.contiguous()
        if dout.data_ptr() % 16:  # a view whose rows begin off a 16-byte boundary
            dout = dout.clone()
        dq, dk, dv = ops_packed.packed_bwd(q, k, v, out, dout, lse,
                                           None if dlse is None else dlse.contiguous(), cu_q, cu_k,
                                           ctx.causal, ctx.scale)
        return dq, dk, dv, None, None, None, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: torch.Tensor | None = None, causal: bool = True,
                     scale: float | None = None, return_lse: bool = False):
    """Attention within each of the sequences packed one behind the other.

    Args:
        q: [Tq, H, D] bf16, D 64 or 128; rows in any strides on 16-byte boundaries.
            For gradients H * D is below 2^24, and a q whose strides reach 2^24
            (beyond 64 heads to a key head, 2^30 over those) is copied.
        k, v: [Tk, Hkv, D] bf16, H a multiple of Hkv, at most 65,536 times: query
            head h attends with key head h // (H // Hkv). Row strides below 2^24.
        cu_q: int32 [B + 1], ascending: sequence b has the rows cu_q[b] ..
            cu_q[b + 1] - 1 of q. Offsets are not checked (they stay on the GPU);
            ones outside the rows are clamped to them.
        cu_k: the same for k and v; None: cu_q. A sequence with more keys than
            queries is a later chunk of a prompt: its last query sees every key.
        causal: query i of n_q sees the keys up to i + n_k - n_q; else all.
        scale: of the scores; None: D ** -0.5. Positive.
        return_lse: also return the [Tq, H] fp32 natural-log LSE.

    Returns:
        out [Tq, H, D] bf16, or (out, lse). Rows that see no key, and rows of no
        sequence, have out 0 and lse -inf. A key that a row does not see does not
        touch its out, whatever it holds. Differentiable in q, k and v (and
        through the LSE) where they require grad, once; the gradients are the same
        bits on every call, and values that are not finite stay within the
        gradients of their sequence.

    The probabilities, and in the backward the gradients of the scores, are rounded
    to bf16 for the matrix products, out and the gradients once at the end; scores,
    softmax sums and the products' sums have 32 bits. At thousands of keys out is
    2.1e-3 from 64 bits by norm and the gradients 2.4e-3, 1.5e-3 of it bf16's own
    rounding.

    Rows that meet a NaN in v, or an infinity in v that the mask hides within their
    tile, are formed key by key, which takes some 200 times as long (what is not
    finite in q and k, and an infinity that they see, costs nothing).
    """
    scale = _scale(scale, q.shape[-1])
    cu_k = cu_q if cu_k is None else cu_k
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _PackedAttention.apply(q, k, v, cu_q, cu_k, causal, scale)
        return (out, lse) if return_lse else out
    res = ops_packed.packed_fwd(q, k, v, cu_q, cu_k, causal, scale, return_lse)
    return (res[0], res[1]) if return_lse else res[0]


def cache_append_(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor,
                  table: torch.Tensor, start: torch.Tensor) -> None:
    """Writes packed new rows into the cache.

    Row cu[b] + i of k and v [T, Hkv, D] (bf16) goes to position start[b] + i of
    sequence b: row position % page of page table[b, position // page]. An e4m3
    cache holds a row as codes times a power of two, the least that brings its
    largest finite magnitude to 448 or less, so the scaling itself rounds
    nothing and a value is off by at most 2^-4 of itself (2^-10 of that power of
    two below 2^-6 of it); NaN and infinities become NaN.

    Rows of no sequence, positions past the table and page numbers outside the
    cache are left out; every other row of the cache stays as it was. Two rows
    written to one place by one call (a page that two sequences share where both
    write): which of them the cache then holds is undefined. A cache that holds
    two of its rows, or their exponents, in one place by a stride of 0, is refused,
    and so is one that holds K where it holds V, unless k and v are one tensor too.

    cu int32 [B + 1], table int32 [B, pages of a sequence], start int32 [B].
    """
    ops_packed.cache_append_(cache.k, cache.v, cache.k_exp, cache.v_exp, k, v, cu, table, start)


def cache_gather(cache: PagedCache, cu: torch.Tensor, table: torch.Tensor,
                 rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [rows, Hkv, D] bf16: positions 0 .. cu[b + 1] - cu[b] - 1 of every
    sequence, packed at cu[b] (the cu_k, k and v of packed_attention). Rows of no
    sequence, positions past the table and pages outside the cache read zeros."""
    k, v = ops_packed.cache_gather(cache.k, cache.v, cache.k_exp, cache.v_exp, cu, table, rows)
    return k, v


def paged_attention(q: torch.Tensor, cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor,
                    scale: float | None = None, return_lse: bool = False):
    """Attention of one new token of every sequence over its cached positions.

    Args:
        q: [B, H, D] bf16, H a multiple of the cache's key heads.
        cache: holds the new token's own row too (append it first).
        table: int32 [B, pages of a sequence], rows in any stride. Entries past a
            sequence's length are not read, but the width sets how a sequence is
            split over the GPU, in parts of up to 1,024 positions, and the workspace,
            4 (D + 4) B H bytes a part. So a table much wider than its sequences
            costs time: one of 1,500 positions 7.9 us in a captured graph with a
            table of its size, 9.0 with one for 8,192, 17.8 for 131,072; 64 of 2,000
            (40 heads on 8) 106, 111 and 143, with 11, 30 and 173 MB. Where a bound on
            the lengths is known, pass table[:, :pages of the longest].
        lengths: int32 [B]: positions 0 .. lengths[b] - 1 are seen (at most the
            table's width). Positions in a page outside the cache draw no weight.
        scale: of the scores; None: D ** -0.5. Positive.
        return_lse: also return the [B, H] fp32 natural-log LSE.

    Returns:
        out [B, H, D] bf16, or (out, lse); out 0 and lse -inf without a key. The
        same bits on every call with these shapes. The probabilities are rounded to
        bf16 for the products, as packed_attention's.
    """
    res = ops_packed.paged_fwd(q, cache.k, cache.v, cache.k_exp, cache.v_exp, table, lengths,
                               _scale(scale, q.shape[-1]), return_lse)
    return (res[0], res[1]) if return_lse else res[0]
