"""A decoder layer's attention for batches: head norms and rotation, and a paged 8-bit KV cache.

W4DecodeModel steps one sequence over a contiguous bf16 cache
(scripts/decode_loop.py:106-124 of the reference, one token at a time). These
entry points are its parts for ragged batches of sequences, as a serving loop
uses them between the projections (w4_gemm_fused, w4_matmul):

  q = kv8_append(cache, k, v, page_table, lengths, row_starts, cos, sin, q=q, ...)
  o = kv8_attention(q, cache, page_table, lengths, row_starts)

A step's rows lie one sequence after another: those of sequence b are
row_starts[b] .. row_starts[b + 1] - 1, and they take the positions behind the
lengths[b] tokens that it held before the step (the caller adds the step's rows
to lengths after the last layer). Token t of sequence b is in page
page_table[b, t // page_size]. Rows behind the last sequence are left alone.
All of it is read on the device, so a step can be captured once in a CUDA graph
and replayed as lengths and pages change. A page, length or position out of
range is never followed: what it belongs to is left out, and device_error()
returns _lib.ERR_KV_RANGE. A sequence of negative length is left out with all
its rows (one without rows is a free slot and no error); attention over a length
that the page table has no room for is over the tokens that it has room for.

Every function runs on the current CUDA stream through the C ABI
(include/w4b200.h); there is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class KV8Cache(NamedTuple):
    """Pages of keys and values in e4m3, with one scale a page and head.

    k and v are float8_e4m3fn [pages, kv_heads, page_size, head_dim], k_scale and
    v_scale float32 [pages, kv_heads]; a stored value is code * scale. page_size
    is 16, 32, 64 or 128, head_dim 64 or 128. kv8_append writes power-of-two
    scales; kv8_attention takes any positive ones (a v_scale below 2^-80 counts as
    2^-80: values of 2^-71 at most).
    """
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64,
              device: torch.device | str = "cuda") -> "KV8Cache":
        """A cache of unwritten pages (their contents are never read)."""
        shape = (pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
                   torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
                   torch.empty(shape[:2], dtype=torch.float32, device=device),
                   torch.empty(shape[:2], dtype=torch.float32, device=device))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                 eps: float = 1e-6, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head and its rotation, in one pass.

    q [rows, heads, head_dim] and k [rows, kv_heads, head_dim], float16 or
    bfloat16, may be views into one q|k|v buffer. A head is normed where it has a
    weight (q_norm, k_norm [head_dim]: x * rsqrt(mean(x^2) + eps) * w), then
    rotated (rotate-half) by row positions[row] of cos and sin [max_pos,
    head_dim], if given. fp32 throughout, rounded once. A row whose position has
    no table row is left unwritten. q_out and k_out may be q and k; an output must
    not overlap an input or the other output otherwise.
    """
    return _lib.torch_module().qk_norm_rope(q, k, cos, sin, positions, q_norm, k_norm, eps, q_out,
                                            k_out)


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
               lengths: torch.Tensor, row_starts: torch.Tensor, cos: torch.Tensor | None = None,
               sin: torch.Tensor | None = None, q: torch.Tensor | None = None,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
               eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes a step's keys and values into the cache, rotated on the way.

    k and v [rows, kv_heads, head_dim] (float16 or bfloat16, views allowed); keys
    are normed (k_norm) and rotated (cos, sin) as in qk_norm_rope, at their
    positions in the sequence. With q [rows, heads, head_dim] its heads are normed
    and rotated in the same launch and returned (into `out` if given, which may be
    q and must not overlap q, k or v otherwise); rows outside every sequence are left unwritten. A row whose position has no
    table row is left out: neither its key nor its value is stored.

    The scale of a block (one page of one head, K and V apart) is the least power
    of two s, within 2^-32 .. 2^120, with max|x| <= 448 s over the block's new
    rows. A block that held rows already keeps its scale where that is larger;
    where it is smaller its rows are rounded again in the new one (exact, but for
    values that become subnormal in e4m3). Infinities are stored as +-448 s and
    NaN as NaN; neither sets a scale. A page that the call writes must stand in the
    table once only.
    """
    return _lib.torch_module().kv8_append(*cache, k, v, page_table, lengths, row_starts, cos, sin, q,
                                          q_norm, k_norm, eps, out)


def kv8_attention(q: torch.Tensor, cache: KV8Cache, page_table: torch.Tensor,
                  lengths: torch.Tensor, row_starts: torch.Tensor, scale: float | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's queries over the cache, which holds the step's own rows already.

    q [rows, heads, head_dim], float16 or bfloat16, heads a multiple of the
    cache's (1 to 16 query heads each). Row i of sequence b sees the tokens
    0 .. lengths[b] + i. scale (finite) defaults to head_dim ** -0.5. Scores,
    exponentials and all sums are in fp32; for their product with the values the
    softmax's weights are rounded to fp16 (by 2^-11 of each, or 2^-39 of the
    largest); the result is rounded once to q's type. Deterministic. Returns [rows, heads,
    head_dim] (`out` if given, which may be q and must not overlap it otherwise);
    rows outside every sequence are left unwritten, and a row whose pages are all
    out of range is zero.

    One of two kernels takes the whole call, by the average number of rows a
    sequence. A step of many single rows and a prompt is faster as two calls over
    parts of the same tensors (with the m single rows first):
      kv8_attention(q[:m], cache, page_table[:m], lengths[:m], row_starts[:m + 1], out=o[:m])
      kv8_attention(q, cache, page_table[m:], lengths[m:], row_starts[m:], out=o)
    """
    return _lib.torch_module().kv8_attention(q, *cache, page_table, lengths, row_starts, scale, out)
