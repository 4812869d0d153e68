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
returns _lib.ERR_KV_RANGE.

Every function runs on the current CUDA stream through the C ABI
(include/w4b200.h); there is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._lib import check
from .kernels import _DTYPE_CODE, _dense16, _on_device, _stream_ptr

_TABLE_CODE = {torch.float16: _lib.W4_F16, torch.bfloat16: _lib.W4_BF16,
               torch.float32: _lib.W4_F32}
_NO_HEADS = _lib.Heads(None, 0, 0, 0)
_workspace_bytes: dict[int, int] = {}


class KV8Cache(NamedTuple):
    """Pages of keys and values in e4m3, with one scale a page and head.

    k and v are float8_e4m3fn [pages, kv_heads, page_size, head_dim], k_scale and
    v_scale float32 [pages, kv_heads]; a stored value is code * scale. page_size
    is 16, 32, 64 or 128, head_dim 64 or 128. kv8_append writes power-of-two
    scales; kv8_attention takes any positive ones.
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


def _cache_desc(cache: KV8Cache) -> _lib.Kv8CacheDesc:
    k, v, ks, vs = cache
    shape, device = k.shape, k.device
    if len(shape) != 4 or v.shape != shape or ks.shape != shape[:2] or vs.shape != shape[:2]:
        raise ValueError(f"cache must be k and v [pages, kv_heads, page_size, head_dim] with scales "
                         f"[pages, kv_heads], got {tuple(shape)}, {tuple(v.shape)}, "
                         f"{tuple(ks.shape)}, {tuple(vs.shape)}")
    if k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn \
            or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise ValueError(f"cache must be float8_e4m3fn with float32 scales, got {k.dtype}, "
                         f"{v.dtype}, {ks.dtype}, {vs.dtype}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if not k.is_cuda or v.device != device or ks.device != device or vs.device != device:
        raise ValueError("cache tensors must be on one CUDA device")
    return _lib.Kv8CacheDesc(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *shape)


def _batch_desc(page_table: torch.Tensor, lengths: torch.Tensor, row_starts: torch.Tensor,
                rows: int, device: torch.device) -> _lib.KvBatch:
    for name, t in (("page_table", page_table), ("lengths", lengths), ("row_starts", row_starts)):
        if t.dtype != torch.int32 or t.device != device:
            raise ValueError(f"{name} must be int32 on {device}, got {t.dtype} on {t.device}")
    seqs = lengths.shape[0] if lengths.dim() == 1 else -1
    if page_table.dim() != 2 or page_table.shape[0] != seqs or row_starts.shape != (seqs + 1,):
        raise ValueError(f"page_table must be [seqs, pages], lengths [seqs] and row_starts "
                         f"[seqs + 1], got {tuple(page_table.shape)}, {tuple(lengths.shape)}, "
                         f"{tuple(row_starts.shape)}")
    stride, width = page_table.stride(0), page_table.shape[1]
    if (width > 1 and page_table.stride(1) != 1) or (seqs > 1 and lengths.stride(0) != 1) \
            or (seqs and row_starts.stride(0) != 1):
        raise ValueError("page_table's rows, lengths and row_starts must be contiguous")
    return _lib.KvBatch(page_table.data_ptr(), stride, width, lengths.data_ptr(),
                        row_starts.data_ptr(), seqs, rows)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t [rows, heads, dim] as the kernels read it: 16-byte aligned, a head's elements together."""
    row, head, elem = t.stride()
    if elem != 1 or (row | head) & 7 or t.data_ptr() & 15 \
            or (t.shape[1] > 1 and head < t.shape[2]) or row < 0:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _heads(t: torch.Tensor) -> _lib.Heads:
    row, head, _ = t.stride()
    return _lib.Heads(t.data_ptr(), row, head, t.shape[1])


def _check_rows(name: str, t: torch.Tensor, like: torch.Tensor, heads: int | None,
                head_dim: int) -> None:
    if t.dim() != 3 or t.shape[0] != like.shape[0] or t.shape[2] != head_dim \
            or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [{like.shape[0]}, {heads or 'heads'}, {head_dim}], got "
                         f"{tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on "
                         f"{t.device}")


def _check_out(name: str, out: torch.Tensor, like: torch.Tensor) -> None:
    _check_rows(name, out, like, like.shape[1], like.shape[2])
    if _rows16(out) is not out or (out.shape[0] > 1 and out.stride(0) < out.shape[2]):
        raise ValueError(f"{name} needs 16-byte aligned heads that do not overlap, got strides "
                         f"{out.stride()}")


def _rope_desc(cos: torch.Tensor | None, sin: torch.Tensor | None, q_norm: torch.Tensor | None,
               k_norm: torch.Tensor | None, eps: float, head_dim: int,
               like: torch.Tensor) -> tuple[_lib.Rope, tuple]:
    """The descriptor, and the tensors that it points to."""
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    code = max_pos = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape[1] != head_dim or cos.shape != sin.shape or not len(cos):
            raise ValueError(f"cos and sin must be [positions, {head_dim}], got "
                             f"{tuple(cos.shape)} and {tuple(sin.shape)}")
        if cos.dtype not in _TABLE_CODE or sin.dtype != cos.dtype or cos.device != like.device \
                or sin.device != like.device:
            raise ValueError(f"cos and sin must be of one type (float16, bfloat16 or float32) on "
                             f"{like.device}, got {cos.dtype}, {sin.dtype}")
        cos, sin = _dense16(cos), _dense16(sin)
        code, max_pos = _TABLE_CODE[cos.dtype], cos.shape[0]
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.shape != (head_dim,) or w.dtype != like.dtype
                              or w.device != like.device):
            raise ValueError(f"{name} must be {like.dtype} [{head_dim}] on {like.device}, got "
                             f"{w.dtype} {tuple(w.shape)} on {w.device}")
    q_norm, k_norm = _dense16(q_norm), _dense16(k_norm)
    return _lib.Rope(_ptr(cos), _ptr(sin), code, max_pos, _ptr(q_norm), _ptr(k_norm), eps), \
        (cos, sin, q_norm, k_norm)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


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
    no table row is left unwritten. q_out and k_out may be q and k.
    """
    if q.dim() != 3 or q.dtype not in _DTYPE_CODE or not q.is_cuda:
        raise ValueError(f"q must be float16 or bfloat16 [rows, heads, head_dim] on a CUDA device, "
                         f"got {q.dtype} {tuple(q.shape)} on {q.device}")
    rows, _, head_dim = q.shape
    _check_rows("k", k, q, None, head_dim)
    rope, keep = _rope_desc(cos, sin, q_norm, k_norm, eps, head_dim, q)
    if cos is not None:
        if positions is None or positions.shape != (rows,) or positions.dtype != torch.int64 \
                or positions.device != q.device:
            raise ValueError(f"positions must be int64 [{rows}] on {q.device}")
        positions = positions.contiguous()
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_out("q_out", q_out, q)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    else:
        _check_out("k_out", k_out, k)
    qs, ks = _rows16(q), _rows16(k)
    with _on_device(q.device):
        check(_lib.load().w4_qk_norm_rope(_heads(qs), _heads(ks), _heads(q_out), _heads(k_out),
                                          _DTYPE_CODE[q.dtype], rows, head_dim, rope,
                                          _ptr(positions), _stream_ptr(q.device)), "qk_norm_rope")
    del keep
    return q_out, k_out


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
    q); rows outside every sequence are left unwritten.

    The scale of a block (one page of one head, K and V apart) is the least power
    of two s, within 2^-32 .. 2^120, with max|x| <= 448 s over the block's new
    rows. A block that held rows already keeps its scale where that is larger;
    where it is smaller its rows are rounded again in the new one (exact, but for
    values that become subnormal in e4m3). Infinities are stored as +-448 s and
    NaN as NaN; neither sets a scale. A page must not belong to two of the
    sequences that the call writes.
    """
    desc = _cache_desc(cache)
    device, kv_heads, head_dim = cache.k.device, desc.kv_heads, desc.head_dim
    if k.dim() != 3 or k.dtype not in _DTYPE_CODE or k.device != device:
        raise ValueError(f"k must be float16 or bfloat16 [rows, {kv_heads}, {head_dim}] on "
                         f"{device}, got {k.dtype} {tuple(k.shape)} on {k.device}")
    _check_rows("k", k, k, kv_heads, head_dim)
    _check_rows("v", v, k, kv_heads, head_dim)
    rope, keep = _rope_desc(cos, sin, q_norm, k_norm, eps, head_dim, k)
    batch = _batch_desc(page_table, lengths, row_starts, k.shape[0], device)
    qd = od = _NO_HEADS
    if q is not None:
        _check_rows("q", q, k, None, head_dim)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=device)
        else:
            _check_out("out", out, q)
        q = _rows16(q)
        qd, od = _heads(q), _heads(out)
    elif out is not None:
        raise ValueError("out is for q")
    k, v = _rows16(k), _rows16(v)
    with _on_device(device):
        check(_lib.load().w4_kv8_append(desc, batch, _heads(k), _heads(v), qd, od,
                                        _DTYPE_CODE[k.dtype], rope, _stream_ptr(device)),
              "kv8_append")
    del keep
    return out


def kv8_attention(q: torch.Tensor, cache: KV8Cache, page_table: torch.Tensor,
                  lengths: torch.Tensor, row_starts: torch.Tensor, scale: float | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's queries over the cache, which holds the step's own rows already.

    q [rows, heads, head_dim], float16 or bfloat16, heads a multiple of the
    cache's (1 to 16 query heads each). Row i of sequence b sees the tokens
    0 .. lengths[b] + i. scale defaults to head_dim ** -0.5. Softmax and sums in
    fp32, rounded once to q's type; deterministic. Returns [rows, heads,
    head_dim] (`out` if given); rows outside every sequence are left unwritten,
    and a row whose pages are all out of range is zero.
    """
    desc = _cache_desc(cache)
    device, head_dim = cache.k.device, desc.head_dim
    if q.dim() != 3 or q.dtype not in _DTYPE_CODE or q.device != device \
            or q.shape[2] != head_dim or q.shape[1] % desc.kv_heads:
        raise ValueError(f"q must be float16 or bfloat16 [rows, n * {desc.kv_heads}, {head_dim}] "
                         f"on {device}, got {q.dtype} {tuple(q.shape)} on {q.device}")
    batch = _batch_desc(page_table, lengths, row_starts, q.shape[0], device)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    else:
        _check_out("out", out, q)
    lib = _lib.load()
    need = _workspace_bytes.get(head_dim)
    if need is None:
        need = _workspace_bytes[head_dim] = int(lib.w4_kv8_attention_workspace_bytes(head_dim))
    q = _rows16(q)
    # the workspace is this call's own: the allocator keeps it apart from other
    # streams' and, during capture, from other graphs'
    ws = torch.empty((need,), dtype=torch.uint8, device=device)
    with _on_device(device):
        check(lib.w4_kv8_attention(desc, batch, _heads(q), _heads(out), _DTYPE_CODE[q.dtype],
                                   head_dim ** -0.5 if scale is None else scale, ws.data_ptr(),
                                   need, _stream_ptr(device)), "kv8_attention")
    return out
