"""64-bit restatement of the batched attention operators (test infrastructure only).

Plain torch in float64 on whatever device the inputs are on, from the operators'
definitions: head norm and rotation, the paged e4m3 cache with a power-of-two
scale a page and head, causal grouped attention over it, and the epilogue of
the W4A16 GEMM. The product never imports it.
"""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def norm_rope(x, weight=None, cos=None, sin=None, eps=1e-6):
    """x [rows, heads, D]; cos and sin [rows, D], each row's own."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if cos is None:
        return x
    cos, sin = cos.double().unsqueeze(1), sin.double().unsqueeze(1)
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos[..., :h] - b * sin[..., :h],
                      b * cos[..., h:] + a * sin[..., h:]], -1)


def least_scale(amax: float) -> float:
    """The least power of two s in 2^-32 .. 2^120 with amax <= 448 s."""
    e = -32
    while e < 120 and amax > math.ldexp(E4M3_MAX, e):
        e += 1
    return math.ldexp(1.0, e)


def to_e4m3(x):
    """Round to nearest even, +-448 beyond the range, NaN kept."""
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float32).to(torch.float8_e4m3fn)


def sequences(lengths, row_starts):
    """(sequence, tokens before, first row, rows) of every sequence with rows."""
    starts = row_starts.tolist()
    return [(b, p, starts[b], starts[b + 1] - starts[b])
            for b, p in enumerate(lengths.tolist()) if starts[b + 1] > starts[b]]


def blocks(lengths, row_starts, page_table, page):
    """(page id, first slot, first row, rows) of every page that a step writes."""
    table = page_table.tolist()
    for b, past, first, n in sequences(lengths, row_starts):
        for j in range(past // page, (past + n - 1) // page + 1):
            lo, hi = max(past, j * page), min(past + n, (j + 1) * page)
            yield table[b][j], lo - j * page, first + lo - past, hi - lo


def positions(lengths, row_starts, rows):
    """Every row's position in its sequence (zero outside every sequence)."""
    out = torch.zeros(rows, dtype=torch.int64)
    for _, past, first, n in sequences(lengths, row_starts):
        out[first:first + n] = past + torch.arange(n)
    return out.to(lengths.device)


def dense(codes, scale, pages, n):
    """The first n tokens of a sequence's pages, [kv_heads, n, D] in float64."""
    pages = torch.as_tensor(pages, device=codes.device)
    x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
    x = x * scale[pages].double()[:, :, None, None]
    return x.transpose(0, 1).reshape(codes.shape[1], -1, codes.shape[3])[:, :n]


def attention(q, cache, page_table, lengths, row_starts, scale=None):
    """(out, sum of weight * |v|, bound on the scores' absolute sums) [rows, heads, D] / [.., 1]."""
    k_cache, v_cache, k_scale, v_scale = cache
    kv, page, D = k_cache.shape[1:]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, reach = torch.zeros_like(out), torch.zeros_like(out[..., :1])
    for b, past, first, n in sequences(lengths, row_starts):
        pages = page_table[b, :-(-(past + n) // page)].tolist()
        k = dense(k_cache, k_scale, pages, past + n)
        v = dense(v_cache, v_scale, pages, past + n)
        x = q[first:first + n].double().view(n, kv, -1, D).permute(1, 2, 0, 3)  # [kv, G, n, D]
        s = (x @ k.transpose(1, 2).unsqueeze(1)) * scale
        r = (x.abs() @ k.abs().transpose(1, 2).unsqueeze(1)) * abs(scale)
        hidden = torch.arange(past + n, device=q.device)[None] > \
            past + torch.arange(n, device=q.device)[:, None]
        w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        seen_v = torch.where(hidden.all(0)[None, :, None], 0.0, v)
        o, a = w @ seen_v.unsqueeze(1), w @ seen_v.abs().unsqueeze(1)
        rows = slice(first, first + n)
        out[rows] = o.permute(2, 0, 1, 3).reshape(n, -1, D)
        size[rows] = a.permute(2, 0, 1, 3).reshape(n, -1, D)
        reach[rows] = r.masked_fill(hidden, 0.0).amax(-1).permute(2, 0, 1).reshape(n, -1, 1)
    return out, size, reach


def gemm(x, w, bias=None, activation=None, residual=None):
    """residual + act(x @ w + bias), w already dequantised to x's type."""
    y = x.double() @ w.double()
    if bias is not None:
        y = y + bias.double()
    if activation == "silu":
        y = y * torch.sigmoid(y)
    elif activation == "gelu":
        y = y * torch.special.ndtr(y)
    elif activation == "swiglu":
        y = y.view(y.shape[0], -1, 2, 32)
        g, u = y[:, :, 0].flatten(1), y[:, :, 1].flatten(1)
        y = g * torch.sigmoid(g) * u
    return y if residual is None else y + residual.double()
