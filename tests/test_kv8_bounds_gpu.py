"""kv8_append and kv8_attention at the borders of their contract: lengths, positions, scales, values.

Bars are those of test_kv8_gpu.py unless a test says otherwise.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

import roofline_decoding_b200 as rd  # noqa: E402
from oracle import kv8_oracle as o  # noqa: E402
from roofline_decoding_b200 import _lib  # noqa: E402
from test_kv8_gpu import (check_attention, fresh_cache, gen, i32, page_tables, randn, starts,  # noqa: E402
                          tables)

DEV = "cuda"


def same_bytes(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def copy_of(cache):
    return rd.KV8Cache(*[t.clone() for t in cache])


# ------------------------------------------------------------------ lengths below zero


@pytest.mark.parametrize("length", [-1, -(2 ** 31)])
@pytest.mark.parametrize("n", [1, 40])  # a warp a block of the cache, a CTA a block
def test_append_leaves_out_a_sequence_of_negative_length(n, length):
    g, page = gen(1), 32
    past = [5, 60, 31]
    table, pages = page_tables(g, past, [n] * 3, page)
    cache = fresh_cache(g, pages, 2, 128, page)
    want = copy_of(cache)
    cos, sin = tables(128, 128, torch.float32)
    q, k, v = randn(g, 3 * n, 4, 128), randn(g, 3 * n, 2, 128), randn(g, 3 * n, 2, 128)
    out, want_q = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
    for b in (0, 2):
        rows = slice(b * n, (b + 1) * n)
        rd.kv8_append(want, k[rows], v[rows], table[b:b + 1], i32([past[b]]), i32([0, n]), cos, sin,
                      q=q[rows], out=want_q[rows])
    assert rd.device_error() == 0
    rd.kv8_append(cache, k, v, table, i32([past[0], length, past[2]]), i32(starts([n] * 3)), cos, sin,
                  q=q, out=out)
    assert rd.device_error() == _lib.ERR_KV_RANGE
    assert same_bytes(cache, want) and torch.equal(out, want_q)


@pytest.mark.parametrize("length", [-1, -(2 ** 31)])
@pytest.mark.parametrize("n", [1, 20, 80])
def test_attention_leaves_out_a_sequence_of_negative_length(n, length):
    g, page = gen(2), 32
    past = [300, 60, 31]
    table, pages = page_tables(g, past, [n] * 3, page)
    cache = fresh_cache(g, pages, 2, 128, page)
    q = randn(g, 3 * n, 4, 128)
    out = torch.full_like(q, 9.0)
    rd.kv8_attention(q, cache, table, i32([past[0], length, past[2]]), i32(starts([n] * 3)), out=out)
    assert rd.device_error() == _lib.ERR_KV_RANGE
    assert torch.all(out[n:2 * n] == 9.0)
    for b in (0, 2):
        rows = slice(b * n, (b + 1) * n)
        check_attention(out[rows], q[rows], cache, table[b:b + 1], i32([past[b]]), i32([0, n]))


def test_a_negative_length_without_rows_is_no_error():
    """A slot of the batch that holds no sequence."""
    g = gen(3)
    table, pages = page_tables(g, [20, 0, 20], [1, 0, 1], 16)
    cache = fresh_cache(g, pages, 2, 64, 16)
    q, k = randn(g, 2, 2, 64), randn(g, 2, 2, 64)
    lengths, rs = i32([20, -1, 20]), i32([0, 1, 1, 2])
    rd.kv8_append(cache, k, k, table, lengths, rs, q=q)
    got = rd.kv8_attention(q, cache, table, lengths, rs)
    assert rd.device_error() == 0
    keep = torch.tensor([0, 2], device=DEV)
    check_attention(got, q, cache, table[keep], i32([20, 20]), i32([0, 1, 2]))


# ------------------------------------------------------------------ positions beyond the tables


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("past,n,max_pos", [
    ([14, 3, 40], [4, 4, 4], 16),     # a warp a block; across max_pos inside a page, before, behind
    ([14, 3, 40], [40, 9, 40], 50),   # a CTA a block; inside the first pages and a later one
    ([0, 45, 48], [60, 6, 20], 48)])  # at a page's end
def test_append_across_the_end_of_the_tables(D, past, n, max_pos):
    """What lies below max_pos is stored, K and V alike, and what lies behind is not."""
    g, page = gen(4), 16
    table, pages = page_tables(g, past, n, page)
    cache = fresh_cache(g, pages, 2, D, page)
    want = copy_of(cache)
    cos, sin = tables(max_pos, D, torch.float32)
    w = randn(g, D, mul=0.2, add=1.0)
    T = sum(n)
    q, k, v = randn(g, T, 4, D), randn(g, T, 2, D, mul=3.0), randn(g, T, 2, D, mul=3.0)
    out, want_q = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
    first = 0
    for b in range(3):
        m = max(0, min(n[b], max_pos - past[b]))
        rows = slice(first, first + m)
        first += n[b]
        if m:
            rd.kv8_append(want, k[rows], v[rows], table[b:b + 1], i32([past[b]]), i32([0, m]), cos, sin,
                          q=q[rows], q_norm=w, k_norm=w, out=want_q[rows])
    assert rd.device_error() == 0
    rd.kv8_append(cache, k, v, table, i32(past), i32(starts(n)), cos, sin, q=q, q_norm=w, k_norm=w,
                  out=out)
    assert rd.device_error() == _lib.ERR_KV_RANGE
    assert same_bytes(cache, want) and torch.equal(out, want_q)


# ------------------------------------------------------------------ outputs over inputs


def test_outputs_over_other_inputs_are_refused():
    g = gen(9)
    cos, sin = tables(32, 64, torch.float32)
    pos = torch.arange(4, device=DEV)
    buf = randn(g, 4, 12, 64)
    q, k, v, rest = buf[:, :2], buf[:, 2:4], buf[:, 4:6], buf[:, 6:8]
    was = buf.clone()
    for bad in (dict(q_out=k), dict(k_out=q), dict(q_out=buf[:, 1:3]), dict(q_out=rest, k_out=rest),
                dict(k_out=buf[:, 3:5]), dict(q_out=buf.view(-1)[512:1024].view(4, 2, 64))):
        with pytest.raises(ValueError, match="overlap"):
            rd.qk_norm_rope(q, k, cos, sin, pos, **bad)
    table, pages = page_tables(g, [0], [4], 16)
    cache = fresh_cache(g, pages, 2, 64, 16)
    lengths, rs = i32([0]), i32([0, 4])
    for bad in (k, v, buf[:, 1:3], buf[:, 5:7]):
        with pytest.raises(ValueError, match="overlap"):
            rd.kv8_append(cache, k, v, table, lengths, rs, cos, sin, q=q, out=bad)
    for bad in (buf[:, 1:3], buf.view(-1)[:512].view(4, 2, 64)):
        with pytest.raises(ValueError, match="overlap"):
            rd.kv8_attention(q, cache, table, lengths, rs, out=bad)
    assert torch.equal(buf, was)


def test_outputs_beside_the_inputs_in_one_buffer_are_taken():
    g = gen(10)
    cos, sin = tables(32, 64, torch.float32)
    pos = torch.arange(4, device=DEV)
    buf = randn(g, 4, 12, 64)
    q, k, v = buf[:, :2], buf[:, 2:4], buf[:, 4:6]
    want = rd.qk_norm_rope(q.clone(), k.clone(), cos, sin, pos)
    got = rd.qk_norm_rope(q, k, cos, sin, pos, q_out=buf[:, 6:8], k_out=buf[:, 8:10])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # every third head, and rows of another buffer's halves
    thirds = randn(g, 4, 9, 64)
    got = rd.qk_norm_rope(thirds[:, ::3], thirds[:, 1::3], cos, sin, pos, q_out=thirds[:, 2::3],
                          k_out=thirds[:, 1::3])
    assert got[0].data_ptr() == thirds[:, 2::3].data_ptr()
    rows = randn(g, 8, 2, 64)
    rd.qk_norm_rope(rows[:4], k, cos, sin, pos, q_out=rows[4:])
    table, pages = page_tables(g, [0], [4], 16)
    cache = fresh_cache(g, pages, 2, 64, 16)
    lengths, rs = i32([0]), i32([0, 4])
    assert torch.equal(rd.kv8_append(cache, k, v, table, lengths, rs, cos, sin, q=q, out=q), want[0])
    one = rd.kv8_attention(q, cache, table, lengths, rs)
    got = rd.kv8_attention(q, cache, table, lengths, rs, out=buf[:, 10:])
    assert torch.equal(got, one)
# ------------------------------------------------------------------ small weights


@pytest.mark.parametrize("past", [200, 900, 20000])  # shares of one CTA, of some, of all
@pytest.mark.parametrize("rows", [1, 3, 64, 130])
def test_small_weights_beside_a_large_one_count_in_both_kernels(rows, past):
    """Weights of 2^-30.6 of the largest, whose value is nothing: P' is 2^-16.6 or more, an fp16
    subnormal with steps of 2^-24, so half a step is 2^-8.4 of it; then the result's rounding."""
    g = gen(5)
    table, pages = page_tables(g, [past], [rows], 64)
    cache = fresh_cache(g, pages, 1, 128, 64)
    cache.k.view(torch.uint8).zero_()
    cache.v.copy_(o.to_e4m3(torch.ones(cache.v.shape, device=DEV)))
    cache.k_scale.fill_(1.0)
    cache.v_scale.fill_(1.0)
    pid = int(table[0, 0])
    cache.k[pid, :, 0, 0] = 240.0
    cache.v[pid, :, 0] = 0.0
    q = torch.zeros((rows, 2, 128), device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    lengths, rs = i32([past]), i32([0, rows])
    got = rd.kv8_attention(q, cache, table, lengths, rs)
    want, _, _ = o.attention(q, cache, table, lengths, rs)
    assert want.abs().min() > 0
    assert torch.all((got.double() - want).abs() <= want.abs() * 2.0 ** -8 * 2)


# ------------------------------------------------------------------ scores beyond 2^20


@pytest.mark.parametrize("rows", [1, 3, 80])
@pytest.mark.parametrize("mul", [1e4, 1e6, 4e6, 1e7, 2e7, 4e7, 1e8, 2e8, 1e9, 1e12, 1e20, 1e30])
def test_the_largest_score_takes_all_however_large(mul, rows):
    """One key's score is 448 / 240 of the next: its value is the result, whatever the steps of
    the scores in fp32 are."""
    g, page, D = gen(11), 16, 64
    for past, at in ((0, 0), (40, 0), (40, 17), (700, 699), (700, 130)):
        table, pages = page_tables(g, [past], [rows], page)
        cache = fresh_cache(g, pages, 1, D, page)
        cache.k.view(torch.uint8).zero_()
        cache.k[:, :, :, 0] = 240.0
        cache.k[int(table[0, at // page]), :, at % page, 0] = 448.0
        cache.k_scale.fill_(1.0)
        q = torch.zeros((rows, 2, D), device=DEV, dtype=torch.bfloat16)
        q[..., 0] = mul
        q[:, 1, 0] *= 0.6
        got = rd.kv8_attention(q, cache, table, i32([past]), i32([0, rows]))
        v = o.dense(cache.v, cache.v_scale, table[0].tolist(), past + 1)[0, at]
        assert torch.all((got.double() - v).abs() <= v.abs() * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -19))


# ------------------------------------------------------------------ value scales


@pytest.mark.parametrize("rows", [1, 3, 80])
@pytest.mark.parametrize("order", ["small first", "large first", "mixed"])
@pytest.mark.parametrize("past", [100, 3000])
def test_value_scales_far_apart(rows, order, past):
    """Equal weights of tokens whose values lie 2^149 apart: each counts in the sum.

    The result is a mean of large values and of (next to them) zeros. A factor that
    flushes loses half of the weights; the bar is the arithmetic's of check_attention
    (weights rounded to fp16, exp2 and log2, the sums) and the result's rounding.
    """
    g, page = gen(6), 16
    table, pages = page_tables(g, [past], [rows], page)
    cache = fresh_cache(g, pages, 1, 64, page)
    at = torch.arange(table.shape[1], device=DEV)
    small = {"small first": at < table.shape[1] // 2, "large first": at >= table.shape[1] // 2,
             "mixed": at % 3 != 1}[order]
    cache.v_scale[table[0].long(), 0] = torch.where(small, 2.0 ** -32, 2.0 ** 117)
    q = torch.zeros((rows, 2, 64), device=DEV, dtype=torch.bfloat16)
    lengths, rs = i32([past]), i32([0, rows])
    got = rd.kv8_attention(q, cache, table, lengths, rs)
    assert rd.device_error() == 0
    want, size, _ = o.attention(q, cache, table, lengths, rs)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -16 + past / 8 * 2.0 ** -24) * size
    assert torch.all((got.double() - want).abs() <= tol)


@pytest.mark.parametrize("rows", [1, 80])
@pytest.mark.parametrize("scale", [0.0, 1e-44, 1e-39, 2.0 ** -126, 2.0 ** -90])
def test_value_scales_that_are_next_to_nothing(rows, scale):
    """Tokens of a block with such a scale keep their weights; their values are nothing."""
    g, page = gen(7), 16
    past = 200
    table, pages = page_tables(g, [past], [rows], page)
    cache = fresh_cache(g, pages, 1, 64, page)
    cache.v_scale[table[0, ::2].long()] = scale
    q = randn(g, rows, 2, 64, mul=0.3)
    lengths, rs = i32([past]), i32([0, rows])
    check_attention(rd.kv8_attention(q, cache, table, lengths, rs), q, cache, table, lengths, rs)
    cache.v_scale.fill_(scale)
    got = rd.kv8_attention(q, cache, table, lengths, rs)
    assert torch.all(got.double().abs() <= 448 * 2.0 ** -80) and rd.device_error() == 0


# ------------------------------------------------------------------ infinite queries


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 80])
@pytest.mark.parametrize("past", [0, 40])
def test_an_infinite_query_against_keys_of_one_sign_is_nan(past, rows, dtype):
    """Every score is -inf: the softmax has no value, and the row is not taken for an empty one."""
    g = gen(8)
    table, pages = page_tables(g, [past], [rows], 16)
    cache = fresh_cache(g, pages, 1, 64, 16)
    cache.k[..., 5] = -3.0
    q = randn(g, rows, 2, 64, dtype=dtype)
    q[0, 1, 5] = float("inf")
    got = rd.kv8_attention(q, cache, table, i32([past]), i32([0, rows]))
    nan = torch.isnan(got)
    assert nan[0, 1].all() and int(nan.sum()) == 64


# ------------------------------------------------------------------ mixed steps


def test_a_mixed_step_as_two_calls():
    """Decoding sequences first, prompts behind: two calls over parts of one step's tensors."""
    g, page, D = gen(12), 16, 128
    past, rows = [300, 7, 1500, 64, 0, 90], [1, 1, 1, 1, 200, 130]
    table, pages = page_tables(g, past, rows, page)
    cache = fresh_cache(g, pages, 2, D, page)
    q = randn(g, sum(rows), 8, D)
    lengths, rs = i32(past), i32(starts(rows))
    out = torch.full_like(q, 9.0)
    rd.kv8_attention(q[:4], cache, table[:4], lengths[:4], rs[:5], out=out[:4])
    assert torch.all(out[4:] == 9.0)
    done = out[:4].clone()
    rd.kv8_attention(q, cache, table[4:], lengths[4:], rs[4:], out=out)
    assert torch.equal(out[:4], done) and rd.device_error() == 0
    check_attention(out, q, cache, table, lengths, rs)
    check_attention(rd.kv8_attention(q, cache, table, lengths, rs), q, cache, table, lengths, rs)
