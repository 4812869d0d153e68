"""Batched attention operators on the GPU: qk_norm_rope, kv8_append, kv8_attention.

Against a float64 restatement (oracle/kv8_oracle.py). Bars, derived from the
arithmetic before the first run (u = 2^-24, half = finfo(type).eps / 2):
  norm + rotation  fp32: the mean square of D terms in a chain of at most 16
      fused adds and 3 exchanges (19 u, halved by the root), root, reciprocal,
      three products and the rotation's two: below 24 u of |x' cos| + |x' sin|;
      then half of the result, plus half a subnormal step (2^-25 for fp16).
  8-bit codes      bit for bit where the input of the rounding is exact (values
      without a rotation); else within half a step, 2^-4 of the value or 2^-10
      of the scale, after the fp32 error above.
  attention        a score's error: D products summed in fp32, D u of the sum of
      |q k| in the exponent; exp2 and its argument 2^-20; P rounded to fp16,
      2^-11 of each weight (and 2^-39 of the largest below fp16's normal range);
      the sums over n tokens, n / 8 u. Each of these is relative to sum w |v|.
      Then half of the result.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

import roofline_decoding_b200 as rd  # noqa: E402
from oracle import kv8_oracle as o  # noqa: E402
from roofline_decoding_b200 import _lib  # noqa: E402

DEV = "cuda"
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16, mul=1.0, add=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * mul + add).to(dtype)


def tables(n, D, dtype):
    inv = 1e4 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(n, device=DEV, dtype=torch.float64), inv)
    a = torch.cat([a, a], -1)
    return a.cos().to(dtype), a.sin().to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(rows, lead=0):
    out = [lead]
    for n in rows:
        out.append(out[-1] + n)
    return out


def check_rope(got, x, weight, cos, sin, dtype):
    want = o.norm_rope(x, weight, cos, sin)
    size = o.norm_rope(x, weight).abs()
    if cos is not None:
        other = size.roll(size.shape[-1] // 2, -1)
        size = size * cos.double().abs()[:, None] + other * sin.double().abs()[:, None]
    tol = 24 * U * size + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -25
    assert got.dtype == dtype and got.shape == x.shape
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), ((got.double() - want).abs() / tol).max().item()


# ------------------------------------------------------------------ norm + rotation


@pytest.mark.parametrize("dtype,table", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"),
                                         ("fp16", "fp32")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads,kv,rows", [(1, 1, 1), (12, 2, 8), (5, 5, 3), (32, 8, 700), (7, 0, 9),
                                           (0, 3, 9)])
@pytest.mark.parametrize("norm", ["both", "q", "k", "none"])
def test_qk_norm_rope(dtype, table, D, heads, kv, rows, norm):
    g, dt = gen(heads * 100 + rows), TYPES[dtype]
    qkv = randn(g, rows, heads + 2 * kv, D, dtype=dt, mul=2.0)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
    cos, sin = tables(400, D, TYPES[table])
    pos = torch.randint(0, 400, (rows,), generator=g, device=DEV)
    wq = randn(g, D, dtype=dt, mul=0.2, add=1.0) if norm in ("both", "q") else None
    wk = randn(g, D, dtype=dt, mul=0.2, add=1.0) if norm in ("both", "k") else None
    got_q, got_k = rd.qk_norm_rope(q, k, cos, sin, pos, q_norm=wq, k_norm=wk)
    check_rope(got_q, q, wq, cos[pos], sin[pos], dt)
    check_rope(got_k, k, wk, cos[pos], sin[pos], dt)
    assert rd.device_error() == 0


def test_qk_norm_rope_without_tables_in_place_and_transposed():
    g, dt = gen(3), torch.bfloat16
    q, k = randn(g, 6, 4, 128), randn(g, 6, 2, 128)
    w = randn(g, 128, mul=0.2, add=1.0)
    got_q, got_k = rd.qk_norm_rope(q, k, q_norm=w)
    check_rope(got_q, q, w, None, None, dt)
    assert torch.equal(got_k, k)  # neither norm nor rotation
    # in place, in a q|k|v buffer; v stays
    cos, sin = tables(16, 128, torch.float32)
    pos = torch.arange(6, device=DEV)
    buf = randn(g, 6, 8, 128)
    was = buf.clone()
    rd.qk_norm_rope(buf[:, :4], buf[:, 4:6], cos, sin, pos, k_norm=w, q_out=buf[:, :4],
                    k_out=buf[:, 4:6])
    check_rope(buf[:, :4], was[:, :4], None, cos[pos], sin[pos], dt)
    check_rope(buf[:, 4:6], was[:, 4:6], w, cos[pos], sin[pos], dt)
    assert torch.equal(buf[:, 6:], was[:, 6:])
    # other orders of storage: heads first, elements apart, a pointer off alignment
    cases = [randn(g, 4, 6, 128).transpose(0, 1), randn(g, 6, 128, 4).transpose(1, 2),
             randn(g, 6 * 4 * 128 + 3)[3:].view(6, 4, 128)]
    for x in cases:
        got, _ = rd.qk_norm_rope(x, k, cos, sin, pos, q_norm=w)
        check_rope(got, x, w, cos[pos], sin[pos], dt)
    out = torch.zeros(4, 6, 128, device=DEV, dtype=dt).transpose(0, 1)
    assert rd.qk_norm_rope(x, k, cos, sin, pos, q_out=out)[0] is out
    check_rope(out, x, None, cos[pos], sin[pos], dt)


def test_qk_norm_rope_zero_rows_and_extreme_values():
    g, dt = gen(4), torch.bfloat16
    w = randn(g, 64, mul=0.2, add=1.0)
    empty = torch.empty((0, 2, 64), device=DEV, dtype=dt)
    q, _ = rd.qk_norm_rope(empty, empty, q_norm=w)
    assert q.shape == (0, 2, 64)
    x = torch.zeros((3, 2, 64), device=DEV, dtype=dt)
    x[1] = 1e-20  # the squares vanish beside eps
    x[2, 0, 5] = float("nan")
    got, _ = rd.qk_norm_rope(x, x, q_norm=w)
    assert torch.all(got[0] == 0)
    check_rope(got[:2], x[:2], w, None, None, dt)
    assert torch.isnan(got[2, 0]).all() and torch.all(got[2, 1] == 0)


def test_positions_outside_the_tables_are_left_out():
    g = gen(5)
    q, k = randn(g, 4, 2, 64), randn(g, 4, 2, 64)
    cos, sin = tables(8, 64, torch.float32)
    pos = torch.tensor([0, 8, -1, 7], device=DEV)
    out_q, out_k = torch.full_like(q, 3.0), torch.full_like(k, 3.0)
    rd.qk_norm_rope(q, k, cos, sin, pos, q_out=out_q, k_out=out_k)
    assert rd.device_error() == _lib.ERR_KV_RANGE and rd.device_error() == 0
    assert torch.all(out_q[1:3] == 3.0) and torch.all(out_k[1:3] == 3.0)
    keep = torch.tensor([0, 3], device=DEV)
    check_rope(out_q[keep], q[keep], None, cos[pos[keep]], sin[pos[keep]], torch.bfloat16)


# ------------------------------------------------------------------ cache


def fresh_cache(g, pages, kv, D, page):
    """A cache in use: random codes, power-of-two scales."""
    def codes():
        return o.to_e4m3(torch.randn((pages, kv, page, D), generator=g, device=DEV) * 100)

    def scales():
        return torch.exp2(torch.randint(-8, -5, (pages, kv), generator=g, device=DEV).float())

    return rd.KV8Cache(codes(), codes(), scales(), scales())


def page_tables(g, past, rows, page, extra=2):
    """Distinct shuffled pages for every sequence, and the number of pages."""
    need = [-(-(p + n) // page) for p, n in zip(past, rows)]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(past), max(max(need), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def check_append(before, after, new, exact, lengths, row_starts, table, scale_before, scale_after):
    """One of K and V: codes and scales of every page, against the definition."""
    page = before.shape[2]
    untouched = torch.ones(before.shape[:3], dtype=torch.bool, device=DEV)
    whole = torch.ones(before.shape[0], dtype=torch.bool, device=DEV)
    for pid, slot, row, n in o.blocks(lengths, row_starts, table, page):
        whole[pid] = False
        untouched[pid, :, slot:slot + n] = False
        for h in range(before.shape[1]):
            x = new[row:row + n, h]
            fin = x.abs()[torch.isfinite(x)]
            amax = fin.max().item() if fin.numel() else 0.0
            s = scale_after[pid, h].item()
            slack = 0.0 if exact else 2.0 ** -19
            old = scale_before[pid, h].item() if slot else 0.0
            assert max(old, o.least_scale(amax * (1 - slack))) <= s <= \
                max(old, o.least_scale(amax * (1 + slack))), (pid, h)
            got = after[pid, h, slot:slot + n]
            if exact:
                want = o.to_e4m3(torch.nan_to_num(x / s, nan=float("nan"), posinf=448.0,
                                                  neginf=-448.0))
                same = (got.float() == want.float()) | (torch.isnan(got.float()) & torch.isnan(x))
                assert same.all()
            else:
                err = (got.double() * s - x).abs()
                assert torch.all(err <= x.abs() * 2.0 ** -4 * (1 + 2.0 ** -10) + s * 2.0 ** -10 * 1.01)
            held = before[pid, h, :slot].float()
            want = o.to_e4m3(held * (old / s)) if s != old else before[pid, h, :slot]
            assert torch.equal(after[pid, h, :slot].float(), want.float())
            untouched[pid, h, :slot] = False
    assert torch.equal(after.view(torch.uint8)[untouched], before.view(torch.uint8)[untouched])
    assert torch.equal(scale_after[whole], scale_before[whole])


def run_append(seed, past, rows, kv=2, heads=6, D=128, page=64, dtype="bf16", table="fp32",
               norm=True, rope=True, lead=0, pad=0, mul=1.5, change=None):
    g, dt = gen(seed), TYPES[dtype]
    T = lead + sum(rows) + pad
    tab, pages = page_tables(g, past, rows, page)
    cache = fresh_cache(g, pages, kv, D, page)
    qkv = randn(g, T, heads + 2 * kv, D, dtype=dt, mul=mul)
    if change:
        change(qkv[:, heads:heads + kv], qkv[:, heads + kv:])
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    cos, sin = tables(max(p + n for p, n in zip(past, rows)) or 1, D, TYPES[table])
    if not rope:
        cos = sin = None
    wq = randn(g, D, dtype=dt, mul=0.2, add=1.0) if norm else None
    wk = randn(g, D, dtype=dt, mul=0.2, add=1.0) if norm else None
    lengths, rs = i32(past), i32(starts(rows, lead))
    was = [t.clone() for t in cache]
    out = torch.full((T, heads, D), 9.0, device=DEV, dtype=dt)
    got = rd.kv8_append(cache, k, v, tab, lengths, rs, cos, sin, q=q if heads else None, q_norm=wq,
                        k_norm=wk, out=out if heads else None)
    assert rd.device_error() == 0
    pos = o.positions(lengths, rs, T)
    c, s = (cos[pos], sin[pos]) if rope else (None, None)
    new_k = o.norm_rope(k, wk, c, s)
    check_append(was[0], cache.k, new_k, not (norm or rope), lengths, rs, tab, was[2], cache.k_scale)
    check_append(was[1], cache.v, v.double(), True, lengths, rs, tab, was[3], cache.v_scale)
    if heads:
        inside = slice(lead, T - pad)
        check_rope(got[inside], q[inside], wq, None if c is None else c[inside],
                   None if s is None else s[inside], dt)
        assert torch.all(out[:lead] == 9.0) and torch.all(out[T - pad:] == 9.0)


@pytest.mark.parametrize("D,page", [(64, 16), (64, 128), (128, 16), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("past,rows", [([0], [1]), ([5, 64, 0, 127], [1, 1, 1, 1]),
                                       ([0, 3, 200], [130, 0, 7]), ([63, 16, 128], [2, 129, 33])])
def test_append(D, page, past, rows):
    run_append(D + page + sum(past), past, rows, D=D, page=page)


@pytest.mark.parametrize("dtype,table", [("bf16", "bf16"), ("fp16", "fp16"), ("fp16", "fp32")])
@pytest.mark.parametrize("norm,rope,heads", [(True, False, 3), (False, True, 4), (False, False, 0)])
def test_append_types_and_parts(dtype, table, norm, rope, heads):
    run_append(11, [30, 0, 1], [3, 70, 1], dtype=dtype, table=table, norm=norm, rope=rope,
               heads=heads, kv=4, page=32)


def test_append_many_sequences_and_padding():
    """More sequences than a scan step, some without rows, rows before and behind them."""
    past = [(37 * i) % 150 for i in range(77)]
    rows = [(5 * i) % 4 if i % 9 else 0 for i in range(77)]
    run_append(21, past, rows, kv=1, heads=2, D=64, page=16, lead=3, pad=5)


@pytest.mark.parametrize("mul", [1e-12, 1e-3, 300.0, 3e30])
def test_append_scales_grow_with_the_values(mul):
    """Tiny values keep the old scale, larger ones round the page's older rows again."""
    run_append(31, [20, 63, 64], [2, 3, 1], norm=False, mul=mul)
    run_append(32, [20, 63, 64], [2, 3, 1], norm=False, rope=False, mul=mul)


def test_append_values_at_the_borders_of_the_scale():
    def change(k, v):
        v.zero_()
        v[0, 0, 0] = 448.0      # scale 1 exactly
        v[0, 1, 0] = 450.0      # the next bf16: scale 2
        v[1, 0, 0] = 7.0 / 16   # 2^-10
        v[2, 1, 3] = 1e-30      # below the least scale's reach
    run_append(41, [0, 0, 0], [1, 1, 1], norm=False, rope=False, change=change)


def test_append_infinities_and_nan():
    def change(k, v):
        v[0, 0, 3], v[0, 0, 4], v[0, 1, 5] = float("inf"), float("-inf"), float("nan")
        k[1, 0, 3], k[1, 1, 9] = float("inf"), float("nan")
    run_append(42, [5, 40], [2, 2], norm=False, rope=False, change=change)


def test_append_step_by_step_is_one_long_append_within_a_step():
    """A token at a time, a page's scale ends where one call over the page puts it."""
    g, D, page, n = gen(51), 128, 32, 80
    table, pages = page_tables(g, [0], [n], page)
    k, v = randn(g, n, 2, D), randn(g, n, 2, D) * torch.linspace(0.01, 4, n, device=DEV).to(
        torch.bfloat16)[:, None, None]
    one, many = (rd.KV8Cache.empty(pages, 2, D, page) for _ in range(2))
    rd.kv8_append(one, k, v, table, i32([0]), i32([0, n]))
    for i in range(n):
        rd.kv8_append(many, k[i:i + 1], v[i:i + 1], table, i32([i]), i32([0, 1]))
    used = table[0].long()
    assert torch.equal(one.k_scale[used], many.k_scale[used])
    assert torch.equal(one.v_scale[used], many.v_scale[used])
    a = o.dense(one.v, one.v_scale, table[0].tolist(), n)
    b = o.dense(many.v, many.v_scale, table[0].tolist(), n)
    # equal but where a value was rounded in a smaller scale first: a step apart at most
    step = a.abs().maximum(b.abs()) * 2.0 ** -3 + \
        one.v_scale.double()[used].amax() * 2.0 ** -9
    assert torch.all((a - b).abs() <= step)
    assert (a == b).double().mean() > 0.9


def test_append_bad_pages_and_positions_are_left_out():
    g, page = gen(61), 16
    cache = fresh_cache(g, 6, 2, 64, page)
    was = [t.clone() for t in cache]
    k, v = randn(g, 5, 2, 64), randn(g, 5, 2, 64)
    q = randn(g, 5, 2, 64)
    # pages 6 and -1 do not exist; sequence 3's second page is outside the table; 4 is fine
    table = i32([[6], [-1], [-2 ** 31], [1], [2]])
    lengths = i32([0, 3, 5, 16, 4])
    rd.kv8_append(cache, k, v, table, lengths, i32([0, 1, 2, 3, 4, 5]))
    assert rd.device_error() == _lib.ERR_KV_RANGE
    changed = [p for p in range(6) if not torch.equal(cache.v.view(torch.uint8)[p],
                                                      was[1].view(torch.uint8)[p])]
    assert changed == [2]
    # a position beyond the tables
    cos, sin = tables(4, 64, torch.float32)
    out = torch.full_like(q, 9.0)
    was = [t.clone() for t in cache]
    rd.kv8_append(cache, k[:1], v[:1], i32([[3]]), i32([4]), i32([0, 1]), cos, sin, q=q[:1],
                  out=out[:1])
    assert rd.device_error() == _lib.ERR_KV_RANGE
    assert torch.all(out == 9.0)
    assert torch.equal(cache.k.view(torch.uint8), was[0].view(torch.uint8))


# ------------------------------------------------------------------ attention


def check_attention(got, q, cache, table, lengths, rs, scale=None, rows=None):
    want, size, reach = o.attention(q, cache, table, lengths, rs, scale)
    D, n = q.shape[2], int((lengths.long() + rs.long().diff()).max())
    rel = 2.0 ** -11 + 2.0 ** -19 + 2 * D * U * reach + n / 8 * U
    vmax = max((cache.v_scale.max() * 448).item(), 0.0)
    tol = torch.finfo(q.dtype).eps / 2 * want.abs() + rel * size + n * 2.0 ** -39 * vmax + 2.0 ** -25
    rows = slice(int(rs[0]), int(rs[-1])) if rows is None else rows
    bad = (got.double() - want).abs()[rows] / tol[rows]
    assert not (bad > 1).any() and not torch.isnan(bad).any(), bad.max().item()


def run_attention(seed, past, rows, heads=6, kv=2, D=128, page=64, dtype="bf16", mul=1.0,
                  lead=0, pad=0, scale=None, tune=None):
    g, dt = gen(seed), TYPES[dtype]
    T = lead + sum(rows) + pad
    table, pages = page_tables(g, past, rows, page)
    cache = fresh_cache(g, pages, kv, D, page)
    q = randn(g, T, heads, D, dtype=dt, mul=mul)
    if tune:
        cache = tune(q, cache) or cache
    lengths, rs = i32(past), i32(starts(rows, lead))
    out = torch.full_like(q, 9.0)
    got = rd.kv8_attention(q, cache, table, lengths, rs, scale=scale, out=out)
    assert got is out and rd.device_error() == 0
    check_attention(got, q, cache, table, lengths, rs, scale)
    assert torch.all(out[:lead] == 9.0) and torch.all(out[T - pad:] == 9.0)
    again = rd.kv8_attention(q, cache, table, lengths, rs, scale=scale)
    assert torch.equal(again[lead:T - pad], out[lead:T - pad])
    return q, cache, table, lengths, rs, out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("past", [0, 1, 14, 15, 16, 31, 32, 33, 127, 128, 700, 5000])
def test_attention_lengths(D, past):
    run_attention(past + D, [past], [1], D=D, page=16 if past % 2 else 64)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 3), (10, 2), (16, 1), (40, 8), (32, 2)])
@pytest.mark.parametrize("rows", [1, 2, 5])
def test_attention_heads(heads, kv, rows):
    run_attention(heads + rows, [40, 333, 0], [rows, rows, rows], heads=heads, kv=kv, page=32)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attention_ragged(page, dtype):
    """Sequences without rows among the others, rows before and behind them."""
    run_attention(page, [1000, 7, 0, 129, 64, 2047], [1, 0, 3, 17, 1, 40], page=page, dtype=dtype,
                  lead=2, pad=3)


def test_attention_many_sequences():
    past = [(131 * i) % 900 for i in range(200)]
    run_attention(7, past, [1 + i % 2 for i in range(200)], heads=4, kv=2, D=64, page=16)


def test_attention_of_a_prompt():
    run_attention(8, [0, 100], [300, 129], heads=8, kv=2)


@pytest.mark.parametrize("mul", [1e-3, 30.0, 1e4])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attention_sharp_and_flat_scores(mul, dtype):
    """From almost uniform weights to one token that takes all, over split sequences."""
    run_attention(9, [3000, 50], [1, 2], mul=mul, dtype=dtype)


def test_attention_scales_of_any_size():
    """Scales that are no powers of two, 2^40 apart from page to page, and a given factor."""
    def tune(q, cache):
        s = torch.exp2(torch.rand(cache.v_scale.shape, generator=gen(1), device=DEV) * 40 - 20)
        return cache._replace(v_scale=s, k_scale=torch.rand_like(s) * 0.02 + 1e-3)
    run_attention(10, [700, 90], [1, 3], page=16, tune=tune, scale=0.31)


def test_attention_negative_and_zero_factor():
    run_attention(12, [200], [2], scale=-0.05)
    run_attention(13, [200], [2], scale=0.0)


def test_attention_one_token_far_below_the_rest_still_counts():
    """Many small weights beside one large one: none is lost to the 16-bit product."""
    def tune(q, cache):
        cache.k.view(torch.uint8).zero_()
        cache.v.copy_(o.to_e4m3(torch.full(cache.v.shape, 1.0, device=DEV)))
        cache.v_scale.fill_(1.0)
        q.zero_()
        q[..., 0] = 1.0
        pid = int(tune.table[0, 0])
        cache.k[pid, :, 0, 0] = 240.0  # e^-21 for every other token
        cache.k_scale.fill_(1.0)
        cache.v[pid, :, 0] = 0.0       # the large weight's value is nothing
    g = gen(14)
    past = 60000
    table, pages = page_tables(g, [past], [1], 64)
    cache = fresh_cache(g, pages, 1, 128, 64)
    tune.table = table
    q = randn(g, 1, 2, 128)
    tune(q, cache)
    got = rd.kv8_attention(q, cache, table, i32([past]), i32([0, 1]))
    want, size, _ = o.attention(q, cache, table, i32([past]), i32([0, 1]))
    # weights of 2^-30.6 of the largest: P' is 2^-16.6, an fp16 subnormal with steps of
    # 2^-24, so half a step is 2^-8.4 of it; then the rounding of the result
    assert want.abs().min() > 0
    assert torch.all((got.double() - want).abs() <= want.abs() * 2.0 ** -8 * 2)


def test_attention_stale_page_contents_are_not_read_into_results():
    """NaN codes behind a sequence's end, and in pages of no sequence."""
    g = gen(15)
    past, rows = [37, 5, 0], [1, 3, 1]
    table, pages = page_tables(g, past, rows, 64)
    cache = fresh_cache(g, pages, 2, 128, 64)
    used = torch.zeros(pages, 64, dtype=torch.bool, device=DEV)
    for b in range(3):
        used[table[b, 0].long(), :past[b] + rows[b]] = True
    for c in (cache.k, cache.v):
        c.view(torch.uint8).copy_(torch.where(used[:, None, :, None], c.view(torch.uint8), 0x7F))
    q = randn(g, 5, 4, 128)
    got = rd.kv8_attention(q, cache, table, i32(past), i32(starts(rows)))
    check_attention(got, q, cache, table, i32(past), i32(starts(rows)))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("where", ["k", "v"])
def test_attention_nan_reaches_only_the_rows_that_see_it(D, where):
    """Token 41 holds a NaN: rows 40.. see it, the rows before do not."""
    g = gen(16)
    past, n, bad = 36, 30, 41
    table, pages = page_tables(g, [past], [n], 16)
    cache = fresh_cache(g, pages, 1, D, 16)
    pid = int(table[0, bad // 16])
    (cache.k if where == "k" else cache.v).view(torch.uint8)[pid, 0, bad % 16, 3] = 0x7F
    q = randn(g, n, 2, D)
    got = rd.kv8_attention(q, cache, table, i32([past]), i32([0, n]))
    clean = rd.KV8Cache(*[t.clone() for t in cache])
    for c in (clean.k, clean.v):
        c.view(torch.uint8)[pid, 0, bad % 16, 3] = 0
    first = bad - past  # the first row that sees it
    check_attention(got, q, clean, table, i32([past]), i32([0, n]), rows=slice(0, first))
    if where == "k":
        assert torch.isnan(got[first:]).all()
    else:
        assert torch.isnan(got[first:, :, 3]).all()
        keep = [d for d in range(D) if d != 3]
        assert not torch.isnan(got[:, :, keep]).any()


def test_attention_infinite_and_nan_queries_stay_in_their_rows():
    g = gen(17)
    table, pages = page_tables(g, [50], [3], 64)
    cache = fresh_cache(g, pages, 2, 128, 64)
    q = randn(g, 3, 4, 128)
    q[0, 1, 7] = float("inf")
    q[2, 3, 7] = float("nan")
    got = rd.kv8_attention(q, cache, table, i32([50]), i32([0, 3]))
    nan = torch.isnan(got).all(-1)
    assert nan[0, 1] and nan[2, 3] and int(nan.sum()) == 2
    assert int(torch.isnan(got).any(-1).sum()) == 2


def test_attention_bad_pages_are_left_out():
    g, page = gen(18), 16
    past, rows = [60, 20, 100], [1, 2, 1]
    table, pages = page_tables(g, past, rows, page)
    cache = fresh_cache(g, pages, 2, 64, page)
    q = randn(g, 4, 4, 64)
    bad = table.clone()
    bad[0, 1], bad[0, 3] = pages, -7       # two of sequence 0's four pages
    bad[1, :] = 2 ** 31 - 1                # all of sequence 1's
    got = rd.kv8_attention(q, cache, bad, i32(past), i32(starts(rows)))
    assert rd.device_error() == _lib.ERR_KV_RANGE
    # sequence 0 over the 32 tokens that are left; as two pages of a shorter one
    short = torch.stack([table[0, 0], table[0, 2]])[None]
    check_attention(got[:1], q[:1], cache, short, i32([31]), i32([0, 1]))
    assert torch.all(got[1:3] == 0)
    check_attention(got[3:], q[3:], cache, table[2:], i32(past[2:]), i32([0, 1]))


def test_attention_length_beyond_the_page_table():
    """A length that the table has no room for: the tokens it has are used, the error is told."""
    g, page = gen(19), 16
    table, pages = page_tables(g, [47], [1], page)
    cache = fresh_cache(g, pages, 1, 64, page)
    q = randn(g, 1, 2, 64)
    for length in (48, 1000, 2 ** 31 - 1):
        got = rd.kv8_attention(q, cache, table, i32([length]), i32([0, 1]))
        assert rd.device_error() == _lib.ERR_KV_RANGE
        check_attention(got, q, cache, table, i32([47]), i32([0, 1]))


def test_attention_cache_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes each for K and V, its last pages in use."""
    kv, page, D = 8, 128, 128
    pages = 2 ** 32 // (kv * page * D) + 40
    cache = rd.KV8Cache.empty(pages, kv, D, page)
    g = gen(20)
    past, rows = [300, 4], [2, 1]
    table = i32([[pages - 1, pages - 2, 5], [pages - 3, 0, 0]])
    k, v = randn(g, 301, kv, D), randn(g, 301, kv, D)
    rd.kv8_append(cache, k[:300], v[:300], table[:1], i32([0]), i32([0, 300]))
    rd.kv8_append(cache, k[:4], v[:4], table[1:], i32([0]), i32([0, 4]))
    rd.kv8_append(cache, k[:3], v[:3], table, i32(past), i32([0, 2, 3]))
    q = randn(g, 3, 16, D)
    got = rd.kv8_attention(q, cache, table, i32(past), i32([0, 2, 3]))
    assert rd.device_error() == 0
    check_attention(got, q, cache, table, i32(past), i32([0, 2, 3]))
    a = o.dense(cache.v, cache.v_scale, table[0].tolist(), 300)
    assert torch.all((a.transpose(0, 1) - v[:300].double()).abs() <=
                     v[:300].double().abs() * 2.0 ** -4 + cache.v_scale[table[0].long()].max() * 2.0 ** -10)


def test_attention_views_other_orders_and_no_rows():
    g = gen(22)
    table, pages = page_tables(g, [90], [3], 64)
    cache = fresh_cache(g, pages, 2, 128, 64)
    lengths, rs = i32([90]), i32([0, 3])
    buf = randn(g, 3, 8, 128)
    for q in (buf[:, :4], randn(g, 4, 3, 128).transpose(0, 1), randn(g, 3, 128, 4).transpose(1, 2)):
        check_attention(rd.kv8_attention(q, cache, table, lengths, rs), q, cache, table, lengths, rs)
    out = torch.zeros(4, 3, 128, device=DEV, dtype=torch.bfloat16).transpose(0, 1)
    rd.kv8_attention(q, cache, table, lengths, rs, out=out)
    check_attention(out, q, cache, table, lengths, rs)
    # a page table that is a part of a wider one
    wide = torch.full((1, 9), -1, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + table.shape[1]] = table
    part = wide[:, 4:4 + table.shape[1]]
    check_attention(rd.kv8_attention(q, cache, part, lengths, rs), q, cache, table, lengths, rs)
    # nothing to do: no rows, no sequences, sequences without rows
    none = rd.kv8_attention(q[:0], cache, table, lengths, i32([0, 0]))
    assert none.shape == (0, 4, 128)
    out = torch.full((3, 4, 128), 9.0, device=DEV, dtype=torch.bfloat16)
    rd.kv8_attention(q, cache, table[:0], lengths[:0], i32([0]), out=out)
    rd.kv8_attention(q, cache, table, lengths, i32([1, 1]), out=out)
    rd.kv8_append(cache, q[:, :2], q[:, 2:4], table, lengths, i32([1, 1]), q=q, out=out)
    assert torch.all(out == 9.0) and rd.device_error() == 0


def test_streams_graphs_and_repeated_calls():
    """Two captured steps on streams of their own, replayed side by side as lengths move on."""
    g, page = gen(23), 32
    sides = []
    for i in range(2):
        past, rows = [40 + i, 3, 200], [1, 1, 1]
        table, pages = page_tables(g, [300] * 3, [0] * 3, page)
        cache = fresh_cache(g, pages, 2, 128, page)
        k, v, q = (randn(g, 3, n, 128) for n in (2, 2, 8))
        cos, sin = tables(400, 128, torch.float32)
        lengths, rs = i32(past), i32(starts(rows))
        s = torch.cuda.Stream()
        sides.append(dict(table=table, cache=cache, k=k, v=v, q=q, cos=cos, sin=sin, lengths=lengths,
                          rs=rs, stream=s))

    def step(x):
        x["q2"] = rd.kv8_append(x["cache"], x["k"], x["v"], x["table"], x["lengths"], x["rs"],
                                x["cos"], x["sin"], q=x["q"])
        x["out"] = rd.kv8_attention(x["q2"], x["cache"], x["table"], x["lengths"], x["rs"])
        x["lengths"] += 1

    torch.cuda.synchronize()
    for x in sides:
        x["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(x["graph"], stream=x["stream"]):
            step(x)
    for _ in range(5):
        for x in sides:
            with torch.cuda.stream(x["stream"]):
                x["graph"].replay()
        torch.cuda.synchronize()
        for x in sides:
            check_attention(x["out"], x["q2"], x["cache"], x["table"], x["lengths"] - 1, x["rs"])
    assert rd.device_error() == 0


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_batched_decoder_layer(dtype):
    """Projections, head norms, rotation, cache and attention of a prompt and two steps after it.

    Every operator is checked against its own 64-bit form on the inputs that the
    run hands it, so the bars stay those of the single operators.
    """
    from test_gemm_fused_gpu import check_gemm, weights

    g, dt = gen(71), TYPES[dtype]
    hidden, heads, kv, D, page, inter = 512, 8, 2, 64, 16, 640
    w_qkv, w_o = weights(g, hidden, (heads + 2 * kv) * D), weights(g, heads * D, hidden)
    w_gu, w_down = weights(g, hidden, 2 * inter), weights(g, inter, hidden)
    b_qkv = randn(g, (heads + 2 * kv) * D, dtype=dt, mul=0.1)
    wq, wk = randn(g, D, dtype=dt, mul=0.1, add=1.0), randn(g, D, dtype=dt, mul=0.1, add=1.0)
    cos, sin = tables(128, D, torch.float32)
    table, pages = page_tables(g, [50, 33, 70], [0, 0, 0], page)
    cache = rd.KV8Cache.empty(pages, kv, D, page)
    past = [0, 0, 0]
    for rows in ([40, 17, 61], [1, 1, 1], [3, 0, 2]):
        T = sum(rows)
        h = randn(g, T, hidden, dtype=dt)
        lengths, rs = i32(past), i32(starts(rows))
        qkv = rd.w4_gemm_fused(h, *w_qkv, bias=b_qkv)
        check_gemm(qkv, h, w_qkv, bias=b_qkv)
        x = qkv.view(T, heads + 2 * kv, D)
        was = [t.clone() for t in cache]
        q = rd.kv8_append(cache, x[:, heads:heads + kv], x[:, heads + kv:], table, lengths, rs, cos,
                          sin, q=x[:, :heads], q_norm=wq, k_norm=wk)
        pos = o.positions(lengths, rs, T)
        check_rope(q, x[:, :heads], wq, cos[pos], sin[pos], dt)
        check_append(was[0], cache.k, o.norm_rope(x[:, heads:heads + kv], wk, cos[pos], sin[pos]),
                     False, lengths, rs, table, was[2], cache.k_scale)
        check_append(was[1], cache.v, x[:, heads + kv:].double(), True, lengths, rs, table, was[3],
                     cache.v_scale)
        a = rd.kv8_attention(q, cache, table, lengths, rs)
        check_attention(a, q, cache, table, lengths, rs)
        a = a.view(T, heads * D)
        h2 = rd.w4_gemm_fused(a, *w_o, residual=h)
        check_gemm(h2, a, w_o, residual=h)
        act = rd.w4_gemm_fused(h2, *w_gu, activation="swiglu")
        check_gemm(act, h2, w_gu, activation="swiglu")
        before = h2.clone()
        rd.w4_gemm_fused(act, *w_down, residual=h2, out=h2)
        check_gemm(h2, act, w_down, residual=before)
        past = [p + n for p, n in zip(past, rows)]
    assert rd.device_error() == 0


def test_a_chain_of_calls_sees_each_others_results():
    """Append, attention and norms back to back with the kernels that write and reuse their inputs."""
    g, page = gen(81), 32
    past, rows = [300, 45, 0, 77], [1, 1, 1, 1]
    table, pages = page_tables(g, past, rows, page)
    cache = fresh_cache(g, pages, 2, 128, page)
    cos, sin = tables(400, 128, torch.float32)
    lengths, rs = i32(past), i32(starts(rows))
    steps = [randn(g, 4, 12, 128) for _ in range(5)]

    def run(behind):
        c = rd.KV8Cache(*[t.clone() for t in cache])
        buf, outs = torch.empty_like(steps[0]), []
        big = torch.randn(4096, 4096, device=DEV)
        torch.cuda.synchronize()
        for x in steps:
            if behind:
                torch.mm(big, big)
            buf.copy_(x)
            q = rd.kv8_append(c, buf[:, 8:10], buf[:, 10:], table, lengths, rs, cos, sin, q=buf[:, :8])
            o1 = rd.kv8_attention(q, c, table, lengths, rs)
            n1, n2 = rd.qk_norm_rope(o1, q[:, :2], cos, sin, lengths.long())
            outs += [q + 0, o1 + 0, n1 + n2.repeat(1, 4, 1)]
            buf.fill_(float("nan"))
            if not behind:
                torch.cuda.synchronize()
        return outs

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b) and not torch.isnan(a).any()


# ------------------------------------------------------------------ many rows a sequence


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("past,rows,heads,kv,page", [
    ([0], [128], 1, 1, 64), ([0], [127], 2, 1, 16), ([5], [129], 3, 1, 32), ([130], [64], 8, 8, 128),
    ([0, 1000, 300], [200, 1, 77], 8, 2, 64), ([4000], [100], 10, 2, 16),
    ([0, 0, 0, 0], [40, 300, 0, 150], 16, 1, 32), ([0], [1500], 5, 1, 64)])
def test_attention_prompts(D, past, rows, heads, kv, page):
    run_attention(sum(rows) + D, past, rows, heads=heads, kv=kv, D=D, page=page)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("mul", [1e-3, 1.0, 30.0, 1e4])
def test_attention_prompts_sharp_and_flat(dtype, mul):
    run_attention(91, [700, 33], [150, 90], heads=4, kv=2, dtype=dtype, mul=mul, lead=1, pad=2)


def test_attention_prompts_scales_of_any_size():
    def tune(q, cache):
        s = torch.exp2(torch.rand(cache.v_scale.shape, generator=gen(1), device=DEV) * 40 - 20)
        return cache._replace(v_scale=s, k_scale=torch.rand_like(s) * 0.02 + 1e-3)
    run_attention(92, [300, 20], [70, 100], page=16, tune=tune, scale=0.31)


def test_attention_prompts_many_short_ones():
    """Items of one tile one after another, some of them empty."""
    rows = [(17 * i) % 23 + 20 if i % 7 else 0 for i in range(90)]
    run_attention(93, [(5 * i) % 40 for i in range(90)], rows, heads=8, kv=2, D=64, page=16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("where", ["k", "v"])
def test_attention_prompts_nan_reaches_only_the_rows_that_see_it(D, where):
    """NaN codes in several items' mixed tiles, of sequences one after another."""
    g, n = gen(94), 100
    past, bad = [36, 0, 200], [41, 63, 290]
    table, pages = page_tables(g, past, [n] * 3, 16)
    cache = fresh_cache(g, pages, 2, D, 16)
    clean = rd.KV8Cache(*[t.clone() for t in cache])
    for b in range(3):
        pid = int(table[b, bad[b] // 16])
        for c, code in ((cache, 0x7F), (clean, 0)):
            (c.k if where == "k" else c.v).view(torch.uint8)[pid, 1, bad[b] % 16, 3 + b] = code
    q = randn(g, 3 * n, 4, D)
    lengths, rs = i32(past), i32([0, n, 2 * n, 3 * n])
    got = rd.kv8_attention(q, cache, table, lengths, rs)
    want = rd.kv8_attention(q, clean, table, lengths, rs)
    check_attention(want, q, clean, table, lengths, rs)
    for b in range(3):
        first, rows = bad[b] - past[b], slice(b * n, (b + 1) * n)
        a, w = got[rows], want[rows]
        assert torch.equal(a[:, :2], w[:, :2])          # the other cache head's rows
        assert torch.equal(a[:first, 2:], w[:first, 2:])
        if where == "k":
            assert torch.isnan(a[first:, 2:]).all()
        else:
            assert torch.isnan(a[first:, 2:, 3 + b]).all()
            keep = [d for d in range(D) if d != 3 + b]
            assert torch.equal(a[:, :, keep], w[:, :, keep])


def test_attention_prompts_bad_pages_and_stale_contents():
    g, page = gen(95), 16
    past, rows = [50, 10], [80, 80]
    table, pages = page_tables(g, past, rows, page)
    cache = fresh_cache(g, pages, 2, 64, page)
    used = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    for b in range(2):
        for t in range(past[b] + rows[b]):
            used[int(table[b, t // page]), t % page] = True
    for c in (cache.k, cache.v):
        c.view(torch.uint8).copy_(torch.where(used[:, None, :, None], c.view(torch.uint8), 0x7F))
    q = randn(g, 160, 4, 64)
    lengths, rs = i32(past), i32([0, 80, 160])
    check_attention(rd.kv8_attention(q, cache, table, lengths, rs), q, cache, table, lengths, rs)
    bad = table.clone()
    bad[1, :] = -5
    got = rd.kv8_attention(q, cache, bad, lengths, rs)
    assert rd.device_error() == _lib.ERR_KV_RANGE
    check_attention(got, q, cache, table, lengths, rs, rows=slice(0, 80))
    assert torch.all(got[80:] == 0)


def test_attention_prompts_agree_with_single_rows():
    """The same rows as one chunk and one at a time, on the two kernels."""
    g = gen(96)
    past, n = 77, 70
    table, pages = page_tables(g, [past], [n], 32)
    cache = fresh_cache(g, pages, 2, 128, 32)
    q = randn(g, n, 8, 128)
    many = rd.kv8_attention(q, cache, table, i32([past]), i32([0, n]))
    for i in (0, 1, 50, n - 1):
        one = rd.kv8_attention(q[i:i + 1], cache, table, i32([past + i]), i32([0, 1]))
        check_attention(many[i:i + 1], q[i:i + 1], cache, table, i32([past + i]), i32([0, 1]))
        check_attention(one, q[i:i + 1], cache, table, i32([past + i]), i32([0, 1]))


@pytest.mark.parametrize("D,page,most", [(128, 64, 30), (64, 16, 17), (128, 16, 3)])
def test_append_hundreds_of_sequences(D, page, most):
    """Sequences beyond one scan step (128), without rows, with a few and with many."""
    past = [(37 * i) % 150 for i in range(301)]
    rows = [(11 * i) % (most + 1) if i % 5 else 0 for i in range(301)]
    run_append(D + most, past, rows, kv=2, heads=2, D=D, page=page, lead=1, pad=2)


@pytest.mark.parametrize("seqs", [33, 128, 129, 300])
@pytest.mark.parametrize("rows", [1, 24])
def test_attention_hundreds_of_sequences(seqs, rows):
    """Shares found four sequences a lane, in one step and in several."""
    past = [(131 * i) % 500 for i in range(seqs)]
    new = [rows - i % 2 if i % 6 else 0 for i in range(seqs)]
    run_attention(seqs + rows, past, new, heads=8, kv=2, D=64, page=16, lead=1, pad=2)


def test_outputs_whose_rows_overlap_are_refused():
    q = torch.zeros(3, 4, 128, device=DEV, dtype=torch.bfloat16)
    for strides in ((128, 128, 1), (256, 128, 1), (128, 256, 1)):
        out = torch.zeros(2048, device=DEV, dtype=torch.bfloat16).as_strided((3, 4, 128), strides)
        with pytest.raises(ValueError, match="overlap"):
            rd.qk_norm_rope(q, q, q_out=out)
    for strides in ((512, 128, 1), (1024, 136, 1), (128, 384, 1)):
        out = torch.zeros(4096, device=DEV, dtype=torch.bfloat16).as_strided((3, 4, 128), strides)
        rd.qk_norm_rope(q, q, q_out=out)


def test_prompts_on_two_streams_and_in_graphs_follow_lengths_and_rows():
    """Captured prompt steps replayed side by side, with items that are cut and that are not."""
    g, page = gen(31), 64
    sides = []
    for i in range(2):
        table, pages = page_tables(g, [6000, 900, 300], [0] * 3, page)
        x = dict(cache=fresh_cache(g, pages, 4, 128, page), table=table, q=randn(g, 300, 8, 128),
                 lengths=i32([0, 0, 0]), rs=i32([0, 0, 0, 0]), stream=torch.cuda.Stream())
        sides.append(x)
    torch.cuda.synchronize()
    for x in sides:
        x["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(x["graph"], stream=x["stream"]):
            x["out"] = rd.kv8_attention(x["q"], x["cache"], x["table"], x["lengths"], x["rs"])
    steps = [([5700, 10, 0], [0, 300, 300, 300]), ([0, 800, 3], [0, 0, 90, 300]),
             ([100, 64, 127], [5, 105, 205, 290]), ([5999, 899, 299], [0, 1, 2, 3]),
             ([4000, 500, 0], [0, 128, 250, 300])]
    for past, rs in steps:
        for x in sides:
            x["lengths"].copy_(i32(past))
            x["rs"].copy_(i32(rs))
            x["out"].fill_(9.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for x in sides:
                with torch.cuda.stream(x["stream"]):
                    x["graph"].replay()
        torch.cuda.synchronize()
        for x in sides:
            check_attention(x["out"], x["q"], x["cache"], x["table"], x["lengths"], x["rs"])
            assert torch.all(x["out"][:rs[0]] == 9.0) and torch.all(x["out"][rs[-1]:] == 9.0)
            eager = rd.kv8_attention(x["q"], x["cache"], x["table"], x["lengths"], x["rs"])
            assert torch.equal(eager[rs[0]:rs[-1]], x["out"][rs[0]:rs[-1]])
    assert rd.device_error() == 0


@pytest.mark.parametrize("past,rows", [(3000, 64), (4096, 256), (0, 40), (15000, 20)])
def test_attention_into_its_own_queries(past, rows):
    """The output over the queries: an item's are read before any of its rows is written."""
    g = gen(past + rows)
    table, pages = page_tables(g, [past], [rows], 64)
    cache = fresh_cache(g, pages, 2, 128, 64)
    q = randn(g, rows, 8, 128)
    lengths, rs = i32([past]), i32([0, rows])
    want = rd.kv8_attention(q, cache, table, lengths, rs)
    got = rd.kv8_attention(q, cache, table, lengths, rs, out=q)
    assert got is q and torch.equal(got, want)
    for n in (1, 3):
        q = randn(g, n, 8, 128)
        rs = i32([0, n])
        want = rd.kv8_attention(q, cache, table, lengths, rs)
        assert torch.equal(rd.kv8_attention(q, cache, table, lengths, rs, out=q), want)
