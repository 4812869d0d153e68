"""Cases of the operators that a decoder layer needs for more than one row at a time.

  gemm       y = residual + act(x @ W4 + bias), or the gated silu(g) * u of interleaved gate and up columns
  norm_rope  RMS norm of every query and key head and its rotation, in one pass
  append     keys (normed, rotated) and values into a paged 8-bit cache, queries normed and rotated beside them
  attention  queries against that cache, grouped heads, ragged rows, causal

`listed()` and `draw()` give cases, `prepare()` their inputs, `run()` one pass,
in elementary torch operations or, with `own`, by the package's entry points,
`exact()` the same outputs in 64 bits, and `work()` the bytes and operations
that a pass cannot do without.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
SCALE_EXP = (-32, 120)  # the block scales are powers of two in this range
EPS = 1e-6


def listed():
    return [
        # q|k|v of one decoding step just past the rows that the GEMV takes, with its bias
        dict(op="gemm", name="gemm bias 17x1536x2048", M=17, K=1536, N=2048, dtype="bf16", bias=True, act="", residual=False),
        # the down projection of a prompt of odd length, the residual stream added
        dict(op="gemm", name="gemm residual 511x8960x1536", M=511, K=8960, N=1536, dtype="fp16", bias=False, act="", residual=True),
        # gate and up of a long prompt, the gated activation in the epilogue
        dict(op="gemm", name="gemm swiglu 2048x4096x14336", M=2048, K=4096, N=14336, dtype="bf16", bias=False, act="swiglu", residual=False),
        # one step of eight sequences, the smallest call
        dict(op="norm_rope", name="norm_rope 8 rows 12/2", rows=8, heads=12, kv_heads=2, head_dim=128, dtype="bf16", table="bf16", norm=True, max_pos=2048),
        # a long prompt of a grouped-head model
        dict(op="norm_rope", name="norm_rope 8191 rows 32/8", rows=8191, heads=32, kv_heads=8, head_dim=128, dtype="bf16", table="fp32", norm=True, max_pos=32768),
        # one new token for each of 64 running sequences
        dict(op="append", name="append 64x1 32/8", seqs=64, rows=1, heads=32, kv_heads=8, head_dim=128, page=64, past=4096, dtype="bf16", table="fp32", norm=True),
        # drafted tokens of a few sequences, short pages, 64-wide heads
        dict(op="append", name="append 5x7 16/16 d64", seqs=5, rows=7, heads=16, kv_heads=16, head_dim=64, page=16, past=300, dtype="fp16", table="fp16", norm=False),
        # prompts written in one go
        dict(op="append", name="append 3x4001 12/2", seqs=3, rows=4001, heads=12, kv_heads=2, head_dim=128, page=64, past=0, dtype="bf16", table="bf16", norm=False),
        # one sequence, one token: the smallest step, latency counts
        dict(op="attention", name="attention 1x1 over 700 12/2", seqs=1, rows=1, heads=12, kv_heads=2, head_dim=128, page=64, past=700, dtype="bf16"),
        # a batch of ragged sequences with three drafted tokens each, 64-wide heads
        dict(op="attention", name="attention 16x3 over 2000 16/4 d64", seqs=16, rows=3, heads=16, kv_heads=4, head_dim=64, page=16, past=2000, dtype="fp16"),
        # a chunk of a prompt over what the cache holds already
        dict(op="attention", name="attention 2x256 over 4096 32/8", seqs=2, rows=256, heads=32, kv_heads=8, head_dim=128, page=64, past=4096, dtype="bf16"),
        # a serving batch of long ragged contexts: the cache is what a step reads
        dict(op="attention", name="attention 32x1 over 32768 32/8", seqs=32, rows=1, heads=32, kv_heads=8, head_dim=128, page=64, past=32768, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "norm_rope", "append", "attention"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "gemm":
        act = rng.choice(["", "silu", "gelu", "swiglu"])
        M, K, N = _log(rng, 1, 2048), 128 * _log(rng, 1, 70), 128 * _log(rng, 1, 112)
        if M * K * N > 2048 * 4096 * 14336:
            M = max(1, 2048 * 4096 * 14336 // (K * N))
        return dict(op=op, M=M, K=K, N=N, dtype=dtype, bias=rng.random() < 0.5, act=act, residual=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 8, 16] if kv_heads < 4 else [1, 2, 4, 5])
    head_dim = rng.choice([64, 128])
    if op == "norm_rope":
        return dict(op=op, rows=_log(rng, 1, 8191), heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                    table=rng.choice([dtype, "fp32"]), norm=rng.random() < 0.7, max_pos=_log(rng, 512, 32768))
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        seqs = _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, rows=min(_log(rng, 1, 4001), 12000 // seqs), heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    past=rng.choice([0, _log(rng, 1, 4096)]), dtype=dtype, table=rng.choice([dtype, "fp32"]), norm=rng.random() < 0.5)
    rows = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 16, 256)])
    past = _log(rng, 1, 32768) if rows <= 8 else _log(rng, 1, 4096)
    seqs = _log(rng, 1, 32) if rows <= 8 else rng.randint(1, 2)
    return dict(op=op, seqs=seqs, rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, past=past, dtype=dtype)


# ------------------------------------------------------------------ inputs


def _ragged(n, most, least):
    """n whole numbers spread over least..most, the first one the largest."""
    return [most if i == 0 else least + int((most - least) * ((0.35 + 0.6180339887 * i) % 1.0)) for i in range(n)]


def _layout(case):
    """New rows of each sequence, and the tokens that it holds before them."""
    rows = [case["rows"]] * case["seqs"] if case["rows"] <= 8 else _ragged(case["seqs"], case["rows"], 1)
    past = _ragged(case["seqs"], case["past"], 0)
    return rows, past


def _tables(max_pos, head_dim, table):
    inv = 1e6 ** (-torch.arange(0, head_dim, 2, device="cuda", dtype=torch.float64) / head_dim)
    angle = torch.outer(torch.arange(max_pos, device="cuda", dtype=torch.float64), inv)
    angle = torch.cat([angle, angle], -1)
    return angle.cos().to(DTYPES[table]), angle.sin().to(DTYPES[table])


def _cache(case, pages, gen):
    """A page pool in use: 8-bit codes, and a power-of-two scale for each page and head."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])

    def codes():
        return (torch.randn(shape, generator=gen, device="cuda") * 100).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)

    def scales():
        return torch.exp2(torch.randint(-8, -5, shape[:2], generator=gen, device="cuda").float())

    return codes(), codes(), scales(), scales()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, mul=1.0, add=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * mul + add).to(dtype)

    s = dict(case)
    if case["op"] == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        wide = N // 2 if case["act"] == "swiglu" else N
        s["x"] = randn(M, K)
        s["packed"] = torch.randint(-(1 << 31), 1 << 31, (K // 8, N), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        s["scales"] = ((0.5 + torch.rand((K // 128, N), generator=gen, device="cuda")) * 0.004).half()
        s["bias_t"] = randn(N, mul=0.5) if case["bias"] else None
        s["residual_t"] = randn(M, wide) if case["residual"] else None
        return s
    H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "norm_rope":
        T = case["rows"]
        s["positions"] = torch.randint(0, case["max_pos"], (T,), generator=gen, device="cuda")
        s["cos"], s["sin"] = _tables(case["max_pos"], D, case["table"])
    else:
        rows, past = _layout(case)
        T = sum(rows)
        need = [-(-(r + p) // case["page"]) for r, p in zip(rows, past)]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
        at = first[:, None] + torch.arange(max(need), device="cuda")[None]
        s["page_table"] = order[at.clamp_(max=pages - 1)].contiguous()
        s["lengths"] = torch.tensor(past, device="cuda", dtype=torch.int32)
        s["row_starts"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], device="cuda", dtype=torch.int32)
        s["k"], s["v"], s["k_scale"], s["v_scale"] = _cache(case, pages, gen)
        if case["op"] == "attention":
            s["q"] = randn(T, H, D)
            return s
        s["cos"], s["sin"] = _tables(max(r + p for r, p in zip(rows, past)), D, case["table"])
    # the rows as the q|k|v projection leaves them: one buffer, the heads side by side
    qkv = randn(T, (H + 2 * KV) * D, mul=1.5).view(T, H + 2 * KV, D)
    s["q"], s["new_k"], s["new_v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    s["q_norm"] = randn(D, mul=0.1, add=1.0) if case["norm"] else None
    s["k_norm"] = randn(D, mul=0.1, add=1.0) if case["norm"] else None
    return s


# ------------------------------------------------------------------ plain forms


def _plain_gemm(s):
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    q = (s["packed"][:, None, :] >> shifts[None, :, None]) & 15
    w = (q - 8).reshape(-1, s["N"]).float() * s["scales"].float().repeat_interleave(128, 0)
    y = s["x"].float() @ w.to(s["x"].dtype).float()
    if s["bias_t"] is not None:
        y = y + s["bias_t"].float()
    if s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif s["act"] == "swiglu":  # gate and up columns alternate in blocks of 32
        y = y.view(s["M"], s["N"] // 64, 2, 32)
        g, u = y[:, :, 0].reshape(s["M"], -1), y[:, :, 1].reshape(s["M"], -1)
        y = g / (1 + torch.exp(-g)) * u
    if s["residual_t"] is not None:
        y = y + s["residual_t"].float()
    return y.to(s["x"].dtype)


def _norm_rope(x, weight, cos, sin):
    """x [T, heads, D] in 32 bits: normed where there is a weight, then rotated."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos.float()[:, None] + turned * sin.float()[:, None]


def _plain_norm_rope(s):
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    return [_norm_rope(s["q"], s["q_norm"], cos, sin).to(s["q"].dtype), _norm_rope(s["new_k"], s["k_norm"], cos, sin).to(s["q"].dtype)]


def _rows(s):
    """Sequence and position of every new row."""
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["row_starts"][1:].long(), row, right=True)
    return seq, s["lengths"].long()[seq] + row - s["row_starts"].long()[seq]


def _power_of_two(amax):
    """The smallest power of two that amax / 448 does not exceed; 448 is 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    return torch.exp2(torch.where(m > 0.875, e - 8, e - 9).clamp(*SCALE_EXP).float())


def _store(new, codes, scale, s, page, slot):
    """New rows [T, heads, D] into the pages; what a page holds already keeps a scale that fits it too."""
    pages, P = codes.shape[0], codes.shape[2]
    flat, bits = scale, codes.view(torch.uint8)
    amax = torch.zeros_like(flat).index_reduce_(0, page, new.abs().amax(-1), "amax")
    # the page that a sequence goes on with: its rows in use are rounded again where its scale grows
    past = s["lengths"].long()
    used = past % P
    last = s["page_table"].long().gather(1, (past // P).clamp(max=s["page_table"].shape[1] - 1)[:, None])[:, 0]
    old = flat[last]
    goes_on = (used > 0) & (s["row_starts"][1:] > s["row_starts"][:-1])
    want = torch.where(goes_on[:, None], torch.maximum(old, _power_of_two(amax[last])), _power_of_two(amax[last]))
    held = codes[last].float() * (old / want)[:, :, None, None]
    keep = (torch.arange(P, device="cuda")[None] < used[:, None]) & goes_on[:, None]
    bits[last] = torch.where(keep[:, None, :, None], held.to(codes.dtype).view(torch.uint8), bits[last])
    flat[page] = _power_of_two(amax[page])
    flat[last] = torch.where((s["row_starts"][1:] > s["row_starts"][:-1])[:, None], want, flat[last])
    bits[page, :, slot] = (new / flat[page][:, :, None]).to(codes.dtype).view(torch.uint8)


def _plain_append(s):
    seq, pos = _rows(s)
    P = s["page"]
    page, slot = s["page_table"].long()[seq, pos // P], pos % P
    cos, sin = s["cos"][pos], s["sin"][pos]
    _store(_norm_rope(s["new_k"], s["k_norm"], cos, sin), s["k"], s["k_scale"], s, page, slot)
    _store(s["new_v"].float(), s["v"], s["v_scale"], s, page, slot)
    return [_norm_rope(s["q"], s["q_norm"], cos, sin).to(s["q"].dtype), s["k"], s["v"], s["k_scale"], s["v_scale"]]


def _plain_attention(s):
    B, KV, D, T = s["seqs"], s["kv_heads"], s["head_dim"], s["q"].shape[0]
    seq, pos = _rows(s)
    within = torch.arange(T, device="cuda") - s["row_starts"].long()[seq]
    most = s["rows"]
    table = s["page_table"].long()

    def gathered(codes, scale):
        x = codes.view(torch.uint8)[table].view(codes.dtype).float() * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(B, KV, -1, D)

    k, v = gathered(s["k"], s["k_scale"]), gathered(s["v"], s["v_scale"])
    q = torch.zeros((B, most, s["heads"], D), device="cuda")
    q[seq, within] = s["q"].float()
    q = q.view(B, most, KV, -1, D).permute(0, 2, 3, 1, 4)  # [B, KV, G, rows, D]
    score = (q.reshape(B, KV, -1, D) @ k.transpose(-1, -2)).view(*q.shape[:4], -1) / math.sqrt(D)
    last = s["lengths"].long()[:, None] + torch.arange(most, device="cuda")[None]
    hidden = torch.arange(k.shape[2], device="cuda") > last[..., None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True))
    score /= score.sum(-1, keepdim=True)
    o = (score.view(B, KV, -1, k.shape[2]) @ v).view(q.shape)
    return o.permute(0, 3, 1, 2, 4).reshape(B, most, s["heads"], D)[seq, within].to(s["q"].dtype)


def run(s):
    if own:
        import roofline_decoding_b200 as rd

        if s["op"] == "gemm":
            return rd.w4_gemm_fused(s["x"], s["packed"], s["scales"], bias=s["bias_t"], activation=s["act"] or None, residual=s["residual_t"])
        if s["op"] == "norm_rope":
            return list(rd.qk_norm_rope(s["q"], s["new_k"], s["cos"], s["sin"], s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS))
        cache = rd.KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if s["op"] == "append":
            q = rd.kv8_append(cache, s["new_k"], s["new_v"], s["page_table"], s["lengths"], s["row_starts"], cos=s["cos"], sin=s["sin"],
                              q=s["q"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
            return [q, s["k"], s["v"], s["k_scale"], s["v_scale"]]
        return rd.kv8_attention(s["q"], cache, s["page_table"], s["lengths"], s["row_starts"])
    return {"gemm": _plain_gemm, "norm_rope": _plain_norm_rope, "append": _plain_append, "attention": _plain_attention}[s["op"]](s)


# ------------------------------------------------------------------ 64 bits


def _exact_gemm(case, s):
    x, N = s["x"].double(), case["N"]
    y = torch.empty((case["M"], N), dtype=torch.float64, device="cuda")
    for n in range(0, N, 2048):
        p = s["packed"][:, n:n + 2048].long() & 0xFFFFFFFF
        q = torch.stack([(p >> (4 * i)) % 16 for i in range(8)], 1).reshape(case["K"], -1)
        scale = s["scales"][:, n:n + 2048].double()
        w = (q - 8).double().view(-1, 128, q.shape[1]) * scale[:, None]
        y[:, n:n + 2048] = x @ w.view(case["K"], -1).to(s["x"].dtype).double()
    if case["bias"]:
        y += s["bias_t"].double()
    if case["act"] == "silu":
        y = y * torch.special.expit(y)
    elif case["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    elif case["act"] == "swiglu":
        gate = [c + i for c in range(0, N, 64) for i in range(32)]
        g, u = y[:, gate], y[:, [c + 32 for c in gate]]
        y = g * torch.special.expit(g) * u
    return y + s["residual_t"].double() if case["residual"] else y


def _exact_rows(x, weight, cos, sin):
    """Each pair (x_d, x_{d + D/2}) as a complex number, scaled to a root mean square of one and turned."""
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    if weight is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos[..., :h] - b * sin[..., :h], b * cos[..., h:] + a * sin[..., h:]], -1)


def _least_power(amax):
    e = SCALE_EXP[0]
    while e < SCALE_EXP[1] and amax > math.ldexp(E4M3_MAX, e):
        e += 1
    return math.ldexp(1.0, e)


def _exact_append(case, s):
    """The pages' values in units of their scale, before they are rounded to 8 bits."""
    rows, past = _layout(case)
    P, table = case["page"], s["page_table"].tolist()
    spots = [(table[b][(past[b] + i) // P], (past[b] + i) % P, past[b] + i) for b in range(case["seqs"]) for i in range(rows[b])]
    page, slot, pos = (torch.tensor(c, device="cuda") for c in zip(*spots))
    cos, sin = s["cos"][pos], s["sin"][pos]
    outs = []
    for new, codes, scale in ((_exact_rows(s["new_k"], s["k_norm"], cos, sin), s["k"], s["k_scale"]), (s["new_v"].double(), s["v"], s["v_scale"])):
        value, scale, start = codes.double(), scale.double().clone(), 0
        for b in range(case["seqs"]):
            mine, start = new[start:start + rows[b]], start + rows[b]
            for p in range(past[b] // P, (past[b] + rows[b] - 1) // P + 1):
                lo, hi = max(p * P, past[b]), min(p * P + P, past[b] + rows[b])
                block, at = mine[lo - past[b]:hi - past[b]], table[b][p]
                want = torch.tensor([_least_power(a) for a in block.abs().amax((0, 2)).tolist()], device="cuda", dtype=torch.float64)
                if lo > p * P:
                    want = torch.maximum(want, scale[at])
                    value[at, :, :lo - p * P] *= (scale[at] / want)[:, None, None]
                scale[at] = want
                value[at, :, lo - p * P:hi - p * P] = block.transpose(0, 1) / want[:, None, None]
        outs.append((value, scale))
    return [_exact_rows(s["q"], s["q_norm"], cos, sin), outs[0][0], outs[1][0], outs[0][1], outs[1][1]]


def _exact_attention(case, s):
    rows, past = _layout(case)
    KV, D, out, start = case["kv_heads"], case["head_dim"], [], 0
    for b in range(case["seqs"]):
        n = past[b] + rows[b]
        pages = s["page_table"][b, :-(-n // case["page"])].long()
        k, v = (c.view(torch.uint8)[pages].view(c.dtype).double() * f[pages].double()[:, :, None, None] for c, f in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        k, v = (x.permute(1, 0, 2, 3).reshape(KV, -1, D)[:, :n] for x in (k, v))
        q = s["q"][start:start + rows[b]].double().view(rows[b], KV, -1, D)
        seen = torch.arange(n, device="cuda")[None] <= past[b] + torch.arange(rows[b], device="cuda")[:, None]
        o = torch.empty_like(q)
        for g in range(q.shape[2]):
            score = (q[:, :, g].transpose(0, 1) @ k.transpose(1, 2)) * D ** -0.5
            o[:, :, g] = (torch.softmax(score.masked_fill(~seen[None], -math.inf), -1) @ v).transpose(0, 1)
        out.append(o.reshape(rows[b], -1, D))
        start += rows[b]
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        return _exact_gemm(case, s)
    if case["op"] == "norm_rope":
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return [_exact_rows(s["q"], s["q_norm"], cos, sin), _exact_rows(s["new_k"], s["k_norm"], cos, sin)]
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["op"] == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        wide = N // 2 if case["act"] == "swiglu" else N
        moved = K * N // 2 + K // 128 * N * 2 + 2 * M * K + 2 * M * wide * (2 if case["residual"] else 1) + 2 * N * case["bias"]
        return {"bytes": moved, "flops": 2 * M * K * N}
    H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
    width = 4 if case.get("table") == "fp32" else 2
    if case["op"] == "norm_rope":
        T = case["rows"]
        table = min(T, case["max_pos"]) * 2 * D * width
        return {"bytes": T * (H + KV) * D * 4 + T * 8 + table + 4 * D * case["norm"], "flops": T * (H + KV) * D * (3 + 3 * case["norm"])}
    rows, past = _layout(case)
    T = sum(rows)
    if case["op"] == "append":
        table = min(T, max(r + p for r, p in zip(rows, past))) * 2 * D * width
        blocks = sum((r + p - 1) // case["page"] - p // case["page"] + 1 for r, p in zip(rows, past))
        moved = T * H * D * 4 + T * KV * 2 * D * 3 + table + blocks * (4 + KV * 8) + 8 * case["seqs"] + 4 * D * case["norm"]
        return {"bytes": moved, "flops": T * ((H + KV) * D * (3 + 3 * case["norm"]) + KV * 2 * D * 2)}
    keys = [r + p for r, p in zip(rows, past)]
    blocks = sum(-(-n // case["page"]) for n in keys)
    pairs = sum(r * p + r * (r + 1) // 2 for r, p in zip(rows, past))
    return {"bytes": sum(keys) * KV * 2 * D + blocks * (4 + KV * 8) + T * H * D * 4 + 8 * case["seqs"], "flops": 4 * pairs * H * D}
