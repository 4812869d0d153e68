"""w4_gemm_fused on the GPU: bias, activation, gated pair and residual in the GEMM's epilogue.

Against a float64 restatement (oracle/kv8_oracle.py gemm) over the 16-bit weights
that the kernel multiplies (dequantize_v1 in x's type). Bars, derived before the
first run: each 16-wide step of the tensor cores adds to the fp32 accumulator
with an error of at most 2^-22 of the largest magnitude on the way, below
sum |x w| (+ |bias|), so K / 16 * 2^-22 * sum |x w| in all; the activations'
slopes are at most 1.13 (silu 1.10), a gated product adds the two sides'
errors each times the other side (the gate's first times 1.10); exp, erfc,
division and products are good to 2^-20; one rounding, half of the result's
epsilon (2^-25 absolute below fp16's normal range).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

import roofline_decoding_b200 as rd  # noqa: E402
from oracle import kv8_oracle as o  # noqa: E402

DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16, mul=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * mul).to(dtype)


def weights(g, K, N):
    return rd.pack_weights((torch.randn((K, N), generator=g, device=DEV) * K ** -0.5).half())


def check_gemm(got, x, packed_scales, bias=None, activation=None, residual=None):
    w = rd.dequantize_v1(*packed_scales, out_dtype=x.dtype)
    want = o.gemm(x, w, bias, activation, residual)
    K = x.shape[1]
    acc = K / 16 * 2.0 ** -22 * (x.double().abs() @ w.double().abs())
    y = o.gemm(x, w, bias)
    if activation == "swiglu":
        halves = [t.view(t.shape[0], -1, 2, 32) for t in (acc, y)]
        (eg, eu), (yg, yu) = [(t[:, :, 0].flatten(1), t[:, :, 1].flatten(1)) for t in halves]
        err = 1.1 * eg * (yu.abs() + eu) + eu * yg.abs() + 2.0 ** -20 * (yg * yu).abs()
    else:
        err = 1.13 * acc + 2.0 ** -20 * y.abs()
    if residual is not None:
        err = err + 2.0 ** -23 * residual.double().abs()
    tol = err + torch.finfo(got.dtype).eps / 2 * (want.abs() + err) + 2.0 ** -25
    assert got.shape == want.shape
    bad = (got.double() - want).abs() / tol
    assert not (bad > 1).any() and not torch.isnan(bad).any(), bad.max().item()


def run(M, K, N, dtype, bias, activation, residual, split_k=None, seed=0, in_place=False):
    g = gen(seed + M + N)
    w = weights(g, K, N)
    x = randn(g, M, K, dtype=dtype)
    wide = N // 2 if activation == "swiglu" else N
    b = randn(g, N, dtype=dtype, mul=0.5) if bias else None
    r = randn(g, M, wide, dtype=dtype) if residual else None
    was = r.clone() if residual else None
    y = rd.w4_gemm_fused(x, *w, bias=b, activation=activation, residual=r, split_k=split_k,
                         out=r if in_place else None)
    check_gemm(y, x, w, b, activation, was)
    assert rd.device_error() == 0
    return x, w, b, was, y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "swiglu"])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (True, True), (False, False)])
@pytest.mark.parametrize("M,K,N", [(1, 128, 128), (17, 256, 384), (130, 512, 256), (300, 384, 640)])
def test_epilogues(M, K, N, dtype, activation, bias, residual):
    run(M, K, N, dtype, bias, activation, residual)


@pytest.mark.parametrize("activation", [None, "gelu", "swiglu"])
@pytest.mark.parametrize("M,K,N,split_k", [
    (40, 512, 384, 1), (40, 512, 384, 3), (200, 1024, 640, 8), (128, 128, 256, 2),  # K slices
    (17, 1536, 2048, None), (128, 2304, 256, None), (511, 8960, 1536, None),  # few tiles: slices
    (140, 384, 128, None), (33, 256, 1152, None),
    (4000, 256, 2432, None),  # 256-column tiles, the last one half filled
    (2048, 1024, 5120, None),  # 160 of them: the last wave's tiles run as K slices
    (600, 2048, 1536, None)])
def test_tiles_and_slices(M, K, N, split_k, activation):
    run(M, K, N, torch.bfloat16, True, activation, True, split_k=split_k)


def test_residual_in_place_and_shared_rows():
    run(77, 256, 384, torch.float16, True, None, True, in_place=True)
    run(77, 256, 384, torch.bfloat16, False, "swiglu", True, in_place=True)
    run(2048, 1024, 5120, torch.bfloat16, True, None, True, in_place=True)


def test_no_epilogue_is_w4_gemm_bit_for_bit():
    """Where both cut K alike: one slice, and grids that fill the SMs."""
    for M, K, N, split_k in ((50, 256, 384, 1), (2048, 1024, 5120, None)):
        x, w, _, _, y = run(M, K, N, torch.float16, False, None, False, split_k=split_k)
        assert torch.equal(y, rd.w4_gemm(x, *w))


def test_other_types_shapes_and_orders():
    g = gen(9)
    w = weights(g, 256, 384)
    x = randn(g, 3, 20, 256, dtype=torch.float16)
    b, r = randn(g, 384, dtype=torch.bfloat16), randn(g, 3, 20, 384, dtype=torch.bfloat16)
    y = rd.w4_gemm_fused(x, *w, bias=b, residual=r, out_dtype=torch.bfloat16)
    assert y.dtype == torch.bfloat16
    check_gemm(y, x.view(60, 256), w, b, None, r.view(60, 384))
    one = rd.w4_gemm_fused(x[0, 0], *w, bias=b, out_dtype=torch.bfloat16)
    assert one.shape == (384,)
    check_gemm(one[None], x[0, :1], w, b)
    # a residual and a bias off alignment, a transposed x
    buf = randn(g, 60 * 384 + 1, dtype=torch.float16)
    odd_b = randn(g, 385, dtype=torch.float16)[1:]
    xt = randn(g, 256, 60, dtype=torch.float16).t()
    y = rd.w4_gemm_fused(xt, *w, bias=odd_b, residual=buf[1:].view(60, 384))
    check_gemm(y, xt, w, odd_b, None, buf[1:].view(60, 384))
    assert rd.w4_gemm_fused(xt[:0], *w).shape == (0, 384)


def test_activations_at_their_ends():
    """Large, small and non-finite sums: no overflow in between, NaN only where the maths has one."""
    g = gen(10)
    w = weights(g, 128, 128)
    x = torch.zeros((6, 128), device=DEV, dtype=torch.bfloat16)
    ends = torch.tensor([0.0, 1e4, -1e4, 3e38, -3e38, float("nan")], device=DEV)
    for act in ("silu", "gelu", "swiglu"):
        wide = 64 if act == "swiglu" else 128
        for e in ends.tolist():
            b = torch.full((128,), e, device=DEV, dtype=torch.bfloat16)
            if act == "swiglu":
                b.view(2, 2, 32)[:, 1] = 1.0
            y = rd.w4_gemm_fused(x, *w, bias=b, activation=act).double()
            want = o.gemm(x, torch.zeros((128, 128), device=DEV), b, act)
            assert y.shape == (6, wide)
            if e != e:
                assert torch.isnan(y).all()
            else:
                assert torch.all((y - want).abs() <= want.abs() * 2.0 ** -8)


def test_rows_behind_the_last_are_untouched_and_streams_and_graphs():
    g = gen(11)
    w = weights(g, 512, 256)
    x, r = randn(g, 130, 512), randn(g, 130, 256)
    out = torch.full((131, 256), 7.0, device=DEV, dtype=torch.bfloat16)
    want = rd.w4_gemm_fused(x, *w, activation="silu", residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rd.w4_gemm_fused(x, *w, activation="silu", residual=r, out=out[:130])
    s.synchronize()
    assert torch.equal(out[:130], want) and torch.all(out[130] == 7.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rd.w4_gemm_fused(x, *w, activation="silu", residual=r)
    x.copy_(randn(g, 130, 512))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, rd.w4_gemm_fused(x, *w, activation="silu", residual=r))


def test_inputs_written_just_before_are_seen():
    """x from a kernel that is still running when the call is made, in plans of one launch,
    of K slices and of two launches, and the result read by the next."""
    g = gen(12)
    for M, K, N in ((40, 512, 384), (300, 1024, 1152), (2048, 1024, 5120)):
        w = weights(g, K, N)
        xs = [randn(g, M, K) for _ in range(4)]
        want = [rd.w4_gemm_fused(x, *w, activation="silu") for x in xs]
        torch.cuda.synchronize()
        buf = torch.zeros((M, K), device=DEV, dtype=torch.bfloat16)
        big = torch.randn(4096, 4096, device=DEV)
        got = []
        for x in xs * 3:
            torch.mm(big, big)  # keeps the stream behind the host
            buf.copy_(x)
            got.append(rd.w4_gemm_fused(buf, *w, activation="silu") + 0)
            buf.fill_(float("nan"))
        for i, y in enumerate(got):
            assert torch.equal(y, want[i % 4]), (M, K, N, i)
