"""w4_gemm_fused at the borders of its contract: outputs over inputs, far gates, empty shapes.

Bars as in test_gemm_fused_gpu.py, unless a test says otherwise.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

import roofline_decoding_b200 as rd  # noqa: E402
from oracle import kv8_oracle as o  # noqa: E402
from test_gemm_fused_gpu import gen, randn, weights  # noqa: E402

DEV = "cuda"


def test_outputs_over_inputs_are_refused():
    g = gen(1)
    w = weights(g, 256, 256)
    bias = randn(g, 256)
    for M in (20, 300):
        buf = randn(g, 2 * M + 8, 256)
        x, was = buf[:M], buf.clone()
        r = randn(g, M + 8, 256)
        bad = [dict(out=x), dict(out=x, residual=x), dict(out=buf[8:M + 8]), dict(out=buf[M - 1:2 * M - 1]),
               dict(out=r[8:], residual=r[:M]), dict(out=r[:M], residual=r[1:M + 1])]
        for kw in bad:
            with pytest.raises(ValueError, match="overlap"):
                rd.w4_gemm_fused(x, *w, bias=bias, **kw)
        assert torch.equal(buf, was)
        # beside them
        want = rd.w4_gemm_fused(x, *w, bias=bias)
        got = rd.w4_gemm_fused(x, *w, bias=bias, out=buf[M:2 * M])
        assert torch.equal(got, want) and torch.equal(buf[:M], was[:M])
    # one row: over the bias, over the scales
    x, b1 = randn(g, 1, 256, dtype=torch.float16), randn(g, 256, dtype=torch.float16)
    with pytest.raises(ValueError, match="overlap"):
        rd.w4_gemm_fused(x, *w, bias=b1, out=b1[None])
    with pytest.raises(ValueError, match="overlap"):
        rd.w4_gemm_fused(x, *w, out=w[1][:1])
    with pytest.raises(ValueError, match="overlap"):
        rd.w4_gemm_fused(x, *w, out=w[0].view(torch.float16)[:1, :256])


@pytest.mark.parametrize("split_k", [1, 2])
@pytest.mark.parametrize("gate", [-80.0, -87.5, -88.0, -88.5, -90.0, -95.0])
def test_silu_of_gates_whose_exponential_is_out_of_range(gate, split_k):
    """silu(-88) is -5.3e-37, not zero: times a large up column it is a number of note.

    exp is good to 2^-17 at arguments this large (half a step of the argument in log2
    units, 2^-18), subnormal exponentials below -87.3 to 2^-149 of themselves.
    """
    g = gen(2)
    w = weights(g, 128, 128)
    x = torch.zeros((3, 128), device=DEV, dtype=torch.bfloat16)
    b = torch.full((128,), gate, device=DEV, dtype=torch.bfloat16)
    zero = torch.zeros((128, 128), device=DEV)
    for act in ("silu", "swiglu"):
        if act == "swiglu":
            b.view(2, 2, 32)[:, 1] = 1e30
        y = rd.w4_gemm_fused(x, *w, bias=b, activation=act, split_k=split_k).double()
        want = o.gemm(x, zero, b, act)
        up = 1e30 if act == "swiglu" else 1.0
        slack = 2.0 ** -149 * abs(gate) * up + (2.0 ** -133 if act == "silu" else 0.0)
        assert torch.all((y - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -16) + slack)


def test_weights_of_no_rows_or_columns_are_refused():
    """y of no K would be residual + act(bias), which no kernel of the library makes."""
    for K, N in ((0, 128), (128, 0)):
        packed = torch.zeros((K // 8, N), dtype=torch.int32, device=DEV)
        scales = torch.zeros((K // 128, N), dtype=torch.float16, device=DEV)
        for M in (0, 5):
            with pytest.raises(ValueError, match="packed must have K > 0"):
                rd.w4_gemm_fused(torch.zeros((M, K), dtype=torch.float16, device=DEV), packed, scales)
