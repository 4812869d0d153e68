"""w4_gemm_fused at the borders of its contract: outputs over inputs, far gates, empty shapes.

Bars as in test_gemm_fused_gpu.py, unless a test says otherwise.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

import roofline_decoding_b200 as rd  # noqa: E402
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
