"""Refusals of the batched attention operators and the GEMM epilogue, before any device work."""
import ctypes

import pytest
import torch

import roofline_decoding_b200 as rd
from oracle import kv8_oracle as o
from roofline_decoding_b200 import _lib

FAKE = 1 << 20  # an aligned address that is never followed


def heads(n=4, ptr=FAKE, row=512, head=128):
    return _lib.Heads(ptr, row, head, n)


def rope(**kw):
    r = _lib.Rope(FAKE, FAKE, _lib.W4_F32, 16, None, None, 1e-6)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def cache(**kw):
    c = _lib.Kv8CacheDesc(FAKE, FAKE, FAKE, FAKE, 10, 2, 64, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    b = _lib.KvBatch(FAKE, 8, 8, FAKE, FAKE, 3, 5)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


BAD_HEADS = [(heads(ptr=None), 1), (heads(ptr=FAKE + 2), 2), (heads(row=508), 2), (heads(head=4), 2),
             (heads(head=64), 1), (heads(row=-512), 1), (heads(n=-1), 1), (heads(n=5000), 1)]
BAD_ROPE = [(rope(cos_table=None), 1), (rope(table_dtype=3), 1), (rope(max_pos=0), 1),
            (rope(cos_table=FAKE + 8), 2), (rope(q_norm=FAKE + 2), 2), (rope(k_norm=FAKE + 4), 2)]
BAD_CACHE = [(cache(k=None), 1), (cache(v_scale=None), 1), (cache(pages=0), 1), (cache(kv_heads=0), 1),
             (cache(page_size=48), 3), (cache(page_size=256), 3), (cache(head_dim=96), 3),
             (cache(v=FAKE + 8), 2)]
BAD_BATCH = [(batch(page_table=None), 1), (batch(lengths=None), 1), (batch(row_starts=None), 1),
             (batch(seqs=-1), 1), (batch(rows=-1), 1), (batch(rows=(1 << 24) + 1), 1),
             (batch(max_pages=0), 1), (batch(table_stride=-1), 1)]


def norm_rope(q=None, k=None, qo=None, ko=None, dtype=1, rows=5, D=128, r=None, pos=FAKE):
    return _lib.load().w4_qk_norm_rope(q or heads(), k or heads(2), qo or heads(), ko or heads(2),
                                       dtype, rows, D, r or rope(), pos, None)


def append(c=None, b=None, k=None, v=None, q=None, qo=None, dtype=1, r=None):
    return _lib.load().w4_kv8_append(c or cache(), b or batch(), k or heads(2), v or heads(2),
                                     q or heads(), qo or heads(), dtype, r or rope(), None)


def attention(c=None, b=None, q=None, out=None, dtype=1, ws=FAKE, size=1 << 30):
    return _lib.load().w4_kv8_attention(c or cache(), b or batch(), q or heads(), out or heads(),
                                        dtype, 0.1, ws, size, None)


def test_norm_rope_refusals():
    for bad, status in BAD_HEADS:
        assert norm_rope(q=bad) == status
        assert norm_rope(ko=bad) == status
    for bad, status in BAD_ROPE:
        assert norm_rope(r=bad) == status
    assert norm_rope(dtype=2) == _lib.W4_ERR_INVALID_ARG
    assert norm_rope(D=96) == _lib.W4_ERR_UNSUPPORTED
    assert norm_rope(D=256) == _lib.W4_ERR_UNSUPPORTED
    assert norm_rope(rows=-1) == _lib.W4_ERR_INVALID_ARG
    assert norm_rope(pos=None) == _lib.W4_ERR_INVALID_ARG
    assert norm_rope(qo=heads(3)) == _lib.W4_ERR_INVALID_ARG
    assert norm_rope(rows=0) == _lib.W4_OK  # nothing to do: no device is touched


def test_append_refusals():
    for bad, status in BAD_CACHE:
        assert append(c=bad) == status
    for bad, status in BAD_BATCH:
        assert append(b=bad) == status
    for bad, status in BAD_HEADS:
        assert append(k=bad) == status
        assert append(qo=bad) == status
    for bad, status in BAD_ROPE:
        assert append(r=bad) == status
    assert append(k=heads(3)) == _lib.W4_ERR_INVALID_ARG
    assert append(v=heads(1)) == _lib.W4_ERR_INVALID_ARG
    assert append(qo=heads(2)) == _lib.W4_ERR_INVALID_ARG
    assert append(dtype=2) == _lib.W4_ERR_INVALID_ARG
    assert append(b=batch(rows=0)) == _lib.W4_OK
    assert append(b=batch(seqs=0)) == _lib.W4_OK


def test_attention_refusals():
    for bad, status in BAD_CACHE:
        assert attention(c=bad) == status
    for bad, status in BAD_BATCH:
        assert attention(b=bad) == status
    for bad, status in BAD_HEADS:
        assert attention(q=bad, out=bad) == status
    assert attention(q=heads(0), out=heads(0)) == _lib.W4_ERR_INVALID_ARG
    assert attention(q=heads(3), out=heads(3)) == _lib.W4_ERR_INVALID_ARG   # 3 over 2
    assert attention(q=heads(34), out=heads(34)) == _lib.W4_ERR_INVALID_ARG  # 17 each
    assert attention(out=heads(2)) == _lib.W4_ERR_INVALID_ARG
    assert attention(dtype=2) == _lib.W4_ERR_INVALID_ARG
    need = _lib.load().w4_kv8_attention_workspace_bytes(128)
    assert attention(size=need - 1) == _lib.W4_ERR_INVALID_ARG
    assert attention(ws=None) == _lib.W4_ERR_INVALID_ARG
    assert attention(ws=FAKE + 8) == _lib.W4_ERR_ALIGNMENT
    assert attention(b=batch(rows=0)) == _lib.W4_OK


def test_gemm_epilogue_refusals():
    lib = _lib.load()

    def call(ops, M=17, K=256, N=128, x=FAKE, y_dtype=1, split_k=0):
        return lib.w4_gemm_fused(x, 1, FAKE, FAKE, FAKE, y_dtype, M, K, N, ops, split_k, None)

    ok = _lib.GemmOps(0, None, None)
    assert call(None) == _lib.W4_ERR_INVALID_ARG
    assert call(_lib.GemmOps(4, None, None)) == _lib.W4_ERR_INVALID_ARG
    assert call(_lib.GemmOps(-1, None, None)) == _lib.W4_ERR_INVALID_ARG
    assert call(_lib.GemmOps(0, FAKE + 2, None)) == _lib.W4_ERR_ALIGNMENT
    assert call(_lib.GemmOps(0, None, FAKE + 8)) == _lib.W4_ERR_ALIGNMENT
    assert call(ok, M=0) == _lib.W4_ERR_INVALID_ARG
    assert call(ok, K=100) == _lib.W4_ERR_INVALID_ARG
    assert call(ok, N=96) == _lib.W4_ERR_INVALID_ARG
    assert call(ok, x=FAKE + 2) == _lib.W4_ERR_ALIGNMENT
    assert call(ok, y_dtype=2) == _lib.W4_ERR_INVALID_ARG
    assert call(ok, split_k=9) == _lib.W4_ERR_INVALID_ARG


def test_python_refusals_without_a_gpu():
    q = torch.zeros((3, 4, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        rd.qk_norm_rope(q, q)
    c = rd.KV8Cache.empty(4, 2, device="cpu")
    assert c.k.shape == (4, 2, 64, 128) and c.k_scale.shape == (4, 2)
    table = torch.zeros((1, 2), dtype=torch.int32)
    lengths, rs = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        rd.kv8_attention(q, c, table, lengths, rs)
    with pytest.raises(ValueError, match="CUDA"):
        rd.kv8_append(c, q[:, :2], q[:, 2:], table, lengths, rs)
    for bad in (c._replace(v=c.v[:3]), c._replace(k_scale=c.k_scale[:, :1]), c._replace(k=c.k[0])):
        with pytest.raises(ValueError, match="cache"):
            rd.kv8_attention(q, bad, table, lengths, rs)
    with pytest.raises(ValueError, match="float8"):
        rd.kv8_attention(q, c._replace(k=c.k.view(torch.uint8)), table, lengths, rs)
    with pytest.raises(ValueError, match="contiguous"):
        rd.kv8_attention(q, c._replace(k=c.k.transpose(2, 3).contiguous().transpose(2, 3)), table,
                         lengths, rs)


def test_structures_have_the_headers_layout():
    assert ctypes.sizeof(_lib.Heads) == 32 and ctypes.sizeof(_lib.Rope) == 48
    assert ctypes.sizeof(_lib.Kv8CacheDesc) == 48 and ctypes.sizeof(_lib.KvBatch) == 48
    assert ctypes.sizeof(_lib.GemmOps) == 24


def test_the_oracles_scale_and_rounding():
    """The 64-bit restatement itself, on values with known answers."""
    assert o.least_scale(448.0) == 1.0 and o.least_scale(448.1) == 2.0
    assert o.least_scale(0.0) == 2.0 ** -32 and o.least_scale(7.0) == 2.0 ** -6
    x = torch.tensor([1.0, 1.0625, 1.1875, 500.0, -1e9, 2.0 ** -9, 2.0 ** -10, 0.0])
    want = [1.0, 1.0, 1.25, 448.0, -448.0, 2.0 ** -9, 0.0, 0.0]
    assert o.to_e4m3(x).float().tolist() == want
    rs = torch.tensor([1, 3, 3, 8], dtype=torch.int32)
    lengths = torch.tensor([15, 4, 0], dtype=torch.int32)
    table = torch.tensor([[3, 1], [0, 0], [2, 0]], dtype=torch.int32)
    assert o.sequences(lengths, rs) == [(0, 15, 1, 2), (2, 0, 3, 5)]
    assert list(o.blocks(lengths, rs, table, 16)) == [(3, 15, 1, 1), (1, 0, 2, 1), (2, 0, 3, 5)]
    assert o.positions(lengths, rs, 9).tolist() == [0, 15, 16, 0, 1, 2, 3, 4, 0]


def test_the_oracles_attention_is_softmax_attention():
    g = torch.Generator().manual_seed(0)
    codes = [o.to_e4m3(torch.randn((3, 2, 16, 64), generator=g) * 50) for _ in range(2)]
    scales = [torch.rand((3, 2), generator=g) * 0.02 for _ in range(2)]
    q = torch.randn((4, 4, 64), generator=g).bfloat16()
    out, size, _ = o.attention(q, (*codes, *scales), torch.tensor([[2, 0]], dtype=torch.int32),
                               torch.tensor([20], dtype=torch.int32),
                               torch.tensor([0, 4], dtype=torch.int32))
    k, v = (torch.cat([c[p].double() * s[p].double()[:, None, None] for p in (2, 0)], 1)
            for c, s in zip(codes, scales))
    for i in range(4):
        for h in range(4):
            kk, vv = k[h // 2, :21 + i], v[h // 2, :21 + i]
            w = torch.softmax(kk @ q[i, h].double() / 8, 0)
            assert torch.allclose(out[i, h], w @ vv, rtol=1e-12, atol=1e-14)
            assert torch.allclose(size[i, h], w @ vv.abs(), rtol=1e-12, atol=1e-14)
