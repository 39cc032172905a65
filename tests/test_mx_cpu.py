"""CPU tests of the expert selection and of the MXFP4 operators: what the C ABI and the Python binding refuse.  None of
these calls reaches a kernel launch."""
import ctypes

import pytest
import torch

A = 1 << 24  # an aligned address that no call here reads


@pytest.fixture(scope="module")
def g():
    import gptoss_moe
    return gptoss_moe


def refused(g, rc, status, text):
    assert rc == getattr(g, "GPTOSS_ERR_" + status)
    assert text in g.lib.gptoss_last_error(), g.lib.gptoss_last_error()


def select(g, cfg=None, **kw):
    c = dict(score=0, top_k=4, num_groups=1, top_groups=1, group_rank=2, renormalize=1, scale=1.0)
    c.update(cfg or {})
    a = dict(logits=A, stride=128, fp32=0, bias=None, T=7, E=128, idx=3 * A, w=4 * A)
    a.update(kw)
    r = g.RoutingConfig(*c.values())
    return g.lib.gptoss_moe_select_experts(a["logits"], a["stride"], a["fp32"], a["bias"], a["T"], a["E"],
                                           None if cfg is False else ctypes.byref(r), a["idx"], a["w"], None)


@pytest.mark.parametrize("cfg, kw, status, text", [
    (dict(score=2), {}, "INVALID", b"score"),
    (dict(top_k=0), {}, "INVALID", b"top_k"),
    (dict(top_k=33), {}, "INVALID", b"top_k"),
    (dict(top_k=5), dict(E=4), "INVALID", b"top_k"),
    (dict(top_k=17, num_groups=8), {}, "INVALID", b"top_k"),  # 16 experts in the one group that stays
    (dict(num_groups=0), {}, "INVALID", b"num_groups"),
    (dict(num_groups=3), {}, "INVALID", b"num_groups"),
    (dict(num_groups=128), {}, "INVALID", b"num_groups"),
    (dict(num_groups=4, top_groups=5), {}, "INVALID", b"top_groups"),
    (dict(top_groups=0), {}, "INVALID", b"top_groups"),
    (dict(group_rank=3), {}, "INVALID", b"group_rank"),
    (dict(group_rank=0), {}, "INVALID", b"group_rank"),
    (dict(scale=float("nan")), {}, "INVALID", b"scale"),
    (dict(scale=float("inf")), {}, "INVALID", b"scale"),
    ({}, dict(E=0), "UNSUPPORTED", b"num_experts"),
    ({}, dict(E=1025, stride=1025), "UNSUPPORTED", b"num_experts"),
    ({}, dict(T=-1), "INVALID", b"num_tokens"),
    ({}, dict(T=(1 << 26) + 1), "UNSUPPORTED", b"num_tokens"),
    ({}, dict(logits=None), "INVALID", b"null"),
    ({}, dict(idx=None), "INVALID", b"null"),
    ({}, dict(w=None), "INVALID", b"null"),
    ({}, dict(logits=A + 1), "INVALID", b"aligned"),
    ({}, dict(logits=A + 2, fp32=1), "INVALID", b"aligned"),
    ({}, dict(bias=A + 2), "INVALID", b"aligned"),
    ({}, dict(stride=127), "INVALID", b"apart"),
    ({}, dict(stride=1 << 62), "INVALID", b"apart"),
    ({}, dict(idx=A + 64), "INVALID", b"overlap"),
    ({}, dict(w=3 * A + 4), "INVALID", b"overlap"),
    ({}, dict(bias=4 * A), "INVALID", b"overlap"),
])
def test_select_refusals(g, cfg, kw, status, text):
    refused(g, select(g, cfg, **kw), status, text)


def test_select_without_a_config_or_tokens(g):
    refused(g, select(g, False), "INVALID", b"cfg")
    assert select(g, T=0, logits=None, idx=None, w=None) == g.GPTOSS_OK


def quantize(g, **kw):
    a = dict(x=A, stride=96, fp32=0, rows=5, K=96, packed=2 * A, scales=3 * A)
    a.update(kw)
    return g.lib.gptoss_mxfp4_quantize(*a.values(), None)


def dequantize(g, **kw):
    a = dict(packed=2 * A, scales=3 * A, rows=5, K=96, x=A, stride=96, fp32=0)
    a.update(kw)
    return g.lib.gptoss_mxfp4_dequantize(*a.values(), None)


@pytest.mark.parametrize("call", [quantize, dequantize])
@pytest.mark.parametrize("kw, status, text", [
    (dict(K=0), "INVALID", b"matrix of"),
    (dict(K=-32), "INVALID", b"matrix of"),
    (dict(K=100), "INVALID", b"multiple of the 32"),
    (dict(rows=-1), "INVALID", b"matrix of"),
    (dict(rows=(1 << 26) + 1), "UNSUPPORTED", b"at most"),
    (dict(K=(1 << 24) + 32), "UNSUPPORTED", b"at most"),
    (dict(x=None), "INVALID", b"null"),
    (dict(packed=None), "INVALID", b"null"),
    (dict(scales=None), "INVALID", b"null"),
    (dict(x=A + 8), "INVALID", b"aligned"),
    (dict(packed=2 * A + 8), "INVALID", b"aligned"),
    (dict(stride=64), "INVALID", b"apart"),
    (dict(stride=100), "INVALID", b"apart"),
    (dict(stride=98, fp32=1), "INVALID", b"apart"),
    (dict(stride=1 << 60), "INVALID", b"apart"),
    (dict(packed=A + 16), "INVALID", b"overlap"),
    (dict(scales=A + 5 * 96 * 2 - 1), "INVALID", b"overlap"),
])
def test_quantize_refusals(g, call, kw, status, text):
    refused(g, call(g, **kw), status, text)


def test_quantize_of_overlapping_results(g):
    refused(g, quantize(g, scales=2 * A + 5 * 48 - 1), "INVALID", b"overlap")


def test_no_rows(g):
    assert quantize(g, rows=0, x=None, packed=None, scales=None) == g.GPTOSS_OK
    assert dequantize(g, rows=0, x=None, packed=None, scales=None) == g.GPTOSS_OK


def product(g, grouped, res=None, **kw):
    r = dict(swiglu=0, alpha=1.702, limit=7.0, fp32=0, out=9 * A, stride=64, op=None, os=None)
    r.update(res or {})
    r = g.Mxfp4Result(*r.values())
    a = dict(a=A, asc=2 * A, a_rows=10, index=None, off=3 * A, E=4, rows=10, w=4 * A, ws=5 * A, bias=6 * A, N=64, K=96)
    a.update(kw)
    where = None if res is False else ctypes.byref(r)
    if grouped:
        return g.lib.gptoss_moe_grouped_mxfp4_matmul(*a.values(), where, None)
    return g.lib.gptoss_mxfp4_matmul(a["a"], a["asc"], a["a_rows"], a["w"], a["ws"], a["bias"], a["N"], a["K"], where, None)


QUANT = dict(out=None, op=9 * A, os=10 * A)


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("res, kw, status, text", [
    (None, dict(K=48), "INVALID", b"multiple of the 32"),
    (None, dict(K=0), "INVALID", b"matrix of"),
    (None, dict(N=0), "INVALID", b"N=0"),
    (None, dict(N=-1), "INVALID", b"matrix of"),
    (None, dict(N=(1 << 24) + 1), "INVALID", b"N="),
    (None, dict(a_rows=-1), "INVALID", b"matrix of"),
    (False, {}, "INVALID", b"result"),
    (dict(swiglu=1), dict(N=63), "INVALID", b"pairs"),
    (dict(swiglu=1, alpha=float("nan")), {}, "INVALID", b"alpha"),
    (dict(swiglu=1, limit=float("nan")), {}, "INVALID", b"limit"),
    (dict(swiglu=1, limit=-1.0), {}, "INVALID", b"limit"),
    (QUANT, dict(N=80), "INVALID", b"multiple of the 32"),
    (dict(QUANT, swiglu=1), dict(N=96), "INVALID", b"multiple of the 32"),
    (dict(QUANT, out=11 * A), {}, "INVALID", b"one of them"),
    (dict(QUANT, os=None), {}, "INVALID", b"null out_packed"),
    (dict(QUANT, op=None), {}, "INVALID", b"null out_packed"),
    (dict(QUANT, op=9 * A + 8), {}, "INVALID", b"aligned"),
    (dict(QUANT, os=9 * A), {}, "INVALID", b"overlaps out_scales"),
    (dict(QUANT, op=A + 16), {}, "INVALID", b"overlap an input"),
    (dict(QUANT, os=5 * A), {}, "INVALID", b"overlap an input"),
    (None, dict(a=None), "INVALID", b"null a"),
    (None, dict(asc=None), "INVALID", b"null a"),
    (None, dict(w=None), "INVALID", b"null w"),
    (None, dict(ws=None), "INVALID", b"null w"),
    (None, dict(a=A + 8), "INVALID", b"aligned"),
    (None, dict(w=4 * A + 4), "INVALID", b"aligned"),
    (None, dict(bias=6 * A + 1), "INVALID", b"aligned"),
    (dict(out=None), {}, "INVALID", b"null out"),
    (dict(out=9 * A + 1), {}, "INVALID", b"aligned"),
    (dict(out=9 * A + 2, fp32=1), {}, "INVALID", b"aligned"),
    (dict(stride=63), {}, "INVALID", b"apart"),
    (dict(stride=1 << 60), {}, "INVALID", b"apart"),
    (dict(out=A), {}, "INVALID", b"overlaps an input"),
    (dict(out=6 * A), {}, "INVALID", b"overlaps an input"),
])
def test_product_refusals(g, grouped, res, kw, status, text):
    refused(g, product(g, grouped, res, **kw), status, text)


@pytest.mark.parametrize("kw, status, text", [
    (dict(E=0), "UNSUPPORTED", b"num_experts"),
    (dict(E=1025), "UNSUPPORTED", b"num_experts"),
    (dict(rows=-1), "INVALID", b"rows"),
    (dict(rows=(1 << 26) + 1), "INVALID", b"rows"),
    (dict(rows=11), "INVALID", b"without row_index"),
    (dict(a_rows=0, index=7 * A), "INVALID", b"no rows"),
    (dict(off=None), "INVALID", b"expert_offsets"),
    (dict(off=3 * A + 2), "INVALID", b"aligned"),
    (dict(index=7 * A + 1), "INVALID", b"aligned"),
    (dict(off=9 * A), "INVALID", b"overlaps an input"),
    (dict(index=9 * A), "INVALID", b"overlaps an input"),
    (dict(rows=1 << 26, a_rows=1 << 26, N=1 << 24), "UNSUPPORTED", b"2^42"),
])
def test_grouped_refusals(g, kw, status, text):
    refused(g, product(g, True, **kw), status, text)


def test_product_of_more_tiles_than_a_launch_holds(g):
    far = {n: (i + 1) << 44 for i, n in enumerate(("a", "asc", "w", "ws", "bias"))}
    refused(g, product(g, False, dict(out=8 << 44, stride=1 << 16), a_rows=1 << 23, N=1 << 16, K=32, **far), "UNSUPPORTED",
            b"columns in one call")


@pytest.mark.parametrize("grouped", [False, True])
def test_alpha(g, grouped):
    """Over ln 2 it has to be finite in 32 bits; without swiglu it does not count."""
    none = dict(a_rows=0, rows=0)
    for alpha in (3e38, -3e38, 1.8e38, float("inf"), -float("inf")):
        refused(g, product(g, grouped, dict(swiglu=1, alpha=alpha), **none), "INVALID", b"alpha")
        assert product(g, grouped, dict(alpha=alpha), **none) == g.GPTOSS_OK
    for alpha in (2.0 ** 127, -2.0 ** 127, 0.0, 1e-40):
        assert product(g, grouped, dict(swiglu=1, alpha=alpha), **none) == g.GPTOSS_OK


def test_products_of_nothing(g):
    assert product(g, False, a_rows=0, a=None, asc=None, w=None, ws=None) == g.GPTOSS_OK
    assert product(g, True, a_rows=0, rows=0, a=None, asc=None, off=None) == g.GPTOSS_OK


# -- the Python binding ------------------------------------------------------
def matrix(g, *shape):
    return g.MXFP4Matrix(torch.zeros((*shape[:-1], shape[-1] // 2), dtype=torch.uint8),
                         torch.zeros((*shape[:-1], shape[-1] // 32), dtype=torch.uint8))


def u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


@pytest.mark.parametrize("packed, scales, text", [
    (u8(4, 16).int(), u8(4, 1), "uint8"), (u8(4, 16), u8(4, 1).int(), "uint8"), (None, u8(4, 1), "uint8"),
    (u8(4, 16), u8(4, 2), "packed must be"), (u8(4, 16), u8(3, 1), "packed must be"), (u8(16), u8(1), "packed must be"),
    (u8(1, 1, 4, 16), u8(1, 1, 4, 1), "packed must be"), (u8(4, 0), u8(4, 0), "positive"),
    (u8(16, 4).T, u8(4, 1), "contiguous"), (u8(4, 32), u8(4, 4)[:, ::2], "contiguous"),
])
def test_matrix_refusals(g, packed, scales, text):
    with pytest.raises(ValueError, match=text):
        g.MXFP4Matrix(packed, scales)


def test_sizes_past_32_bits(g):
    """Of matrices without memory: a size that the C calls cannot hold is refused and not cut short."""
    meta = dict(dtype=torch.uint8, device="meta")
    for shape in ((1 << 31, 32), (1 << 33, 32), (1, 1 << 32), (1 << 32, 1, 32)):
        with pytest.raises(ValueError, match="too large"):
            g.MXFP4Matrix(torch.empty((*shape[:-1], shape[-1] // 2), **meta), torch.empty((*shape[:-1], shape[-1] // 32), **meta))
    for shape in (((1 << 32) + 8, 32), (8, 1 << 32)):
        with pytest.raises(ValueError, match="too large"):
            g.mxfp4_quantize(torch.empty(shape, dtype=BF, device="meta"))
        with pytest.raises(ValueError, match="too large"):
            g.select_experts(torch.empty(shape, dtype=BF, device="meta"), 4)
    m = g.MXFP4Matrix(torch.empty((1 << 20, 1 << 12, 16), **meta), torch.empty((1 << 20, 1 << 12, 1), **meta))
    with pytest.raises(ValueError, match="too large"):
        g.mxfp4_dequantize(m)


def test_matrix_is_fixed(g):
    m = matrix(g, 3, 4, 64)
    assert m.shape == (3, 4, 64) and (m.experts, m.rows, m.K) == (3, 4, 64) and matrix(g, 4, 64).shape == (4, 64)
    with pytest.raises(AttributeError, match="fixed"):
        m.packed = u8(1)
    with pytest.raises(AttributeError, match="fixed"):
        del m.scales


BF = torch.bfloat16


@pytest.mark.parametrize("call, text", [
    (lambda g: g.select_experts([1.0], 1), "torch.Tensor"),
    (lambda g: g.select_experts(torch.zeros(3, 8, dtype=torch.float16), 1), "dtype"),
    (lambda g: g.select_experts(torch.zeros(8), 1), "2-D"),
    (lambda g: g.select_experts(torch.zeros(8, 3).T, 1), "contiguous rows"),
    (lambda g: g.select_experts(torch.zeros(1, 8).expand(3, 8), 1), "contiguous rows"),
    (lambda g: g.select_experts(torch.zeros(3, 8), 1, score="max"), "score"),
    (lambda g: g.select_experts(torch.zeros(3, 8), -1), "top_k"),
    (lambda g: g.select_experts(torch.zeros(3, 8), 1 << 32), "top_k"),
    (lambda g: g.select_experts(torch.zeros(3, 8), 1, num_groups=1 << 33), "num_groups"),
    (lambda g: g.select_experts(torch.zeros(3, 8), 1, bias=torch.zeros(7)), "bias"),
    (lambda g: g.select_experts(torch.zeros(3, 8), 1, bias=torch.zeros(8, dtype=BF)), "bias"),
    (lambda g: g.select_experts(torch.zeros(3, 8), 1, out=(torch.zeros(3, 1), torch.zeros(3, 1))), "indices"),
    (lambda g: g.select_experts(torch.zeros(3, 8), 1), "GPU"),
    (lambda g: g.mxfp4_quantize(torch.zeros(3, 32, dtype=torch.float16)), "dtype"),
    (lambda g: g.mxfp4_quantize(torch.zeros(3, 33)), "multiple of 32"),
    (lambda g: g.mxfp4_quantize(torch.zeros(3, 0)), "multiple of 32"),
    (lambda g: g.mxfp4_quantize(torch.zeros(2, 3, 32)), "2-D"),
    (lambda g: g.mxfp4_quantize(torch.zeros(3, 32), out=matrix(g, 3, 64)), "shape"),
    (lambda g: g.mxfp4_quantize(torch.zeros(3, 32), out=torch.zeros(3, 32)), "MXFP4Matrix"),
    (lambda g: g.mxfp4_quantize(torch.zeros(3, 32)), "GPU"),
    (lambda g: g.mxfp4_dequantize(torch.zeros(3, 32)), "MXFP4Matrix"),
    (lambda g: g.mxfp4_dequantize(matrix(g, 3, 32), dtype=torch.float16), "dtype"),
    (lambda g: g.mxfp4_dequantize(matrix(g, 3, 32), out=torch.zeros(3, 64)), "shape"),
    (lambda g: g.mxfp4_dequantize(matrix(g, 2, 3, 32), out=torch.zeros(2, 3, 32)), "2-D"),
    (lambda g: g.mxfp4_dequantize(matrix(g, 3, 32)), "GPU"),
    (lambda g: g.mxfp4_matmul(torch.zeros(3, 32), matrix(g, 4, 32)), "MXFP4Matrix"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 2, 4, 32)), "stack"),
    (lambda g: g.mxfp4_matmul(matrix(g, 2, 3, 32), matrix(g, 4, 32)), "stack"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 64)), "K="),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 32), bias=torch.zeros(3, dtype=BF)), "bias"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 32), bias=torch.zeros(4)), "bias"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 32), dtype=torch.float16), "dtype"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 32), out=torch.zeros(3, 5)), "shape"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 32), quantize=True), "multiple of 32"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 64, 32), quantize=True, out=torch.zeros(3, 64)), "MXFP4Matrix"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 64, 32), swiglu=True, quantize=True, out=matrix(g, 3, 64)),
     "shape"),
    (lambda g: g.mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 32)), "GPU"),
    (lambda g: g.grouped_mxfp4_matmul(matrix(g, 3, 32), matrix(g, 4, 32), torch.zeros(5).int(), 3), "stack"),
    (lambda g: g.grouped_mxfp4_matmul(matrix(g, 3, 32), matrix(g, 2, 4, 32), torch.zeros(4).int(), 3), "offsets"),
    (lambda g: g.grouped_mxfp4_matmul(matrix(g, 3, 32), matrix(g, 2, 4, 32), torch.zeros(3), 3), "offsets"),
    (lambda g: g.grouped_mxfp4_matmul(matrix(g, 3, 32), matrix(g, 2, 4, 32), torch.zeros(3).int(), -1), "rows"),
    (lambda g: g.grouped_mxfp4_matmul(matrix(g, 3, 32), matrix(g, 2, 4, 32), torch.zeros(3).int(), 3,
                                      row_index=torch.zeros(2).int()), "row_index"),
    (lambda g: g.grouped_mxfp4_matmul(matrix(g, 3, 32), matrix(g, 2, 4, 32), torch.zeros(3).int(), 3,
                                      bias=torch.zeros(4, dtype=BF)), "bias"),
    (lambda g: g.grouped_mxfp4_matmul(matrix(g, 3, 32), matrix(g, 2, 4, 32), torch.zeros(3).int(), 3), "GPU"),
])
def test_binding_refusals(g, call, text):
    with pytest.raises(ValueError, match=text):
        call(g)
