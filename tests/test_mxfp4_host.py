"""What the calls on MXFP4 rows and the root-mean-square norm refuse, without a device: through the C ABI with addresses that nothing
reads, and through tennis_amd.capi with tensors of the host."""
import ctypes

import pytest

AT = 1 << 20          # an address that nothing reads


@pytest.fixture(scope="module")
def capi():
    from tennis_amd import capi as c
    c.lib()
    return c


def said(capi):
    return capi.lib().tsx_last_error().decode()


def refused(capi, f, args, word):
    assert f(*args) == -1 and word in said(capi), (args, said(capi))


def test_quantize_refuses(capi):
    f = capi.lib().tsx_quantize_mxfp4
    good = dict(rows=4, cols=40, x=AT, type=0, stride=40, codes=AT, codes_stride=20, scales=AT, scales_stride=2, stream=None)
    assert f(*dict(good, rows=0, x=None, codes=None, scales=None).values()) == 0
    for change, word in ((dict(rows=-1), "-1 rows"), (dict(cols=0), "0 columns"), (dict(cols=(1 << 30) + 1), "columns"), (dict(type=3), "element type 3"),
                         (dict(type=4), "element type 4"), (dict(stride=39), "overlap"), (dict(codes_stride=19), "overlap"), (dict(scales_stride=1), "overlap"),
                         (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(x=AT + 2), "multiple"), (dict(x=AT + 1, type=1), "multiple")):
        refused(capi, f, dict(good, **change).values(), word)


def test_dequantize_refuses(capi):
    f = capi.lib().tsx_dequantize_mxfp4
    good = dict(rows=4, cols=40, codes=AT, codes_stride=20, scales=AT, scales_stride=2, out=AT, type=2, stride=40, stream=None)
    assert f(*dict(good, rows=0).values()) == 0
    for change, word in ((dict(rows=-1), "-1 rows"), (dict(cols=0), "0 columns"), (dict(type=3), "element type 3"), (dict(stride=39), "overlap"),
                         (dict(codes_stride=19), "overlap"), (dict(scales_stride=1), "overlap"), (dict(codes=None), "null"), (dict(scales=None), "null"),
                         (dict(out=None), "null"), (dict(out=AT + 1), "multiple")):
        refused(capi, f, dict(good, **change).values(), word)
    f = capi.lib().tsx_dequantize_tokens
    good = dict(rows=4, cols=40, q=AT, q_stride=40, scales=AT, out=AT, type=2, stride=40, stream=None)
    assert f(*dict(good, rows=0).values()) == 0
    for change, word in ((dict(rows=-1), "-1 rows"), (dict(cols=0), "0 columns"), (dict(type=3), "element type 3"), (dict(stride=39), "overlap"), (dict(q_stride=39), "overlap"),
                         (dict(q=None), "null"), (dict(scales=None), "null"), (dict(out=None), "null"), (dict(out=AT + 1), "multiple"), (dict(scales=AT + 2), "multiple")):
        refused(capi, f, dict(good, **change).values(), word)


def gemm(capi, **change):
    g = dict(m=4, n=8, k=256, x_type=2, out_type=2, act=0, slope=0.0, x_dev=AT, x_stride=256, x_scales_dev=None, x_scales_stride=8, packed_w_dev=AT, bias_dev=None,
             out_dev=AT, out_stride=8)
    g.update(change)
    return capi.Mxfp4Gemm(**g)


def test_product_refuses(capi):
    L = capi.lib()
    many = dict(m=1000, n=1000, out_stride=1000)
    assert L.tsx_gemm_mxfp4_workspace_bytes(ctypes.byref(gemm(capi, **many))) == 1000 * (128 + 8)
    assert L.tsx_gemm_mxfp4_workspace_bytes(ctypes.byref(gemm(capi, m=100))) == 0      # the product quantizes few rows itself
    codes = dict(x_type=4, x_stride=128, x_scales_dev=AT)
    assert L.tsx_gemm_mxfp4_workspace_bytes(ctypes.byref(gemm(capi, m=100, **codes))) == 0
    assert L.tsx_gemm_mxfp4_workspace_bytes(ctypes.byref(gemm(capi, m=100, **dict(codes, x_dev=AT + 1)))) == 100 * (128 + 8)
    assert L.tsx_gemm_mxfp4(ctypes.byref(gemm(capi, m=0)), None, 0, None) == 0
    for change, word in ((dict(m=-1), "extents"), (dict(n=0), "extents"), (dict(k=0), "extents"), (dict(m=1 << 28), "2^28"), (dict(n=1 << 24, out_stride=1 << 24), "2^24"),
                         (dict(k=1 << 21, x_stride=1 << 21), "2^21"), (dict(x_type=3), "element type"), (dict(x_type=5), "element type"), (dict(out_type=3), "output type"),
                         (dict(out_type=4), "output type"), (dict(act=3), "activation 3"), (dict(act=6), "activation 6"), (dict(x_stride=255), "overlap"), (dict(out_stride=7), "overlap"),
                         (dict(codes, x_stride=127), "overlap"), (dict(codes, x_scales_stride=7), "overlap"), (dict(x_dev=None), "null"), (dict(packed_w_dev=None), "null"),
                         (dict(out_dev=None), "null"), (dict(codes, x_scales_dev=None), "scales"), (dict(packed_w_dev=AT + 8), "aligned"), (dict(x_dev=AT + 1), "multiple"),
                         (dict(out_dev=AT + 1), "multiple"), (dict(bias_dev=AT + 2), "multiple")):
        refused(capi, L.tsx_gemm_mxfp4, (ctypes.byref(gemm(capi, **change)), AT, 1 << 30, None), word)
    assert L.tsx_gemm_mxfp4(None, AT, 1 << 30, None) == -1
    g = gemm(capi, **many)
    assert L.tsx_gemm_mxfp4(ctypes.byref(g), AT, 16, None) == -2 and "workspace" in said(capi)
    assert L.tsx_gemm_mxfp4(ctypes.byref(g), None, 1 << 30, None) == -2
    assert L.tsx_gemm_mxfp4(ctypes.byref(g), AT + 4, 1 << 30, None) == -1 and "aligned" in said(capi)
    assert L.tsx_gemm_mxfp4_workspace_bytes(ctypes.byref(gemm(capi, k=0))) == 0


def test_weights_refuse(capi):
    L = capi.lib()
    assert L.tsx_gemm_mxfp4_packed_weight_bytes(1, 1) == 4 * 4 * (2048 + 128)
    assert L.tsx_gemm_mxfp4_packed_weight_bytes(0, 1) == 0 and L.tsx_gemm_mxfp4_packed_weight_bytes(1 << 21, 1) == 0
    good = dict(k=64, n=4, codes=AT, codes_stride=32, scales=AT, scales_stride=2, packed=AT, stream=None)
    for change, word in ((dict(k=0), "K = 0"), (dict(n=0), "0 columns"), (dict(k=1 << 21), "2^21"), (dict(n=1 << 24), "2^24"), (dict(codes_stride=31), "overlap"),
                         (dict(scales_stride=1), "overlap"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(packed=None), "null"), (dict(packed=AT + 8), "aligned")):
        refused(capi, L.tsx_gemm_mxfp4_pack_weights, dict(good, **change).values(), word)


def norm(capi, **change):
    g = dict(rows=3, cols=40, type=1, x_dev=AT, x_stride=40, residual_dev=AT, residual_stride=40, sum_dev=AT, sum_stride=40, weight_dev=None, epsilon=1e-6)
    g.update(change)
    return capi.RmsNorm(**g)


def test_norm_refuses(capi):
    L = capi.lib()
    rows = lambda g: L.tsx_rms_norm_rows(ctypes.byref(g), AT, 40, None)            # noqa: E731
    tokens = lambda g: L.tsx_rms_norm_tokens(ctypes.byref(g), AT, AT, None)        # noqa: E731
    mxfp4 = lambda g: L.tsx_rms_norm_mxfp4(ctypes.byref(g), AT, AT, None)          # noqa: E731
    for call in (rows, tokens, mxfp4):
        assert call(norm(capi, rows=0, x_dev=None)) == 0
        for change, word in ((dict(rows=-1), "-1 rows"), (dict(cols=0), "0 columns"), (dict(cols=(1 << 30) + 1), "columns"), (dict(type=3), "element type"),
                             (dict(epsilon=-1.0), "epsilon"), (dict(epsilon=float("nan")), "epsilon"), (dict(epsilon=float("inf")), "epsilon"), (dict(x_stride=39), "overlap"),
                             (dict(residual_stride=39), "overlap"), (dict(sum_stride=39), "overlap"), (dict(x_dev=None), "null"), (dict(sum_dev=None), "place for the sum"),
                             (dict(x_dev=AT + 1), "multiple"), (dict(residual_dev=AT + 1), "multiple"), (dict(sum_dev=AT + 1), "multiple"), (dict(weight_dev=AT + 2), "multiple")):
            assert call(norm(capi, **change)) == -1 and word in said(capi), (change, said(capi))
    for call in (lambda: L.tsx_rms_norm_rows(ctypes.byref(norm(capi)), None, 40, None), lambda: L.tsx_rms_norm_tokens(ctypes.byref(norm(capi)), AT, None, None),
                 lambda: L.tsx_rms_norm_mxfp4(ctypes.byref(norm(capi)), None, AT, None)):
        assert call() == -1 and "null" in said(capi)
    assert L.tsx_rms_norm_rows(ctypes.byref(norm(capi)), AT, 39, None) == -1 and "overlap" in said(capi)
    assert L.tsx_rms_norm_rows(ctypes.byref(norm(capi)), AT + 1, 40, None) == -1 and "multiple" in said(capi)
    assert L.tsx_rms_norm_tokens(ctypes.byref(norm(capi)), AT, AT + 2, None) == -1 and "multiple" in said(capi)


def test_python_calls_refuse(capi):
    import torch
    x, b = torch.zeros(4, 64), torch.zeros((4, 32), dtype=torch.uint8)
    for call in (lambda: capi.quantize_mxfp4(x), lambda: capi.quantize_mxfp4([1.0]), lambda: capi.dequantize_mxfp4(b, b[:, :2]), lambda: capi.rms_norm(x),
                 lambda: capi.rms_norm_tokens(x), lambda: capi.rms_norm_mxfp4(x), lambda: capi.TokenGemmMxfp4(b, b[:, :2]),
                 lambda: capi.dequantize_tokens(x.to(torch.int8), x[:, 0])):
        with pytest.raises(capi.TsxError, match="device tensor"):
            call()
    for k in (0, -1):
        with pytest.raises(capi.TsxError, match="values"):
            capi.dequantize_mxfp4(b, b[:, :2], k=k)
    with pytest.raises(capi.TsxError, match="output type"):
        capi.dequantize_mxfp4(b, b[:, :2], dtype=torch.int8)
