"""What the calls on tokens and the group norm refuse, without a device: through the C ABI with addresses that nothing reads, and
through tennis_amd.capi with tensors of the host."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def capi():
    from tennis_amd import capi as c
    c.lib()
    return c


AT = 1 << 20          # an address that nothing reads


def said(capi):
    return capi.lib().tsx_last_error().decode()


def test_quantize_tokens_refuses(capi):
    f = capi.lib().tsx_quantize_tokens
    assert f(0, 8, None, 0, 8, None, 8, None, None) == 0                       # no rows: nothing to do
    for args, word in (((-1, 8, AT, 0, 8, AT, 8, AT), "-1 rows"), ((4, 0, AT, 0, 8, AT, 8, AT), "0 columns"), ((4, 8, AT, 3, 8, AT, 8, AT), "element type 3"),
                       ((4, 8, AT, 7, 8, AT, 8, AT), "element type 7"), ((4, 8, AT, 0, 7, AT, 8, AT), "overlap"), ((4, 8, AT, 0, 8, AT, 7, AT), "overlap"),
                       ((4, 8, None, 0, 8, AT, 8, AT), "null"), ((4, 8, AT, 0, 8, None, 8, AT), "null"), ((4, 8, AT, 0, 8, AT, 8, None), "null"),
                       ((4, 8, AT + 2, 0, 8, AT, 8, AT), "multiple"), ((4, 8, AT + 1, 1, 8, AT, 8, AT), "multiple"), ((4, 8, AT, 1, 8, AT, 8, AT + 2), "multiple"),
                       ((1, (1 << 30) + 1, AT, 0, 1 << 31, AT, 1 << 31, AT), "columns")):
        assert f(*args, None) == -1 and word in said(capi), (args, said(capi))


def gemm(capi, **change):
    g = dict(m=4, n=8, k=16, x_type=2, out_type=2, act=0, slope=0.0, x_dev=AT, x_stride=16, x_scales_dev=None, packed_w_dev=AT, w_scales_dev=AT,
             bias_dev=None, out_dev=AT, out_stride=8)
    g.update(change)
    return capi.TokenGemm(**g)


def test_product_refuses(capi):
    L = capi.lib()
    need = L.tsx_gemm_i8_tokens_workspace_bytes(ctypes.byref(gemm(capi, m=100)))
    assert need >= 100 * 16 + 100 * 4
    assert L.tsx_gemm_i8_tokens(ctypes.byref(gemm(capi, m=0)), None, 0, None) == 0
    for change, word in ((dict(m=-1), "extents"), (dict(n=0), "extents"), (dict(m=1 << 28), "below 2^28"), (dict(n=1 << 24, out_stride=1 << 24), "below 2^28"), (dict(k=0), "extents"), (dict(k=1 << 17, x_stride=1 << 17), "2^17"),
                         (dict(x_type=4), "element type"), (dict(out_type=3), "output type"), (dict(act=3), "activation 3"), (dict(act=6), "activation 6"),
                         (dict(x_stride=15), "overlap"), (dict(out_stride=7), "overlap"), (dict(x_dev=None), "null"), (dict(packed_w_dev=None), "null"),
                         (dict(w_scales_dev=None), "null"), (dict(out_dev=None), "null"), (dict(x_type=3), "scales"), (dict(packed_w_dev=AT + 8), "aligned"),
                         (dict(x_dev=AT + 1), "multiple"), (dict(out_dev=AT + 1), "multiple")):
        g = gemm(capi, **change)
        assert L.tsx_gemm_i8_tokens(ctypes.byref(g), AT, 1 << 30, None) == -1 and word in said(capi), (change, said(capi))
    assert L.tsx_gemm_i8_tokens(None, AT, 1 << 30, None) == -1
    assert L.tsx_gemm_i8_tokens(ctypes.byref(gemm(capi, m=100)), AT, 16, None) == -2 and "workspace" in said(capi)
    assert L.tsx_gemm_i8_tokens(ctypes.byref(gemm(capi, m=100)), None, 1 << 30, None) == -2
    assert L.tsx_gemm_i8_tokens(ctypes.byref(gemm(capi, m=100)), AT + 4, 1 << 30, None) == -1 and "aligned" in said(capi)
    assert L.tsx_gemm_i8_tokens_workspace_bytes(ctypes.byref(gemm(capi, k=0))) == 0


def norm(capi, **change):
    g = dict(n=2, c=16, groups=4, type=1, pixels=9, image_stride=144, pixel_stride=16, x_dev=AT, weight_dev=None, bias_dev=None, epsilon=1e-5, act=0,
             slope=0.0)
    g.update(change)
    return capi.GroupNorm(**g)


def test_group_norm_refuses(capi):
    L = capi.lib()
    plain = lambda g: L.tsx_group_norm_nhwc(ctypes.byref(g), AT, AT, 1 << 30, None)                      # noqa: E731
    tokens = lambda g: L.tsx_group_norm_tokens_nhwc(ctypes.byref(g), AT, AT, AT, 1 << 30, None)          # noqa: E731
    for call in (plain, tokens):
        assert call(norm(capi, n=0)) == 0 and call(norm(capi, pixels=0)) == 0
        for change, word in ((dict(n=-1), "extents"), (dict(c=0), "extents"), (dict(groups=0), "extents"), (dict(pixels=-1), "extents"),
                             (dict(groups=5), "5 groups"), (dict(c=8200, groups=1, pixel_stride=8200), "at most 8192"), (dict(type=3), "element type"),
                             (dict(n=65536), "65536 images"), (dict(pixels=1 << 30), "pixels"), (dict(pixel_stride=(1 << 26) + 1), "2^26"), (dict(pixel_stride=15), "overlap"), (dict(image_stride=-1), "negative"), (dict(act=3), "activation 3"),
                             (dict(epsilon=-1.0), "epsilon"), (dict(epsilon=float("nan")), "epsilon"), (dict(x_dev=None), "null"), (dict(x_dev=AT + 1), "multiple")):
            assert call(norm(capi, **change)) == -1 and word in said(capi), (change, said(capi))
    g = norm(capi, pixels=1 << 20, image_stride=16 << 20)
    assert L.tsx_group_norm_workspace_bytes(ctypes.byref(g)) > 0
    assert L.tsx_group_norm_nhwc(ctypes.byref(g), AT, AT, 4, None) == -2 and "workspace" in said(capi)
    assert L.tsx_group_norm_nhwc(ctypes.byref(g), AT, None, 1 << 30, None) == -2
    assert L.tsx_group_norm_nhwc(ctypes.byref(g), AT, AT + 4, 1 << 30, None) == -1 and "aligned" in said(capi)
    assert L.tsx_group_norm_nhwc(ctypes.byref(norm(capi)), None, AT, 1 << 30, None) == -1 and "null" in said(capi)
    assert L.tsx_group_norm_tokens_nhwc(ctypes.byref(norm(capi)), AT, None, AT, 1 << 30, None) == -1 and "null" in said(capi)
    assert L.tsx_group_norm_workspace_bytes(ctypes.byref(norm(capi, groups=5))) == 0


def test_other_calls_do_not_take_silu(capi):
    """5 stays an unknown activation where it was one."""
    assert "silu" not in capi._ACT
    assert capi.lib().tsx_add_f32(AT, AT, 4, 5, 0.0, AT, None) == -1 and "activation" in said(capi)


def test_python_calls_refuse(capi):
    import torch
    x = torch.zeros(4, 16)
    for call in (lambda: capi.quantize_tokens(x), lambda: capi.quantize_tokens([1.0]), lambda: capi.group_norm(x, 4), lambda: capi.group_norm_tokens(x, 4),
                 lambda: capi.TokenGemmI8(torch.zeros((4, 4), dtype=torch.int8), torch.ones(4))):
        with pytest.raises(capi.TsxError, match="device tensor"):
            call()
    for act in ("mish", "gelu", 5):
        with pytest.raises(capi.TsxError, match="activation"):
            capi.group_norm(x, 4, act=act)
