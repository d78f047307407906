"""The calls on tokens and on channels-last tensors against their definitions in 64 bits: rows quantized by their own largest
magnitude, the int8 product with scales for each token and channel, group norm with an activation, and its int8 tokens.

Bars.  u = 2^-24 is half a step of fp32 relative to the value, h that of the output's type (eps / 2, and the type's smallest
step absolute).  int8 values and sums of int8 products are exact."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["f32", "f16", "bf16"]
ACTS = [None, "relu", "leaky_relu", "silu", "mish_fast"]


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "this test needs the MI355X"
    return t


@pytest.fixture(scope="module")
def capi():
    from tennis_amd import capi as c
    c.lib()
    return c


def dtype(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def values(torch, rng, shape, name, spread=1.0):
    """Rows of different size on the device, and the same values in 64 bits."""
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[:-1] + (1,)))
    t = torch.from_numpy(x).to(dtype(torch, name))
    return t.cuda(), t.double().numpy()


def tokens64(x):
    """(q, scale) by the definition; the division's result in fp32 is that of 64 bits rounded again (53 >= 2 * 24 + 2 bits)."""
    with np.errstate(over="ignore"):
        top = np.abs(x).max(-1, keepdims=True)
        lift = np.where(top < 2.0 ** -64, 2.0 ** 64, 1.0)
        finite = np.isfinite(top)
        r = np.where(finite & (top > 0), 127.0 / np.where(finite & (top > 0), top * lift, 1.0), 0.0).astype(np.float32).astype(np.float64)
        q = np.rint(np.where(finite, np.where(np.isfinite(x), x, 0.0) * lift * r, 0.0))
        scale = np.where(finite, np.where(finite, top, 0.0) / 127.0, np.nan).astype(np.float32)
    return q.astype(np.int8), scale[..., 0]


def act64(y, act, slope=0.1):
    if act == "relu":
        return np.maximum(y, 0.0)
    if act == "leaky_relu":
        return np.where(y > 0, y, float(np.float32(slope)) * y)
    with np.errstate(over="ignore"):
        if act == "silu":
            return y / (1.0 + np.exp(-y))
        if act == "mish_fast":
            return y * np.tanh(np.logaddexp(y, 0.0))
    return y


def after_act(y, act, error):
    """The error of act(y) in fp32 where y is off by `error`.  ReLU and LeakyReLU: the error again, and one rounding.  SiLU and Mish
    have slopes within 1.1.  Their own arithmetic: an exponential and a reciprocal (each within a step, 2 u), the exponential's
    argument rounded (|y| u of the exponential, at most a quarter of |y| of the result's slope) and three more roundings of a quotient
    of at most 1: 8 u |y| + u y^2 / 2, and Mish 12 u |y| for its two more."""
    if act in ("silu", "mish_fast"):
        return 1.1 * error + (12 * np.abs(y) + y * y / 2) * U
    return error + np.abs(y) * U


def close(torch, got, want, error, name):
    """`error` in fp32 ahead of the one rounding to the output's type."""
    t = dtype(torch, name)
    h = torch.finfo(t).eps / 2
    tiny = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}[name]
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    off = np.abs(got - want) - (error * (1 + h) + h * np.abs(want) + tiny)
    assert not np.isnan(got).any() and off.max(initial=-1.0) <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


# ---------------------------------------------------------------- rows to int8

@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 4096), (3, 7), (5, 8), (300, 64), (65, 511), (64, 512), (33, 513), (7, 2047), (5, 2049), (3, 8192), (2, 8197),
                                 (2, 32768), (2, 32771), (2, 70001)])
def test_quantize_tokens(torch, capi, name, m, k):
    rng = np.random.default_rng(m + k)
    x, x64 = values(torch, rng, (m, k), name)
    q, s = capi.quantize_tokens(x)
    eq, es = tokens64(x64)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and s.shape == (m,)
    assert np.array_equal(q.cpu().numpy(), eq) and np.array_equal(s.cpu().numpy(), es)
    assert (np.abs(eq).max(1) == 127).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,k", [(3000, 1), (1000, 8), (999, 9), (777, 31), (700, 128), (700, 129), (600, 1000), (600, 4096), (513, 4000), (2000, 600)])
def test_quantize_many_tokens(torch, capi, name, m, k):
    """Several rows to a wavefront, and one."""
    rng = np.random.default_rng(m + k)
    x, x64 = values(torch, rng, (m, k + 3), name)
    q, s = capi.quantize_tokens(x[:, 1:k + 1])
    eq, es = tokens64(x64[:, 1:k + 1])
    assert np.array_equal(q.cpu().numpy(), eq) and np.array_equal(s.cpu().numpy(), es)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_tokens_strides(torch, capi, name):
    rng = np.random.default_rng(4)
    wide, wide64 = values(torch, rng, (37, 300), name)
    three, three64 = values(torch, rng, (4, 5, 96), name)
    for x, x64 in ((wide[:, 3:204], wide64[:, 3:204]), (wide[::3, :130], wide64[::3, :130]), (wide.t(), wide64.T), (wide[5, 1:], wide64[5, 1:]),
                   (three, three64), (three[:, 1:4, 5:77], three64[:, 1:4, 5:77]), (three.transpose(0, 1), three64.transpose(1, 0, 2)),
                   (wide[:1, :64].expand(6, 64), np.repeat(wide64[:1, :64], 6, 0)), (three[:0], three64[:0])):
        q, s = capi.quantize_tokens(x)
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        if x.numel():
            eq, es = tokens64(x64)
            assert np.array_equal(q.cpu().numpy(), eq) and np.array_equal(s.cpu().numpy(), es)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_tokens_special_rows(torch, capi, name):
    """Zeros, ties, infinities, NaN, the smallest and largest numbers; every row by itself."""
    t = dtype(torch, name)
    big, small = torch.finfo(t).max, {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}[name]
    rows = [[0.0] * 9, [-0.0] * 9, [127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 3.5, 126.5], [math.inf, 1, 2, 3, 4, 5, 6, 7, 8],
            [1, 2, 3, math.nan, 5, 6, 7, 8, -math.inf], [big, -big, big / 2, big / 4, 0, 1, -1, big, big], [small, -small, 0, 0, 0, 0, 0, 0, small],
            [8 * small, 3 * small, -5 * small, small, 0, 0, 0, 0, 0], [1e-3, 1, -1, 0, 0, 0, 0, 0, -0.0], [-63.5, 31.75, 0.25, 0.75, 1.25, 0, 0, 0, 0]]
    x = torch.tensor(rows, dtype=torch.float64).to(t)
    q, s = capi.quantize_tokens(x.cuda())
    eq, es = tokens64(x.double().numpy())
    assert np.array_equal(q.cpu().numpy(), eq)
    assert np.array_equal(s.cpu().numpy(), es, equal_nan=True)
    assert np.isnan(es[3]) and np.isnan(es[4]) and es[0] == 0


# ---------------------------------------------------------------- the product

def product64(q, sx, w, sw, bias, act):
    p = (q.astype(np.float64) @ w.astype(np.float64).T) * sw.astype(np.float64) * sx.astype(np.float64)[..., None]
    y = p if bias is None else p + bias.astype(np.float64)
    # the sum to fp32, two products: 3 u of p; the bias: u of the sum
    return act64(y, act), after_act(y, act, 3.01 * U * np.abs(p) + (0 if bias is None else U * (np.abs(y) + 3.01 * U * np.abs(p))))


def weights(torch, rng, n, k):
    w = rng.integers(-127, 128, (n, k)).astype(np.int8)
    sw = (rng.uniform(0.5, 1.5, n) / (60 * math.sqrt(k))).astype(np.float32)
    return w, sw, rng.standard_normal(n).astype(np.float32)


PRODUCTS = [(1, 1, 1), (1, 64, 64), (1, 4096, 1024), (2, 33, 5), (7, 1000, 2048), (16, 100, 4100), (31, 31, 31), (32, 32, 128), (33, 33, 129), (64, 130, 256),
            (127, 129, 127), (128, 128, 128), (129, 257, 384), (197, 777, 1500), (300, 40, 700), (513, 200, 65), (256, 512, 1024), (1024, 768, 512)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(torch, capi, name, m, n, k):
    rng = np.random.default_rng(m + n + k)
    w, sw, bias = weights(torch, rng, n, k)
    x, x64 = values(torch, rng, (m, k), name, 0.3)
    q, sx = tokens64(x64)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())
    act = ACTS[(m + n) % len(ACTS)]
    want, error = product64(q, sx, w, sw, bias, act)
    out = layer(x, act=act, slope=0.1)
    assert out.dtype == x.dtype
    close(torch, out, want, error, name)
    # its own tokens, quantized ahead, are the same bits
    qd, sd = capi.quantize_tokens(x)
    assert torch.equal(layer(qd, x_scales=sd, act=act, slope=0.1, out_dtype=x.dtype), out)


@pytest.mark.parametrize("kernel", "01234")
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (5, 17, 64), (33, 31, 100), (64, 130, 192), (65, 129, 257), (130, 70, 1040), (257, 257, 640), (300, 520, 2048), (260, 100, 48)])
def test_every_product_kernel(torch, capi, monkeypatch, kernel, m, n, k):
    """Each kernel on sizes that end inside its tiles and K of fewer and more chunks than it keeps in flight: the same bits."""
    rng = np.random.default_rng(m + n + k)
    w, sw, bias = weights(torch, rng, n, k)
    q = rng.integers(-128, 128, (m, k)).astype(np.int8)
    sx = rng.uniform(0.01, 0.1, m).astype(np.float32)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())
    x, s = torch.from_numpy(q).cuda(), torch.from_numpy(sx).cuda()
    monkeypatch.setenv("TSX_TOKENS_KERNEL", kernel)
    for name, act in zip(TYPES, ("silu", None, "leaky_relu")):
        want, error = product64(q, sx, w, sw, bias, act)
        got = layer(x, x_scales=s, act=act, slope=0.1, out_dtype=dtype(torch, name))
        close(torch, got, want, error, name)
        monkeypatch.delenv("TSX_TOKENS_KERNEL")
        assert torch.equal(got, layer(x, x_scales=s, act=act, slope=0.1, out_dtype=got.dtype))
        monkeypatch.setenv("TSX_TOKENS_KERNEL", kernel)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40, 40960), (2, 33, 20479), (3, 20, 9000), (5, 20, 8192), (9, 50, 4551), (20, 70, 2048), (32, 40, 1279), (17, 16, 7)])
def test_product_quantizes_few_tokens_itself(torch, capi, name, m, n, k):
    """Rows that one workgroup's threads hold and rows read in turns, shared by all, several or one of its wavefronts."""
    rng = np.random.default_rng(m + k)
    w, sw, bias = weights(torch, rng, n, k)
    x, x64 = values(torch, rng, (m, k), name, 0.3)
    x[m - 1, k // 2] = math.inf
    q, sx = tokens64(x.double().cpu().numpy())
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())
    out = layer(x)
    assert out[m - 1].isnan().all()
    if m > 1:
        want, error = product64(q[:-1], sx[:-1], w, sw, bias, None)
        close(torch, out[:-1], want, error, name)


def test_product_of_the_longest_rows(torch, capi):
    """The largest sums: 127 * 127 * (2^17 - 1) is 2 % short of what 32 bits hold."""
    k = (1 << 17) - 1
    for m in (2, 40):
        q = torch.full((m, k), 127, dtype=torch.int8, device="cuda")
        layer = capi.TokenGemmI8(torch.full((3, k), 127, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))
        assert (layer(q, x_scales=torch.ones(m, device="cuda")) == float(np.float32(127 * 127 * k))).all()
    with pytest.raises(capi.TsxError, match="2\\^17"):
        capi.TokenGemmI8(torch.ones((3, k + 1), dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))(torch.ones((2, k + 1), device="cuda"))


def test_product_of_many_short_tokens(torch, capi):
    """More groups of tokens than a launch has places along its second axis; 32-bit offsets would end at 2^31 bytes of rows and outputs."""
    rng = np.random.default_rng(13)
    for m, n, k in ((1 << 21, 16, 64), ((1 << 21) + 77, 1040, 1040)):
        w, sw, bias = weights(torch, rng, n, k)
        layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())
        q = torch.randint(-128, 128, (m, k), dtype=torch.int8, device="cuda")
        sx = torch.rand(m, device="cuda") * 0.1 + 0.01
        out = layer(q, x_scales=sx, out_dtype=torch.bfloat16)
        at = torch.tensor([0, 1, 255, 256, m // 2, m - 257, m - 256, m - 2, m - 1], device="cuda")
        want, error = product64(q[at].cpu().numpy(), sx[at].cpu().numpy(), w, sw, bias, None)
        close(torch, out[at], want, error, "bf16")
        for first in range(0, m, 1 << 19):       # the same by parts
            assert torch.equal(out[first:first + (1 << 19)], layer(q[first:first + (1 << 19)], x_scales=sx[first:first + (1 << 19)], out_dtype=torch.bfloat16))


def test_product_of_rows_far_apart(torch, capi):
    """int8 tokens at strides on both sides of the longest that a tile reads in place, the last of them behind 2^32 bytes."""
    rng = np.random.default_rng(14)
    w, sw, _ = weights(torch, rng, 40, 64)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda())
    for m, stride in ((300, 1 << 23), (300, (1 << 23) + 16), (2, 1 << 31)):
        whole = torch.empty((m - 1) * stride + 64, dtype=torch.int8, device="cuda")
        x = whole.as_strided((m, 64), (stride, 1))
        q = torch.from_numpy(rng.integers(-128, 128, (m, 64)).astype(np.int8)).cuda()
        x.copy_(q)
        s = torch.ones(m, device="cuda")
        assert torch.equal(layer(x, x_scales=s), layer(q, x_scales=s))


@pytest.mark.parametrize("m", [1, 16, 70])
def test_rows_without_a_number_and_activations(torch, capi, m):
    """ReLU and LeakyReLU make 0 of a NaN, the others keep it, in the products and in the norm."""
    layer = capi.TokenGemmI8(torch.ones((33, 24), dtype=torch.int8, device="cuda"), torch.ones(33, device="cuda"))
    x = torch.full((m, 24), math.nan, device="cuda")
    planes = torch.full((2, m, 24), math.nan, device="cuda")
    for act in ACTS:
        for y in (layer(x, act=act, slope=0.1), capi.group_norm(planes, 3, act=act, slope=0.1)):
            assert (y == 0).all() if act in ("relu", "leaky_relu") else y.isnan().all()
        q, s = capi.group_norm_tokens(planes, 3, act=act, slope=0.1)
        assert (q == 0).all() and ((s == 0).all() if act in ("relu", "leaky_relu") else s.isnan().all())


def test_layers_are_copied_and_stored(torch, capi):
    import copy
    import io
    import pickle
    rng = np.random.default_rng(15)
    w, sw, bias = weights(torch, rng, 30, 50)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())
    x, _ = values(torch, rng, (7, 50), "bf16", 0.3)
    want = layer(x)
    for other in (copy.copy(layer), copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        assert torch.equal(other(x), want)
    buf = io.BytesIO()
    torch.save({"q": layer.w, "s": layer.w_scales, "b": layer.bias}, buf)
    buf.seek(0)
    state = torch.load(buf, weights_only=True)
    assert torch.equal(capi.TokenGemmI8(state["q"], state["s"], state["b"])(x), want)


def test_tensors_of_other_kinds(torch, capi):
    """Views that stand for their negation, leaves that want gradients, vectors of another type, calls that carry no gradient."""
    rng = np.random.default_rng(16)
    z = torch.complex(torch.randn(6, 48, device="cuda"), torch.randn(6, 48, device="cuda"))
    x = z.conj().imag
    assert x.is_neg()
    for a, b in ((capi.quantize_tokens(x), capi.quantize_tokens(x.clone())), (capi.group_norm_tokens(x, 4), capi.group_norm_tokens(x.clone(), 4))):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(capi.group_norm(x, 4), capi.group_norm(x.clone(), 4))
    w, sw, bias = weights(torch, rng, 30, 48)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda().double(), torch.from_numpy(bias).cuda().double())
    assert torch.equal(layer(x), layer(x.clone()))
    leaf = torch.randn(6, 48, device="cuda", requires_grad=True)
    for y in (layer(leaf), capi.group_norm(leaf, 4, torch.ones(48, device="cuda", requires_grad=True)), capi.quantize_tokens(leaf)[1]):
        assert not y.requires_grad


def test_product_refuses_on_the_device(torch, capi):
    layer = capi.TokenGemmI8(torch.ones((5, 16), dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"))
    x, q = torch.ones((3, 16), device="cuda"), torch.ones((3, 16), dtype=torch.int8, device="cuda")
    for call in (lambda: layer(x[:, :15]), lambda: layer(q), lambda: layer(x, x_scales=torch.ones(3, device="cuda")), lambda: layer(q, x_scales=torch.ones(2, device="cuda")),
                 lambda: layer(x, out_dtype=torch.int8), lambda: layer(x.double()), lambda: layer(x, act="mish"), lambda: layer(x.cpu()), lambda: layer(torch.ones((), device="cuda")),
                 lambda: capi.quantize_tokens(x[:, :0]), lambda: capi.quantize_tokens(q), lambda: capi.group_norm(x, 5), lambda: capi.group_norm(x, 0), lambda: capi.group_norm(x, -4),
                 lambda: capi.group_norm(x, (1 << 32) + 4), lambda: capi.group_norm(x[:, :0], 1), lambda: capi.group_norm(x[0], 4), lambda: capi.group_norm(x, 4, torch.ones(15, device="cuda")),
                 lambda: capi.group_norm(x, 4, epsilon=math.nan), lambda: capi.group_norm(torch.ones((1, 8193), device="cuda"), 1),
                 lambda: capi.group_norm(torch.ones((65536, 1), device="cuda"), 1), lambda: capi.group_norm_tokens(x, 4, None, torch.ones(17, device="cuda"))):
        with pytest.raises(capi.TsxError):
            call()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 50, 70), (40, 136, 200), (130, 200, 140)])
def test_product_types_and_activations(torch, capi, act, out, m, n, k):
    rng = np.random.default_rng(9)
    w, sw, bias = weights(torch, rng, n, k)
    q = rng.integers(-127, 128, (m, k)).astype(np.int8)
    sx = rng.uniform(0.01, 0.1, m).astype(np.float32)
    for b in (None, bias):
        want, error = product64(q, sx, w, sw, b, act)
        for transpose in (True, False):
            wd = torch.from_numpy(w if transpose else np.ascontiguousarray(w.T)).cuda()
            layer = capi.TokenGemmI8(wd, torch.from_numpy(sw).cuda(), None if b is None else torch.from_numpy(b).cuda(), transpose=transpose)
            got = layer(torch.from_numpy(q).cuda(), x_scales=torch.from_numpy(sx).cuda(), act=act, slope=0.1, out_dtype=dtype(torch, out))
            close(torch, got, want, error, out)


def test_product_strides(torch, capi):
    rng = np.random.default_rng(10)
    w, sw, _ = weights(torch, rng, 72, 128)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda())
    for rows in (6, 90):
        wide, wide64 = values(torch, rng, (rows, 5, 300), "bf16", 0.3)
        whole = torch.from_numpy(rng.integers(-128, 128, (rows, 333)).astype(np.int8)).cuda()
        sx = torch.from_numpy(rng.uniform(0.01, 0.1, rows).astype(np.float32)).cuda()
        for x in (wide[:, :, 7:135], wide[:, 2, 100:228], wide[0, 0, :128], wide.transpose(0, 1)[..., :128], wide[:0, :, :128]):
            out = layer(x)
            assert out.shape == x.shape[:-1] + (72,)
            assert torch.equal(out, layer(x.contiguous()))
        for at in (0, 1, 16, 17):
            x = whole[:, at:at + 128]
            assert torch.equal(layer(x, x_scales=sx), layer(x.contiguous(), x_scales=sx))
        aligned = torch.empty((rows, 384), dtype=torch.int8, device="cuda")[:, 128:256].copy_(whole[:, :128])
        assert torch.equal(layer(aligned, x_scales=sx), layer(whole[:, :128].contiguous(), x_scales=sx))


def test_product_writes_its_rows_only(torch, capi):
    """Columns behind the last one, rows behind the last token and a wider output's other columns stay as they were."""
    import ctypes
    rng = np.random.default_rng(11)
    for m, n, k in ((5, 37, 64), (40, 37, 64), (130, 131, 64)):
        w, sw, _ = weights(torch, rng, n, k)
        layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda())
        x, _ = values(torch, rng, (m, k), "f16", 0.3)
        for t, code in ((torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)):
            want = layer(x, out_dtype=t)
            wide = torch.full((m + 2, n + 9), 7.0, dtype=t, device="cuda")
            at = wide[1:, 3:]
            g = capi.TokenGemm(m, n, k, 1, code, 0, 0.0, capi._ptr(x), k, None, capi._ptr(layer.packed), capi._ptr(layer.w_scales), None,
                               capi._ptr(at), n + 9)
            nbytes = capi.lib().tsx_gemm_i8_tokens_workspace_bytes(ctypes.byref(g))
            ws = torch.empty(nbytes + 16, dtype=torch.uint8, device="cuda")
            capi.check(capi.lib().tsx_gemm_i8_tokens(ctypes.byref(g), capi._ptr(ws), nbytes, capi._stream()))
            assert torch.equal(wide[1:m + 1, 3:n + 3], want)
            wide[1:m + 1, 3:n + 3] = 7.0
            assert (wide == 7.0).all()


def test_product_rows_without_a_number(torch, capi):
    """A row with an infinity or NaN is NaN, the others do not notice; a row of zeros is the activation of the bias."""
    rng = np.random.default_rng(12)
    w, sw, bias = weights(torch, rng, 48, 200)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())
    for m in (4, 70):
        x, _ = values(torch, rng, (m, 200), "f32", 0.3)
        want = layer(x)
        x[1, 3] = math.inf
        x[2, 199] = math.nan
        x[3] = 0
        got = layer(x)
        assert got[1:3].isnan().all() and torch.equal(got[0], want[0]) and torch.equal(got[4:], want[4:])
        assert np.array_equal(got[3].cpu().numpy(), bias)


def test_product_from_float(torch, capi):
    rng = np.random.default_rng(13)
    w, w64 = values(torch, rng, (50, 90), "bf16", 0.0)
    x, x64 = values(torch, rng, (9, 90), "f32", 0.0)
    q, s = tokens64(w64)
    qx, sx = tokens64(x64)
    want, error = product64(qx, sx, q, s, None, None)
    close(torch, capi.TokenGemmI8.from_float(w)(x), want, error, "f32")


# ---------------------------------------------------------------- group norm

def norm64(x, groups, weight, bias, eps, act):
    """The norm in 64 bits and what fp32 may be off ahead of the activation: statistics merged in any order, each of at most `terms`
    sums in a row."""
    n, c = x.shape[0], x.shape[-1]
    v = x.reshape(n, -1, groups, c // groups)
    mean = v.mean((1, 3), keepdims=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdims=True)
    r = 1 / np.sqrt(var + eps)
    y = ((v - mean) * r).reshape(x.shape)
    w, b = (1.0 if weight is None else weight.astype(np.float64)), (0.0 if bias is None else bias.astype(np.float64))
    z = y * w + b
    # A thread adds up to 256 values around the first of them, merges follow; a sum is off by (terms) u of the sum of its terms'
    # magnitudes, which are within the group's range around its mean: 600 u of that range for the mean, and relative to the
    # variance 2 * 600 u of range^2 / var at the outside.  Typical is the square root of that; ranges here are a few deviations.
    span = np.abs(v - mean).max((1, 3), keepdims=True)
    top = np.abs(v).max((1, 3), keepdims=True)
    terms = 600.0
    mean_off = U * (top + terms * np.sqrt(var))
    relative = U * (8 + terms / 4) + 0 * span
    off = ((mean_off + 2 * U * np.abs(v)) * r + np.abs((v - mean) * r) * relative).reshape(x.shape)
    return act64(z, act), after_act(z, act, off * np.abs(w) + U * (np.abs(y * w) * 2 + np.abs(z)))


NORMS = [((2, 8, 8, 1280), 32), ((1, 1, 1, 32), 8), ((3, 1, 64), 64), ((2, 5, 7, 30), 3), ((1, 37, 29, 15), 5), ((4, 33, 10), 1), ((2, 16, 16, 320), 32),
         ((1, 64, 48, 96), 32), ((5, 3, 3, 7), 7), ((2, 100, 1), 1), ((3, 17, 2), 2), ((1, 9, 9, 2560), 32), ((2, 4, 4, 4096), 32), ((1, 6, 8191), 1),
         ((1, 300, 1030), 10), ((2, 12), 4), ((1, 128, 128, 128), 32), ((20, 40, 24), 6), ((1, 3, 5000), 8), ((2, 11, 13, 1025), 5), ((1, 70, 50, 3), 1), ((1, 3, 3, 809), 1), ((3, 9, 9, 51), 1),
         ((8, 10, 10, 7), 1), ((1, 89, 89, 1059), 3), ((2, 5, 127, 138), 2), ((1, 2, 2, 8190), 3),
         ((1, 2, 8192), 8192), ((2, 3, 8192), 4096), ((1, 40, 8192), 1)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape,groups", NORMS)
def test_group_norm(torch, capi, name, shape, groups):
    rng = np.random.default_rng(sum(shape))
    c = shape[-1]
    x64 = rng.standard_normal(shape) * rng.uniform(0.5, 2.0, c) + rng.standard_normal(c)
    x = torch.from_numpy(x64).to(dtype(torch, name))
    x64 = x.double().numpy()
    w, b = (1 + 0.2 * rng.standard_normal(c)).astype(np.float32), (0.2 * rng.standard_normal(c)).astype(np.float32)
    act = ACTS[sum(shape) % len(ACTS)]
    want, error = norm64(x64, groups, w, b, 1e-5, act)
    got = capi.group_norm(x.cuda(), groups, torch.from_numpy(w).cuda(), torch.from_numpy(b).cuda(), 1e-5, act=act, slope=0.1)
    assert got.dtype == x.dtype
    close(torch, got, want, error, name)
    if name != "f16":
        want, error = norm64(x64, groups, None, None, 0.3, None)
        close(torch, capi.group_norm(x.cuda(), groups, epsilon=0.3), want, error, name)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("name", TYPES)
def test_group_norm_activations(torch, capi, name, act):
    rng = np.random.default_rng(21)
    x = torch.from_numpy(rng.standard_normal((2, 50, 48)) * 3).to(dtype(torch, name))
    w, b = (4 * rng.standard_normal(48)).astype(np.float32), rng.standard_normal(48).astype(np.float32)
    want, error = norm64(x.double().numpy(), 6, w, b, 1e-5, act)
    close(torch, capi.group_norm(x.cuda(), 6, torch.from_numpy(w).cuda(), torch.from_numpy(b).cuda(), act=act, slope=0.1), want, error, name)


def test_group_norm_strides(torch, capi):
    rng = np.random.default_rng(22)
    for name in TYPES:
        whole = torch.from_numpy(rng.standard_normal((3, 10, 12, 80))).to(dtype(torch, name)).cuda()
        planes = whole.permute(0, 3, 1, 2).contiguous(memory_format=torch.channels_last)
        for x in (whole[..., :48], whole[..., 5:70], whole[::2], whole[:, :, 3:9], whole[:, 2:7], planes.permute(0, 2, 3, 1), whole.transpose(1, 2),
                  whole[1:2].expand(4, 10, 12, 80), whole[..., ::2], whole[:0], whole[:, :0]):
            groups = 5 if x.shape[-1] % 5 == 0 else 4
            out = capi.group_norm(x, groups, act="silu")
            assert out.shape == x.shape and out.is_contiguous()
            # strides choose other ways to share the work, not other sums by more than their rounding
            want, error = norm64(x.double().cpu().numpy(), groups, None, None, 1e-5, "silu") if x.numel() else (np.zeros(x.shape), np.zeros(x.shape))
            close(torch, out, want, error, name)


@pytest.mark.parametrize("name", TYPES)
def test_group_norm_far_from_zero(torch, capi, name):
    """A mean a thousand deviations from zero, and one value a thousand deviations from the mean: sums of squares would cancel."""
    rng = np.random.default_rng(23)
    x = torch.from_numpy(rng.standard_normal((2, 40, 40, 16)) + 1000.0).to(dtype(torch, name))
    want, error = norm64(x.double().numpy(), 4, None, None, 1e-5, None)
    close(torch, capi.group_norm(x.cuda(), 4), want, error, name)
    x = torch.from_numpy(rng.standard_normal((2, 40, 40, 16))).to(dtype(torch, name))
    x[0, 0, 0, 0] = 1000.0
    x[1, 20, 3, 9] = -1000.0
    want, error = norm64(x.double().numpy(), 4, None, None, 1e-5, None)
    close(torch, capi.group_norm(x.cuda(), 4), want, error, name)


def test_group_norm_in_place(torch, capi):
    """Through the C ABI the result may take the tensor's place, in one launch and in two."""
    import ctypes
    rng = np.random.default_rng(25)
    for shape, groups in (((2, 8, 8, 320), 32), ((1, 5, 9, 60), 4), ((1, 200, 200, 24), 4), ((2, 90, 91, 13), 1), ((3, 1, 8192), 1)):
        for name, code in (("f32", 0), ("f16", 1), ("bf16", 2)):
            x = torch.from_numpy(rng.standard_normal(shape)).to(dtype(torch, name)).cuda()
            want = capi.group_norm(x, groups, act="silu")
            c = shape[-1]
            pixels = x[0].numel() // c
            g = capi.GroupNorm(shape[0], c, groups, code, pixels, pixels * c, c, capi._ptr(x), None, None, 1e-5, 5, 0.0)
            nbytes = capi.lib().tsx_group_norm_workspace_bytes(ctypes.byref(g))
            ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
            capi.check(capi.lib().tsx_group_norm_nhwc(ctypes.byref(g), capi._ptr(x), capi._ptr(ws), nbytes, capi._stream()))
            assert torch.equal(x, want)


def test_group_norm_of_large_images(torch, capi):
    """Outputs that go past the caches, and images of more than 2^32 bytes, channels in odd numbers among them."""
    for shape, groups, name in (((1, 1200, 1300, 40), 5, "bf16"), ((1, 1, (1 << 28) + 3, 9), 3, "bf16"), ((1, 1, (1 << 26) + 5, 24), 2, "f32")):
        x = torch.randn(shape, device="cuda", dtype=dtype(torch, name)).mul_(2).add_(0.5)
        out = capi.group_norm(x, groups, epsilon=1e-5)
        q, s = capi.group_norm_tokens(x, groups)
        d = shape[-1] // groups
        for g in range(groups):
            part = x[..., g * d:(g + 1) * d]
            count = part.numel()
            mean = sum(p.double().sum() for p in part.flatten(1, 2).split(1 << 24, 1)) / count
            variance = sum((p.double() - mean).square().sum() for p in part.flatten(1, 2).split(1 << 24, 1)) / count
            pixels = out.shape[1] * out.shape[2]
            for at in (0, pixels // 2, pixels - 1000):
                xs = part.flatten(1, 2)[:, at:at + 1000].double()
                want = ((xs - mean) / torch.sqrt(variance + 1e-5)).cpu().numpy()
                # the bar of norm64: threads add up to 2400 values here, sqrt(2400) / 2 roundings' worth, and 10^5 threads' errors average
                close(torch, out.flatten(1, 2)[:, at:at + 1000, g * d:(g + 1) * d], want, (600 + 160 * np.abs(want)) * U, name)
                got = q.flatten(1, 2)[:, at:at + 1000, g * d:(g + 1) * d].double() * s.flatten(1, 2)[:, at:at + 1000, None].double()
                step = s.flatten(1, 2)[:, at:at + 1000, None].double().cpu().numpy()
                assert (np.abs(got.cpu().numpy() - want) <= 0.501 * step + (600 + 160 * np.abs(want)) * U).all()


def test_group_norm_of_constants(torch, capi):
    """No variance: the bias, whatever the constant; epsilon keeps the rest finite."""
    for c, groups in ((64, 8), (15, 3)):
        x = torch.full((2, 9, 9, c), 3.0, device="cuda")
        b = torch.linspace(-1, 1, c, device="cuda")
        assert torch.equal(capi.group_norm(x, groups, None, b), b.expand(2, 9, 9, c))
        q, s = capi.group_norm_tokens(x, groups)
        assert (q == 0).all() and (s == 0).all()


def test_group_norm_nan_stays_in_its_group(torch, capi):
    rng = np.random.default_rng(24)
    for shape in ((2, 6, 6, 32), (2, 100, 100, 32)):
        x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()
        want = capi.group_norm(x, 4)
        x[0, 3, 3, 9] = math.nan
        x[1, 2, 2, 31] = math.inf
        got = capi.group_norm(x, 4)
        assert got[0, ..., 8:16].isnan().all() and got[1, ..., 24:].isnan().all()
        assert torch.equal(got[0, ..., :8], want[0, ..., :8]) and torch.equal(got[0, ..., 16:], want[0, ..., 16:]) and torch.equal(got[1, ..., :24], want[1, ..., :24])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape,groups", NORMS)
def test_group_norm_tokens(torch, capi, name, shape, groups):
    rng = np.random.default_rng(sum(shape) + 1)
    c = shape[-1]
    x = torch.from_numpy(rng.standard_normal(shape) * rng.uniform(0.5, 2.0, c) + rng.standard_normal(c)).to(dtype(torch, name))
    w, b = (1 + 0.2 * rng.standard_normal(c)).astype(np.float32), (0.2 * rng.standard_normal(c)).astype(np.float32)
    act = ACTS[(sum(shape) + 2) % len(ACTS)]
    want, error = norm64(x.double().numpy(), groups, w, b, 1e-5, act)
    q, s = capi.group_norm_tokens(x.cuda(), groups, torch.from_numpy(w).cuda(), torch.from_numpy(b).cuda(), 1e-5, act=act, slope=0.1)
    q, s = q.cpu().numpy().astype(np.float64), s.cpu().numpy().astype(np.float64)
    top = np.abs(want).max(-1)
    assert (np.abs(s * 127 - top) <= error.max(-1) + 2 * U * top).all()
    # half a step of the token's scale, and what the norm itself may be off (twice: the scale's too)
    assert (np.abs(q * s[..., None] - want) <= 0.5001 * s[..., None] + 2 * error + error.max(-1)[..., None]).all()
    assert (np.abs(q).max(-1)[top > 0] == 127).all()


# ---------------------------------------------------------------- a run of them together

@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape,groups,n", [((2, 8, 8, 320), 32, 960), ((1, 5, 9, 60), 4, 61), ((3, 1, 128), 8, 64), ((2, 20, 24, 130), 13, 260)])
def test_norm_tokens_product(torch, capi, name, shape, groups, n):
    """The block they make: norm, tokens, projection, and the projection's output normed again; the same product by hand."""
    rng = np.random.default_rng(n)
    c = shape[-1]
    x = torch.from_numpy(rng.standard_normal(shape)).to(dtype(torch, name)).cuda()
    w, sw, bias = weights(torch, rng, n, c)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())
    q, s = capi.group_norm_tokens(x, groups, act="silu")
    out = layer(q, x_scales=s, act="silu", out_dtype=x.dtype)
    want, error = product64(q.cpu().numpy(), s.cpu().numpy(), w, sw, bias, "silu")
    close(torch, out, want, error, name)
    assert torch.equal(capi.quantize_tokens(out)[0], capi.quantize_tokens(out.contiguous().clone())[0])
    again = capi.group_norm(out, 1, act="relu")
    want, error = norm64(out.double().cpu().numpy(), 1, None, None, 1e-5, "relu")
    close(torch, again, want, error, name)


def test_streams_graphs_and_repeats(torch, capi):
    """The block on a stream of its own and in two captured graphs replayed side by side, again and again, between eager calls:
    the same bits every time."""
    rng = np.random.default_rng(31)
    w, sw, bias = weights(torch, rng, 200, 96)
    layer = capi.TokenGemmI8(torch.from_numpy(w).cuda(), torch.from_numpy(sw).cuda(), torch.from_numpy(bias).cuda())

    def block(x):
        q, s = capi.group_norm_tokens(x, 8, act="silu")
        return layer(q, x_scales=s, out_dtype=x.dtype), layer(capi.group_norm(x, 8, act="relu")), capi.quantize_tokens(x)[0]

    for pixels in (3, 4000):
        xs = [torch.from_numpy(rng.standard_normal((2, pixels, 96))).to(torch.bfloat16).cuda() for _ in range(4)]
        want = [block(x) for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        held, graphs = [xs[0].clone(), xs[1].clone()], []
        for x, stream in zip(held, streams):
            with torch.cuda.stream(stream):
                for _ in range(2):
                    block(x)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = block(x)
            graphs.append((graph, out))
        for turn in range(4):
            for i in range(2):
                held[i].copy_(xs[(turn + i) % 4])
            torch.cuda.synchronize()
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i][0].replay()
            eager = block(xs[turn])
            torch.cuda.synchronize()
            for a, b in zip(eager, want[turn]):
                assert torch.equal(a, b)
            for i in range(2):
                for a, b in zip(graphs[i][1], want[(turn + i) % 4]):
                    assert torch.equal(a, b), (pixels, turn, i)
