"""Rows in microscaled 4-bit floating point against their definition in 64 bits: quantization and back, and the product on every kernel.

Codes and scales are compared bit for bit.  Products of two such values are exact in fp32, and so are sums of them where their magnitudes
together stay below 2^24 of their common step: there the product is compared bit for bit, too.  Otherwise: u = 2^-24; an instruction adds
64 products (128 of the one for few tokens) to a sum within 2 u of the magnitudes that meet there, eight partial sums and a bias are
joined within u each."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["f32", "f16", "bf16"]
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([GRID, -GRID])
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


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


def quantized64(x):
    """(code of each value, scale byte of each block) of x [m][k] in 64 bits."""
    m, k = x.shape
    padded = np.zeros((m, -(-k // 32) * 32))
    padded[:, :k] = x
    b = padded.reshape(m, -1, 32)
    fine = np.isfinite(b).all(-1)
    top = np.where(fine, np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1), 1.0)
    scale = np.where(top > 0, np.maximum(np.frexp(top)[1] - 1 - 2, -127), -127)
    size = np.abs(np.where(fine[..., None], b, 0.0)) * 2.0 ** -scale[..., None].astype(np.float64)
    code = np.zeros(b.shape, np.int64)
    for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):      # ties to even codes
        code += (size > border) if i % 2 == 0 else (size >= border)
    code += 8 * np.signbit(np.where(fine[..., None], b, 0.0))
    return code.reshape(m, -1)[:, :k], np.where(fine, scale + 127, 255).astype(np.uint8)


def packed(code):
    m, k = code.shape
    even = np.zeros((m, k + k % 2), np.int64)
    even[:, :k] = code
    return (even[:, 0::2] | even[:, 1::2] << 4).astype(np.uint8)


def unpacked(codes, k):
    return np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)[:, :k].astype(np.int64)


def values64(code, scales):
    """What codes [m][k] and scale bytes stand for."""
    k = code.shape[1]
    by = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return VALUES[code] * np.repeat(by, 32, 1)[:, :k]


def as_type(torch, x, name):
    """64-bit values as the type holds them: (device tensor, in 64 bits)."""
    t = torch.from_numpy(x).to(dtype(torch, name))
    return t.cuda(), t.double().numpy()


def check_quantized(torch, capi, x, x64, name):
    codes, scales = capi.quantize_mxfp4(x)
    m, k = x64.shape
    ec, es = quantized64(x64)
    assert codes.dtype == scales.dtype == torch.uint8 and codes.shape == (m, (k + 1) // 2) and scales.shape == (m, (k + 31) // 32)
    assert np.array_equal(scales.cpu().numpy(), es)
    assert np.array_equal(codes.cpu().numpy(), packed(ec))
    for to in (name, "f32"):
        back = capi.dequantize_mxfp4(codes, scales, k=k, dtype=dtype(torch, to)).cpu()
        want = torch.from_numpy(values64(ec, es)).to(torch.float32).to(dtype(torch, to))
        assert back.shape == (m, k) and torch.equal(torch.isnan(back), torch.isnan(want)) and torch.equal(back.nan_to_num(nan=1.0), want.nan_to_num(nan=1.0))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 7), (1, 8), (2, 9), (1, 4096), (3, 31), (5, 32), (300, 33), (65, 511), (64, 512), (33, 513), (7, 2047), (2, 32771),
                                 (4000, 1), (1111, 40), (777, 1000), (513, 4096), (4099, 4160), (9000, 2050)])
def test_quantize(torch, capi, name, m, k):
    rng = np.random.default_rng(m + k)
    x = rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)) + 2 * rng.standard_normal((1, k)))
    x, x64 = as_type(torch, x, name)
    check_quantized(torch, capi, x, x64, name)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_every_scale_and_border(torch, capi, name):
    """Each power of two as a block's scale, with values on, just below and just above every border."""
    e = {"f32": (-149, 128), "bf16": (-133, 128), "f16": (-24, 16)}[name]
    sixteenths = np.concatenate([np.arange(0, 128), np.arange(1, 128)]) / 16.0
    rows = []
    for power in range(e[0] - 2, e[1] - 2):
        for part in np.array_split(sixteenths, 9):
            near = np.concatenate([part, -part * (1 + 2.0 ** -8), part * (1 - 2.0 ** -8)])[:31]
            rows.append(np.concatenate([near * 2.0 ** power, np.zeros(31 - len(near)), [4.0 * 2.0 ** power]]))
    with np.errstate(over="ignore"):
        x, x64 = as_type(torch, np.array(rows), name)
    check_quantized(torch, capi, x, x64, name)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_special_blocks(torch, capi, name):
    t = dtype(torch, name)
    big, small = torch.finfo(t).max, SMALLEST[name]
    rows = np.zeros((9, 70))
    rows[1] = -0.0
    rows[2, 3], rows[2, 40] = math.inf, 5.0
    rows[3, 69], rows[3, 1] = math.nan, 2.0
    rows[4, :] = big
    rows[5, ::2], rows[5, 1::2] = small, -3 * small
    rows[6, :33] = np.arange(33) * small
    rows[7, 31], rows[7, 32] = -math.inf, -6.0
    rows[8, 0], rows[8, 1] = 1.0, small
    x, x64 = as_type(torch, rows, name)
    check_quantized(torch, capi, x, x64, name)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_strides(torch, capi, name):
    rng = np.random.default_rng(4)
    wide, wide64 = as_type(torch, rng.standard_normal((37, 300)), name)
    three, three64 = as_type(torch, rng.standard_normal((4, 5, 96)), name)
    for x, x64 in ((wide[:, 3:204], wide64[:, 3:204]), (wide[::3, :130], wide64[::3, :130]), (wide.t(), wide64.T), (wide[5:6, 1:], wide64[5:6, 1:]),
                   (wide[:1, :64].expand(6, 64), np.repeat(wide64[:1, :64], 6, 0))):
        check_quantized(torch, capi, x, x64, name)
    for x, x64 in ((three, three64), (three[:, 1:4, 5:77], three64[:, 1:4, 5:77]), (three.transpose(0, 1), three64.transpose(1, 0, 2)), (three[:0], three64[:0])):
        codes, scales = capi.quantize_mxfp4(x)
        assert codes.shape == x.shape[:-1] + (x.shape[-1] // 2,) and scales.shape == x.shape[:-1] + (-(-x.shape[-1] // 32),) or x.shape[-1] % 2
        if x.numel():
            ec, es = quantized64(x64.reshape(-1, x64.shape[-1]))
            assert np.array_equal(codes.cpu().numpy().reshape(len(ec), -1), packed(ec)) and np.array_equal(scales.cpu().numpy().reshape(len(es), -1), es)
        assert capi.dequantize_mxfp4(codes, scales, k=x.shape[-1]).shape == x.shape
    # codes and scales at strides of their own, at odd addresses
    codes, scales = capi.quantize_mxfp4(wide)
    room = torch.zeros((37, 161), dtype=torch.uint8, device="cuda")
    room[:, 3:153] = codes
    scale_room = torch.zeros((37, 13), dtype=torch.uint8, device="cuda")
    scale_room[:, 1:11] = scales
    assert torch.equal(capi.dequantize_mxfp4(room[:, 3:153], scale_room[:, 1:11]), capi.dequantize_mxfp4(codes, scales))


def test_rows_behind_the_last_value_stay(torch, capi):
    """Bytes of a wider buffer beside and behind the rows are left as they were."""
    x = torch.randn((5, 41), device="cuda")
    codes = torch.full((7, 30), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((7, 5), 0xCD, dtype=torch.uint8, device="cuda")
    capi.check(capi.lib().tsx_quantize_mxfp4(5, 41, x.data_ptr(), 0, 41, codes.data_ptr(), 30, scales.data_ptr(), 5, capi._stream()))
    ec, es = capi.quantize_mxfp4(x)
    assert torch.equal(codes[:5, :21], ec) and torch.equal(scales[:5, :2], es)
    assert (codes[:, 21:] == 0xAB).all() and (codes[5:] == 0xAB).all() and (scales[:, 2:] == 0xCD).all() and (scales[5:] == 0xCD).all()
    out = torch.full((7, 50), 3.0, device="cuda")
    capi.check(capi.lib().tsx_dequantize_mxfp4(5, 41, ec.data_ptr(), 21, es.data_ptr(), 2, out.data_ptr(), 0, 50, capi._stream()))
    assert torch.equal(out[:5, :41], capi.dequantize_mxfp4(ec, es, k=41)) and (out[:, 41:] == 3.0).all() and (out[5:] == 3.0).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (2, 3, 4096), (70, 1001), (2100, 4100)])
def test_dequantize_tokens(torch, capi, name, shape):
    """One fp32 product a value, rounded to the type once more."""
    torch.manual_seed(3)
    q = torch.randint(-128, 128, shape, dtype=torch.int8)
    scales = torch.rand(shape[:-1]) * 0.01
    scales.view(-1)[0] = math.nan
    got = capi.dequantize_tokens(q.cuda(), scales.cuda(), dtype=dtype(torch, name)).cpu()
    want = (q.float() * scales[..., None]).to(dtype(torch, name))
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
    wide = torch.zeros(shape[:-1] + (shape[-1] + 5,), dtype=torch.int8, device="cuda")
    wide[..., 3:3 + shape[-1]] = q.cuda()
    assert torch.equal(capi.dequantize_tokens(wide[..., 3:3 + shape[-1]], scales.cuda()).nan_to_num(nan=7.0), (q.float() * scales[..., None]).cuda().nan_to_num(nan=7.0))


# ---------------------------------------------------------------- the product

KERNELS = ["0", "1", "2", "3", "4", "5"]


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
    """The error of act(y) in fp32 where y is off by `error`: slopes within 1.1, and their own exponential, reciprocal and roundings."""
    if act in ("silu", "mish_fast"):
        return 1.1 * error + (12 * np.abs(y) + y * y / 2) * U
    return error + np.abs(y) * U


def random_rows(rng, m, k, scales=(126, 130)):
    """Random codes [m][k] and scale bytes: what they stand for is a multiple of 2^-2 of a step ..."""
    return rng.integers(0, 16, (m, k)), rng.integers(*scales, (m, -(-k // 32))).astype(np.uint8)


def device(torch, code, scales):
    return torch.from_numpy(packed(code)).cuda(), torch.from_numpy(scales).cuda()


SHAPES = [(1, 1, 1), (1, 16, 32), (1, 33, 31), (2, 17, 33), (5, 300, 129), (16, 64, 128), (16, 1000, 2048), (17, 40, 65), (33, 129, 1500), (64, 65, 256), (65, 64, 384),
          (100, 200, 300), (129, 257, 1000), (255, 300, 640), (300, 513, 4096), (513, 255, 96)]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_is_exact(torch, capi, monkeypatch, kernel, m, n, k):
    """Sums that fp32 holds, rounded once: every kernel, on codes."""
    monkeypatch.setenv("TSX_MXFP4_KERNEL", kernel)
    rng = np.random.default_rng(m * n + k)
    xc, xs = random_rows(rng, m, k)
    wc, ws = random_rows(rng, n, k)
    x, w = values64(xc, xs), values64(wc, ws)
    assert (np.abs(x) @ np.abs(w).T).max() < 2.0 ** 20      # in steps of 2^-4: 24 bits
    layer = capi.TokenGemmMxfp4(*device(torch, wc, ws), k=k)
    x_dev, s_dev = device(torch, xc, xs)
    for name in TYPES:
        got = layer(x_dev, x_scales=s_dev, out_dtype=dtype(torch, name))
        want = torch.from_numpy(x @ w.T).float().to(dtype(torch, name))
        assert got.dtype == dtype(torch, name) and torch.equal(got.cpu(), want), name


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_of_floats(torch, capi, name, m, n, k):
    """Rows quantized by the call: the same bits as from codes."""
    rng = np.random.default_rng(m + n + k)
    x, x64 = as_type(torch, rng.standard_normal((m, k + 3)) * np.exp(rng.standard_normal((m, 1))), name)
    x, x64 = x[:, 1:k + 1], x64[:, 1:k + 1]
    w = rng.standard_normal((n, k))
    bias = rng.standard_normal(n).astype(np.float32)
    layer = capi.TokenGemmMxfp4.from_float(torch.from_numpy(w).float().cuda(), torch.from_numpy(bias).cuda())
    xv, wv = (values64(*quantized64(v)) for v in (x64, w.astype(np.float32).astype(np.float64)))
    exact, size = xv @ wv.T + bias, np.abs(xv) @ np.abs(wv).T + np.abs(bias)
    error = (2 * (k // 64 + 2) + 9) * U * size
    codes = capi.quantize_mxfp4(x)
    for act in (None, "relu", "leaky_relu", "silu", "mish_fast"):
        for out in (layer(x, act=act, slope=0.1), layer(codes[0], x_scales=codes[1], act=act, slope=0.1, out_dtype=dtype(torch, name))):
            want, e = act64(exact, act), after_act(exact, act, error)
            h = torch.finfo(dtype(torch, name)).eps / 2
            off = np.abs(out.double().cpu().numpy() - want) - (e * (1 + h) + h * np.abs(want) + SMALLEST[name])
            assert off.max() <= 0, (act, off.max())


@pytest.mark.parametrize("kernel", KERNELS)
def test_product_of_special_rows(torch, capi, monkeypatch, kernel):
    """A block that is not a number makes its row or column so and no other; rows of zeros; the least and largest scales."""
    monkeypatch.setenv("TSX_MXFP4_KERNEL", kernel)
    rng = np.random.default_rng(8)
    m, n, k = 70, 90, 200
    xc, xs = random_rows(rng, m, k)
    wc, ws = random_rows(rng, n, k)
    xs[3, 6], xs[69, 0], ws[17, 2], ws[89, 6] = 255, 255, 255, 255
    xc[5], xs[5] = 0, 0
    xs[7], xs[8] = 0, 250
    ws[9], ws[10] = 250, 3
    xc[7], wc[9] = rng.integers(1, 8, k), rng.integers(1, 8, k)      # positive: their sum does not cancel
    layer = capi.TokenGemmMxfp4(*device(torch, wc, ws), k=k)
    got = layer(device(torch, xc, xs)[0], x_scales=device(torch, xc, xs)[1]).double().cpu().numpy()
    want = values64(xc, xs) @ values64(wc, ws).T
    nan = np.zeros((m, n), bool)
    nan[[3, 69]] = True
    nan[:, [17, 89]] = True
    size = np.abs(values64(xc, xs)) @ np.abs(values64(wc, ws)).T
    with np.errstate(invalid="ignore"):
        beyond = size > 2.0 ** 127      # sums on their way leave fp32, in both directions: an infinity, or one less another
        assert beyond[8, 9] and not np.isfinite(got[8, 9]) and not np.delete(np.delete(beyond, 8, 0), 9, 1).any()
        assert np.array_equal(np.isnan(got)[~beyond], nan[~beyond])
        fine = ~nan & ~beyond
        # behind 2^-126 the matrix cores may keep nothing
        assert (np.abs(got - want)[fine] <= 20 * U * size[fine] + 2.0 ** -126).all()
        assert (got[5][~nan[5]] == 0).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 40, 200), (16, 300, 1500), (60, 64, 256), (300, 2000, 640)])
def test_product_of_floats_beside_bad_rows(torch, capi, name, m, n, k):
    """Infinities and NaN in rows that the call quantizes: those rows are not numbers, the others what they are alone."""
    torch.manual_seed(m)
    layer = capi.TokenGemmMxfp4.from_float(torch.randn((n, k), device="cuda"), torch.randn(n, device="cuda"))
    x = torch.randn((m, k)).to(dtype(torch, name))
    good = x.clone()
    bad = sorted({0, m - 1, m // 2})
    for row, (at, value) in zip(bad, ((0, math.inf), (k - 1, math.nan), (k // 2, -math.inf))):
        x[row, at], good[row] = value, 0.0
    got, want = layer(x.cuda()).cpu(), layer(good.cuda()).cpu()
    for row in range(m):
        assert torch.isnan(got[row]).all() if row in bad else torch.equal(got[row], want[row]), row


@pytest.mark.parametrize("name", TYPES)
def test_two_streams_at_once(torch, capi, name):
    """One layer, calls in turn on two streams that nothing orders: each with a workspace of its own."""
    layer = capi.TokenGemmMxfp4.from_float(torch.randn((3000, 520), device="cuda"))
    inputs = [torch.randn((m, 520), device="cuda").to(dtype(torch, name)) for m in (700, 650)]
    want = [layer(x) for x in inputs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer(inputs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_product_of_strided_rows(torch, capi):
    """Rows and scales at strides of their own, aligned and not, read in place and copied."""
    rng = np.random.default_rng(9)
    n, k = 130, 256
    wc, ws = random_rows(rng, n, k)
    layer = capi.TokenGemmMxfp4(*device(torch, wc, ws))
    for m in (1, 7, 100, 300):
        xc, xs = random_rows(rng, m, k)
        codes, scales = device(torch, xc, xs)
        want = torch.from_numpy(values64(xc, xs) @ values64(wc, ws).T).float()
        for wide, at, s_wide, s_at in ((128, 0, 8, 0), (160, 16, 12, 4), (160, 1, 12, 4), (129, 0, 8, 0), (160, 16, 11, 1), (144, 8, 9, 0)):
            room = torch.full((m, wide), 0x77, dtype=torch.uint8, device="cuda")
            room[:, at:at + 128] = codes
            s_room = torch.full((m, s_wide), 255, dtype=torch.uint8, device="cuda")
            s_room[:, s_at:s_at + 8] = scales
            got = layer(room[:, at:at + 128], x_scales=s_room[:, s_at:s_at + 8])
            assert torch.equal(got.cpu(), want), (m, wide, at, s_wide, s_at)
    xc, xs = random_rows(rng, 12, k)
    codes, scales = device(torch, xc, xs)
    got = layer(codes.view(3, 4, 128), x_scales=scales.view(3, 4, 8))
    assert got.shape == (3, 4, n) and torch.equal(got.view(12, n), layer(codes, x_scales=scales))
    assert layer(codes[:0], x_scales=scales[:0]).shape == (0, n) and layer(torch.zeros((0, k), device="cuda")).shape == (0, n)
    # weights at strides of their own
    room = torch.zeros((n, 140), dtype=torch.uint8, device="cuda")
    room[:, 5:133] = device(torch, wc, ws)[0]
    other = capi.TokenGemmMxfp4(room[:, 5:133], device(torch, wc, ws)[1])
    assert torch.equal(other.packed, layer.packed)


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("k", [1, 31, 129, 1023])
def test_codes_behind_odd_rows_are_not_used(torch, capi, m, k):
    """The upper half of an odd row's last byte may hold anything, in rows and in weights."""
    rng = np.random.default_rng(k)
    xc, xs = random_rows(rng, m, k)
    wc, ws = random_rows(rng, 50, k)
    (codes, scales), (w_codes, w_scales) = device(torch, xc, xs), device(torch, wc, ws)
    want = torch.from_numpy(values64(xc, xs) @ values64(wc, ws).T).float()
    codes[:, -1] |= 0x70
    w_codes[:, -1] |= 0xF0
    assert torch.equal(capi.TokenGemmMxfp4(w_codes, w_scales, k=k)(codes, x_scales=scales).cpu(), want)
    assert torch.equal(capi.dequantize_mxfp4(codes, scales, k=k).cpu(), torch.from_numpy(values64(xc, xs)).float())


@pytest.mark.parametrize("kernel,m,n,k", [("3", 1, 40, 5888), ("3", 130, 140, 6016), ("3", 300, 129, 6144), ("4", 3, 300, 4096), ("4", 257, 130, 3584), ("4", 300, 513, 4480),
                                          (None, 2048, 4096, 4352)])
def test_product_of_long_rows_with_scales_apart(torch, capi, monkeypatch, kernel, m, n, k):
    """Scales of long rows, which are turned first: exact sums, from rows at strides of their own too, of which nothing behind the scales is used."""
    if kernel:
        monkeypatch.setenv("TSX_MXFP4_KERNEL", kernel)
    rng = np.random.default_rng(m + k)
    xc, xs = random_rows(rng, m, k, scales=(126, 128))
    wc, ws = random_rows(rng, n, k, scales=(126, 128))      # values of at most 6, in steps of 1/4
    assert k * 36 * 16 < 2 ** 24
    layer = capi.TokenGemmMxfp4(*device(torch, wc, ws))
    codes, scales = device(torch, xc, xs)
    x, w = (torch.from_numpy(values64(*v)).cuda() for v in ((xc, xs), (wc, ws)))
    want = (x @ w.t().contiguous()).float()
    assert torch.equal(layer(codes, x_scales=scales), want)
    room = torch.full((m + 1, k // 32 + 12), 255, dtype=torch.uint8, device="cuda")
    room[:m, 4:4 + k // 32] = scales
    assert torch.equal(layer(codes, x_scales=room[:m, 4:4 + k // 32]), want)


@pytest.mark.parametrize("m,n,k,name", [(8300, 4099, 96, "bf16"), (4096, 8192, 130, "f16"), (5000, 4096, 256, "f32"), (70000, 130, 64, "bf16")])
def test_large_outputs(torch, capi, m, n, k, name):
    """Many tiles, inside and across the edges, outputs of more than the caches hold: exact sums again."""
    rng = np.random.default_rng(k)
    wc, ws = random_rows(rng, n, k)
    xc, xs = random_rows(rng, m, k)
    layer = capi.TokenGemmMxfp4(*device(torch, wc, ws), k=k)
    codes, scales = device(torch, xc, xs)
    bias = torch.randint(-8, 8, (n,)).float().cuda()
    layer.bias = bias
    x, w = (torch.from_numpy(values64(*v)).cuda() for v in ((xc, xs), (wc, ws)))
    want = ((x @ w.t().contiguous()) + bias.double()).clamp(min=0.0).float().to(dtype(torch, name))
    assert torch.equal(layer(codes, x_scales=scales, act="relu", out_dtype=dtype(torch, name)), want)


def test_product_leaves_its_inputs_and_repeats(torch, capi):
    """The same bits from call to call, inputs as they were."""
    x = torch.randn((100, 1000), device="cuda").bfloat16()
    layer = capi.TokenGemmMxfp4.from_float(torch.randn((300, 1000), device="cuda"))
    before, first = x.clone(), layer(x)
    for _ in range(5):
        assert torch.equal(layer(x), first)
    assert torch.equal(x, before)


def test_product_on_other_streams_and_in_a_graph(torch, capi):
    layer = capi.TokenGemmMxfp4.from_float(torch.randn((512, 640), device="cuda"))
    inputs = [torch.randn((m, 640), device="cuda").half() for m in (1, 40, 300)]
    want = [layer(x) for x in inputs]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [layer(x) for x in inputs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    fixed = [x.clone() for x in inputs]
    with torch.cuda.graph(graph):
        outs = [layer(x) for x in fixed]
        outs.append(layer(*capi.quantize_mxfp4(fixed[2]), out_dtype=torch.float16))
        outs.append(capi.dequantize_mxfp4(*capi.quantize_mxfp4(fixed[1])))
    for turn in range(3):
        for f in fixed:
            f.copy_(torch.randn_like(f))
        graph.replay()
        torch.cuda.synchronize()
        eager = [layer(x) for x in fixed]
        eager += [layer(*capi.quantize_mxfp4(fixed[2]), out_dtype=torch.float16), capi.dequantize_mxfp4(*capi.quantize_mxfp4(fixed[1]))]
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), turn


def test_long_rows(torch, capi):
    """K of many chunks, on tiles and on few tokens; and a buffer of more than 2^31 values."""
    rng = np.random.default_rng(2)
    for m, n, k in ((3, 20, 40000), (80, 70, 33000)):
        xc, xs = random_rows(rng, m, k, (127, 128))
        wc, ws = random_rows(rng, n, k, (127, 128))
        x, w = values64(xc, xs), values64(wc, ws)
        assert (np.abs(x) @ np.abs(w).T).max() < 2.0 ** 22      # in steps of 2^-2
        layer = capi.TokenGemmMxfp4(*device(torch, wc, ws), k=k)
        codes, scales = device(torch, xc, xs)
        assert torch.equal(layer(codes, x_scales=scales).cpu(), torch.from_numpy(x @ w.T).float())
    big = torch.zeros((66000, 33000), dtype=torch.bfloat16, device="cuda")
    big[-2:] = torch.randn((2, 33000), device="cuda").bfloat16()
    codes, scales = capi.quantize_mxfp4(big)
    ec, es = capi.quantize_mxfp4(big[-2:].clone())
    assert torch.equal(codes[-2:], ec) and torch.equal(scales[-2:], es) and not codes[:-2].any()
    back = capi.dequantize_mxfp4(codes, scales, dtype=torch.bfloat16)
    assert torch.equal(back[-2:], capi.dequantize_mxfp4(ec, es, dtype=torch.bfloat16)) and not back[:-2].any()


def test_python_calls_refuse(torch, capi):
    """What the calls say about operands that do not fit each other."""
    codes, scales = capi.quantize_mxfp4(torch.randn((6, 70), device="cuda"))
    layer = capi.TokenGemmMxfp4(codes, scales, k=70)
    x = torch.randn((4, 70), device="cuda")
    xc, xs = capi.quantize_mxfp4(x)
    for call, word in ((lambda: capi.dequantize_mxfp4(codes, scales, k=72), "shape"), (lambda: capi.dequantize_mxfp4(codes, scales[:, :2]), "shape"),
                       (lambda: capi.dequantize_mxfp4(codes[:5], scales), "shape"), (lambda: capi.dequantize_mxfp4(codes, scales.float()), "float32"),
                       (lambda: capi.TokenGemmMxfp4(codes, scales, k=64), "shape"), (lambda: capi.TokenGemmMxfp4(codes[0], scales[0]), "shape"),
                       (lambda: capi.TokenGemmMxfp4(codes, scales, bias=torch.zeros(5, device="cuda")), "values"), (lambda: layer(x[:, :69]), "weights of 70"),
                       (lambda: layer(xc), "come with their scales"), (lambda: layer(x, x_scales=xs), "come with their scales"), (lambda: layer(xc, x_scales=xs[:, :2]), "shape"),
                       (lambda: layer(xc, x_scales=xs[:3]), "shape"), (lambda: layer(x, act="mish"), "activation"), (lambda: layer(x, out_dtype=torch.int8), "output type"),
                       (lambda: layer(x.double()), "float64"), (lambda: capi.quantize_mxfp4(x.to(torch.int8)), "int8"), (lambda: capi.quantize_mxfp4(x[:, :0]), "shape"),
                       (lambda: capi.rms_norm(x, torch.ones(69, device="cuda")), "values"), (lambda: capi.rms_norm(x, residual=x.half()), "float16"),
                       (lambda: capi.rms_norm(x, residual=x[:3]), "residual of shape"), (lambda: capi.rms_norm(x, epsilon=-1.0), "epsilon"),
                       (lambda: capi.rms_norm_tokens(x[:, :0]), "shape"), (lambda: capi.dequantize_tokens(x.to(torch.int8), x[:3, 0]), "values"),
                       (lambda: capi.dequantize_tokens(x.to(torch.int8), None), "scales")):
        with pytest.raises(capi.TsxError, match=word):
            call()
