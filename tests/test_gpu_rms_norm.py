"""Root-mean-square norm of rows, with the residual's addition: to its own type, to int8 tokens and to MXFP4 rows, and the products
behind them.

u = 2^-24.  The sum of squares has only positive terms: two chains of at most 16 fused steps in a thread, a join, six between lanes,
16 between wavefronts, 40 roundings in all; its mean two more; the root halves that, 21 u, and adds two (v_rsq_f32 is within a step);
y is two products: 25 u, taken as R = 30 u.  int8 codes do not depend on the root: they are the definition's bits."""
import math

import numpy as np
import pytest

from tests.test_gpu_mxfp4 import SMALLEST, TYPES, U, VALUES, dtype, quantized64, unpacked, values64
from tests.test_gpu_tokens import tokens64

pytestmark = pytest.mark.gpu

R = 30 * U
EPS = 1e-6


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


def inputs(torch, rng, m, k, name, residual=True):
    t = dtype(torch, name)
    x = torch.from_numpy(rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))).to(t)
    r = torch.from_numpy(rng.standard_normal((m, k))).to(t) if residual else None
    w = torch.from_numpy(1.0 + 0.3 * rng.standard_normal(k)).float()
    return x, r, w


def summed(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def norm64(h, w, epsilon=EPS):
    h = h.double().numpy()
    with np.errstate(all="ignore"):
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + float(np.float32(epsilon)))
        return y if w is None else y * w.double().numpy()


def cuda(*t):
    return [None if v is None else v.cuda() for v in t]


def same(torch, a, b):
    return torch.equal(a.cpu(), b.cpu())


def check_rows(torch, capi, x, r, w, name, epsilon=EPS):
    dx, dr, dw = cuda(x, r, w)
    out = capi.rms_norm(dx, dw, epsilon, residual=dr)
    h = summed(x, r)
    if r is not None:
        out, total = out
        assert total.dtype == x.dtype and same(torch, total, h)
    want = norm64(h, w, epsilon)
    half = torch.finfo(dtype(torch, name)).eps / 2
    got = out.double().cpu().numpy()
    assert out.dtype == x.dtype and got.shape == want.shape
    zeros = np.broadcast_to((epsilon == 0.0) & (h.double().numpy() == 0).all(-1, keepdims=True), want.shape)      # 0 / 0, in the formula too
    off = (np.abs(got - want) - ((R + half * (1 + R)) * np.abs(want) + SMALLEST[name]))[~zeros]
    assert np.array_equal(np.isnan(got), zeros) and off.max() <= 0, off.max()


def check_tokens(torch, capi, x, r, w, epsilon=EPS):
    dx, dr, dw = cuda(x, r, w)
    q, scales, *total = capi.rms_norm_tokens(dx, dw, epsilon, residual=dr)
    h = summed(x, r)
    assert len(total) == (r is not None) and all(same(torch, t, h) for t in total)
    v = h.float() if w is None else h.float() * w
    eq, _ = tokens64(v.double().numpy())
    assert q.dtype == torch.int8 and q.shape == x.shape and np.array_equal(q.cpu().numpy(), eq)
    want = np.abs(norm64(h, w, epsilon)).max(-1) / 127.0
    assert scales.dtype == torch.float32 and scales.shape == x.shape[:-1]
    zeros = (epsilon == 0.0) & (h.double().numpy() == 0).all(-1)
    got = scales.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), zeros) and (np.abs(got - want) <= (R + 2 * U) * want + 2.0 ** -149)[~zeros].all()


def check_mxfp4(torch, capi, x, r, w, epsilon=EPS):
    dx, dr, dw = cuda(x, r, w)
    codes, scales, *total = capi.rms_norm_mxfp4(dx, dw, epsilon, residual=dr)
    h = summed(x, r)
    m, k = x.shape
    assert len(total) == (r is not None) and all(same(torch, t, h) for t in total)
    assert codes.shape == (m, (k + 1) // 2) and scales.shape == (m, (k + 31) // 32)
    y = norm64(h, w, epsilon)
    low, high = quantized64(y * (1 - R))[1], quantized64(y * (1 + R))[1]
    s = scales.cpu().numpy()
    assert ((s == low) | (s == high)).all()
    by = np.repeat(2.0 ** (s.astype(np.float64) - 127), 32, 1)[:, :k]
    code = unpacked(codes.cpu().numpy(), k)
    got = np.abs(VALUES[code])
    def nearest(size):
        place = np.zeros(size.shape, np.int64)
        for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
            place += (size > border) if i % 2 == 0 else (size >= border)
        return VALUES[place]
    assert (nearest(np.abs(y) / by * (1 - R)) <= got).all() and (got <= nearest(np.abs(y) / by * (1 + R))).all()
    assert np.array_equal(code >= 8, np.signbit(y))


SIZES = [(1, 1), (3, 2), (2, 7), (5, 8), (70, 31), (9, 33), (200, 128), (65, 129), (64, 512), (33, 513), (7, 1000), (5, 1025), (1, 2048), (3, 2049), (1, 4096), (64, 4096),
         (2, 4100), (1, 8192), (2, 8197), (1, 16384), (2, 16390), (1, 40001), (600, 600), (513, 1024), (700, 2047), (520, 4096)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,k", SIZES)
def test_norm(torch, capi, name, m, k):
    rng = np.random.default_rng(m + k)
    x, r, w = inputs(torch, rng, m, k, name)
    check_rows(torch, capi, x, r, w, name)
    check_rows(torch, capi, x, None, None, name)
    check_tokens(torch, capi, x, r, w)
    check_tokens(torch, capi, x, None, None)
    check_mxfp4(torch, capi, x, r, w)
    check_mxfp4(torch, capi, x, None, None)


@pytest.mark.parametrize("m,k,name", [(1100001, 7, "bf16"), (1100003, 1, "f16"), (270001, 20, "bf16"), (140001, 40, "bf16"), (40001, 200, "f16"),
                                      (66001, 100, "f16"), (16999, 300, "f32"), (17003, 700, "bf16"), (4500, 2000, "f16"), (4501, 2500, "bf16"), (4500, 2200, "f32"),
                                      (4501, 3500, "bf16"), (1100, 5000, "f16"), (1027, 8000, "f32"), (600, 9001, "bf16"), (530, 17000, "f16")])
def test_many_rows(torch, capi, m, k, name):
    """More rows than a launch has workgroups: these take several, one behind the other; a few of them in 2^-70 and 2^70 steps in fp32 and bf16."""
    rng = np.random.default_rng(k)
    x, r, w = inputs(torch, rng, m, k, name)
    if name != "f16":
        for part in (x, r):
            part[7::997] *= 2.0 ** 70
            part[8::991] *= 2.0 ** -70
    check_rows(torch, capi, x, r, w, name, 0.0)
    check_tokens(torch, capi, x, r, w, 0.0)
    check_mxfp4(torch, capi, x, None, w, 0.0)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [5, 100, 1000, 4096, 20000])
def test_strides(torch, capi, name, k):
    """Rows of x and of the residual at strides of their own, at odd addresses; more axes; none at all."""
    rng = np.random.default_rng(k)
    x, r, w = inputs(torch, rng, 12, k, name)
    wide_x, wide_r = torch.zeros((12, k + 9), dtype=x.dtype, device="cuda"), torch.zeros((24, k + 3), dtype=x.dtype, device="cuda")
    wide_x[:, 1:k + 1], wide_r[::2, 3:] = x.cuda(), r.cuda()
    w_room = torch.zeros(k + 1, device="cuda")
    w_room[1:] = w.cuda()
    dx, dr, dw = cuda(x, r, w)
    for call in (capi.rms_norm, capi.rms_norm_tokens, capi.rms_norm_mxfp4):
        want = call(dx, dw, EPS, residual=dr)
        for got in (call(wide_x[:, 1:k + 1], w_room[1:], EPS, residual=wide_r[::2, 3:]), call(dx.t().contiguous().t(), dw, EPS, residual=dr)):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = call(dx.view(3, 4, k), dw, EPS, residual=dr.view(3, 4, k))
        assert all(a.shape[:2] == (3, 4) and torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
        got = call(dx[:0], dw, EPS, residual=dr[:0])
        assert all(t.shape[0] == 0 for t in got)
        one = call(dx[0], dw, EPS, residual=dr[0])
        assert all(torch.equal(a, b) for a, b in zip(one, call(dx[:1].clone(), dw, EPS, residual=dr[:1].clone()))) or one[0].shape != dx[:1].shape
    assert torch.equal(capi.rms_norm(dx, dw.double()), capi.rms_norm(dx, dw)) or name      # another type of the weight is converted


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [3, 40, 700, 5000, 17000])
def test_sizes_that_leave_fp32_when_squared(torch, capi, name, k):
    """Rows of the largest and smallest numbers: scaled, not lost."""
    if name == "f16":
        big, small = 65504.0, 2.0 ** -24
    else:
        big, small = 2.0 ** 127, SMALLEST[name]
    rng = np.random.default_rng(k)
    rows = rng.uniform(0.5, 1.0, (6, k)) * rng.choice([-1.0, 1.0], (6, k))
    rows[0] *= big
    rows[1] = np.where(np.arange(k) == k // 2, big, rows[1])
    rows[2] *= small * 64
    rows[3] = np.where(np.arange(k) == k - 1, small, 0.0)
    rows[4] *= 2.0 ** -60 if name != "f16" else 2.0 ** -10
    x = torch.from_numpy(rows).to(dtype(torch, name))
    for epsilon in (0.0, 1e-6, 1e-37):
        check_rows(torch, capi, x, None, None, name, epsilon)
        h = x.double().numpy()
        q, scales = capi.rms_norm_tokens(x.cuda(), None, epsilon)
        assert np.array_equal(q.cpu().numpy(), tokens64(h)[0])
        want = np.abs(norm64(x, None, epsilon)).max(-1) / 127.0
        assert (np.abs(scales.double().cpu().numpy() - want) <= (R + 2 * U) * want + 2.0 ** -149).all()
        check_mxfp4(torch, capi, x, None, None, epsilon)


@pytest.mark.parametrize("k", [24, 700, 5000, 17000])
def test_weights_that_leave_fp32_times_the_row(torch, capi, k):
    """Rows and weights whose products are beyond fp32 or below its normal numbers, where the norm itself is not."""
    rng = np.random.default_rng(k)
    x = torch.from_numpy(rng.standard_normal((3, k)) * np.array([[1e15], [1e-17], [1.0]])).float()
    x[1, ::2] *= 1e-19
    for size in (1e25, 1e-9):
        w = torch.from_numpy(size * (1.0 + 0.3 * rng.standard_normal(k))).float()
        for name in ("f32", "bf16"):
            check_rows(torch, capi, x.to(dtype(torch, name)), None, w, name, 0.0)
        check_mxfp4(torch, capi, x, None, w, 0.0)
    q, scales = capi.rms_norm_tokens(x.cuda(), torch.full((k,), 1e25, device="cuda"))
    assert torch.isnan(scales).tolist() == [True, False, False]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [6, 100, 1000, 9000, 17000])
def test_rows_of_infinities_and_zeros(torch, capi, name, k):
    """What the formula gives, row by row: neighbours are untouched."""
    rows = np.ones((6, k))
    rows[0] = 0.0
    rows[1, k // 2] = math.inf
    rows[2, k - 1] = math.nan
    rows[3, 0], rows[3, k - 1] = -math.inf, math.nan
    rows[5] = -0.0
    x = torch.from_numpy(rows).to(dtype(torch, name)).cuda()
    for epsilon in (0.0, EPS):
        y = capi.rms_norm(x, None, epsilon).double().cpu().numpy()
        with np.errstate(all="ignore"):
            want = rows / np.sqrt((rows * rows).mean(-1, keepdims=True) + epsilon)
        assert np.array_equal(np.isnan(y), np.isnan(want))
        # ones: 1 / sqrt(1 + epsilon)
        assert np.allclose(np.nan_to_num(y), np.nan_to_num(want), rtol=2.0 ** -8, atol=0)
        q, scales = capi.rms_norm_tokens(x, None, epsilon)
        bad = np.isnan(want).any(-1)
        assert np.array_equal(np.isnan(scales.cpu().numpy()), bad)
        assert not q.cpu().numpy()[bad].any() and (q.cpu().numpy()[4] == 127).all()
        codes, s = capi.rms_norm_mxfp4(x, None, epsilon)
        blocks = np.array([[np.isnan(row[at:at + 32]).any() for at in range(0, k, 32)] for row in want])
        assert np.array_equal(s.cpu().numpy() == 255, blocks)
        back = capi.dequantize_mxfp4(codes, s, k=k).cpu().numpy()
        # a number just below a power of two is close to 8 steps, which become 6
        assert (back[4] >= 0.75).all() and (back[4] <= 1.0).all()


def test_sum_in_place(torch, capi):
    """The sum may be written over x or over the residual."""
    import ctypes
    for rows, k in ((3, 100), (2, 4096), (700, 1024), (2, 30000)):
        x, r = torch.randn((rows, k), device="cuda").bfloat16(), torch.randn((rows, k), device="cuda").bfloat16()
        w = torch.rand(k, device="cuda")
        want, total = capi.rms_norm(x, w, EPS, residual=r)
        for into in (0, 1):
            a, b, out = x.clone(), r.clone(), torch.empty_like(x)
            place = (a, b)[into]
            g = capi.RmsNorm(rows, k, 2, a.data_ptr(), k, b.data_ptr(), k, place.data_ptr(), k, w.data_ptr(), EPS)
            capi.check(capi.lib().tsx_rms_norm_rows(ctypes.byref(g), out.data_ptr(), k, capi._stream()))
            assert torch.equal(out, want) and torch.equal(place, total)


def test_memory_beside_the_rows_stays(torch, capi):
    import ctypes
    rows, k = 5, 43
    x, r = torch.randn((rows, k), device="cuda").half(), torch.randn((rows, k), device="cuda").half()
    want, total = capi.rms_norm(x, None, EPS, residual=r)
    out, kept = torch.full((7, 60), 9.0, device="cuda").half(), torch.full((7, 60), 9.0, device="cuda").half()
    g = capi.RmsNorm(rows, k, 1, x.data_ptr(), k, r.data_ptr(), k, kept.data_ptr(), 60, None, EPS)
    capi.check(capi.lib().tsx_rms_norm_rows(ctypes.byref(g), out.data_ptr(), 60, capi._stream()))
    assert torch.equal(out[:5, :43], want) and torch.equal(kept[:5, :43], total)
    for t in (out, kept):
        assert (t[:, 43:] == 9).all() and (t[5:] == 9).all()
    q, scales = torch.full((7 * 43,), 5, dtype=torch.int8, device="cuda"), torch.full((7,), 5.0, device="cuda")
    capi.check(capi.lib().tsx_rms_norm_tokens(ctypes.byref(g), q.data_ptr(), scales.data_ptr(), capi._stream()))
    eq, es = capi.rms_norm_tokens(total, None, EPS)
    assert torch.equal(q[:5 * 43].view(5, 43), eq) and torch.equal(scales[:5], es) and (q[5 * 43:] == 5).all() and (scales[5:] == 5).all()
    codes, bytes_ = torch.full((7 * 22,), 0xEE, dtype=torch.uint8, device="cuda"), torch.full((14,), 0xEE, dtype=torch.uint8, device="cuda")
    capi.check(capi.lib().tsx_rms_norm_mxfp4(ctypes.byref(g), codes.data_ptr(), bytes_.data_ptr(), capi._stream()))
    ec, es = capi.rms_norm_mxfp4(total, None, EPS)
    assert torch.equal(codes[:110].view(5, 22), ec) and torch.equal(bytes_[:10].view(5, 2), es) and (codes[110:] == 0xEE).all() and (bytes_[10:] == 0xEE).all()


@pytest.mark.parametrize("m", [1, 16, 100])
def test_layers_in_a_run(torch, capi, m):
    """Two layers of a network as they would be used: norm with the residual, product, the next norm on the sum; int8 and MXFP4, eager, on
    another stream and as a graph."""
    rng = np.random.default_rng(m)
    k, n = 512, 512
    x, r, w = inputs(torch, rng, m, k, "bf16")
    x, r, w = cuda(x, r, w)
    first = capi.TokenGemmI8.from_float(torch.randn((n, k), device="cuda"))
    second = capi.TokenGemmMxfp4.from_float(torch.randn((k, n), device="cuda"))

    def run(x, r):
        q, scales, h = capi.rms_norm_tokens(x, w, EPS, residual=r)
        y = first(q, x_scales=scales, act="silu", out_dtype=torch.bfloat16)
        codes, blocks, h = capi.rms_norm_mxfp4(y, w, EPS, residual=h)
        y = second(codes, x_scales=blocks, out_dtype=torch.bfloat16)
        return capi.rms_norm(y, w, EPS, residual=h)

    want = run(x, r)
    # step by step, from what the single calls are tested to give
    h = summed(x, r)
    q, scales = capi.rms_norm_tokens(h, w, EPS)
    y = first(q, x_scales=scales, act="silu", out_dtype=torch.bfloat16)
    h = summed(y, h)
    codes, blocks = capi.rms_norm_mxfp4(h, w, EPS)
    y = second(codes, x_scales=blocks, out_dtype=torch.bfloat16)
    assert torch.equal(want[1], summed(y, h)) and torch.equal(want[0], capi.rms_norm(want[1], w, EPS))
    xv = torch.from_numpy(values64(unpacked(codes.cpu().numpy(), k), blocks.cpu().numpy())).float().cuda()
    wv = capi.dequantize_mxfp4(*capi.quantize_mxfp4(torch.eye(k, device="cuda")))      # the identity is exact in this format
    assert torch.equal(wv, torch.eye(k, device="cuda")) and torch.equal(capi.TokenGemmMxfp4.from_float(wv)(codes, x_scales=blocks), xv)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = run(x, r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    gx, gr = x.clone(), r.clone()
    with torch.cuda.graph(graph):
        got = run(gx, gr)
    for turn in range(3):
        gx.copy_(torch.randn_like(gx))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run(gx, gr))), turn
