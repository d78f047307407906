"""Statistics of the channels-last group norm where fp32 sums lose them: means far from zero, single values and blocks of pixels far from
the rest, means that drift along an image; on images of up to a thousand pixels a thread, in one launch and in two, with their definition in
64 bits.

Bars.  u = 2^-24 is half a step of fp32 relative to the value.  Ahead of the rounding to the output's type, (x - mean) r is off by

* the mean's error times r.  Means of threads, of chunks and of the group are each rounded once, to within u of a magnitude that is at
  most the group's mean or, on average, its deviation; sums of differences from a value of the group are within some roundings of the
  average difference: u (4 |mean| + 8 deviations).
* relative errors: the difference, the product's sum, 1 / count and its product, epsilon's sum and the root (a step, 2 u), half of those
  under it: 6 u.  Sums of squares: a thread's roundings average with those of all others, the last merges of up to 16 in a row do not: 16 u of
  the variance, 8 u here; 10 u with what is left of the average.
* a thread's mean rounded where it is far from zero: (u |mean| r)^2 of the variance.
* a value far from the rest that is the first of a batch of eight: the squares of seven differences from it, each within 10 u, less the
  square of their sum / 8, within 18 u of the squares, leaves an eighth of the squares or more: 8 * 29 u of the variance, 116 u here."""
import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


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


def image(torch, kind, shape, groups, name):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    c, n = shape[-1], shape[0]
    pixels = math.prod(shape[1:-1])
    x = torch.randn((n, pixels, groups, c // groups), generator=g, device="cuda")
    if kind == "far":
        x += 1000.0
    elif kind == "drift":
        x = x * 0.03 + 1000.0 + torch.linspace(0, 1, pixels, device="cuda").view(1, -1, 1, 1)
    elif kind == "block":        # of pixels: what a chunk of them has, or less
        x[:, :max(1, pixels // 256)] += 1000.0
    elif kind == "outlier":      # in front of zeros, of small values and of a constant
        for k in range(groups):
            if k % 3 == 0:
                x[:, :, k] = 0.0
            elif k % 3 == 1:
                x[:, :, k] *= 1e-3
            else:
                x[:, :, k] = 0.25
            x[:, 0, k, 0] = 1000.0 * (1 + k / 7)
    return x.reshape(shape).to(dtype(torch, name))


def norm64(torch, x, groups, epsilon, kind):
    """The norm in 64 bits and what fp32 may be off it."""
    v = x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups).double()
    mean = v.mean((1, 3), keepdim=True)
    v -= mean
    variance = (v * v).mean((1, 3), keepdim=True)
    r = 1.0 / torch.sqrt(variance + epsilon)
    v *= r
    relative = U * (16 + (116 if kind == "outlier" else 0)) + (U * mean.abs() * r) ** 2
    error = v.abs() * relative
    error += U * (4 * mean.abs() + 8 * variance.sqrt()) * r
    return v.view(x.shape), error.view(x.shape)


SHAPES = [((1, 2048, 2048, 128), 32), ((300, 64, 64, 64), 8), ((1, 300, 512, 1025), 5), ((1, 1700, 1700, 3), 1), ((2, 40, 40, 15), 5), ((1, 130, 130, 16), 4),
          ((1, 9000, 320), 32), ((2, 40, 40, 16), 4), ((2, 8, 8, 1280), 32)]


@pytest.mark.parametrize("kind", ["normal", "far", "drift", "block", "outlier"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_statistics(torch, capi, shape, groups, name, kind):
    epsilon = 1e-12
    x = image(torch, kind, shape, groups, name)
    want, error = norm64(torch, x, groups, epsilon, kind)
    got = capi.group_norm(x, groups, epsilon=epsilon)
    h = torch.finfo(x.dtype).eps / 2
    off = (got.double() - want).abs_() - (error * (1 + h) + h * want.abs() + TINY[name])
    assert not got.isnan().any() and float(off.max()) <= 0, (float(off.max()), int(off.argmax()))
    del got, off
    q, s = capi.group_norm_tokens(x, groups, epsilon=epsilon)
    top, most, s = want.abs().amax(-1), error.amax(-1), s.double()
    assert bool(((s * 127 - top).abs() <= most + 2 * U * top).all())
    # half a step of the token's scale, and what the norm may be off, in the value and in the scale
    assert bool(((q.double() * s[..., None] - want).abs() <= 0.5001 * s[..., None] + 2 * error + most[..., None]).all())


def test_statistics_of_many_images(torch, capi):
    """One chunk an image where there are images for all CUs: threads of 500 rows each."""
    x = image(torch, "outlier", (2, 500, 4096), 32, "bf16")
    want, error = norm64(torch, x, 32, 1e-12, "outlier")
    h = torch.finfo(x.dtype).eps / 2
    for i in range(2):
        got = capi.group_norm(x[i:i + 1].expand(256, 500, 4096), 32, epsilon=1e-12)
        assert torch.equal(got[0], got[255])
        off = (got[0].double() - want[i]).abs() - (error[i] * (1 + h) + h * want[i].abs() + TINY["bf16"])
        assert float(off.max()) <= 0


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 8), ((2, 130, 130, 16), 4), ((2, 40, 40, 15), 5), ((300, 64, 64, 64), 8)])
def test_statistics_that_leave_fp32(torch, capi, shape, groups, name):
    """A group whose squares leave fp32 is NaN, in one launch and in two, and nothing finite in its place; the others do not notice.  Up to there
    the norm is that of smaller values."""
    x = image(torch, "normal", shape, groups, name)
    d = shape[-1] // groups
    bias = torch.linspace(-1, 1, shape[-1], device="cuda")
    want, (q, s) = capi.group_norm(x, groups, None, bias), capi.group_norm_tokens(x, groups)
    for size in (1e20, 1e25, 1e30, 1e37):
        y = x.clone()
        y[1, ..., d:2 * d] *= size
        got = capi.group_norm(y, groups, None, bias)
        assert got[1, ..., d:2 * d].isnan().all()
        got[1, ..., d:2 * d] = want[1, ..., d:2 * d]
        assert torch.equal(got, want)
        qt, st = capi.group_norm_tokens(y, groups)
        assert (qt[1] == 0).all() and st[1].isnan().all() and torch.equal(qt[0], q[0]) and torch.equal(st[0], s[0])
    # 67600 squares of at most (6e15)^2 are within 3.4e38
    y = x * 1e15
    want, error = norm64(torch, y, groups, 1e-5, "normal")
    got = capi.group_norm(y, groups)
    h = torch.finfo(x.dtype).eps / 2
    assert float(((got.double() - want).abs() - (error * (1 + h) + h * want.abs() + TINY[name])).max()) <= 0
