"""The int8 form of the root-mean-square norm where products of a row's values with the weight leave fp32's normal numbers and y does not, and
where y leaves fp32.

Codes are the definition's bits of h w rounded to 24 bits, whatever their exponent: a power of two in front of both changes none.  A scale is the
largest |y| over 127 within R and two more roundings, or a step of the subnormal numbers."""
import math

import numpy as np
import pytest

from tests.test_gpu_mxfp4 import U, dtype
from tests.test_gpu_rms_norm import R, norm64
from tests.test_gpu_tokens import tokens64

pytestmark = pytest.mark.gpu

COLS = [1, 5, 24, 700, 1030, 5000, 17000]


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


def products24(h, w):
    """h w of fp32 numbers rounded to 24 bits, each row times a power of two that makes its largest lie in [1, 2).  The product is exact in 64 bits."""
    part, e = np.frexp(h * w)
    top = np.where(part == 0, -10000, e).max(-1, keepdims=True)
    top = np.where(top == -10000, 0, top)
    return np.ldexp(np.rint(np.ldexp(part, 24)), e - top + 1 - 24)


def rows(rng, m, k):
    return rng.uniform(0.25, 1.0, (m, k)) * rng.choice([-1.0, 1.0], (m, k))


def check_tokens(torch, capi, x, w, epsilon, residual=None):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    q, scales, *total = capi.rms_norm_tokens(x.cuda(), w.cuda(), epsilon, residual=None if residual is None else residual.cuda())
    assert all(torch.equal(t.cpu(), h) for t in total)
    assert np.array_equal(q.cpu().numpy(), tokens64(products24(h.double().numpy(), w.double().numpy()))[0])
    want = np.abs(norm64(h, w, epsilon)).max(-1) / 127.0
    assert (np.abs(scales.double().cpu().numpy() - want) <= (R + 2 * U) * want + 2.0 ** -149).all()


@pytest.mark.parametrize("name,size,of_weight,epsilon", [("f32", -59, -91, 0.0), ("bf16", -59, -91, 0.0), ("f16", -18, -112, 0.0), ("f32", -20, -114, 0.0),
                                                         ("f32", -55, -62, 0.0), ("bf16", -25, -100, 1e-6), ("bf16", -30, -95, 1e-6)])
@pytest.mark.parametrize("k", COLS)
def test_small_products(torch, capi, k, name, size, of_weight, epsilon):
    """Rows whose mean square needs no scaling, weights so small that h w is no normal number; the rows beside them are ordinary."""
    rng = np.random.default_rng(k - size)
    x = torch.from_numpy(rows(rng, 6, k) * np.array([[2.0 ** size]] * 5 + [[2.0 ** (size + 12)]])).to(dtype(torch, name))
    w = torch.from_numpy(rng.uniform(0.5, 1.0, k) * 2.0 ** of_weight).float()
    check_tokens(torch, capi, x, w, epsilon)
    x[2] = 0.0
    if epsilon:
        check_tokens(torch, capi, x, w, epsilon, torch.zeros_like(x))


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("k", COLS)
def test_products_of_scaled_rows(torch, capi, k, name):
    """Rows whose mean square is below fp32's normal numbers, and weights that bring h w back into range: what the scaled row times the weight
    would leave is no matter.  Rows whose mean square is above it, likewise."""
    rng = np.random.default_rng(k)
    for sizes, of_weight in (((-70, -80, -100, -62), 100), ((-70, -120), 60), ((-100, -110, -126), 126), ((80, 100, 120), -120), ((70, 126), -20), ((-90, -120), -20)):
        x = torch.from_numpy(rows(rng, len(sizes), k) * 2.0 ** np.array(sizes)[:, None]).to(dtype(torch, name))
        w = torch.from_numpy(rng.uniform(0.5, 1.0, k) * 2.0 ** of_weight).float()
        check_tokens(torch, capi, x, w, 0.0)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("k", [300, 5000, 17000])
def test_rows_whose_norm_leaves_fp32(torch, capi, k, name):
    """One value alone in its row: y is the root of the columns' count times the weight.  Where that is beyond fp32 the token has no scale, as a row
    with an infinity; the rows beside it do not notice."""
    rng = np.random.default_rng(k)
    values = rows(rng, 5, k)
    values[1] = values[3] = 0.0
    values[1, k // 3], values[3, k - 1] = 0.125, -0.5
    x = torch.from_numpy(values).to(dtype(torch, name))
    w = torch.full((k,), 2.0 ** 124)
    q, scales = capi.rms_norm_tokens(x.cuda(), w.cuda(), 0.0)
    assert torch.isnan(scales).tolist() == [False, True, False, True, False]
    q, scales = q.cpu().numpy(), scales.double().cpu().numpy()
    others = [0, 2, 4]
    assert not q[[1, 3]].any() and np.array_equal(q[others], tokens64(products24(x.double().numpy(), w.double().numpy()))[0][others])
    want = np.abs(norm64(x, w, 0.0)).max(-1)[others] / 127.0
    assert (np.abs(scales[others] - want) <= (R + 2 * U) * want).all()
    y = capi.rms_norm(x.cuda().float(), w.cuda(), 0.0).cpu()
    assert math.isinf(y[1, k // 3]) and math.isinf(y[3, k - 1]) and torch.isfinite(y[others]).all()


@pytest.mark.parametrize("m,k,name", [(66001, 100, "bf16"), (17003, 700, "f32"), (4501, 2500, "bf16"), (4500, 2200, "f32"), (1027, 8000, "bf16"), (530, 17000, "f32")])
def test_scaled_and_ordinary_rows_in_turn(torch, capi, m, k, name):
    """Workgroups that take several rows: scaled and ordinary ones behind each other, with a residual, so that the sum is written and read again."""
    rng = np.random.default_rng(m)
    sizes = 2.0 ** np.array([-59, 20, -75, 3, 0, 70])[np.arange(m) % 6][:, None]
    x, r = (torch.from_numpy(rows(rng, m, k) * sizes).to(dtype(torch, name)) for _ in range(2))
    x[5::7], r[5::7] = 0.0, 0.0
    w = torch.from_numpy(rng.uniform(0.5, 1.0, k) * 2.0 ** -91).float()
    check_tokens(torch, capi, x, w, 2.0 ** -140, r)


@pytest.mark.parametrize("k", [3, 700, 17000])
def test_weights_of_zeros(torch, capi, k):
    """y is zeros: codes and scales are, too; without epsilon a row of zeros is NaN."""
    x = torch.from_numpy(rows(np.random.default_rng(k), 4, k)).bfloat16()
    x[2] = 0.0
    for epsilon in (0.0, 1e-6):
        q, scales = capi.rms_norm_tokens(x.cuda(), torch.zeros(k, device="cuda"), epsilon)
        assert not q.any() and torch.isnan(scales).tolist() == [False, False, epsilon == 0.0, False] and not scales.nan_to_num(nan=0.0).any()
