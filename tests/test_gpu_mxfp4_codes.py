"""Every code under every scale byte back to every type: the definition's value, rounded once, to nearest even, beyond the largest number to an
infinity; NaN under 255.  Conversions are compared bit for bit, the sign of zeros too."""
import numpy as np
import pytest

from tests.test_gpu_mxfp4 import TYPES, VALUES, dtype, packed

pytestmark = pytest.mark.gpu


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


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [32, 31, 16])
def test_every_code_and_scale(torch, capi, name, k):
    """Codes in turn from a place that goes by the row, so that each is met at each place of a byte and of a piece."""
    scales = np.arange(256, dtype=np.uint8)
    code = (np.arange(k)[None, :] + np.arange(256)[:, None] // 16 + 3 * np.arange(256)[:, None]) % 16
    code = np.concatenate([code, (code + 7) % 16])
    scales = np.concatenate([scales, scales])
    codes = packed(code)
    got = capi.dequantize_mxfp4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales[:, None]).cuda(), k=k, dtype=dtype(torch, name)).cpu()
    with np.errstate(over="ignore"):
        exact = VALUES[code] * np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))[:, None]
    # a value has two significant bits: in fp32 it is exact, or beyond it; then one rounding to the type
    want = torch.from_numpy(exact).float().to(dtype(torch, name))
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan) and nan.any(1).sum() == 2
    whole = {4: torch.int32, 2: torch.int16}[got.element_size()]
    assert torch.equal(got.view(whole)[~nan], want.view(whole)[~nan])
