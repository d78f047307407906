"""Rows of floats whose products are streams over the weights, where K is longer than all of a workgroup's wavefronts request at once: LDS, weights and
rows of later turns, row ends inside and behind them.

The rows hold values of the format, so that quantizing changes none of them, and all sums are whole numbers of steps of 1/4 below 2^24: every result is
exact in fp32, whatever the order of its sums."""
import numpy as np
import pytest

from tests.test_gpu_mxfp4 import TYPES, device, dtype, random_rows, values64

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
@pytest.mark.parametrize("m,n,k", [(m, n, k) for m, n in ((1, 40), (3, 17), (4, 200)) for k in (4096, 4097, 8192, 8200, 16385, 20000)] +
                         [(m, n, k) for m, n in ((5, 40), (16, 33), (20, 16)) for k in (2048, 2049, 4100, 4225, 9001, 20000)] + [(2, 130, 1025), (4, 16, 3972)])
def test_long_streams(torch, capi, monkeypatch, name, m, n, k):
    monkeypatch.setenv("TSX_MXFP4_KERNEL", "0")
    rng = np.random.default_rng(m * n + k)
    xc, xs = random_rows(rng, m, k, (127, 128))
    wc, ws = random_rows(rng, n, k, (127, 128))
    x, w = values64(xc, xs), values64(wc, ws)
    assert 16 * 36 * k < 2 ** 24
    layer = capi.TokenGemmMxfp4(*device(torch, wc, ws), k=k)
    want = torch.from_numpy(x @ w.T).float()
    wide = torch.full((m, k + 10), float("nan"), device="cuda").to(dtype(torch, name))       # what lies beside the rows is not used
    wide[:, 3:k + 3] = torch.from_numpy(x).to(dtype(torch, name)).cuda()
    got = layer(wide[:, 3:k + 3], out_dtype=torch.float32)
    assert got.shape == (m, n) and torch.equal(got.cpu(), want)
    codes, scales = capi.quantize_mxfp4(wide[:, 3:k + 3])
    assert torch.equal(layer(codes, x_scales=scales).cpu(), want)
    assert torch.equal(layer(wide[:, 3:k + 3].contiguous()).cpu(), want.to(dtype(torch, name)))
