"""The root-mean-square norm of a single row given as a tensor of one axis, and with weights of other types than fp32, by value."""
import pytest

from tests.test_gpu_mxfp4 import TYPES, dtype

pytestmark = pytest.mark.gpu

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


def forms(capi):
    return capi.rms_norm, capi.rms_norm_tokens, capi.rms_norm_mxfp4


def every(result):
    return result if isinstance(result, tuple) else (result,)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [1, 5, 100, 1000, 4096, 20000])
def test_one_axis(torch, capi, name, k):
    torch.manual_seed(k)
    x, r = (torch.randn(k, device="cuda").to(dtype(torch, name)) for _ in range(2))
    w = 1.0 + 0.3 * torch.randn(k, device="cuda")
    shapes = {capi.rms_norm: [(k,)], capi.rms_norm_tokens: [(k,), ()], capi.rms_norm_mxfp4: [((k + 1) // 2,), ((k + 31) // 32,)]}
    for call in forms(capi):
        for residual in (None, r):
            got = every(call(x, w, EPS, residual=residual))
            want = every(call(x.view(1, k), w, EPS, residual=None if residual is None else r.view(1, k)))
            assert [tuple(t.shape) for t in got] == shapes[call] + ([] if residual is None else [(k,)])
            assert len(got) == len(want) and all(a.dtype == b.dtype and torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [5, 100, 1000, 4096, 20000])
def test_weights_of_other_types(torch, capi, name, k):
    """Weights are converted to fp32: what fp16, bf16 and 64 bits hold of fp32 numbers gives the results of those numbers."""
    torch.manual_seed(k)
    x, r = (torch.randn((12, k), device="cuda").to(dtype(torch, name)) for _ in range(2))
    for kind in (torch.float64, torch.float16, torch.bfloat16):
        w = (1.0 + 0.3 * torch.randn(k, device="cuda")).to(kind).float()
        for call in forms(capi):
            for residual in (None, r):
                want = every(call(x, w, EPS, residual=residual))
                assert not torch.equal(want[0], every(call(x, None, EPS, residual=residual))[0])
                got = every(call(x, w.to(kind), EPS, residual=residual))
                assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
