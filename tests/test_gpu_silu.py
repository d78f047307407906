"""SiLU of given fp32 numbers, through the product on tokens and through the group norm, against 64 bits.

A product of one column of ones, w_scales = v, is act(1 * v * 1); a norm with the weight 0 and the bias v is act(v).

Bars.  u = 2^-24.  exp(-x) = 2^t (1 + r): the exponential within a step (2 u), 1 + r and the product u each; the sum with 1 u; the reciprocal
within a step, 2 u; the product with x u: 8 u of the value where exp(-x) is most of the sum, less elsewhere.  Below -87 the reciprocal leaves the
normal numbers; the value is less than 10^-35 there."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KERNELS = [(1, "0"), (40, "0"), (40, "1"), (40, "2"), (40, "3"), (40, "4")]


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


def numbers(count):
    rng = np.random.default_rng(count)
    size = np.exp(rng.uniform(np.log(1e-6), np.log(87.0), count))
    return np.concatenate([size, -size, np.linspace(-87, 87, count), [0.0, -0.0, 100.0, 1e30, 3e38]]).astype(np.float32)


def silu64(x):
    x = x.astype(np.float64)
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-x))


def check(torch, got, x, name):
    want = silu64(x)
    half = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]
    bar = 8.01 * U * np.abs(want)
    if name != "f32":        # the exponential's argument rounded, |x| u of it, and the rounding to the type
        bar = (bar + np.abs(x * want) * U) * (1 + half) + half * np.abs(want) + 2.0 ** (-25 if name == "f16" else -134)
    off = np.abs(got.double().cpu().numpy() - want) - bar
    assert off.max() <= 0, (off.max(), x[off.argmax()], got.flatten()[off.argmax()])


@pytest.mark.parametrize("m,kernel", KERNELS)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_silu_of_products(torch, capi, monkeypatch, name, m, kernel):
    monkeypatch.setenv("TSX_TOKENS_KERNEL", kernel)
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]
    x = numbers(20000)
    if name == "f16":
        x = x[np.abs(x) < 60000]
    layer = capi.TokenGemmI8(torch.ones((len(x), 1), dtype=torch.int8, device="cuda"), torch.from_numpy(x).cuda())
    out = layer(torch.ones((m, 1), dtype=torch.int8, device="cuda"), x_scales=torch.ones(m, device="cuda"), act="silu", out_dtype=t)
    assert torch.equal(out, out[:1].expand_as(out))
    check(torch, out[0], x, name)


@pytest.mark.parametrize("shape", [(2, 4, 4), (1, 130, 130)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_silu_of_norms(torch, capi, name, shape):
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]
    x = numbers(2000)
    x = x[np.abs(x) < 60000][:5984]
    data = torch.randn(shape + (len(x),), device="cuda").to(t)
    out = capi.group_norm(data, 32 if len(x) % 32 == 0 else 1, torch.zeros(len(x), device="cuda"), torch.from_numpy(x).cuda(), act="silu")
    assert torch.equal(out, out[:1, :1, :1].expand_as(out))
    check(torch, out[0, 0, 0], x, name)


def test_silu_of_infinities(torch, capi):
    """x / (1 + exp(-x)) as it is written: its limit to the right, no number where it is infinite over infinite; far to the left 0."""
    x = torch.tensor([float("inf"), float("nan"), float("-inf"), -1e30, -3e38, -200.0, -1000.0], device="cuda")
    layer = capi.TokenGemmI8(torch.ones((7, 1), dtype=torch.int8, device="cuda"), x)
    for t in (torch.float32, torch.bfloat16):
        for m in (1, 40):
            out = layer(torch.ones((m, 1), dtype=torch.int8, device="cuda"), x_scales=torch.ones(m, device="cuda"), act="silu", out_dtype=t)
            assert (out[:, 0] == float("inf")).all() and out[:, 1:3].isnan().all() and (out[:, 3:] == 0).all()
