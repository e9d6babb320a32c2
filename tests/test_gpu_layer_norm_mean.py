"""DeviceLayerNorm of rows that lie far from 0 and vary little or not at all, for every shape of the kernels: what is
normalised is the distance from the mean, and it is wrong by roundings of such distances, not of the mean."""
import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu

EPS = 1e-5
# one wave (16, 32 and 64 lanes, one and two octets), several waves of every shape, rows through the caches
WIDTHS = [5, 96, 200, 500, 1000, 1500, 2000, 3000, 4000, 5000, 6000, 8000, 12000, 20000, 36000]


@pytest.fixture(scope="module")
def lcpp(gpu):
    import lc_parallel_primitive_amd as m

    return m


def near_mean(s, w, b, eps):
    """(y, mean, rstd) in 64 bits and bounds of y, of the mean before it is stored and of rstd.

    The kernel takes a first mean m, at most p = CHAIN roundings of the mean's size off, then the mean of the
    differences s - m (each rounded once, CHAIN roundings of their mean size in the sum) and their squares around it:
    no later rounding is of anything larger than a difference |s - m| <= |s - mean| + p."""
    u, chain = ref.U32, ref.CHAIN
    mean = s.mean(1, keepdim=True)
    c = s - mean
    var = (c * c).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    y = c * rstd * w + b
    p = chain * u * s.abs().mean(1, keepdim=True)
    size = c.abs().mean(1, keepdim=True) + p
    e_mean = u * (chain + 4) * size
    e_centred = e_mean + 2 * u * (c.abs() + p)
    # the squares' sum, its less n rest^2 (rest at most p, wrong by e_mean), each difference's rounding
    e_var = u * (chain + 12) * (var + p * p) + 2 * p * e_mean + 4 * u * (var + p * p)
    rel = 0.5 * e_var / (var + eps) + 6 * u
    bound = w.abs() * rstd * (e_centred + c.abs() * (rel + 3 * u)) * 1.01 + 2 * u * (y.abs() + b.abs())
    return y, mean[:, 0], rstd[:, 0], bound, e_mean[:, 0], (rel * rstd)[:, 0] * 1.01


def check_forward(lcpp, x, add):
    nrows, cols = x.shape
    dtype = {torch.float32: "float32", torch.bfloat16: "bfloat16"}[x.dtype]
    g = torch.Generator()
    g.manual_seed(cols)
    w, b = ref.rows(g, (cols,), "float32", shift=1.0, scale=0.3), ref.rows(g, (cols,), "float32", scale=0.3)
    y = torch.empty_like(x)
    mean, rstd = torch.empty(nrows, device="cuda"), torch.empty(nrows, device="cuda")
    m = lcpp.DeviceLayerNorm()
    if add:
        s = torch.empty_like(x)
        m.AddForward(torch.zeros_like(x), x, s, y, w, b, EPS, mean, rstd)
        assert torch.equal(s, x)
    else:
        m.Forward(x, y, w, b, EPS, mean, rstd)
    want, mu, rs, bound, e_mean, e_rstd = near_mean(ref.host(x), ref.host(w), ref.host(b), EPS)
    ref.check(y, want, bound, dtype, "y")
    ref.check(mean, mu, e_mean, "float32", "mean")
    ref.check(rstd, rs, e_rstd, "float32", "rstd")
    return mean


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("add", [False, True])
def test_constant_rows(lcpp, dtype, cols, add):
    """y is the bias, and the mean the constant itself: its error is far under half a step of it."""
    log(f"layer norm, constant rows of {cols} {dtype}, add {add}")
    values = torch.tensor([1432.48, 14667.6, 41216.0, -49999.9, 1000.1, 3.1], dtype=ref.TYPES[dtype])
    x = values[:, None].expand(-1, cols).contiguous().cuda()
    mean = check_forward(lcpp, x, add)
    assert torch.equal(mean.cpu(), values.float())


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("add", [False, True])
def test_rows_that_vary_by_some_steps_of_their_size(lcpp, cols, add):
    log(f"layer norm, nearly constant rows of {cols}, add {add}")
    g = torch.Generator()
    g.manual_seed(cols + 1)
    far = torch.tensor([1e3, -7e3, 5e4, 2e5, 33.3], dtype=torch.float64)[:, None]
    x = (far + torch.randn(5, cols, generator=g, dtype=torch.float64) * 2.0**-20 * far.abs()).float().cuda()
    check_forward(lcpp, x, add)


@pytest.mark.parametrize("cols", [1000, 5000, 20000, 36000])
def test_an_infinite_row_has_an_infinite_mean(lcpp, cols):
    """One infinity in a row: its mean is that infinity, its outputs NaN; the rows beside it are what they are alone."""
    log(f"layer norm, an infinity in a row of {cols}")
    g = torch.Generator()
    g.manual_seed(cols)
    x = ref.rows(g, (3, cols), "float32")
    clean = x.clone()
    x[1, cols // 3] = -float("inf")
    out = []
    for v in (x, clean):
        y, mean, rstd = torch.empty_like(v), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
        lcpp.DeviceLayerNorm().Forward(v, y, None, None, EPS, mean, rstd)
        out.append((y, mean))
    assert out[0][1][1] == -float("inf") and torch.isnan(out[0][0][1]).all()
    for r in (0, 2):
        assert torch.equal(out[0][0][r], out[1][0][r]) and out[0][1][r] == out[1][1][r]
