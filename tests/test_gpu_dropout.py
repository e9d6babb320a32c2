"""DeviceDropout: the generator's bits exactly, types, odd widths and strides, what is dropped never shows, the backward
pass, the device counter, and the shares of what is kept."""
import math

import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lcpp(gpu):
    import lc_parallel_primitive_amd as m

    return m


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("nrows,cols", [(1, 1), (1, 7), (3, 8), (2, 9), (65, 63), (7, 1001), (300, 20), (2, 4099)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_against_definition(lcpp, dtype, nrows, cols, p):
    log(f"dropout {dtype} {nrows} x {cols} p {p}")
    g = gen(cols)
    seed, offset = 0xFEDCBA9876543210 - cols, (3 << 32) + 11
    x = ref.rows(g, (nrows, cols), dtype, cols % 3, offset=cols % 2)
    r = ref.rows(g, (nrows, cols), dtype, 1)
    y = torch.full((nrows, cols), 7.0, dtype=x.dtype, device="cuda")
    m = lcpp.DeviceDropout()
    want, keep = ref.dropped(ref.host(x), p, seed, offset)
    m.Forward(x, y, p, seed, offset)
    ref.check(y, want, ref.U32 * 2 * want.abs(), dtype, "y")
    assert torch.equal(y.cpu() == 0, (want == 0))  # exactly the same places
    m.Forward(x, y, p, seed, offset, d_residual=r)
    ref.check(y, want + ref.host(r), ref.U32 * (2 * want.abs() + (want + ref.host(r)).abs()), dtype, "y + residual")
    dy, dx = ref.rows(g, (nrows, cols), dtype), torch.empty_like(y)
    m.Backward(dy, dx, p, seed, offset)
    back, _ = ref.dropped(ref.host(dy), p, seed, offset)
    ref.check(dx, back, ref.U32 * 2 * back.abs(), dtype, "dx")
    # the counter's other half: a device integer added to the offset
    c = torch.tensor([offset - 4], dtype=torch.int64, device="cuda")
    again = torch.empty_like(y)
    m.Forward(x, again, p, seed, 4, d_residual=r, d_offset=c)
    assert torch.equal(again, y)
    # in place
    over = x.clone()
    m.Forward(over, over, p, seed, offset, d_residual=r)
    assert torch.equal(over, y)


def test_what_is_dropped_never_shows(lcpp):
    log("dropout of NaN, infinities and largest values")
    n, seed = 4096, 99
    _, keep = ref.dropped(torch.ones(2, n, dtype=torch.float64), 0.5, seed, 0)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        x = torch.ones(2, n, dtype=torch.bfloat16)
        x[~keep] = bad
        y = torch.empty(2, n, dtype=torch.bfloat16, device="cuda")
        lcpp.DeviceDropout().Forward(x.cuda(), y, 0.5, seed)
        assert torch.equal(y.cpu() == 2.0, keep) and torch.equal(y.cpu() == 0.0, ~keep)


def test_same_bits_as_in_the_layer_norm(lcpp):
    """The fused sum and the separate calls drop the same elements: widths of one and of several waves."""
    for cols in (77, 1536, 8200, 40000):
        log(f"dropout in the layer norm, {cols}")
        g = gen(cols)
        x, r = ref.rows(g, (9, cols), "float32"), ref.rows(g, (9, cols), "float32")
        s, y, apart = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        lcpp.DeviceLayerNorm().AddForward(x, r, s, y, p=0.25, seed=5, offset=6)
        lcpp.DeviceDropout().Forward(x, apart, 0.25, 5, 6, d_residual=r)
        assert torch.equal(s, apart)


def test_shares(lcpp):
    """2^24 elements: the kept share, that of neighbours kept together, and that of one place under two offsets, each
    within six standard deviations of what independent choices give."""
    rows, cols, p = 4096, 4096, 0.3
    log("dropout shares")
    x = torch.ones(rows, cols, device="cuda")
    a, b = torch.empty_like(x), torch.empty_like(x)
    m = lcpp.DeviceDropout()
    m.Forward(x, a, p, 1234, 0)
    m.Forward(x, b, p, 1234, 1)
    q = 1 - round(p * 65536) / 65536
    ka, kb = a != 0, b != 0
    n = rows * cols

    def near(share, expect, count):
        assert abs(float(share) - expect) <= 6 * math.sqrt(expect * (1 - expect) / count), (float(share), expect)

    near(ka.double().mean(), q, n)
    near((ka & kb).double().mean(), q * q, n)
    near((ka[:, 1:] & ka[:, :-1]).double().mean(), q * q, n / 2)  # (pairs share elements)
    near((ka[1:] & ka[:-1]).double().mean(), q * q, n / 2)
    assert abs(float(a.double().mean()) - 1) <= 6 * math.sqrt((1 - q) / q / n)


def test_many_octets(lcpp):
    """More octets than one grid has threads, rows of an odd number of octets: the stepped row and column are right."""
    rows, cols = 5003, 4001
    log(f"dropout {rows} x {cols}")
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    y = torch.empty_like(x)
    lcpp.DeviceDropout().Forward(x, y, 0.5, 77, 3)
    for r in (0, 1, 2500, 4097, 5002):
        one = torch.empty(r + 1, cols, dtype=x.dtype, device="cuda")
        lcpp.DeviceDropout().Forward(x[: r + 1], one, 0.5, 77, 3)
        assert torch.equal(one[r], y[r])
    bits = ref.philox_bits(3, cols, 77, 3)
    assert torch.equal(y[:3].cpu() != 0, bits >= 32768)


def test_strides_past_32_bits(lcpp):
    log("dropout, rows 2^30 apart")
    base = torch.ones(2 * (1 << 30) + 1000, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((3, 1000), (1 << 30, 1))
    y, tight = torch.empty(3, 1000, dtype=x.dtype, device="cuda"), torch.empty(3, 1000, dtype=x.dtype, device="cuda")
    m = lcpp.DeviceDropout()
    m.Forward(x.contiguous(), tight, 0.5, 1)
    m.Forward(x, y, 0.5, 1)
    assert torch.equal(y, tight)


def test_refusals(lcpp):
    m = lcpp.DeviceDropout()
    x = torch.zeros(4, 32, device="cuda")
    y = torch.zeros_like(x)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(lcpp.LcppError):
            m.Forward(x, y, p, 1)
    with pytest.raises(TypeError):
        m.Forward(x.double(), y.double(), 0.1, 1)
    with pytest.raises(TypeError):
        m.Forward(x, y.half(), 0.1, 1)
    with pytest.raises(ValueError):
        m.Forward(x, y[:, :31], 0.1, 1)
    with pytest.raises(ValueError):
        m.Forward(x, y[:1].expand(4, 32), 0.1, 1)
    with pytest.raises(ValueError):
        m.Forward(x, y, 0.1, 1, d_residual=x[:3])
    with pytest.raises(ValueError):
        m.Forward(x, y, 0.1, 1, d_offset=torch.zeros(1, dtype=torch.int32, device="cuda"))
    m.Forward(x[:0], y[:0], 0.1, 1)
