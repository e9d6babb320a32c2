"""DeviceLayerNorm against its definition in 64 bits: types, widths around every kernel's limits, strides and alignments,
rows that lie far from 0 or are constant, masks of NaN rows, gradients against the formula and against differences."""
import itertools

import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu

EPS = 1e-5
# one octet, one wave, and the limits of each shape of the kernels, each from both sides
WIDTHS = [1, 7, 8, 9, 64, 500, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096, 4097, 5001, 8192, 8193, 16384, 16385, 32768,
          32769, 40000]


@pytest.fixture(scope="module")
def lcpp(gpu):
    import lc_parallel_primitive_amd as m

    return m


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def weights(g, n, wt):
    return ref.rows(g, (n,), wt, shift=1.0, scale=0.3), ref.rows(g, (n,), wt, scale=0.3)


def temp_for(lcpp, x, rows, cols):
    return torch.empty(lcpp.DeviceLayerNorm.GetBackwardTempStorageBytes(x.dtype, rows, cols), dtype=torch.uint8, device="cuda")


def run_case(lcpp, dtype, wt, nrows, cols, pad=0, offset=0, shift=0.25, scale=1.0, affine=True, seed=1):
    log(f"layer norm {dtype} weights {wt} {nrows} x {cols} pad {pad} offset {offset} shift {shift}")
    g = gen(seed + cols)
    x = ref.rows(g, (nrows, cols), dtype, pad, shift, scale, offset)
    w, b = weights(g, cols, wt) if affine else (None, None)
    dy = ref.rows(g, (nrows, cols), dtype, 0, 0.0, 0.5)
    y, dx = ref.rows(g, (nrows, cols), dtype, pad, offset=offset), ref.rows(g, (nrows, cols), dtype, pad + 1)
    mean, rstd = torch.full((nrows,), 7.0, device="cuda"), torch.full((nrows,), 7.0, device="cuda")
    m = lcpp.DeviceLayerNorm()
    m.Forward(x, y, w, b, EPS, mean, rstd)
    one = torch.ones(cols, dtype=torch.float64)
    w64, b64 = (ref.host(w), ref.host(b)) if affine else (one, one * 0)
    x64 = ref.host(x)
    want, mu, rs, bound, e_mean, e_rstd = ref.norm(x64, w64, b64, EPS)
    ref.check(y, want, bound, dtype, "y")
    ref.check(mean, mu[:, 0], e_mean[:, 0], "float32", "mean")
    ref.check(rstd, rs[:, 0], e_rstd[:, 0], "float32", "rstd")
    wt = wt if affine else dtype
    dw, db = (torch.full((cols,), 7.0, dtype=ref.TYPES[wt], device="cuda") for _ in range(2))
    m.Backward(temp_for(lcpp, x, nrows, cols), dy, x, w, mean, rstd, dx, dw, db)
    ds, gw, gb, bound, bw, bb = ref.norm_grad(x64, w64, ref.host(mean)[:, None], ref.host(rstd)[:, None], ref.host(dy), nrows)
    ref.check(dx, ds, bound, dtype, "dx")
    ref.check(dw, gw, bw, wt, "dw")
    ref.check(db, gb, bb, wt, "db")
    return x, y, dx, dw, db


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype,wt", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16")])
def test_widths(lcpp, dtype, wt, cols):
    run_case(lcpp, dtype, wt, 5, cols)


@pytest.mark.parametrize("cols", [4103, 5119, 5120, 5127, 5128])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_edges_of_the_five_eighths_group(lcpp, dtype, cols):
    run_case(lcpp, dtype, "float32", 9, cols, pad=1)


@pytest.mark.parametrize("nrows", [1, 2, 3, 4, 63, 513, 2050])
@pytest.mark.parametrize("cols", [40, 700, 1536, 5000])
def test_rows(lcpp, nrows, cols):
    run_case(lcpp, "bfloat16", "bfloat16", nrows, cols)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (3, 5), (8, 0), (17, 3)])
def test_strides_and_alignment(lcpp, dtype, pad, offset):
    for cols in (96, 1003, 4500, 20000):
        run_case(lcpp, dtype, "float32", 6, cols, pad, offset)


def test_no_weight(lcpp):
    run_case(lcpp, "float32", "float32", 9, 777, affine=False)


@pytest.mark.parametrize("shift,scale", [(1000.0, 1.0), (0.0, 1e-4), (-30.0, 1e3), (3.0, 0.0)])
def test_far_small_large_and_constant_rows(lcpp, shift, scale):
    for cols in (130, 3000, 36000):
        run_case(lcpp, "float32", "float32", 4, cols, shift=shift, scale=scale)


def test_nothing_leaves_a_row(lcpp):
    """A row of NaN, infinities or the type's largest values changes no other row, forward or backward."""
    for cols, dtype in itertools.product((100, 1500, 9000, 33000), ("float32", "bfloat16")):
        log(f"layer norm with a poisoned row, {dtype} {cols}")
        g = gen(3)
        x = ref.rows(g, (7, cols), dtype)
        clean = x.clone()
        x[2] = float("nan")
        x[4, 5] = float("inf")
        x[5] = torch.finfo(x.dtype).min
        w, b = weights(g, cols, "float32")
        dy = ref.rows(g, (7, cols), dtype)
        m = lcpp.DeviceLayerNorm()
        out = []
        for v in (x, clean):
            y, dx = torch.empty_like(v), torch.empty_like(v)
            mean, rstd = torch.empty(7, device="cuda"), torch.empty(7, device="cuda")
            m.Forward(v, y, w, b, EPS, mean, rstd)
            m.Backward(None, dy, v, w, mean, rstd, dx)
            out.append((y, dx))
        for got, want in zip(*out):
            for r in (0, 1, 3, 6):
                assert torch.equal(got[r], want[r])
            assert torch.isnan(got[2]).all()


def test_empty(lcpp):
    m = lcpp.DeviceLayerNorm()
    w = torch.ones(50, device="cuda")
    x = torch.empty(0, 50, device="cuda")
    dw, db = torch.full((50,), 3.0, device="cuda"), torch.full((50,), 3.0, device="cuda")
    stat = torch.empty(0, device="cuda")
    m.Forward(x, x.clone(), w, w, EPS, stat, stat)
    m.Backward(None, x, x, w, stat, stat, x.clone(), dw, db)  # sums over no rows
    assert not dw.any() and not db.any()
    y = torch.empty(6, 0, device="cuda")
    m.Forward(y, y.clone())


@pytest.mark.parametrize("dtype,wt", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("cols", [8, 100, 513, 1025, 2049, 5001, 16385, 33001])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_add(lcpp, dtype, wt, cols, p):
    """residual + dropout(x), the norm of the stored sum, and back; the sum's own bits decide the norm's input."""
    nrows, pad, seed, offset = 5, 3, (0xDEAD << 40) + cols, (5 << 33) + 1
    log(f"layer norm add {dtype} {nrows} x {cols} p {p}")
    g = gen(cols)
    x, r = (ref.rows(g, (nrows, cols), dtype, pad, 0.1) for _ in range(2))
    w, b = weights(g, cols, wt)
    s, y = torch.empty_like(x), torch.empty(nrows, cols, dtype=x.dtype, device="cuda")
    mean, rstd = torch.empty(nrows, device="cuda"), torch.empty(nrows, device="cuda")
    m = lcpp.DeviceLayerNorm()
    m.AddForward(x, r, s, y, w, b, EPS, mean, rstd, p=p, seed=seed, offset=offset)
    d64, keep = ref.dropped(ref.host(x), p, seed, offset)
    s64 = ref.host(r) + d64
    ref.check(s, s64, 2 * ref.U32 * (ref.host(r).abs() + d64.abs()), dtype, "sum")
    stored, w64 = ref.host(s), ref.host(w)
    want, mu, rs, bound, e_mean, e_rstd = ref.norm(stored, w64, ref.host(b), EPS)
    ref.check(y, want, bound, dtype, "y")
    ref.check(mean, mu[:, 0], e_mean[:, 0], "float32", "mean")
    dy, extra = ref.rows(g, (nrows, cols), dtype, 0, 0.0, 0.5), ref.rows(g, (nrows, cols), dtype, 1)
    dres, dx = torch.empty_like(y), torch.empty_like(x)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    t = temp_for(lcpp, x, nrows, cols)
    m.AddBackward(t, dy, extra, s, w, mean, rstd, dres, dx, dw, db, p=p, seed=seed, offset=offset)
    ds, gw, gb, bound, bw, bb = ref.norm_grad(stored, w64, ref.host(mean)[:, None], ref.host(rstd)[:, None], ref.host(dy), nrows)
    total = ds + ref.host(extra)
    bound = bound + ref.U32 * (ds.abs() + total.abs())
    ref.check(dres, total, bound, dtype, "dresidual")
    cut = int(p * 65536 + 0.5)
    scale = 65536 / (65536 - cut)
    ref.check(dx, torch.where(keep, total * scale, 0.0), bound * scale + 2 * ref.U32 * total.abs() * scale, dtype, "dx")
    ref.check(dw, gw, bw, wt, "dw")
    ref.check(db, gb, bb, wt, "db")
    # what is not wanted is not written, and no other result changes
    only = torch.full_like(dx, 7.0)
    m.AddBackward(None, dy, extra, s, w, mean, rstd, None, only, p=p, seed=seed, offset=offset)
    assert torch.equal(only, dx)
    m.AddBackward(t, dy, None, s, w, mean, rstd, dres, None, dw, None, p=p, seed=seed, offset=offset)
    ref.check(dres, ds, bound, dtype, "ds without the residual path's gradient")
    ref.check(dw, gw, bw, wt, "dw alone")


def test_in_place_and_repeated(lcpp):
    """Outputs in the place of inputs, and the same bits from every call."""
    for cols in (333, 2048, 20001):
        log(f"layer norm in place, {cols}")
        g = gen(cols)
        x = ref.rows(g, (700, cols), "bfloat16")
        dy = ref.rows(g, (700, cols), "bfloat16")
        w, b = weights(g, cols, "float32")
        mean, rstd = torch.empty(700, device="cuda"), torch.empty(700, device="cuda")
        m = lcpp.DeviceLayerNorm()
        y, dx = torch.empty_like(x), torch.empty_like(x)
        t = temp_for(lcpp, x, 700, cols)
        grads = [torch.empty(cols, device="cuda") for _ in range(6)]
        m.Forward(x, y, w, b, EPS, mean, rstd)
        m.Backward(t, dy, x, w, mean, rstd, dx, grads[0], grads[1])
        t.fill_(255)
        m.Backward(t, dy, x, w, mean, rstd, dx, grads[2], grads[3])
        over = dy.clone()
        m.Backward(t, over, x, w, mean, rstd, over, grads[4], grads[5])
        assert torch.equal(over, dx)
        for i in (2, 4):
            assert torch.equal(grads[i], grads[0]) and torch.equal(grads[i + 1], grads[1])
        here = x.clone()
        m.Forward(here, here, w, b, EPS)
        assert torch.equal(here, y)
        # residual + x over the residual
        s, y2 = x.clone(), torch.empty_like(x)
        m.AddForward(dy, s, s, y2, w, b, EPS)
        assert torch.equal(s, (x.float() + dy.float()).bfloat16())


@pytest.mark.parametrize("cols", [24, 600, 3000])
def test_gradient_against_differences(lcpp, cols):
    """dL/dx, dL/dw, dL/db along random directions, L = sum(y c).  With a step of 2^-6 the central difference is off by
    step^2 / 6 times the third derivative (of the order of the first: 4e-5), and by the roundings of y, 2^-22 each and
    independent, over the step: together under 1e-3 of |gradient| |direction|."""
    log(f"layer norm differences, {cols}")
    g = gen(cols)
    n, step = 6, 2.0**-6
    x, c = ref.rows(g, (n, cols), "float32"), ref.rows(g, (n, cols), "float32")
    w, b = weights(g, cols, "float32")
    m = lcpp.DeviceLayerNorm()
    mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    y = torch.empty_like(x)

    def loss(x, w, b):
        m.Forward(x, y, w, b, EPS, mean, rstd)
        return float((y.double() * c.double()).sum())

    loss(x, w, b)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    m.Backward(temp_for(lcpp, x, n, cols), c, x, w, mean, rstd, dx, dw, db)
    args = [x, w, b]
    for i, grad in enumerate((dx, dw, db)):
        d = torch.randn(grad.shape, generator=g).cuda()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * d, args[i] - step * d
        got = (loss(*up) - loss(*down)) / (2 * step)
        want = float((grad.double() * d.double()).sum())
        assert abs(got - want) <= 1e-3 * float(grad.double().norm() * d.double().norm()), (i, got, want)


def test_strides_past_32_bits(lcpp):
    """Rows 2^30 elements apart: the third lies past 2^31 elements."""
    log("layer norm, rows 2^30 apart")
    base = torch.empty(2 * (1 << 30) + 1000, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((3, 1000), (1 << 30, 1))
    x.copy_(torch.randn(3, 1000, generator=gen(1)))
    y, tight = torch.empty(3, 1000, dtype=x.dtype, device="cuda"), torch.empty(3, 1000, dtype=x.dtype, device="cuda")
    m = lcpp.DeviceLayerNorm()
    m.Forward(x.contiguous(), tight)
    m.Forward(x, y)
    assert torch.equal(y, tight)
    m.Forward(x, x)
    assert torch.equal(x.contiguous(), tight)


def test_a_row_wider_than_the_launches(lcpp):
    # more columns than one launch's workgroups take at 64 each: the gradients' sums go round
    cols = (1 << 26) + 70
    log(f"layer norm backward, one row of {cols}")
    g = torch.Generator(device="cuda").manual_seed(5)
    x, dy = (torch.randn(1, cols, generator=g, device="cuda") for _ in range(2))
    mean, rstd = torch.tensor([0.125], device="cuda"), torch.tensor([0.75], device="cuda")
    dx, dw, db = torch.empty_like(x), torch.full((cols,), 7.0, device="cuda"), torch.full((cols,), 7.0, device="cuda")
    lcpp.DeviceLayerNorm().Backward(temp_for(lcpp, x, 1, cols), dy, x, None, mean, rstd, dx, dw, db)
    torch.cuda.synchronize()
    want = dy[0].double() * ((x[0].double() - 0.125) * 0.75)
    # three roundings of a product, each of 2^-24
    assert bool(((dw.double() - want).abs() <= 4 * 2.0**-24 * want.abs()).all())
    assert torch.equal(db, dy[0])


def test_refusals(lcpp):
    m = lcpp.DeviceLayerNorm()
    x = torch.zeros(4, 32, device="cuda")
    y, w = torch.zeros_like(x), torch.zeros(32, device="cuda")
    s = torch.zeros(4, device="cuda")
    with pytest.raises(TypeError):
        m.Forward(x.int(), y)
    with pytest.raises(TypeError):
        m.Forward(x, y.bfloat16())
    with pytest.raises(TypeError):
        m.Forward(x, y, w.bfloat16())  # weights narrower than the rows
    with pytest.raises(TypeError):
        m.Forward(x, y, w, w, EPS, s.double())
    with pytest.raises(ValueError):
        m.Forward(x, y[:3])
    with pytest.raises(ValueError):
        m.Forward(x, y, w[:31])
    with pytest.raises(ValueError):
        m.Forward(x, y, w, w, EPS, s[:3], s)
    with pytest.raises(ValueError):
        m.Forward(x.t(), y.t())
    with pytest.raises(ValueError):
        m.Forward(x, y[:1].expand(4, 32))  # rows of an output that overlap
    with pytest.raises(lcpp.LcppError):
        m.Forward(x, y, eps=-1.0)
    with pytest.raises(lcpp.LcppError) as e:
        m.Backward(torch.empty(256, dtype=torch.uint8, device="cuda"), x, x, w, s, s, y, w.clone(), None)
    assert e.value.status == -2
    with pytest.raises(lcpp.LcppError):
        m.Backward(None, x, x, w, None, s, y)
    with pytest.raises(lcpp.LcppError):
        m.AddForward(x, x, y, y.clone(), p=1.5)
    # inputs may repeat a row
    m.Forward(x[:1].expand(4, 32), y, w, w)
