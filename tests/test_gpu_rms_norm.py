"""RMS norm against its definition in 64 bits: sizes around every layout's edges, strides, places, 8-bit outputs with
scales, values that are not finite, gradients against the formula and against differences."""
import pytest
import torch

import block_ref as ref
import expert_ref as eref
from conftest import log

pytestmark = pytest.mark.gpu
EPS = 1e-6


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def weights(g, cols, dtype):
    return (torch.randn(cols, generator=g, dtype=torch.float64) * 0.3 + 1).to(ref.TYPES[dtype]).cuda()


SIZES = [(1, 1), (3, 7), (5, 8), (1, 127), (33, 128), (7, 129), (9, 250), (4, 263), (65, 512), (3, 1000), (2, 1027), (31, 1536),
         (5, 2047), (3, 2055), (7, 4096), (2, 5001), (3, 6150), (2, 8199), (2, 16391), (1, 33000), (600, 96), (2000, 72), (1000, 1024)]


@pytest.mark.parametrize("dtype,wdtype", [("bfloat16", "float32"), ("float16", "float16"), ("float32", "float32")])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward_backward(gpu, rows, cols, dtype, wdtype):
    import lc_parallel_primitive_amd as lcpp

    log(f"rms {rows} x {cols} {dtype} {wdtype}")
    g = gen(rows * 7 + cols)
    for add, pad, offset in ((False, 0, 0), (True, 3, 1)):
        x, y = ref.rows(g, (rows, cols), dtype, pad, 0.2, 1.5, offset), ref.rows(g, (rows, cols), dtype, pad, offset=offset)
        w = weights(g, cols, wdtype)
        rstd = torch.empty(rows, device="cuda")
        norm = lcpp.DeviceRMSNorm()
        s = x
        if add:
            r, s = ref.rows(g, (rows, cols), dtype, 5), ref.rows(g, (rows, cols), dtype, 1)
            norm.AddForward(x, r, s, y, w, EPS, rstd)
            assert torch.equal(s, (r.float() + x.float()).to(s.dtype))
        else:
            norm.Forward(x, y, w, EPS, rstd)
        hs, hw = ref.host(s), ref.host(w)
        want, want_rstd, rel, rel_rstd = eref.rms(hs, hw, EPS)
        ref.check(y, want, rel * want.abs(), dtype, "y")
        ref.check(rstd, want_rstd[:, 0], rel_rstd * want_rstd[:, 0], "float32", "rstd")
        dy, dx = ref.rows(g, (rows, cols), dtype, pad), ref.rows(g, (rows, cols), dtype, pad, offset=offset)
        dsum = ref.rows(g, (rows, cols), dtype, 2) if add else None
        dw = torch.empty_like(w)
        temp = torch.empty(norm.GetBackwardTempStorageBytes(x.dtype, rows, cols), dtype=torch.uint8, device="cuda")
        norm.Backward(temp, dy, s, w, rstd, dx, dw, d_grad_sum=dsum)
        ds, hdw, b, bw = eref.rms_grad(hs, hw, ref.host(rstd)[:, None], ref.host(dy), None if dsum is None else ref.host(dsum))
        ref.check(dx, ds, b, dtype, "dx")
        ref.check(dw, hdw, bw, wdtype, "dw")
        # without the weights' gradient and without weights
        dx2 = torch.empty_like(x)
        norm.Backward(None, dy, s, w, rstd, dx2, None, d_grad_sum=dsum)
        assert torch.equal(dx2, dx)
        y2 = torch.empty_like(x)
        norm.Forward(s, y2, None, EPS)
        want = eref.rms(hs, torch.ones(()).double(), EPS)[0]
        ref.check(y2, want, rel * want.abs(), dtype, "y without weights")


QSIZES = [(1, 1, 128), (3, 31, 32), (2, 32, 32), (5, 33, 32), (9, 127, 64), (33, 128, 128), (4, 129, 128), (3, 130, 512),
          (7, 250, 256), (5, 255, 32), (4, 263, 64), (4, 263, 0), (2, 1000, 512), (3, 1027, 128), (3, 1027, 0), (2, 1543, 256),
          (3, 2048, 128), (2, 2055, 32), (5, 4096, 128), (2, 5001, 64), (2, 5001, 0), (2, 8199, 512), (2, 16391, 128), (2, 16391, 0),
          (1, 33001, 32), (1, 33001, 0), (700, 96, 32), (70, 1536, 128)]


@pytest.mark.parametrize("dtype,qdtype", [("bfloat16", torch.float8_e4m3fn), ("float16", torch.float8_e5m2),
                                          ("float32", torch.float8_e4m3fn)])
@pytest.mark.parametrize("rows,cols,group", QSIZES)
def test_eight_bits(gpu, rows, cols, group, dtype, qdtype):
    import lc_parallel_primitive_amd as lcpp

    log(f"rms quant {rows} x {cols} group {group} {dtype} {qdtype}")
    g = gen(rows * 11 + cols + group)
    parts = -(-cols // group) if group else 1
    norm = lcpp.DeviceRMSNorm()
    for add, transposed, with_out in ((False, False, True), (True, True, False)):
        x = ref.rows(g, (rows, cols), dtype, 1)
        w = weights(g, cols, dtype)
        q = torch.zeros(rows, cols + 3, dtype=torch.uint8, device="cuda").view(qdtype)[:, :cols]
        scales = torch.empty((parts, rows) if transposed else (rows, parts), device="cuda")
        scales = scales.t() if transposed else scales
        y = torch.empty_like(x) if with_out else None
        s = x
        if add:
            r, s = ref.rows(g, (rows, cols), dtype), torch.empty(rows, cols, dtype=x.dtype, device="cuda")
            norm.AddForward(x, r, s, y, w, EPS, None, q, scales, group)
        else:
            norm.Forward(x, y, w, EPS, None, q, scales, group)
        want, _, rel, _ = eref.rms(ref.host(s), ref.host(w), EPS)
        if with_out:
            ref.check(y, want, rel * want.abs(), dtype, "y")
        eref.check_quantised(q, scales, want, rel, group, f"add {add}")


@pytest.mark.parametrize("cols,group", [(300, 128), (300, 0), (40000, 128), (40000, 0)])
def test_eight_bits_of_odd_values(gpu, cols, group):
    """Zeros, values too small for a scale of their own, infinities and NaN, each in a row (and a group) of its own."""
    import lc_parallel_primitive_amd as lcpp

    x = torch.ones(5, cols, device="cuda")
    x[0] = 0
    x[1] = 2.0**-130  # (eps is what rstd is made of)
    x[2, 5] = float("inf")
    x[3, 3] = float("nan")
    q = torch.empty(5, cols, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(5, -(-cols // group) if group else 1, device="cuda")
    w = torch.full((cols,), 1e-3, device="cuda")
    lcpp.DeviceRMSNorm().Forward(x, None, w, EPS, None, q, scales, group)
    values = q.float().cpu()
    smallest = torch.tensor(2.0**-100) / 448
    assert torch.all(values[:2] == 0) and torch.allclose(scales[:2].cpu(), smallest, rtol=2e-7, atol=0)
    # a row with an infinity has rstd 0: 0 everywhere but in its place, whose group is NaN
    g = group or cols
    assert torch.isnan(scales[2, 0]) and torch.all(torch.isnan(values[2, :g])) and torch.all(values[2, g:] == 0)
    assert torch.all(torch.isnan(values[3])) and torch.all(torch.isnan(scales[3]))
    assert torch.all(values[4] == 448)


def test_zero_rows_and_large_values(gpu):
    import lc_parallel_primitive_amd as lcpp

    x = torch.zeros(2, 100, device="cuda")
    x[1] = 1e18
    y, rstd = torch.empty_like(x), torch.empty(2, device="cuda")
    lcpp.DeviceRMSNorm().Forward(x, y, None, EPS, rstd)
    assert torch.all(y[0] == 0) and torch.allclose(y[1], torch.ones(100, device="cuda"), rtol=1e-5)
    x[1] = 1e30  # (the squares pass float32's range)
    lcpp.DeviceRMSNorm().Forward(x, y, None, EPS, rstd)
    assert torch.all(y == 0) and float(rstd[1]) == 0


@pytest.mark.parametrize("cols", [72, 777, 2048, 9000, 20001])
def test_in_place(gpu, cols):
    """Outputs exactly over an input: out over in, sum over residual and over in, ds over dy."""
    import lc_parallel_primitive_amd as lcpp

    norm, g = lcpp.DeviceRMSNorm(), gen(cols)
    rows = 700
    x, r = ref.rows(g, (rows, cols), "bfloat16"), ref.rows(g, (rows, cols), "bfloat16")
    w = weights(g, cols, "bfloat16")
    y, s = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty(rows, device="cuda")
    norm.AddForward(x, r, s, y, w, EPS, rstd)
    for over in ("residual", "in"):
        a, b = x.clone(), r.clone()
        out = torch.empty_like(x)
        norm.AddForward(a, b, b if over == "residual" else a, out, w, EPS)
        assert torch.equal(b if over == "residual" else a, s) and torch.equal(out, y)
    z, y = s.clone(), torch.empty_like(x)
    norm.Forward(s, y, w, EPS)
    norm.Forward(z, z, w, EPS)
    assert torch.equal(z, y)
    dy, dsum = ref.rows(g, (rows, cols), "bfloat16"), ref.rows(g, (rows, cols), "bfloat16")
    temp = torch.empty(norm.GetBackwardTempStorageBytes(x.dtype, rows, cols), dtype=torch.uint8, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    norm.Backward(temp, dy, s, w, rstd, dx, dw, dsum)
    for over in range(3):
        t = [dy.clone(), s.clone(), dsum.clone()]
        dw2 = torch.empty_like(w)
        norm.Backward(temp, t[0], t[1], w, rstd, t[over], dw2, t[2])
        assert torch.equal(t[over], dx) and torch.equal(dw2, dw)


def test_gradient_by_differences(gpu):
    """The formula's gradients against central differences of the 64-bit forward pass, and the kernel's against both."""
    import lc_parallel_primitive_amd as lcpp

    g = gen(3)
    rows, cols = 4, 37
    s = torch.randn(rows, cols, generator=g, dtype=torch.float64)
    w = torch.randn(cols, generator=g, dtype=torch.float64)
    dy = torch.randn(rows, cols, generator=g, dtype=torch.float64)
    s, w, dy = (v.float().double() for v in (s, w, dy))
    f = lambda a, b: float((eref.rms(a, b, EPS)[0] * dy).sum())  # noqa: E731
    h = 1e-5
    norm = lcpp.DeviceRMSNorm()
    x, wd = s.float().cuda(), w.float().cuda()
    y, rstd, dx, dw = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty_like(x), torch.empty_like(wd)
    norm.Forward(x, y, wd, EPS, rstd)
    temp = torch.empty(norm.GetBackwardTempStorageBytes(x.dtype, rows, cols), dtype=torch.uint8, device="cuda")
    norm.Backward(temp, dy.float().cuda(), x, wd, rstd, dx, dw)
    # the difference quotient is off by h^2 of the third derivative (about 10 here) and 1e-16 / h of the values
    for i, j in ((0, 0), (1, 5), (3, 36), (2, 20)):
        e = torch.zeros_like(s)
        e[i, j] = h
        assert abs((f(s + e, w) - f(s - e, w)) / (2 * h) - float(dx[i, j])) < 1e-5
    for j in (0, 17, 36):
        e = torch.zeros_like(w)
        e[j] = h
        assert abs((f(s, w + e) - f(s, w - e)) / (2 * h) - float(dw[j])) < 1e-5


def test_nothing(gpu):
    import lc_parallel_primitive_amd as lcpp

    norm = lcpp.DeviceRMSNorm()
    for rows, cols in ((0, 64), (4, 0)):
        x = torch.empty(rows, cols, device="cuda")
        norm.Forward(x, torch.empty_like(x), torch.ones(cols, device="cuda"), EPS, torch.empty(rows, device="cuda"))
        dw = torch.full((cols,), 7.0, device="cuda")
        norm.Backward(None, x, x, torch.ones(cols, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x), dw)
        assert torch.all(dw == 0)
