"""The argument checks of the RMS norm, router, token sort and product entry points, without a GPU: every refusal comes
before any launch, and the size queries are host arithmetic."""
import ctypes

import pytest
import torch

F32, BF16, F16, E4, E5 = 2, 6, 7, 8, 9
A, B, C, D, E, G, ODD = 4096, 8192, 12288, 16384, 20480, 24576, 4097  # addresses that no call reads


@pytest.fixture(scope="module")
def L():
    import lc_parallel_primitive_amd as lcpp

    return lcpp.lib()


def norm(L, t=BF16, wt=F32, x=A, xs=64, r=None, w=B, eps=1e-6, s=None, ss=64, y=C, ys=64, rstd=D, qt=E4, q=None, qs=64, sc=None, sr=1,
         sg=1, group=128, rows=4, cols=64):
    return L.lcpp_rms_norm_forward(t, wt, x, xs, r, 64, w, eps, s, ss, y, ys, rstd, qt, q, qs, sc, sr, sg, group, rows, cols, None)


Q = dict(q=E, sc=G)


@pytest.mark.parametrize("change,status", [
    (dict(t=0), -3), (dict(t=E4), -3), (dict(wt=F16), -3), (dict(t=F32, wt=BF16), -3), (dict(x=None), -1), (dict(x=ODD), -1),
    (dict(y=None), -1), (dict(w=B + 2), -1), (dict(rstd=D + 2), -1), (dict(ys=63), -1), (dict(eps=-1.0), -1),
    (dict(eps=float("nan")), -1), (dict(rows=1 << 32), -1), (dict(cols=(1 << 30) + 1, ys=1 << 31), -1), (dict(r=B), -1),
    (dict(r=B, s=C), -1), (dict(r=B, s=E, ss=63), -1), (dict(s=E), -1), (dict(**Q, qt=BF16), -3), (dict(**Q, qt=10), -3),
    (dict(**Q, group=100), -1), (dict(**Q, group=16), -1), (dict(**Q, group=1024), -1), (dict(**Q, qs=63), -1),
    (dict(q=E), -1), (dict(q=E, sc=G + 2), -1), (dict(**Q, sr=0), -1), (dict(**Q, group=32, sr=1, sg=0), -1),
    (dict(**Q, group=32, sr=1, sg=1), -1), (dict(**Q, group=32, sr=1, sg=3), -1), (dict(q=A, sc=G), -1), (dict(q=C, sc=G), -1),
    (dict(q=E, sc=D), -1), (dict(rows=0), 0), (dict(cols=0), 0), (dict(rows=0, x=None, y=None), 0),
])
def test_norm_forward(L, change, status):
    assert norm(L, **change) == status


def norm_backward(L, temp=A, tb=1 << 30, t=BF16, wt=F32, dy=B, gs=None, x=C, rstd=D, dx=E, dxs=64, dw=G, rows=4, cols=64):
    return L.lcpp_rms_norm_backward(t, wt, temp, tb, dy, 64, gs, 64, x, 64, None, rstd, dx, dxs, dw, rows, cols, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=3), -3), (dict(wt=7), -3), (dict(dy=None), -1), (dict(x=None), -1), (dict(rstd=None), -1), (dict(dx=None), -1),
    (dict(dxs=8), -1), (dict(temp=None), -1), (dict(temp=A + 128), -1), (dict(tb=255), -2), (dict(tb=256 + 4 * 64 * 4 - 1), -2),
    (dict(dw=G + 2), -1), (dict(gs=ODD), -1), (dict(dx=G), -1), (dict(rows=1 << 33), -1), (dict(cols=0), 0),
    (dict(rows=0, dw=None, temp=None), 0),
])
def test_norm_backward(L, change, status):
    assert norm_backward(L, **change) == status


def router(L, t=BF16, score=0, scale=1.0, l=A, ids=B, w=C, bias=None, tokens=4, experts=8, k=2):
    return L.lcpp_router_forward(t, score, 1, scale, l, experts, bias, ids, w, tokens, experts, k, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=1), -3), (dict(t=E4), -3), (dict(score=2), -1), (dict(score=-1), -1), (dict(scale=float("nan")), -1), (dict(l=None), -1),
    (dict(l=ODD), -1), (dict(ids=None), -1), (dict(ids=B + 2), -1), (dict(w=None), -1), (dict(w=B), -1), (dict(bias=C + 1), -1),
    (dict(experts=1025), -1), (dict(experts=128, k=65), -1), (dict(k=9), -1), (dict(tokens=1 << 31), -1),
    (dict(tokens=1 << 30, k=2), -1), (dict(tokens=0), 0), (dict(k=0), 0),
])
def test_router_forward(L, change, status):
    assert router(L, **change) == status


def test_router_backward(L):
    def call(t=BF16, score=1, l=A, ids=B, g=C, dl=D, ds=8, tokens=4, experts=8, k=2):
        return L.lcpp_router_backward(t, score, 0, 1.0, l, 8, ids, g, dl, ds, tokens, experts, k, None)

    for bad in (dict(score=7), dict(l=None), dict(ids=None), dict(g=None), dict(g=C + 2), dict(dl=None), dict(dl=ODD), dict(ds=7),
                dict(experts=2000, ds=2000), dict(k=9)):
        assert call(**bad) == -1, bad
    assert call(t=0) == -3
    assert call(tokens=0) == 0


def test_sort(L):
    def call(temp=A, tb=1 << 30, ids=B, tokens=100, k=4, experts=8, pos=C, off=D, src=E):
        return L.lcpp_token_sort(temp, tb, ids, tokens, k, experts, pos, off, src, None)

    for bad in (dict(ids=None), dict(ids=B + 2), dict(pos=None), dict(off=None), dict(off=D + 1), dict(src=E + 3), dict(experts=0),
                dict(experts=1025), dict(tokens=1 << 31), dict(tokens=1 << 30), dict(pos=D), dict(src=C), dict(src=D), dict(src=B),
                dict(off=B), dict(temp=A + 8), dict(temp=None, tokens=10000)):
        assert call(**bad) == -1, bad
    assert call(tokens=10000, tb=300) == -2
    b = ctypes.c_size_t()
    for tokens, k, experts, want in ((0, 8, 16, 0), (512, 8, 16, 0), (4096, 1, 1024, 0), (4097, 1, 16, 256 + 256),
                                     (32768, 8, 256, 256 + 128 * 256 * 4), (1 << 28, 4, 256, 256 + 128 * 256 * 4)):
        assert L.lcpp_token_sort_temp_bytes(tokens, k, experts, ctypes.byref(b)) == 0
        assert b.value == want, (tokens, k, experts, b.value)
    assert L.lcpp_token_sort_temp_bytes(1 << 31, 1, 8, ctypes.byref(b)) == -1
    assert L.lcpp_token_sort_temp_bytes(10, 1, 1025, ctypes.byref(b)) == -1
    assert L.lcpp_token_sort_temp_bytes(10, 1, 8, None) == -1


def spread(L, t=BF16, x=A, p=B, w=None, y=C, ys=64, o=None, d=None, rows=8, tokens=4, k=2, cols=64):
    return L.lcpp_token_spread(t, x, 64, p, w, y, ys, o, 64, d, rows, tokens, k, cols, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=3), -3), (dict(t=5), -3), (dict(t=10), -3), (dict(t=E4, w=D), -3), (dict(t=0, d=D, o=E), -3), (dict(x=None), -1),
    (dict(x=ODD), -1), (dict(p=None), -1), (dict(p=B + 2), -1), (dict(y=None), -1), (dict(y=ODD), -1), (dict(ys=63), -1),
    (dict(w=D + 1), -1), (dict(d=D), -1), (dict(d=D + 2, o=E), -1), (dict(y=D, d=D, o=E), -1), (dict(y=A), -1), (dict(k=65), -1),
    (dict(rows=1 << 31), -1), (dict(tokens=1 << 31), -1), (dict(cols=1 << 31, ys=1 << 31), -1), (dict(tokens=0), 0), (dict(k=0), 0),
    (dict(cols=0), 0), (dict(rows=0), 0),
])
def test_spread(L, change, status):
    assert spread(L, **change) == status


def test_sum(L):
    def call(t=BF16, x=A, rows=8, p=B, w=None, r=None, y=C, ys=64, o=None, d=None, tokens=4, k=2, cols=64):
        return L.lcpp_token_sum(t, x, 64, rows, p, w, r, 64, y, ys, o, 64, d, tokens, k, cols, None)

    for bad in (dict(x=None), dict(p=None), dict(y=None), dict(y=ODD), dict(ys=63), dict(w=D + 2), dict(r=ODD), dict(d=D), dict(y=A),
                dict(d=C, o=E), dict(d=D, o=E, r=G), dict(k=65), dict(cols=1 << 31, ys=1 << 31)):
        assert call(**bad) == -1, bad
    assert call(t=E4) == -3 and call(t=0) == -3
    assert call(tokens=0) == 0 and call(cols=0) == 0


def product(L, t=BF16, x=A, w=B, off=C, ot=BF16, y=D, ys=32, sx=None, sw=None, rows=10, experts=3, n=32, m=64):
    return L.lcpp_expert_product(t, x, m, w, m, n * m, off, ot, y, ys, sx, 1, 1, sw, rows, experts, n, m, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=0), -3), (dict(t=E5), -3), (dict(ot=F32), -3), (dict(t=E4, ot=E4, sx=E, sw=G), -3), (dict(x=None), -1), (dict(x=ODD), -1),
    (dict(w=None), -1), (dict(off=None), -1), (dict(off=C + 2), -1), (dict(y=None), -1), (dict(y=ODD), -1), (dict(ys=31), -1),
    (dict(sx=E), -1), (dict(sw=E), -1), (dict(t=E4), -1), (dict(t=E4, sx=E), -1), (dict(t=E4, sx=E, sw=G + 1), -1), (dict(y=A), -1),
    (dict(y=B), -1), (dict(experts=1025), -1), (dict(rows=1 << 31), -1), (dict(n=(1 << 30) + 1, ys=1 << 31), -1), (dict(rows=0), 0),
    (dict(experts=0), 0), (dict(n=0), 0),
])
def test_product(L, change, status):
    assert product(L, **change) == status


def test_product_backward(L):
    def call(t=BF16, dy=A, x=B, w=C, off=D, dx=E, dxs=64, wt=BF16, dw=G, dws=64, dwe=64 * 32, rows=10, experts=3, n=32, m=64):
        return L.lcpp_expert_product_backward(t, dy, 32, x, 64, w, 64, 2048, off, dx, dxs, wt, dw, dws, dwe, rows, experts, n, m, None)

    for bad in (dict(dy=None), dict(x=None), dict(w=None), dict(off=None), dict(dx=ODD), dict(dxs=63), dict(dw=ODD), dict(dws=63),
                dict(dwe=2047), dict(dx=G), dict(dx=A), dict(dx=C), dict(dx=B), dict(dw=B), dict(dw=A), dict(experts=1025)):
        assert call(**bad) == -1, bad
    assert call(t=E4) == -3 and call(wt=F16) == -3
    assert call(experts=0) == 0 and call(m=0) == 0
    assert call(dx=None, dw=None) == 0


# ------------------------------------------------------------ the Python classes
def test_host_tensors():
    """A tensor that is not on the GPU is refused before its address reaches a kernel."""
    import lc_parallel_primitive_amd as m

    x, w, i = torch.zeros(4, 32), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    off = torch.zeros(4, dtype=torch.int32)
    mats = torch.zeros(3, 8, 32)
    for call in (lambda: m.DeviceRMSNorm().Forward(x, x.clone(), stream=0),
                 lambda: m.DeviceRMSNorm().AddForward(x, x, x, x, stream=0),
                 lambda: m.DeviceRMSNorm().Backward(None, x, x, None, torch.zeros(4), x, stream=0),
                 lambda: m.DeviceExpertRouter().Forward(x, i, w, stream=0),
                 lambda: m.DeviceExpertRouter().Backward(x, i, w, x, stream=0),
                 lambda: m.DeviceTokenSort().Sort(None, i, 3, i.clone(), off, stream=0),
                 lambda: m.DeviceTokenSort().Dispatch(x, i, torch.zeros(8, 32), stream=0),
                 lambda: m.DeviceTokenSort().DispatchBackward(torch.zeros(8, 32), i, x, stream=0),
                 lambda: m.DeviceTokenSort().Combine(torch.zeros(8, 32), i, w, x, stream=0),
                 lambda: m.DeviceTokenSort().CombineBackward(x, torch.zeros(8, 32), i, w, torch.zeros(8, 32), w, stream=0),
                 lambda: m.DeviceExpertProduct().Forward(x, mats, off, torch.zeros(4, 8), stream=0),
                 lambda: m.DeviceExpertProduct().Backward(torch.zeros(4, 8), x, mats, off, x, mats.clone(), stream=0)):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()


@pytest.mark.gpu
def test_python_refusals(gpu):
    import lc_parallel_primitive_amd as m

    dev = "cuda"
    x, y = torch.zeros(4, 256, device=dev), torch.zeros(4, 256, device=dev)
    q, s = torch.zeros(4, 256, device=dev).to(torch.float8_e4m3fn), torch.zeros(4, 2, device=dev)
    i, w = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.zeros(4, 2, device=dev)
    off = torch.zeros(4, dtype=torch.int32, device=dev)
    mats = torch.zeros(3, 8, 256, device=dev)
    norm, router, order, product = m.DeviceRMSNorm(), m.DeviceExpertRouter(), m.DeviceTokenSort(), m.DeviceExpertProduct()
    for error, call in (
            (ValueError, lambda: norm.Forward(x, None)),
            (ValueError, lambda: norm.Forward(x, y[:3])),
            (TypeError, lambda: norm.Forward(x, y.half())),
            (TypeError, lambda: norm.Forward(x.double(), y.double())),
            (ValueError, lambda: norm.Forward(x.t(), y.t())),
            (ValueError, lambda: norm.Forward(x, y, torch.zeros(255, device=dev))),
            (ValueError, lambda: norm.Forward(x, None, d_quant=q)),
            (ValueError, lambda: norm.Forward(x, None, d_quant=q, d_scales=s, group=64)),
            (TypeError, lambda: norm.Forward(x, None, d_quant=q, d_scales=s.half())),
            (TypeError, lambda: norm.Forward(x, None, d_quant=x.half(), d_scales=s)),
            (m.LcppError, lambda: norm.Forward(x, None, d_quant=q, d_scales=s[:, :1].expand(4, 2))),
            (m.LcppError, lambda: norm.Forward(x, None, d_quant=q, d_scales=torch.zeros(4, 3, device=dev), group=100)),
            (ValueError, lambda: router.Forward(x, i, w, score="tanh")),
            (ValueError, lambda: router.Forward(x, i[:3], w)),
            (TypeError, lambda: router.Forward(x, i.long(), w)),
            (TypeError, lambda: router.Forward(x, i, w.half())),
            (ValueError, lambda: router.Forward(x, i, w, d_bias=torch.zeros(255, device=dev))),
            (m.LcppError, lambda: router.Forward(torch.zeros(4, 1025, device=dev), i, w)),
            (ValueError, lambda: order.Sort(None, i, 3, i[:3].clone(), off)),
            (ValueError, lambda: order.Sort(None, i, 4, i.clone(), off)),
            (m.LcppError, lambda: order.Sort(None, i, 3, i, i.flatten())),
            (ValueError, lambda: order.Dispatch(x, i[:3], torch.zeros(8, 256, device=dev))),
            (ValueError, lambda: order.Dispatch(x, i, torch.zeros(8, 255, device=dev))),
            (TypeError, lambda: order.Dispatch(x, i, torch.zeros(8, 256, device=dev, dtype=torch.half))),
            (TypeError, lambda: order.Dispatch(x.double(), i, torch.zeros(8, 256, device=dev).double())),
            (TypeError, lambda: order.Dispatch(q, i, torch.zeros(8, 256, device=dev).to(q.dtype), w)),
            (ValueError, lambda: order.DispatchBackward(torch.zeros(8, 256, device=dev), i, y, w, None, w.clone())),
            (ValueError, lambda: order.Combine(torch.zeros(8, 255, device=dev), i, w, y)),
            (ValueError, lambda: order.Combine(torch.zeros(8, 256, device=dev), i, w[:3], y)),
            (ValueError, lambda: product.Forward(x, mats[0], off, torch.zeros(4, 8, device=dev))),
            (ValueError, lambda: product.Forward(x, mats, off[:3], torch.zeros(4, 8, device=dev))),
            (TypeError, lambda: product.Forward(x, mats.half(), off, torch.zeros(4, 8, device=dev))),
            (TypeError, lambda: product.Forward(x, mats, off, torch.zeros(4, 8, device=dev, dtype=torch.half))),
            (ValueError, lambda: product.Forward(x, mats, off, torch.zeros(4, 8, device=dev), s, s)),
            (ValueError, lambda: product.Forward(q, mats.to(q.dtype), off, torch.zeros(4, 8, device=dev))),
            (ValueError, lambda: product.Forward(q, mats.to(q.dtype), off, torch.zeros(4, 8, device=dev), s, s)),
            (ValueError, lambda: product.Backward(torch.zeros(4, 8, device=dev), x, mats, off, None, mats[:1].expand(3, 8, 256))),
            (TypeError, lambda: product.Backward(torch.zeros(4, 8, device=dev), x, mats, off, None, mats.half())),
    ):
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()
