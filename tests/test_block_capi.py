"""The argument checks of the layer norm, dropout and recurrence entry points, without a GPU: every refusal comes before
any launch, and the size queries are host arithmetic."""
import ctypes

import pytest

F32, BF16, F16 = 2, 6, 7
P, ODD = 4096, 4097  # addresses that no call reads


@pytest.fixture(scope="module")
def L():
    import lc_parallel_primitive_amd as lcpp

    return lcpp.lib()


def norm(L, t=BF16, wt=F32, x=P, xs=64, w=P, b=P, eps=1e-5, y=P, ys=64, mean=P, rstd=P, rows=4, cols=64):
    return L.lcpp_layer_norm_forward(t, wt, x, xs, w, b, eps, y, ys, mean, rstd, rows, cols, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=0), -3), (dict(t=5), -3), (dict(t=99), -3), (dict(t=-1), -3), (dict(wt=F16), -3), (dict(t=F32, wt=BF16), -3),
    (dict(x=None), -1), (dict(y=None), -1), (dict(x=ODD), -1), (dict(w=P + 2), -1), (dict(mean=P + 2), -1),
    (dict(ys=63), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(rows=1 << 32), -1),
    (dict(cols=(1 << 30) + 1, ys=1 << 31), -1), (dict(rows=0), 0), (dict(cols=0), 0), (dict(rows=0, x=None, y=None), 0),
])
def test_norm_forward(L, change, status):
    assert norm(L, **change) == status


def add_forward(L, t=BF16, p=0.1, r=P, s=P, ss=64, rows=0):
    return L.lcpp_layer_norm_add_forward(t, F32, P, 64, r, 64, p, 1, 2, None, P, P, 1e-5, s, ss, P, 64, P, P, rows, 64, None)


def test_norm_add_forward(L):
    assert add_forward(L) == 0
    for bad in (dict(p=-0.1), dict(p=1.01), dict(p=float("nan")), dict(r=None, rows=2), dict(s=None, rows=2), dict(ss=10, rows=2)):
        assert add_forward(L, **bad) == -1, bad
    assert add_forward(L, t=1) == -3


def norm_backward(L, temp=P, tb=1 << 30, t=BF16, wt=F32, dy=P, x=P, mean=P, rstd=P, dx=P, dxs=64, dw=P, db=P, rows=4, cols=64):
    return L.lcpp_layer_norm_backward(t, wt, temp, tb, dy, 64, x, 64, P, mean, rstd, dx, dxs, dw, db, rows, cols, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=3), -3), (dict(wt=7), -3), (dict(dy=None), -1), (dict(x=None), -1), (dict(mean=None), -1), (dict(rstd=None), -1),
    (dict(dx=None), -1), (dict(dxs=8), -1), (dict(temp=None), -1), (dict(temp=P + 128), -1), (dict(tb=255), -2),
    (dict(dw=P + 2), -1), (dict(rows=1 << 33), -1), (dict(cols=0), 0), (dict(rows=0, dw=None, db=None), 0),
])
def test_norm_backward(L, change, status):
    assert norm_backward(L, **change) == status


def test_norm_backward_temp(L):
    b = ctypes.c_size_t()
    sizes = []
    for rows in (0, 1, 300, 512, 513, 1 << 20):
        assert L.lcpp_layer_norm_backward_temp_bytes(BF16, rows, 1000, ctypes.byref(b)) == 0
        sizes.append(b.value)
    assert sizes[0] == 0 and sizes[1] == 256 + 8192 and sizes[3] == sizes[5] == 256 + 512 * 8000
    assert L.lcpp_layer_norm_backward_temp_bytes(BF16, 1 << 32, 10, ctypes.byref(b)) == -1
    assert L.lcpp_layer_norm_backward_temp_bytes(1, 10, 10, ctypes.byref(b)) == -3
    assert L.lcpp_layer_norm_backward_temp_bytes(BF16, 10, 10, None) == -1
    assert norm_backward(L, tb=256 + 4 * 2 * 64 * 4 - 1) == -2


def dropout(L, t=BF16, x=P, r=None, y=P, ys=64, rows=4, cols=64, p=0.1):
    return L.lcpp_dropout(t, x, 64, r, 64, y, ys, rows, cols, p, 1, 2, None, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=4), -3), (dict(x=None), -1), (dict(y=None), -1), (dict(y=ODD), -1), (dict(r=ODD), -1), (dict(ys=1), -1),
    (dict(p=2.0), -1), (dict(p=float("nan")), -1), (dict(rows=1 << 32), -1), (dict(cols=1 << 31), -1), (dict(rows=0), 0),
    (dict(cols=0), 0),
])
def test_dropout(L, change, status):
    assert dropout(L, **change) == status


def recurrence(L, t=BF16, g=2, temp=P, tb=1 << 40, gate=P, x=P, y=P, ys=(64, 64 * 500), n=3, length=500, c=64, begin=None,
               end=None, rows=0, h0=P):
    return L.lcpp_recurrence_forward(t, g, temp, tb, gate, 64, 64 * 500, x, 64, 64 * 500, y, *ys, h0, P, P, n, length, c, begin,
                                     end, rows, None)


@pytest.mark.parametrize("change,status", [
    (dict(t=0), -3), (dict(t=8), -3), (dict(g=3), -1), (dict(g=-1), -1), (dict(gate=None), -1), (dict(x=None), -1),
    (dict(y=None), -1), (dict(y=ODD), -1), (dict(h0=P + 1), -1), (dict(ys=(63, 64 * 500)), -1), (dict(ys=(64, 3)), -1),
    (dict(begin=P), -1), (dict(end=P), -1), (dict(begin=P, end=ODD), -1), (dict(temp=None), -1), (dict(temp=P + 8), -1),
    (dict(tb=1000), -2), (dict(length=1 << 31), -1), (dict(n=1 << 33), -1), (dict(n=1 << 20, length=1 << 20), -1),
    (dict(n=0), 0), (dict(c=0), 0),
])
def test_recurrence_forward(L, change, status):
    assert recurrence(L, **change) == status


def test_recurrence_backward(L):
    def call(saved=P, dy=P, dg=P, dx=P, dgs=64, t=BF16, n=3):
        return L.lcpp_recurrence_backward(t, 0, P, 1 << 40, P, 64, 32000, P, 64, 32000, saved, dy, 64, 32000, dg, dgs, 32000, dx, 64,
                                          32000, P, P, n, 500, 64, None, None, 0, None)

    for bad in (dict(saved=None), dict(dy=None), dict(dg=None), dict(dx=None), dict(dx=ODD), dict(dgs=5)):
        assert call(**bad) == -1, bad
    assert call(t=5) == -3
    assert call(n=0) == 0


def test_recurrence_queries(L):
    b, r = ctypes.c_size_t(), ctypes.c_uint64()
    for length, rows in ((0, 1), (1, 1), (128, 1), (129, 2), (1280, 10)):
        assert L.lcpp_recurrence_checkpoint_rows(length, ctypes.byref(r)) == 0 and r.value == rows
    assert L.lcpp_recurrence_checkpoint_rows(1 << 31, ctypes.byref(r)) == -1
    assert L.lcpp_recurrence_checkpoint_rows(1, None) == -1
    # one tile needs no state; more need a word of 8 bytes for each lane's channel and tile
    assert L.lcpp_recurrence_temp_bytes(7, 128, 1000, ctypes.byref(b)) == 0 and b.value == 0
    assert L.lcpp_recurrence_temp_bytes(7, 129, 1000, ctypes.byref(b)) == 0 and b.value == 256 + 7 * 2 * 1024 * 8
    assert L.lcpp_recurrence_temp_bytes(1, 1 << 32, 1, ctypes.byref(b)) == -1
    assert L.lcpp_recurrence_temp_bytes(1, 1, 1, None) == -1


def test_recurrence_step(L):
    def call(t=BF16, g=2, gate=P, x=P, s=P, s2=P, slots=P, pool=9, y=P, ys=64, n=4, c=64):
        return L.lcpp_recurrence_step(t, g, gate, 64, x, 64, s, s2, slots, pool, y, ys, n, c, None)

    for bad in (dict(gate=None), dict(x=None), dict(s=None), dict(s2=None), dict(y=None), dict(ys=4), dict(g=5),
                dict(slots=P + 2), dict(slots=None, pool=3), dict(pool=1 << 32), dict(s=P + 2)):
        assert call(**bad) == -1, bad
    assert call(t=1) == -3
    assert call(n=0) == 0 and call(c=0) == 0


def test_other_entry_points_refuse_the_new_types(L):
    b = ctypes.c_size_t()
    for t in (BF16, F16):
        assert L.lcpp_reduce_temp_bytes(t, 100, ctypes.byref(b)) == -3
        assert L.lcpp_scan_temp_bytes(t, 100, ctypes.byref(b)) == -3
        assert L.lcpp_radix_sort_keys_temp_bytes(t, 100, ctypes.byref(b)) == -3
        assert L.lcpp_reduce_sum(t, None, 0, P, P, 10, None) == -3
