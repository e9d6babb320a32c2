"""A workspace kept for larger calls holds what an earlier call left in its status word: a later call that does not need
the workspace must not report that as its own."""
import pytest
import torch

from conftest import log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lcpp(gpu):
    import lc_parallel_primitive_amd as m

    return m


def stale():
    return torch.full((4096,), 255, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("length", [0, 1, 16, 17, 65, 128])
def test_recurrences_of_one_tile(lcpp, length, packed):
    log(f"recurrence of {length} rows on a stale workspace, packed {packed}")
    n, c = 3, 70
    shape = (n * length, c) if packed else (n, length, c)
    where = {}
    if packed:
        at = torch.arange(n, dtype=torch.int32) * length
        where = dict(d_begin_offsets=at.cuda(), d_end_offsets=(at + length).cuda(), max_length=length)
    x, y, dg, dx = (torch.zeros(shape, device="cuda") for _ in range(4))
    h0, hT, dh0 = (torch.ones(n, c, device="cuda") for _ in range(3))
    saved = torch.zeros(n, 1, c, device="cuda")
    m = lcpp.DeviceGatedRecurrence().create(debug_stream=torch.cuda.current_stream())
    temp = stale()
    m.Forward(temp, x, x, y, "sigmoid", h0, hT, saved, **where)
    assert int(temp[:4].view(torch.int32)[0]) == 0
    temp = stale()
    m.Backward(temp, x, x, saved, x, dg, dx, "sigmoid", h0, dh0, **where)
    assert int(temp[:4].view(torch.int32)[0]) == 0
    assert bool((temp[256:] == 255).all())


def test_recurrences_of_nothing(lcpp):
    log("recurrence of no sequences on a stale workspace")
    m = lcpp.DeviceGatedRecurrence().create(debug_stream=torch.cuda.current_stream())
    for shape in ((0, 300, 5), (2, 300, 0)):
        x = torch.zeros(shape, device="cuda")
        saved = torch.zeros(shape[0], 3, shape[2], device="cuda")
        m.Forward(stale(), x, x, x.clone(), "sigmoid", d_checkpoints=saved)
        m.Backward(stale(), x, x, saved, x, x.clone(), x.clone(), "sigmoid")


def test_layer_norm_gradients_over_no_rows(lcpp):
    log("layer norm of no rows on a stale workspace")
    m = lcpp.DeviceLayerNorm().create(debug_stream=torch.cuda.current_stream())
    w = torch.ones(50, device="cuda")
    x, stat = torch.empty(0, 50, device="cuda"), torch.empty(0, device="cuda")
    for dw, db in ((w.clone(), w.clone()), (w.clone(), None), (None, w.clone())):
        temp = stale()
        m.Backward(temp, x, x, w, stat, stat, x.clone(), dw, db)
        assert int(temp[:4].view(torch.int32)[0]) == 0
        temp = stale()
        m.AddBackward(temp, x, None, x, w, stat, stat, x.clone(), x.clone(), dw, db)
        assert int(temp[:4].view(torch.int32)[0]) == 0
        assert not any(bool(v.any()) for v in (dw, db) if v is not None)


def test_layer_norm_gradients_of_nothing(lcpp):
    log("layer norm of no columns on a stale workspace")
    m = lcpp.DeviceLayerNorm().create(debug_stream=torch.cuda.current_stream())
    x, stat = torch.empty(0, 50, device="cuda"), torch.empty(0, device="cuda")
    m.Backward(stale(), x, x, None, stat, stat, x.clone())
    m.AddBackward(stale(), x, None, x, None, stat, stat, x.clone(), x.clone())
    x, w, stat = torch.empty(4, 0, device="cuda"), torch.empty(0, device="cuda"), torch.ones(4, device="cuda")
    m.Backward(stale(), x, x, w, stat, stat, x.clone(), w.clone(), w.clone())
    m.AddBackward(stale(), x, None, x, w, stat, stat, x.clone(), x.clone(), w.clone(), w.clone())
