"""Rows of types that are only copied: any of 1, 2 or 4 bytes."""
import pytest
import torch

from conftest import log

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint16, torch.int16, torch.uint32, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz,
                                   torch.float8_e8m0fnu, torch.float8_e5m2])
@pytest.mark.parametrize("cols", [1, 7, 16, 130])
def test_dispatch_of_other_types(gpu, cols, dtype):
    import lc_parallel_primitive_amd as lcpp

    log(f"dispatch {cols} columns of {dtype}")
    size = dtype.itemsize
    g = torch.Generator()
    g.manual_seed(cols)
    top = 2 if dtype == torch.bool else 256
    x = torch.randint(0, top, (9, cols * size), generator=g, dtype=torch.uint8).cuda()
    positions = torch.randperm(18, generator=g).to(torch.int32).view(9, 2).cuda()
    positions[3, 1] = -1
    out = torch.zeros(18, cols * size, dtype=torch.uint8, device="cuda")
    lcpp.DeviceTokenSort().Dispatch(x.view(dtype), positions, out.view(dtype))
    want = torch.zeros_like(out)
    for t in range(9):
        for p in positions[t].tolist():
            if p >= 0:
                want[p] = x[t]
    assert torch.equal(out, want)


def test_dispatch_refuses_weights_of_other_types(gpu):
    import lc_parallel_primitive_amd as lcpp

    x, out = (torch.zeros(n, 16, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for n in (4, 8))
    i, w = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    with pytest.raises(TypeError):
        lcpp.DeviceTokenSort().Dispatch(x, i, out, w)
    for dtype in (torch.int64, torch.float64, torch.complex64):
        with pytest.raises(TypeError):
            lcpp.DeviceTokenSort().Dispatch(torch.zeros(4, 16, device="cuda").to(dtype), i, torch.zeros(8, 16, device="cuda").to(dtype))
