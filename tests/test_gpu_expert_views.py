"""Views as outputs of the products: matrices side by side in the rows of one another, results whose rows begin anywhere."""
import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("outputs,inputs,pad", [(96, 64, 0), (33, 51, 0), (264, 136, 8)])
def test_matrices_side_by_side(gpu, outputs, inputs, pad, dtype):
    import lc_parallel_primitive_amd as lcpp

    log(f"matrices side by side {outputs} x {inputs} {dtype} pad {pad}")
    g = torch.Generator()
    g.manual_seed(outputs)
    lengths = [30, 0, 50, 7]
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    m = lcpp.DeviceExpertProduct()
    x, dy = ref.rows(g, (87, inputs), dtype), ref.rows(g, (87, outputs), dtype)
    w = ref.rows(g, (4, outputs, inputs), dtype)
    want = torch.empty_like(w)
    m.Backward(dy, x, w, offsets, None, want)
    wide = torch.full((outputs, 4, inputs + pad), 5.0, dtype=w.dtype, device="cuda")
    m.Backward(dy, x, w, offsets, None, wide.transpose(0, 1)[:, :, :inputs])
    assert torch.equal(wide.transpose(0, 1)[:, :, :inputs], want) and torch.all(wide[:, :, inputs:] == 5.0)
    # and read from there
    side = torch.empty(outputs, 4, inputs, dtype=w.dtype, device="cuda").transpose(0, 1)
    side.copy_(w)
    y, out = (torch.empty(87, outputs, dtype=w.dtype, device="cuda") for _ in range(2))
    m.Forward(x, w, offsets, y)
    m.Forward(x, side, offsets, out)
    assert torch.equal(out, y)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("offset,pad", [(1, 3), (8, 8), (3, 5)])
def test_results_anywhere(gpu, offset, pad, dtype):
    """Whole and partly empty tiles of 256 x 256 into rows of any alignment, from operands of whole chunks."""
    import lc_parallel_primitive_amd as lcpp

    log(f"results at {offset} of rows {pad} longer, {dtype}")
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    dt = ref.TYPES[dtype]
    lengths = [5000, 0, 300, 5001, 256]
    rows, cols, depth = sum(lengths), 2056, 72
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    m = lcpp.DeviceExpertProduct()
    x, w = (torch.randint(-3, 4, s, generator=g, device="cuda").to(dt) for s in ((rows, depth), (5, cols, depth)))
    across = w.transpose(1, 2).contiguous()
    want = torch.empty(rows, cols, dtype=dt, device="cuda")
    m.Forward(x, w, offsets, want)
    assert torch.equal(want[5000:5300], (x[5000:5300].float() @ across[2].float()).to(dt))
    for call in (lambda y: m.Forward(x, w, offsets, y), lambda y: m.Backward(x, None, across, offsets, y)):
        wide = torch.full((rows, cols + pad), 5.0, dtype=dt, device="cuda")
        flat = torch.full((wide.numel() + offset,), 5.0, dtype=dt, device="cuda")
        call(flat[offset:].view_as(wide)[:, :cols])
        got = flat[offset:].view_as(wide)
        assert torch.equal(got[:, :cols], want) and torch.all(got[:, cols:] == 5.0) and torch.all(flat[:offset] == 5.0)
