"""The RMS norm's 8-bit outputs where out / scale lies exactly half way between two values of the 8-bit type: the even one."""
import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu
QMAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def halves(qdtype):
    """The middles of neighbouring normal values below the type's largest, exact in 32 bits, as (middles, the even neighbours)."""
    values = torch.arange(256, dtype=torch.uint8).view(qdtype).float()
    values = values[torch.isfinite(values) & (values >= 2.0**-6)].sort().values
    low, high = values[:-1].double(), values[1:].double()
    # the even one of two neighbours has a 0 as its last bit: bit patterns rise with the values
    even_low = (low.float().to(qdtype).view(torch.uint8) & 1) == 0
    return (low + high) / 2, torch.where(even_low, low, high)


@pytest.mark.parametrize("qdtype", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("group", [128, 512, 0])
@pytest.mark.parametrize("cols,add", [(512, False), (1536, True), (2055, False), (20000, False)])
def test_ties(gpu, cols, add, group, qdtype):
    import lc_parallel_primitive_amd as lcpp

    log(f"rms ties {cols} group {group} {qdtype} add {add}")
    g = torch.Generator()
    g.manual_seed(cols + group)
    rows = 200
    middles, evens = halves(qdtype)
    # Scales of 16 significant bits: the largest value, QMAX of one, has 19 and a middle times one at most 20, so all are exact
    # in 32 bits.  eps = 1 beside squares below 2^-50 makes rstd exactly 1: out is the input.
    size = group or cols
    parts = -(-cols // size)
    scale = torch.randint(2**15, 2**16, (rows, parts), generator=g).double() * (2.0**-50 if QMAX[qdtype] < 500 else 2.0**-57)
    pick = torch.randint(0, middles.numel(), (rows, cols), generator=g)
    sign = torch.randint(0, 2, (rows, cols), generator=g).double() * 2 - 1
    each = scale.repeat_interleave(size, 1)[:, :cols]
    x, want = sign * middles[pick] * each, sign * evens[pick]
    first = torch.arange(parts) * size  # the group's largest value is its first one
    x[:, first], want[:, first] = QMAX[qdtype] * scale, torch.tensor(QMAX[qdtype]).double()
    assert torch.equal(x.float().double(), x) and float((x * x).mean(1).max()) < 2.0**-50
    x = x.float().cuda()
    q = torch.empty(rows, cols, dtype=qdtype, device="cuda")
    scales = torch.empty(rows, parts, device="cuda")
    norm, s = lcpp.DeviceRMSNorm(), torch.empty_like(x)
    if add:
        norm.AddForward(x, torch.zeros_like(x), s, None, None, 1.0, None, q, scales, group)
    else:
        norm.Forward(x, None, None, 1.0, None, q, scales, group)
    assert torch.equal(ref.host(scales), scale)
    got = q.float().cpu().double()
    wrong = got != want
    assert not bool(wrong.any()), f"{int(wrong.sum())} of {wrong.numel()} ties go the wrong way, the first {got[wrong][:4]} for {want[wrong][:4]}"


@pytest.mark.parametrize("qdtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_zeros_keep_their_sign(gpu, qdtype):
    import lc_parallel_primitive_amd as lcpp

    x = torch.ones(3, 128, device="cuda")
    x[:, 1], x[:, 2] = -0.0, 0.0
    q, scales = torch.empty(3, 128, dtype=qdtype, device="cuda"), torch.empty(3, 1, device="cuda")
    lcpp.DeviceRMSNorm().Forward(x, None, None, 1e-6, None, q, scales)
    bits = q.view(torch.uint8).cpu()
    assert bool((bits[:, 1] == 0x80).all()) and bool((bits[:, 2] == 0).all())
