"""Copies, sums and dots of more tokens than one round of workgroups takes, and the sort of very many pairs."""
import pytest
import torch

from conftest import log

pytestmark = pytest.mark.gpu


def test_more_tokens_than_workgroups(gpu):
    """2^20 workgroups of 32 narrow tokens, or of one wide one, and some more: small whole numbers, exactly."""
    import lc_parallel_primitive_amd as lcpp

    m = lcpp.DeviceTokenSort()
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    tokens, cols = 2**25 + 77, 8
    log(f"rows {tokens} x 1, {cols} columns")
    positions = torch.randperm(tokens, generator=g, device="cuda", dtype=torch.int32).view(tokens, 1)
    positions[5] = -1
    x = torch.randint(-3, 4, (tokens, cols), generator=g, device="cuda", dtype=torch.int8)
    rows = torch.full((tokens, cols), 7, dtype=torch.int8, device="cuda")
    m.Dispatch(x, positions, rows)
    back = rows[positions.flatten().long().clamp(min=0)]
    back[5] = x[5]
    assert torch.equal(back, x)
    del back
    x, rows = x.bfloat16(), rows.bfloat16()
    w = torch.randint(1, 3, (tokens, 1), generator=g, device="cuda").float()
    out, dw = torch.full_like(x, 9.0), torch.full((tokens, 1), 9.0, device="cuda")
    m.Combine(rows, positions, w, out, x)
    want = x.float() * (1 + w)
    want[5] = x[5].float()
    assert torch.equal(out, want.bfloat16())
    m.Dispatch(x, positions, rows, w)
    m.DispatchBackward(rows, positions, out, w, x, dw)
    want = x.float() * w * w
    dots = (x.float() * x.float()).sum(1, keepdim=True) * w
    want[5], dots[5] = 0, 0
    assert torch.equal(out, want.bfloat16()) and torch.equal(dw, dots)


def test_more_wide_tokens_than_workgroups(gpu):
    """Rows of 1032 columns of one long vector, each a place behind the one before."""
    import lc_parallel_primitive_amd as lcpp

    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    tokens, cols = 2**20 + 9, 1032
    log(f"dots of {tokens} x 1, {cols} columns")
    a, b = (torch.randint(-3, 4, (tokens + cols,), generator=g, device="cuda").bfloat16() for _ in range(2))
    few, many = a.as_strided((tokens, cols), (1, 1)), b.as_strided((tokens, cols), (1, 1))
    positions = (torch.arange(tokens, device="cuda", dtype=torch.int32).flip(0)).view(tokens, 1).contiguous()
    dots = torch.full((tokens, 1), 9.0, device="cuda")
    lcpp.DeviceTokenSort().CombineBackward(few, many, positions, None, None, dots)
    for at in range(0, tokens, 1 << 16):
        z = min(tokens, at + (1 << 16))
        want = (few[at:z].float() * many[tokens - z:tokens - at].flip(0).float()).sum(1)
        assert torch.equal(dots[at:z, 0], want), at


def test_very_many_pairs(gpu):
    import lc_parallel_primitive_amd as lcpp

    tokens, k, experts = 2**25 + 39, 2, 300
    log(f"sort {tokens} x {k} of {experts}")
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    ids = torch.randint(-1, experts + 1, (tokens, k), generator=g, device="cuda", dtype=torch.int32)
    m = lcpp.DeviceTokenSort()
    positions, sources = torch.full_like(ids, -9), torch.full((tokens * k,), -9, dtype=torch.int32, device="cuda")
    offsets = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    temp = torch.empty(m.GetTempStorageBytes(tokens, k, experts), dtype=torch.uint8, device="cuda")
    m.Sort(temp, ids, experts, positions, offsets, sources)
    flat = ids.flatten()
    good = (flat >= 0) & (flat < experts)
    counts = torch.bincount(flat[good], minlength=experts)
    assert torch.equal(offsets[1:].long(), counts.cumsum(0)) and int(offsets[0]) == 0
    used = int(offsets[-1])
    pair = sources[:used].long()
    key = flat[pair].long()
    # in the experts' order, each expert's in their own, and every one of them once
    assert bool(((key[1:] > key[:-1]) | ((key[1:] == key[:-1]) & (pair[1:] > pair[:-1]))).all())
    assert bool((sources[used:] == -9).all()) and bool((positions.flatten()[~good] == -1).all())
    assert torch.equal(positions.flatten()[pair].long(), torch.arange(used, device="cuda"))
