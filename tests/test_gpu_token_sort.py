"""Tokens sorted by expert, dispatched, combined and their gradients: places exactly, sums in 64 bits."""
import numpy as np
import pytest
import torch

import block_ref as ref
import expert_ref as eref
from conftest import log

pytestmark = pytest.mark.gpu


def sort(lcpp, ids, experts, with_sources=True):
    m = lcpp.DeviceTokenSort()
    n = ids.size
    d = torch.from_numpy(ids).cuda()
    positions = torch.full(ids.shape, -9, dtype=torch.int32, device="cuda")
    offsets = torch.full((experts + 1,), -9, dtype=torch.int32, device="cuda")
    sources = torch.full((n,), -9, dtype=torch.int32, device="cuda") if with_sources else None
    tb = m.GetTempStorageBytes(*ids.shape, experts)
    temp = torch.full((tb,), 255, dtype=torch.uint8, device="cuda") if tb else None
    m.Sort(temp, d, experts, positions, offsets, sources)
    return positions, offsets, sources


def drawn_ids(seed, tokens, k, experts, kind):
    rng = np.random.default_rng(seed)
    if kind == "one":
        return np.full((tokens, k), experts - 1, dtype=np.int32)
    if kind == "none":
        return np.full((tokens, k), -1, dtype=np.int32)
    ids = rng.integers(0, experts, (tokens, k)).astype(np.int32)
    if kind == "skewed":
        ids = np.minimum(ids, rng.integers(0, experts, (tokens, k))).astype(np.int32) // 2
    if kind == "foreign":
        ids[rng.random((tokens, k)) < 0.3] = -1
        ids[rng.random((tokens, k)) < 0.1] = experts
        ids[rng.random((tokens, k)) < 0.05] = np.iinfo(np.int32).min
        ids[rng.random((tokens, k)) < 0.05] = np.iinfo(np.int32).max
    return ids


SIZES = [(1, 1, 1), (1, 8, 128), (7, 3, 2), (48, 8, 128), (63, 1, 3), (65, 1, 5), (511, 2, 7), (513, 8, 64), (1000, 4, 60), (1024, 4, 1000),
         (2048, 8, 256), (2049, 8, 256), (5000, 6, 160), (20001, 3, 8), (32768, 8, 256), (40000, 10, 512), (70000, 8, 1024),
         (600001, 2, 16)]


@pytest.mark.parametrize("kind", ["even", "skewed", "foreign", "one", "none"])
@pytest.mark.parametrize("tokens,k,experts", SIZES)
def test_sort(gpu, tokens, k, experts, kind):
    import lc_parallel_primitive_amd as lcpp

    log(f"sort {tokens} x {k} of {experts} {kind}")
    ids = drawn_ids(tokens + k, tokens, k, experts, kind)
    want = eref.sorted_pairs(ids, experts)
    positions, offsets, sources = sort(lcpp, ids, experts)
    np.testing.assert_array_equal(offsets.cpu().numpy(), want[1])
    np.testing.assert_array_equal(positions.cpu().numpy(), want[0])
    got = sources.cpu().numpy()
    np.testing.assert_array_equal(got[:len(want[2])], want[2])
    assert np.all(got[len(want[2]):] == -9)  # rows behind the last are left alone
    positions, offsets, _ = sort(lcpp, ids, experts, with_sources=False)
    np.testing.assert_array_equal(positions.cpu().numpy(), want[0])


def test_sort_of_nothing(gpu):
    import lc_parallel_primitive_amd as lcpp

    positions, offsets, sources = sort(lcpp, np.zeros((0, 4), dtype=np.int32), 9)
    assert offsets.tolist() == [0] * 10


def case(seed, tokens, k, experts, kind="even"):
    ids = drawn_ids(seed, tokens, k, experts, kind)
    positions, offsets, sources = eref.sorted_pairs(ids, experts)
    return torch.from_numpy(positions).cuda(), len(sources), sources


ROWS = [(1, 1, 1, 1), (3, 2, 5, 7), (5, 4, 8, 8), (9, 8, 16, 64), (17, 3, 9, 200), (33, 6, 64, 513), (20, 10, 32, 1000), (12, 16, 40, 1024),
        (7, 20, 64, 1031), (9, 33, 64, 2048), (5, 64, 64, 515), (40, 8, 128, 2055), (16, 4, 8, 4096), (3, 8, 256, 8200), (700, 2, 4, 96)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("kind", ["even", "foreign"])
@pytest.mark.parametrize("tokens,k,experts,cols", ROWS)
def test_rows(gpu, tokens, k, experts, cols, kind, dtype):
    import lc_parallel_primitive_amd as lcpp

    log(f"rows {tokens} x {k} of {experts}, {cols} columns, {kind} {dtype}")
    m = lcpp.DeviceTokenSort()
    g = torch.Generator()
    g.manual_seed(cols + tokens)
    positions, used, sources = case(tokens, tokens, k, experts, kind)
    T, U = ref.TYPES[dtype], ref.U[dtype]
    many = tokens * k
    pad = cols % 3
    at = positions.cpu().long()
    has = at >= 0
    w = torch.randn(tokens, k, generator=g).cuda()
    wh = torch.where(has, ref.host(w), torch.zeros(()).double())
    x, y = ref.rows(g, (tokens, cols), dtype, pad, offset=1), ref.rows(g, (many, cols), dtype, pad)
    hx, hy = ref.host(x), ref.host(y)
    parts = torch.where(has[:, :, None], hy[at.clamp(min=0)], torch.zeros(()).double())

    # there: copies are exact, a product is rounded to 32 bits and then to the type
    for weights in (None, w):
        out = torch.full((many, cols + 2), 3.0, dtype=T, device="cuda")[:, 1:cols + 1]
        m.Dispatch(x, positions, out, weights)
        src = torch.from_numpy(sources.astype(np.int64))
        want = x.float()[(src // k).cuda()] * (1.0 if weights is None else w.flatten()[src.cuda()][:, None])
        assert torch.equal(out[:used], want.to(T))
        assert torch.all(out[used:] == 3.0)
    # ... and its gradient
    for weights in (None, w):
        dx = torch.empty(tokens, cols + pad, dtype=T, device="cuda")[:, :cols]
        m.DispatchBackward(y, positions, dx, weights)
        terms = parts if weights is None else parts * wh[:, :, None]
        ref.check(dx, terms.sum(1), ref.U32 * (k + 2) * terms.abs().sum(1), dtype, "dispatch's dx")
    dw, dx2 = torch.full((tokens, k), 5.0, device="cuda"), torch.empty_like(dx)
    m.DispatchBackward(y, positions, dx2, w, x, dw)
    ref.check(dx2, terms.sum(1), ref.U32 * (k + 2) * terms.abs().sum(1), dtype, "dispatch's dx beside dw")
    dots, size = (parts * hx[:, None]).sum(2), (parts * hx[:, None]).abs().sum(2)
    # (a thread's columns of 8200 over 256 threads: 40, six steps over lanes, four waves)
    ref.check(dw, dots, ref.U32 * 64 * size, "float32", "dispatch's dw")

    # back
    r = ref.rows(g, (tokens, cols), dtype, 1)
    for weights, residual in ((w, None), (w, r), (None, r)):
        out = torch.empty(tokens, cols, dtype=T, device="cuda")
        m.Combine(y, positions, weights, out, residual)
        terms = parts if weights is None else parts * wh[:, :, None]
        want, size = terms.sum(1), terms.abs().sum(1)
        if residual is not None:
            want, size = want + ref.host(r), size + ref.host(r).abs()
        ref.check(out, want, ref.U32 * (k + 2) * size, dtype, "combined")
    over = r.clone()
    m.Combine(y, positions, None, over, over)
    assert torch.equal(over, out)
    # ... and its gradient
    dy = torch.full((many, cols), 3.0, dtype=T, device="cuda")
    dw = torch.full((tokens, k), 5.0, device="cuda")
    m.CombineBackward(x, y, positions, w, dy, dw)
    want = x.float()[(src // k).cuda()] * w.flatten()[src.cuda()][:, None]
    assert torch.equal(dy[:used], want.to(T)) and torch.all(dy[used:] == 3.0)
    ref.check(dw, dots, ref.U32 * 64 * (parts * hx[:, None]).abs().sum(2), "float32", "combine's dw")
    only = torch.empty_like(dw)
    m.CombineBackward(x, y, positions, w, None, only)
    assert torch.equal(only, dw)
    dy2 = torch.full((many, cols), 3.0, dtype=T, device="cuda")
    m.CombineBackward(x, None, positions, w, dy2)
    assert torch.equal(dy2, dy)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.uint8, torch.int8, torch.int16, torch.int32])
@pytest.mark.parametrize("cols", [1, 5, 15, 16, 17, 130, 1024, 1500, 4099])
def test_copies_of_other_types(gpu, cols, dtype):
    import lc_parallel_primitive_amd as lcpp

    positions, used, sources = case(cols, 50, 3, 7, "foreign")
    g = torch.Generator()
    g.manual_seed(cols)
    e = torch.empty(0, dtype=dtype).element_size()
    x = torch.randint(0, 255, (50, (cols + 1) * e), generator=g, dtype=torch.uint8).cuda().view(dtype)[:, 1:]
    out = torch.zeros(150, (cols + 2) * e, dtype=torch.uint8, device="cuda").view(dtype)[:, 1:cols + 1]
    lcpp.DeviceTokenSort().Dispatch(x, positions, out)
    src = torch.from_numpy(sources.astype(np.int64) // 3).cuda()
    bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(bits(out)[:used], bits(x)[src]) and torch.all(bits(out)[used:] == 0)


def test_positions_out_of_range_and_values_of_no_pair(gpu):
    """Positions past the rows that there are count nothing; what lies in rows of no pair, or beside pairs of no row, is
    not read into any sum."""
    import lc_parallel_primitive_amd as lcpp

    m = lcpp.DeviceTokenSort()
    x = torch.ones(3, 40, device="cuda")
    y = torch.full((4, 40), float("nan"), device="cuda")
    y[2] = 2.0
    positions = torch.tensor([[2, -1], [4, 1 << 30], [-5, 9]], dtype=torch.int32, device="cuda")
    w = torch.full((3, 2), float("nan"), device="cuda")
    w[0, 0] = 0.5
    out, dw = torch.full((3, 40), 7.0, device="cuda"), torch.full((3, 2), 7.0, device="cuda")
    m.Combine(y, positions, w, out)
    assert torch.equal(out, torch.tensor([1.0, 0.0, 0.0], device="cuda")[:, None].expand(3, 40))
    dy = torch.full((4, 40), 7.0, device="cuda")
    m.CombineBackward(x, y, positions, w, dy, dw)
    assert torch.equal(dw, torch.tensor([[80.0, 0], [0, 0], [0, 0]], device="cuda"))
    assert torch.all(dy[2] == 0.5) and torch.all(dy[[0, 1, 3]] == 7.0)
    m.Dispatch(x, positions, dy)
    assert torch.all(dy[2] == 1.0) and torch.all(dy[[0, 1, 3]] == 7.0)


def test_no_columns_tokens_or_rows(gpu):
    import lc_parallel_primitive_amd as lcpp

    m = lcpp.DeviceTokenSort()
    p = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    dw = torch.full((3, 2), 7.0, device="cuda")
    m.CombineBackward(torch.empty(3, 0, device="cuda"), torch.empty(6, 0, device="cuda"), p, None, torch.empty(6, 0, device="cuda"), dw)
    assert torch.all(dw == 0)
    out = torch.full((3, 9), 7.0, device="cuda")
    m.Combine(torch.empty(0, 9, device="cuda"), p, None, out)
    assert torch.all(out == 0)
    m.Dispatch(torch.empty(0, 9, device="cuda"), p[:0], out)
    m.Dispatch(out, p, torch.empty(0, 9, device="cuda"))
    none = torch.empty(3, 0, dtype=torch.int32, device="cuda")
    m.Combine(out, none, None, out.clone().fill_(7.0), out)
