"""DeviceGatedRecurrence over many tiles: the state before a tile is made of the tiles before it one after the other, so
the bits are those of that order, whichever of their words a tile found first, and the same at every call."""
import numpy as np
import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu

TILE = 128


@pytest.fixture(scope="module")
def lcpp(gpu):
    import lc_parallel_primitive_amd as m

    return m


def buffers(lcpp, n, t, c):
    b = lcpp.DeviceGatedRecurrence.GetTempStorageBytes(n, t, c)
    temp = torch.full((b,), 255, dtype=torch.uint8, device="cuda")
    return temp, torch.empty(n, lcpp.DeviceGatedRecurrence.GetCheckpointRows(t), c, device="cuda")


@pytest.mark.parametrize("n,tiles,c", [(1, 400, 64), (3, 60, 130), (1, 9, 1000)])
def test_one_rounding_a_tile(lcpp, n, tiles, c):
    """Inputs of 0, and one row of a tile whose gate is not 1: the state is the initial one times one gate after the
    other, rounded to 32 bits at each, as numpy computes it; products of gates would be rounded differently."""
    log(f"recurrence, {tiles} tiles of one factor each, {n} x {c}")
    t = tiles * TILE - 5
    rng = np.random.default_rng(tiles)
    factor = rng.uniform(0.97, 1.03, size=(n, tiles, c)).astype(np.float32)
    h0, dhT = (rng.standard_normal((n, c)).astype(np.float32) for _ in range(2))
    gate = torch.ones(n, t, c)
    gate[:, 37::TILE] = torch.from_numpy(factor)
    gate, zero = gate.cuda(), torch.zeros(n, t, c, device="cuda")
    after, h = np.empty((n, tiles, c), np.float32), h0
    for k in range(tiles):
        h = after[:, k] = h * factor[:, k]
    before, e = np.empty((n, tiles, c), np.float32), dhT  # the gradient before each factor's row
    for k in range(tiles - 1, -1, -1):
        e = before[:, k] = e * factor[:, k]
    temp, saved = buffers(lcpp, n, t, c)
    m = lcpp.DeviceGatedRecurrence()
    y, dg, dx = (torch.empty_like(zero) for _ in range(3))
    hT, dh0 = torch.empty(n, c, device="cuda"), torch.empty(n, c, device="cuda")
    for _ in range(3):
        m.Forward(temp, gate, zero, y, "decay", torch.from_numpy(h0).cuda(), hT, saved)
        m.Backward(temp, gate, zero, saved, zero, dg, dx, "decay", torch.from_numpy(dhT).cuda(), dh0)
        assert np.array_equal(y[:, 37::TILE].cpu().numpy(), after)
        assert np.array_equal(y[:, TILE - 6::TILE].cpu().numpy(), after)
        assert np.array_equal(hT.cpu().numpy(), after[:, -1])
        assert np.array_equal(dx[:, 36::TILE].cpu().numpy(), before)
        assert np.array_equal(dx[:, 0::TILE].cpu().numpy(), before)
        assert np.array_equal(dh0.cpu().numpy(), before[:, 0])


@pytest.mark.parametrize("kind", ["decay", "log", "sigmoid"])
@pytest.mark.parametrize("n,t,c,dtype", [(1, 30000, 64, "float32"), (5, 5000, 333, "bfloat16"), (40, 1000, 130, "float16")])
def test_the_same_bits_at_every_call(lcpp, kind, n, t, c, dtype):
    log(f"recurrence, repeated, {kind} {n} x {t} x {c} {dtype}")
    g = torch.Generator()
    g.manual_seed(t)
    gate = ref.rows(g, (n, t, c), dtype)
    a = torch.exp(-1 / torch.exp(torch.rand(n, t, c, generator=g) * 8))
    gate.copy_({"decay": a, "log": torch.log(a), "sigmoid": torch.randn(n, t, c, generator=g) + 4}[kind])
    x, dy = ref.rows(g, (n, t, c), dtype), ref.rows(g, (n, t, c), dtype)
    h0, dhT = torch.randn(n, c, generator=g).cuda(), torch.randn(n, c, generator=g).cuda()
    temp, saved = buffers(lcpp, n, t, c)
    m = lcpp.DeviceGatedRecurrence()
    first = None
    for _ in range(6):
        y, dg, dx, hT, dh0 = (torch.full_like(v, 7.0) for v in (x, x, x, h0, h0))
        m.Forward(temp, gate, x, y, kind, h0, hT, saved)
        m.Backward(temp, gate, x, saved, dy, dg, dx, kind, dhT, dh0)
        got = (y, dg, dx, hT, dh0, saved.clone())
        first = first or got
        for p, q in zip(got, first):
            assert torch.equal(p, q)
