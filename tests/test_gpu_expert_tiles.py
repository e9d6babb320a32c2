"""The experts' products with many tiles: every size of tile, several tiles to a workgroup, whole ones next to partly empty
ones, experts without rows between others, sums of one to five stages.  Values are small whole numbers, so that every product
and sum is exact and results are compared bit by bit."""
import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
T = {**ref.TYPES, "float8_e4m3fn": E4M3}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def whole(g, shape, dtype, pad=0):
    """-3 .. 3 in rows `pad` elements further apart than they are long."""
    view = torch.empty(*shape[:-1], shape[-1] + pad, dtype=dtype, device="cuda")[..., :shape[-1]]
    view.copy_(torch.randint(-3, 4, shape, generator=g, device="cuda").float())
    return view


def offsets_of(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()


def each(lengths):
    at = 0
    for e, n in enumerate(lengths):
        yield e, slice(at, at + n)
        at += n


def uneven(experts, rows, seed):
    """Lengths that add up to rows: some of 0, of 1 and around the tiles' edges, the rest uneven."""
    g = torch.Generator()
    g.manual_seed(seed)
    some = [0, 1, 255, 0, 256, 257, 64, 0, 129, 127][:experts - 2]
    share = torch.rand(experts - len(some), generator=g) + 0.1
    lengths = [int(v) for v in share / share.sum() * (rows - sum(some))]
    lengths[0] += rows - sum(some) - sum(lengths)
    return [v for pair in zip(lengths, some) for v in pair] + lengths[len(some):] + some[len(lengths):]


# What the host's rule takes on 256 CUs (tiles of 128 x 128 past 819 are large ones; up to 32 rows an expert 32 x 128).
# name: (lengths, columns of the results, [sums])
WAYS = {
    "256, whole columns": (uneven(12, 11000, 1), 2048, [64, 200]),
    "256, partial columns": (uneven(14, 10007, 2), 2056, [32, 72, 192]),
    "256, one expert": ([9000], 2304, [136]),
    "128, a second tile": (uneven(10, 2600, 3), 4104, [40, 128, 192]),
    "128, eight tiles": ([49] * 1000 + [60, 0, 50, 49], 520, [64, 136]),
    "32, six tiles": ([1 + i * 7 % 47 for i in range(200)], 1032, [32, 64, 136, 200, 320]),
    "32, empty experts": ([0, 0, 33, 0, 1] * 80, 2048, [96, 256]),
}


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("way", WAYS)
def test_rows(gpu, way, dtype):
    """Forward, and the gradient of the rows."""
    import lc_parallel_primitive_amd as lcpp

    lengths, cols, sums = WAYS[way]
    rows, experts, dt = sum(lengths), len(lengths), T[dtype]
    m, offsets = lcpp.DeviceExpertProduct(), offsets_of(lengths)
    for depth in sums:
        log(f"tiles {way}: {rows} rows of {experts}, {cols} of {depth} {dtype}")
        g = gen(depth)
        x, w = whole(g, (rows, depth), dt), whole(g, (experts, cols, depth), dt)
        y = torch.full((rows + 3, cols), 5.0, dtype=dt, device="cuda")
        m.Forward(torch.cat([x, x.new_full((3, depth), float("nan"))]), w, offsets, y)
        across = w.transpose(1, 2).contiguous()
        dx = torch.full((rows + 3, cols), 5.0, dtype=dt, device="cuda")
        m.Backward(torch.cat([x, x.new_full((3, depth), float("nan"))]), None, across, offsets, dx)
        for e, s in each(lengths):
            want = (x[s].float() @ across[e].float()).to(dt)
            assert torch.equal(y[s], want), f"expert {e}: {int((y[s] != want).sum())} values of {want.numel()}"
            assert torch.equal(dx[s], want), f"gradient, expert {e}: {int((dx[s] != want).sum())} values of {want.numel()}"
        assert torch.all(y[rows:] == 5.0) and torch.all(dx[rows:] == 5.0)


# (lengths, outputs, inputs)
MATRICES = {
    "256, partial": ([0, 1, 63, 64, 65, 0, 128, 200, 7, 300, 0, 90], 1288, 1032),
    "256, whole": ([70, 0, 0, 129, 64, 1], 2048, 2560),
    "128, a second tile": ([0, 40, 129, 64, 0, 65, 200, 1, 0], 1032, 1032),
    "128, few experts": ([500, 0, 333], 2056, 2048),
}


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("way", MATRICES)
def test_matrices(gpu, way, dtype):
    import lc_parallel_primitive_amd as lcpp

    lengths, outputs, inputs = MATRICES[way]
    rows, experts, dt = sum(lengths), len(lengths), T[dtype]
    log(f"tiles of matrices {way}: {rows} rows of {experts}, {outputs} x {inputs} {dtype}")
    g = gen(outputs)
    x, dy = whole(g, (rows, inputs), dt), whole(g, (rows, outputs), dt)
    w = torch.zeros((), dtype=dt, device="cuda").expand(experts, outputs, inputs).contiguous()
    for wide in (False, True):
        dw = torch.full(w.shape, 5.0, dtype=torch.float32 if wide else dt, device="cuda")
        lcpp.DeviceExpertProduct().Backward(dy, x, w, offsets_of(lengths), None, dw)
        for e, s in each(lengths):
            want = (dy[s].float().t().contiguous() @ x[s].float()).to(dw.dtype)
            assert torch.equal(dw[e], want), f"expert {e}, wide {wide}: {int((dw[e] != want).sum())} values"


def test_more_matrices_than_are_listed(gpu):
    """19200 tiles of 256 x 256, which are past the 512 chunks that the XCDs are dealt by what they have to do."""
    import lc_parallel_primitive_amd as lcpp

    experts, size = 300, 2048
    lengths = [i % 5 * 16 + i % 3 for i in range(experts)]
    log(f"tiles of matrices: {experts} experts of {size} x {size}")
    g = gen(9)
    x, dy = whole(g, (sum(lengths), size), torch.bfloat16), whole(g, (sum(lengths), size), torch.bfloat16)
    w = torch.zeros(1, size, size, dtype=torch.bfloat16, device="cuda").expand(experts, size, size)
    dw = torch.full((experts, size, size), 5.0, dtype=torch.bfloat16, device="cuda")
    lcpp.DeviceExpertProduct().Backward(dy, x, w, offsets_of(lengths), None, dw)
    for e, s in each(lengths):
        want = (dy[s].float().t().contiguous() @ x[s].float()).bfloat16()
        assert torch.equal(dw[e], want), f"expert {e}"


EIGHT = {
    "256, whole columns": (uneven(12, 11000, 4), 2048, [128, 400]),
    "256, partial columns": (uneven(14, 10007, 5), 2064, [64, 272]),
    "128, a second tile": (uneven(10, 2600, 6), 4104, [16, 256, 400]),
    "128, eight tiles": ([49] * 1000 + [60, 0, 50, 49], 520, [144]),
    "32, several tiles": ([1 + i * 7 % 47 for i in range(200)], 1032, [128, 528]),
    "32, empty experts": ([0, 0, 33, 0, 1] * 80, 2048, [384]),
    "registers": (uneven(10, 2600, 7), 4101, [131, 300]),
}


@pytest.mark.parametrize("out", ["bfloat16", "float32"])
@pytest.mark.parametrize("way", EIGHT)
def test_eight_bits(gpu, way, out):
    """Scales are powers of two: their products are exact too."""
    import lc_parallel_primitive_amd as lcpp

    lengths, cols, sums = EIGHT[way]
    rows, experts, dt = sum(lengths), len(lengths), T[out]
    for depth in sums:
        log(f"tiles in 8 bits {way}: {rows} rows of {experts}, {cols} of {depth} -> {out}")
        g = gen(depth + 1)
        parts = -(-depth // 128)
        x, w = whole(g, (rows, depth), E4M3), whole(g, (experts, cols, depth), E4M3)
        sx = torch.exp2(torch.randint(-2, 2, (rows, parts), generator=g, device="cuda").float())
        sw = torch.exp2(torch.randint(-2, 2, (experts, -(-cols // 128), parts), generator=g, device="cuda").float())
        y = torch.full((rows + 3, cols), 5.0, dtype=dt, device="cuda")
        # (rows behind the last: scales of NaN)
        more = torch.zeros(rows + 3, depth, dtype=torch.uint8, device="cuda").view(E4M3)
        more_scales = torch.full((rows + 3, parts), float("nan"), device="cuda")
        more[:rows].copy_(x)
        more_scales[:rows] = sx
        lcpp.DeviceExpertProduct().Forward(more, w, offsets_of(lengths), y, more_scales, sw)
        fx = x.float() * sx.repeat_interleave(128, 1)[:, :depth]
        for e, s in each(lengths):
            scale = sw[e].repeat_interleave(128, 0)[:cols].repeat_interleave(128, 1)[:, :depth]
            want = (fx[s] @ (w[e].float() * scale).t().contiguous()).to(dt)
            assert torch.equal(y[s], want), f"expert {e}: {int((y[s] != want).sum())} values of {want.numel()}"
        assert torch.all(y[rows:] == 5.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_registers(gpu, dtype):
    """Operands that are not whole chunks, several tiles to a workgroup, in all three products."""
    import lc_parallel_primitive_amd as lcpp

    dt, m = T[dtype], lcpp.DeviceExpertProduct()
    lengths = uneven(10, 2600, 8)
    rows, experts, offsets = sum(lengths), len(lengths), offsets_of(lengths)
    for cols, depth, pad in ((4099, 51, 0), (4104, 136, 1)):
        log(f"tiles by way of registers: {rows} rows of {experts}, {cols} of {depth} {dtype}, pad {pad}")
        g = gen(cols)
        x, w = whole(g, (rows, depth), dt, pad), whole(g, (experts, cols, depth), dt)
        y, dx = (torch.full((rows, cols), 5.0, dtype=dt, device="cuda") for _ in range(2))
        across = w.transpose(1, 2).contiguous()
        m.Forward(x, w, offsets, y)
        m.Backward(x, None, across, offsets, dx)
        for e, s in each(lengths):
            want = (x[s].float() @ across[e].float()).to(dt)
            assert torch.equal(y[s], want) and torch.equal(dx[s], want), f"expert {e}"
    lengths = [0, 40, 129, 64, 0, 65, 200, 1, 0]
    x, dy = whole(gen(1), (sum(lengths), 1031), dt), whole(gen(2), (sum(lengths), 1033), dt)
    dw = torch.full((len(lengths), 1033, 1031), 5.0, dtype=dt, device="cuda")
    m.Backward(dy, x, torch.zeros_like(dw), offsets_of(lengths), None, dw)
    for e, s in each(lengths):
        assert torch.equal(dw[e], (dy[s].float().t().contiguous() @ x[s].float()).to(dt)), f"expert {e}"


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("outputs,inputs", [(48, 64), (33, 51), (264, 136)])
def test_one_gradient_alone(gpu, outputs, inputs, dtype):
    """Either gradient without the other is the same, of the matrices' type and in 32 bits."""
    import lc_parallel_primitive_amd as lcpp

    log(f"one gradient alone {outputs} x {inputs} {dtype}")
    dt, m = T[dtype], lcpp.DeviceExpertProduct()
    lengths = [17, 0, 140, 3]
    g = torch.Generator()
    g.manual_seed(inputs)
    x, dy, w = (ref.rows(g, s, dtype) for s in ((160, inputs), (160, outputs), (4, outputs, inputs)))
    for kind in (dt, torch.float32):
        dx, dw = torch.empty_like(x), torch.empty(w.shape, dtype=kind, device="cuda")
        m.Backward(dy, x, w, offsets_of(lengths), dx, dw)
        alone_x, alone_w = torch.empty_like(dx), torch.empty_like(dw)
        m.Backward(dy, x, w, offsets_of(lengths), None, alone_w)
        m.Backward(dy, None, w, offsets_of(lengths), alone_x)
        assert torch.equal(alone_w, dw) and torch.equal(alone_x, dx)
        for e, s in each(lengths):
            want = (dy[s].double().t().contiguous() @ x[s].double()).cpu()
            size = (dy[s].double().abs().t().contiguous() @ x[s].double().abs()).cpu()
            ref.check(alone_w[e], want, ref.U32 * (160 + 1) * size, dtype if kind == dt else "float32", f"expert {e}")
