"""DeviceGatedRecurrence over many packed sequences of very different lengths: temp storage and checkpoints of the sizes
that the packed queries give and not a byte more, every sequence against its definition in 64 bits, and the same bits
as the sequence gives alone."""
import pytest
import torch

import block_ref as ref
from conftest import log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lcpp(gpu):
    import lc_parallel_primitive_amd as m

    return m


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def lengths(kind, g):
    """Sequence lengths in the order of the rows."""
    def short(n, most):
        return torch.randint(0, most, (n,), generator=g).tolist()

    if kind == "one long first":
        return [5000] + short(300, 150)
    if kind == "one long last":
        return short(300, 150) + [5000]
    if kind == "two blocks of the list":
        return short(255, 300) + [1300, 0, 700] + short(40, 300)
    if kind == "one long, all others empty":
        return [0] * 130 + [2000] + [0] * 500
    if kind == "many of one tile":
        return short(2000, 100) + [129]
    if kind == "all alike":
        return [400] * 70
    if kind == "around the tiles":
        return [127, 128, 129, 255, 256, 257, 1, 0, 384, 385] * 9
    if kind == "a few long ones":
        return [3000, 2999, 0, 4097]
    raise ValueError(kind)


def guarded(n, dtype, shape):
    """A tensor of `shape`, and the 4096 bytes behind it (a pattern that no call may touch)."""
    size = torch.empty((), dtype=dtype).element_size()
    flat = torch.full((n * size + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    return flat[:n * size].view(dtype).view(shape), flat[n * size:]


KINDS = ["one long first", "one long last", "two blocks of the list", "one long, all others empty", "many of one tile",
         "all alike", "around the tiles", "a few long ones"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("channels,dtype,gate", [(64, "float32", "decay"), (130, "bfloat16", "sigmoid"), (257, "float16", "log"),
                                                 (1100, "bfloat16", "log")])
def test_sequences_of_all_lengths(lcpp, kind, channels, dtype, gate):
    g = gen(channels)
    lens = lengths(kind, g)
    n, c, longest = len(lens), channels, max(lens)
    end = torch.tensor(lens).cumsum(0) + 7  # rows of no sequence before and behind
    begin = end - torch.tensor(lens)
    order = torch.randperm(n, generator=g)  # the sequences are not in the order of their rows
    begin, end, lens = begin[order].tolist(), end[order].tolist(), [lens[i] for i in order.tolist()]
    rows = max(end) + 5
    log(f"recurrence packed, {kind}: {n} sequences, {rows} rows x {c} {dtype} {gate}")
    a = torch.exp(-1 / torch.exp(torch.rand(rows, c, generator=g) * 6))
    gt = {"decay": a, "log": torch.log(a), "sigmoid": torch.randn(rows, c, generator=g) * 2 + 1.5}[gate].to(ref.TYPES[dtype]).cuda()
    x, dy = ref.rows(g, (rows, c), dtype), ref.rows(g, (rows, c), dtype)
    h0, dhT = torch.randn(n, c, generator=g).cuda(), torch.randn(n, c, generator=g).cuda()
    m = lcpp.DeviceGatedRecurrence()
    nbytes = m.GetTempStorageBytes(n, longest, c, rows)
    assert nbytes <= 256 + (rows // 128 + n) * (-(-c // 128) * 128 * 8 + 32) + 512
    temp, behind_temp = guarded(nbytes, torch.uint8, (nbytes,))
    held = m.GetPackedCheckpointRows(n, longest, rows)
    assert held <= rows // 128 + n
    saved, behind_saved = guarded(held * c, torch.float32, (held, c))
    y, dg, dx = (torch.full_like(x, 7.0) for _ in range(3))
    hT, dh0 = torch.full((n, c), 7.0, device="cuda"), torch.full((n, c), 7.0, device="cuda")
    where = dict(d_begin_offsets=torch.tensor(begin, dtype=torch.int32).cuda(),
                 d_end_offsets=torch.tensor(end, dtype=torch.int32).cuda(), max_length=longest)
    m.Forward(temp, gt, x, y, gate, h0, hT, saved, **where)
    if nbytes:
        temp.fill_(0x5A)
    m.Backward(temp, gt, x, saved, dy, dg, dx, gate, dhT, dh0, **where)
    torch.cuda.synchronize()
    assert bool((behind_temp == 0xA5).all()) and bool((behind_saved == 0xA5).all())
    if nbytes:
        assert int(temp[:4].view(torch.int32)[0]) == 0  # the status word
    covered = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for b, e in zip(begin, end):
        covered[b:e] = True
    for v in (y, dg, dx):
        assert bool((v[~covered] == 7.0).all())
    # all sequences: the same bits as alone
    pick = sorted(range(n), key=lambda s: -lens[s])[:4] + torch.randperm(n, generator=g)[:12].tolist()
    for s in pick:
        b, e = begin[s], end[s]
        one = [torch.full((1, e - b, c), 7.0, dtype=x.dtype, device="cuda") for _ in range(3)]
        o_hT, o_dh0 = torch.empty(1, c, device="cuda"), torch.empty(1, c, device="cuda")
        tb = m.GetTempStorageBytes(1, e - b, c)
        t1 = torch.empty(tb, dtype=torch.uint8, device="cuda") if tb else None
        s1 = torch.empty(1, m.GetCheckpointRows(e - b), c, device="cuda")
        view = [v[b:e][None] for v in (gt, x, dy)]
        m.Forward(t1, view[0], view[1], one[0], gate, h0[s:s + 1], o_hT, s1)
        m.Backward(t1, view[0], view[1], s1, view[2], one[1], one[2], gate, dhT[s:s + 1], o_dh0)
        for got, want in zip((y, dg, dx), one):
            assert torch.equal(got[b:e], want[0]), (s, b, e)
        assert torch.equal(hT[s], o_hT[0]) and torch.equal(dh0[s], o_dh0[0]), (s, b, e)
    # some against the definition
    for s in pick[2:8]:
        b, e = begin[s], end[s]
        h = ref.host(h0[s])
        hs, al, share, errs = ref.recurrence(gate, ref.host(gt[b:e]), ref.host(x[b:e]), h)
        zero = torch.zeros(c, dtype=torch.float64)
        ref.check(y[b:e], hs, errs, dtype, f"y of sequence {s}")
        ref.check(hT[s], hs[-1] if e > b else h, errs[-1] if e > b else zero, "float32", f"final state {s}")
        wg, wx, wh, bg, bx, bh = ref.recurrence_grad(gate, ref.host(gt[b:e]), ref.host(x[b:e]), h, hs, errs, al, share,
                                                     ref.host(dy[b:e]), ref.host(dhT[s]))
        ref.check(dg[b:e], wg, bg, dtype, f"dg of sequence {s}")
        ref.check(dx[b:e], wx, bx, dtype, f"dx of sequence {s}")
        ref.check(dh0[s], wh, bh, "float32", f"dh0 of sequence {s}")
    # every sequence's end: the final state is the last row's before it is rounded to the rows' type
    some = [s for s in range(n) if lens[s]]
    ends = torch.tensor([end[s] - 1 for s in some], device="cuda")
    assert torch.equal(hT[some].to(x.dtype), y[ends])
    empty = [s for s in range(n) if not lens[s]]
    assert torch.equal(hT[empty], h0[empty]) and torch.equal(dh0[empty], dhT[empty])


def test_longer_than_max_length_and_past_the_rows(lcpp):
    """Sequences are cut at max_length and at the tensors' rows; those that begin behind the rows are empty."""
    log("recurrence packed, clipped offsets")
    g = gen(4)
    rows, c, longest = 1000, 70, 300
    gt, x = torch.rand(rows, c, generator=g).cuda(), ref.rows(g, (rows, c), "float32")
    begin = torch.tensor([0, 400, 800, 1000, 1 << 31, 4000000000, 350], dtype=torch.int64)
    end = torch.tensor([350, 650, 5000, 1200, (1 << 31) + 9, 4100000000, 340], dtype=torch.int64)
    spans = [(0, 300), (400, 650), (800, 1000), (0, 0), (0, 0), (0, 0), (0, 0)]
    h0, hT = torch.randn(7, c, generator=g).cuda(), torch.empty(7, c, device="cuda")
    y = torch.full_like(x, 7.0)
    m = lcpp.DeviceGatedRecurrence()
    temp = torch.empty(m.GetTempStorageBytes(7, longest, c, rows), dtype=torch.uint8, device="cuda")
    off = [(v - (v >= 1 << 31).long() * (1 << 32)).to(torch.int32).cuda() for v in (begin, end)]
    m.Forward(temp, gt, x, y, "decay", h0, hT, d_begin_offsets=off[0], d_end_offsets=off[1], max_length=longest)
    covered = torch.zeros(rows, dtype=torch.bool)
    for s, (b, e) in enumerate(spans):
        covered[b:e] = True
        hs, _, _, errs = ref.recurrence("decay", ref.host(gt[b:e]), ref.host(x[b:e]), ref.host(h0[s]))
        ref.check(y[b:e], hs, errs, "float32", f"y of sequence {s}")
        if e == b:
            assert torch.equal(hT[s], h0[s])
    assert bool((y.cpu()[~covered] == 7.0).all())


def test_refusals(lcpp):
    m = lcpp.DeviceGatedRecurrence()
    x = torch.zeros(600, 32, device="cuda")
    y = torch.zeros_like(x)
    begin, end = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((3,), 200, dtype=torch.int32, device="cuda")
    where = dict(d_begin_offsets=begin, d_end_offsets=end, max_length=200)
    temp = torch.empty(m.GetTempStorageBytes(3, 200, 32, 600), dtype=torch.uint8, device="cuda")
    with pytest.raises(lcpp.LcppError) as e:
        m.Forward(temp[:-256], x, x, y, "decay", **where)
    assert e.value.status == -2
    held = m.GetPackedCheckpointRows(3, 200, 600)
    with pytest.raises(ValueError):
        m.Forward(temp, x, x, y, "decay", d_checkpoints=torch.empty(held - 1, 32, device="cuda"), **where)
    with pytest.raises(ValueError):
        m.Backward(temp, x, x, torch.empty(held * 32 - 1, device="cuda"), x, y, y.clone(), "decay", **where)
