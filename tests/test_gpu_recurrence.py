"""DeviceGatedRecurrence against its definition in 64 bits: gates, types, lengths around the tiles' limits, odd channel
counts, strides, packed sequences with empty ones, states, gradients against the formula and against differences,
single tokens, and look-back waits that give up."""
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


def gates(g, kind, shape, dtype, pad=0, offset=0):
    """Gates whose memory is from one to some hundred steps long."""
    t = ref.rows(g, shape, dtype, pad, offset=offset)
    if kind == "sigmoid":
        t.copy_(torch.randn(shape, generator=g) * 2 + 1.5)
    else:
        a = torch.exp(-1 / torch.exp(torch.rand(shape, generator=g) * 6))
        t.copy_(torch.log(a) if kind == "log" else a * torch.where(torch.rand(shape, generator=g) < 0.02, -1.0, 1.0))
    return t


def temp_for(lcpp, sequences, length, channels):
    n = lcpp.DeviceGatedRecurrence.GetTempStorageBytes(sequences, length, channels)
    return torch.full((n,), 255, dtype=torch.uint8, device="cuda") if n else None


def saved_for(lcpp, sequences, length, channels):
    return torch.full((sequences, lcpp.DeviceGatedRecurrence.GetCheckpointRows(length), channels), 9.0, device="cuda")


def run_case(lcpp, kind, dtype, spans, shape, packed, pad=0, offset=0, states=True, backward=True):
    """spans: (sequence, first row, end) of every sequence in the flattened rows of `shape`."""
    log(f"recurrence {kind} {dtype} {tuple(shape)} packed {packed} pad {pad} offset {offset}")
    c, n = shape[-1], len(spans)
    g = gen(c + 7 * sum(shape))
    gt = gates(g, kind, shape, dtype, pad, offset)
    x = ref.rows(g, shape, dtype, pad + 1)
    y = ref.rows(g, shape, dtype, pad, offset=offset)
    dy = ref.rows(g, shape, dtype)
    h0 = torch.randn(n, c, generator=g).cuda() if states else None
    hT = torch.full((n, c), 7.0, device="cuda")
    longest = max((e - b for _, b, e in spans), default=0)
    where = {}
    if packed:
        where = dict(d_begin_offsets=torch.tensor([b for _, b, _ in spans], dtype=torch.int32).cuda(),
                     d_end_offsets=torch.tensor([e for _, _, e in spans], dtype=torch.int32).cuda(), max_length=longest)
    m = lcpp.DeviceGatedRecurrence()
    temp, saved = temp_for(lcpp, n, longest, c), saved_for(lcpp, n, longest, c)
    untouched = y.clone()
    m.Forward(temp, gt, x, y, kind, h0, hT, saved, **where)
    dg, dx = torch.full(shape, 7.0, dtype=x.dtype, device="cuda"), ref.rows(g, shape, dtype, 2)
    dx_before = dx.clone()
    dhT = torch.randn(n, c, generator=g).cuda() if states else None
    dh0 = torch.full((n, c), 7.0, device="cuda")
    if backward:
        m.Backward(temp, gt, x, saved, dy, dg, dx, kind, dhT, dh0, **where)
    flat = [ref.host(v).reshape(-1, c) for v in (gt, x, y, dy, dg, dx, untouched, dx_before)]
    covered = torch.zeros(flat[0].shape[0], dtype=torch.bool)
    for s, b, e in spans:
        covered[b:e] = True
        zero = torch.zeros(c, dtype=torch.float64)
        h = ref.host(h0[s]) if states else zero
        hs, a, share, errs = ref.recurrence(kind, flat[0][b:e], flat[1][b:e], h)
        ref.check(flat[2][b:e], hs, errs, dtype, f"y of sequence {s}")
        ref.check(hT[s], hs[-1] if e > b else h, errs[-1] if e > b else zero, "float32", f"final state {s}")
        if not backward:
            continue
        end = ref.host(dhT[s]) if states else zero
        wg, wx, wh, bg, bx, bh = ref.recurrence_grad(kind, flat[0][b:e], flat[1][b:e], h, hs, errs, a, share, flat[3][b:e], end)
        ref.check(flat[4][b:e], wg, bg, dtype, f"dg of sequence {s}")
        ref.check(flat[5][b:e], wx, bx, dtype, f"dx of sequence {s}")
        ref.check(dh0[s], wh, bh, "float32", f"dh0 of sequence {s}")
    # rows of no sequence are left alone
    assert torch.equal(flat[2][~covered], flat[6][~covered])
    if backward:
        assert bool((flat[4][~covered] == 7.0).all()) and torch.equal(flat[5][~covered], flat[7][~covered])


def even(n, t):
    return [(s, s * t, (s + 1) * t) for s in range(n)]


@pytest.mark.parametrize("kind", ["decay", "log", "sigmoid"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 64, 65, 127, 128, 129, 255, 257, 513, 1000])
def test_lengths(lcpp, kind, dtype, length):
    run_case(lcpp, kind, dtype, even(2, length), (2, length, 70), False)


@pytest.mark.parametrize("channels", [1, 2, 3, 63, 64, 65, 66, 127, 128, 129, 255, 300])
@pytest.mark.parametrize("kind,dtype", [("sigmoid", "bfloat16"), ("decay", "float32")])
def test_channels(lcpp, kind, dtype, channels):
    for length in (5, 40, 300):
        run_case(lcpp, kind, dtype, even(3, length), (3, length, channels), False)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (5, 3), (64, 2)])
def test_strides_and_alignment(lcpp, dtype, pad, offset):
    for channels in (33, 131):
        run_case(lcpp, "sigmoid", dtype, even(2, 200), (2, 200, channels), False, pad, offset)


@pytest.mark.parametrize("kind", ["decay", "log", "sigmoid"])
def test_packed(lcpp, kind):
    """Sequences of all lengths one behind the other, empty ones among them, rows between them that belong to none, in
    an order that is not that of the rows."""
    lens, at, spans = [0, 1, 300, 2, 0, 128, 129, 16, 17, 700], 3, []
    for i, n in enumerate(lens):
        spans.append((0, at, at + n))
        at += n + (i % 3)
    order = [3, 0, 9, 1, 2, 8, 4, 5, 7, 6]
    spans = [(k,) + spans[i][1:] for k, i in enumerate(order)]
    for dtype, channels in (("float32", 130), ("bfloat16", 64)):
        run_case(lcpp, kind, dtype, spans, (at + 5, channels), True)
    run_case(lcpp, kind, "float16", [(0, 4, 4), (1, 2, 2)], (9, 40), True)  # nothing but empty sequences


def test_no_states(lcpp):
    run_case(lcpp, "sigmoid", "float32", even(3, 400), (3, 400, 96), False, states=False)
    run_case(lcpp, "log", "bfloat16", [(0, 0, 250), (1, 250, 250), (2, 250, 260)], (260, 96), True, states=False)


def test_time_major_and_repeated_gate(lcpp):
    """(length, sequences, channels) through transposed views; a gate that repeats its row for every time and sequence."""
    log("recurrence, time major")
    g = gen(5)
    n, t, c = 3, 290, 132
    gt = gates(g, "sigmoid", (c,), "float32").expand(n, t, c)
    x = ref.rows(g, (t, n, c), "float32").transpose(0, 1)
    y = torch.empty(t, n, c, device="cuda").transpose(0, 1)
    m = lcpp.DeviceGatedRecurrence()
    m.Forward(temp_for(lcpp, n, t, c), gt, x, y, "sigmoid")
    for s in range(n):
        hs, _, _, errs = ref.recurrence("sigmoid", ref.host(gt[s]), ref.host(x[s]), torch.zeros(c, dtype=torch.float64))
        ref.check(y[s], hs, errs, "float32", f"sequence {s}")


def test_nothing_leaves_a_sequence(lcpp):
    """NaN and infinities in one sequence, and in rows past a packed sequence's end, change no other row or gradient;
    inside a sequence they reach the later rows of their own channel only."""
    log("recurrence with poisoned rows")
    g = gen(11)
    t, c, kind = 600, 130, "sigmoid"
    spans = torch.tensor([[0, 200], [230, 500], [500, 590]], dtype=torch.int32)
    b, e = spans[:, 0].contiguous().cuda(), spans[:, 1].contiguous().cuda()
    gt, x, dy = gates(g, kind, (t, c), "float32"), ref.rows(g, (t, c), "float32"), ref.rows(g, (t, c), "float32")
    m = lcpp.DeviceGatedRecurrence()

    def run(gt, x, dy):
        y, dg, dx = (torch.zeros(t, c, device="cuda") for _ in range(3))
        saved = saved_for(lcpp, 3, 270, c)
        w = dict(d_begin_offsets=b, d_end_offsets=e, max_length=270)
        m.Forward(temp_for(lcpp, 3, 270, c), gt, x, y, kind, d_checkpoints=saved, **w)
        m.Backward(temp_for(lcpp, 3, 270, c), gt, x, saved, dy, dg, dx, kind, **w)
        return y, dg, dx

    clean = run(gt, x, dy)
    bad = [v.clone() for v in (gt, x, dy)]
    for v in bad:
        v[200:230] = float("nan")
        v[590:] = float("inf")
    for got, want in zip(run(*bad), clean):
        assert torch.equal(got, want)
    x2 = x.clone()
    x2[300, 7] = float("nan")
    y, dg, dx = run(gt, x2, dy)
    same = torch.ones(t, c, dtype=torch.bool, device="cuda")
    same[300:500, 7] = False
    assert torch.equal(y[same], clean[0][same]) and torch.isnan(y[~same]).all()
    assert torch.equal(dx, clean[2])  # dx depends on the gates alone
    same[300:500, 7] = False
    assert torch.equal(dg[same], clean[1][same])


def test_saturated_gates(lcpp):
    """Gates at both ends: a of exactly 0 and 1, sigmoids of +-100, exp of -1000; nothing overflows."""
    log("recurrence with saturated gates")
    t, c = 300, 66
    for kind, values in (("decay", [0.0, 1.0]), ("log", [0.0, -1000.0, -1e30]), ("sigmoid", [100.0, -100.0, 1e30, -1e30])):
        g = gen(3)
        pick = torch.randint(0, len(values), (1, t, c), generator=g)
        gt = torch.tensor(values)[pick].cuda()
        x, dy = ref.rows(g, (1, t, c), "float32"), ref.rows(g, (1, t, c), "float32")
        y, dg, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        m = lcpp.DeviceGatedRecurrence()
        saved = saved_for(lcpp, 1, t, c)
        m.Forward(temp_for(lcpp, 1, t, c), gt, x, y, kind, d_checkpoints=saved)
        m.Backward(temp_for(lcpp, 1, t, c), gt, x, saved, dy, dg, dx, kind)
        zero = torch.zeros(c, dtype=torch.float64)
        a, share = ref.gate_values(kind, ref.host(gt[0]))
        h, hs = zero, []
        for i in range(t):
            h = a[i] * h + share[i] * ref.host(x[0, i])
            hs.append(h)
        # a and 1 - a are 0 and 1 to 1e-40: at most 300 sums of values under 5
        assert float((ref.host(y[0]) - torch.stack(hs)).abs().max()) <= 300 * 300 * 5 * ref.U32
        assert torch.isfinite(dg).all() and torch.isfinite(dx).all()
        if kind == "sigmoid":
            assert float(dg.abs().max()) <= 1e-30


def test_long_memory(lcpp):
    """100 000 rows of a decay that never forgets: the sum of all inputs, through 782 tiles."""
    log("recurrence, 100000 rows")
    t, c = 100_000, 64
    g = gen(2)
    x = ref.rows(g, (1, t, c), "float32")
    y, hT = torch.empty_like(x), torch.empty(1, c, device="cuda")
    one = torch.ones(1, 1, 1, device="cuda").expand(1, t, c)
    one = one.contiguous()
    m = lcpp.DeviceGatedRecurrence()
    m.Forward(temp_for(lcpp, 1, t, c), one, x, y, "decay", None, hT)
    want = torch.cumsum(ref.host(x), 1)
    # chains of 16 rows, 8 waves and 782 tiles: each rounding is of a sum under 6 sqrt(t)
    assert float((ref.host(y) - want).abs().max()) <= (16 + 8 + 782) * ref.U32 * 6 * t**0.5
    assert torch.equal(hT, y[:, -1])


def test_in_place_and_repeated(lcpp):
    log("recurrence in place")
    g = gen(9)
    n, t, c, kind = 4, 700, 190, "sigmoid"
    gt, x, dy = gates(g, kind, (n, t, c), "bfloat16"), ref.rows(g, (n, t, c), "bfloat16"), ref.rows(g, (n, t, c), "bfloat16")
    y, dg, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    m = lcpp.DeviceGatedRecurrence()
    temp, saved = temp_for(lcpp, n, t, c), saved_for(lcpp, n, t, c)
    m.Forward(temp, gt, x, y, kind, d_checkpoints=saved)
    m.Backward(temp, gt, x, saved, dy, dg, dx, kind)
    over = x.clone()
    m.Forward(temp, gt, over, over, kind)
    assert torch.equal(over, y)
    og, ox = gt.clone(), x.clone()
    m.Backward(temp, og, ox, saved, dy, og, ox, kind)
    assert torch.equal(og, dg) and torch.equal(ox, dx)
    assert int(temp[:4].view(torch.int32)[0]) == 0  # the status word


@pytest.mark.parametrize("channels", [129, 257, 1025, 2049])
def test_in_place_with_an_odd_channel(lcpp, channels):
    """The last channel's lane reads its neighbour's channel too, which another workgroup may already have written."""
    log(f"recurrence in place, {channels} channels")
    g = gen(channels)
    n, t, kind = 6, 400, "log"
    gt, x, dy = (gates(g, kind, (n, t, channels), "bfloat16"), ref.rows(g, (n, t, channels), "bfloat16"),
                 ref.rows(g, (n, t, channels), "bfloat16"))
    h0, dhT = torch.randn(n, channels, generator=g).cuda(), torch.randn(n, channels, generator=g).cuda()
    y, dg, dx, hT, dh0 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(h0), torch.empty_like(h0)
    m = lcpp.DeviceGatedRecurrence()
    temp, saved = temp_for(lcpp, n, t, channels), saved_for(lcpp, n, t, channels)
    m.Forward(temp, gt, x, y, kind, h0, hT, saved)
    m.Backward(temp, gt, x, saved, dy, dg, dx, kind, dhT, dh0)
    for _ in range(3):
        over, state = x.clone(), h0.clone()
        m.Forward(temp, gt, over, over, kind, state, state, saved)
        assert torch.equal(over, y) and torch.equal(state, hT)
        og, od, back = gt.clone(), dy.clone(), dhT.clone()
        m.Backward(temp, og, x, saved, od, og, od, kind, back, back)
        assert torch.equal(og, dg) and torch.equal(od, dx) and torch.equal(back, dh0)


@pytest.mark.parametrize("kind", ["decay", "log", "sigmoid"])
def test_gradient_against_differences(lcpp, kind):
    """dL along random directions, L = sum(y c) + sum(hT d).  h depends on a gate as a polynomial or exponential of it:
    with a step of 2^-9 (gates) or 2^-4 (inputs, in which h is linear) the central difference is off by step^2 / 6 of
    the third derivative, which a memory of at most 20 steps makes up to 400 times the first (2.6e-4), and by y's
    roundings, 2^-21 each and independent, over the step (2.4e-4): together under 5e-3 of |gradient| |direction|."""
    log(f"recurrence differences, {kind}")
    g = gen(21)
    n, t, c = 2, 300, 70
    a = 0.5 + 0.45 * torch.rand(n, t, c, generator=g)
    gt = {"decay": a, "log": torch.log(a), "sigmoid": torch.log(a / (1 - a))}[kind].cuda()
    x, w = ref.rows(g, (n, t, c), "float32"), ref.rows(g, (n, t, c), "float32")
    h0, d = torch.randn(n, c, generator=g).cuda(), torch.randn(n, c, generator=g).cuda()
    y, hT = torch.empty_like(x), torch.empty_like(h0)
    m = lcpp.DeviceGatedRecurrence()
    temp, saved = temp_for(lcpp, n, t, c), saved_for(lcpp, n, t, c)

    def loss(gt, x, h0):
        m.Forward(temp, gt, x, y, kind, h0, hT, saved)
        return float((y.double() * w.double()).sum() + (hT.double() * d.double()).sum())

    loss(gt, x, h0)
    dg, dx, dh0 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(h0)
    m.Backward(temp, gt, x, saved, w, dg, dx, kind, d, dh0)
    args = [gt, x, h0]
    for i, (grad, step) in enumerate(((dg, 2.0**-9), (dx, 2.0**-4), (dh0, 2.0**-4))):
        v = torch.randn(grad.shape, generator=g).cuda()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * v, args[i] - step * v
        got = (loss(*up) - loss(*down)) / (2 * step)
        want = float((grad.double() * v.double()).sum())
        assert abs(got - want) <= 5e-3 * float(grad.double().norm() * v.double().norm()), (i, got, want)


@pytest.mark.parametrize("kind", ["decay", "log", "sigmoid"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("n,c", [(1, 1), (3, 7), (5, 64), (64, 2048), (300, 131)])
def test_step(lcpp, kind, dtype, n, c):
    log(f"recurrence step {kind} {dtype} {n} x {c}")
    g = gen(n + c)
    pool = n + 3
    gt, x = gates(g, kind, (n, c), dtype, 3), ref.rows(g, (n, c), dtype, 1, offset=1)
    state = torch.randn(pool, c, generator=g).cuda()
    slots = torch.randperm(pool, generator=g)[:n].to(torch.int32)
    if n > 2:
        slots[1], slots[2] = -1, pool + 5  # padding
    out = torch.full((n, c), 7.0, dtype=x.dtype, device="cuda")
    nxt = state.clone()
    m = lcpp.DeviceGatedRecurrence()
    m.Step(gt, x, state, nxt, out, kind, d_slots=slots.cuda())
    want_state = ref.host(state)
    named = []
    for i, s in enumerate(slots.tolist()):
        if not 0 <= s < pool:
            assert not out[i].any()
            continue
        named.append(s)
        hs, _, _, errs = ref.recurrence(kind, ref.host(gt[i])[None], ref.host(x[i])[None], want_state[s])
        ref.check(out[i], hs[0], errs[0], dtype, f"out of {i}")
        ref.check(nxt[s], hs[0], errs[0], "float32", f"state of {i}")
    others = [s for s in range(pool) if s not in named]
    assert torch.equal(nxt[others], state[others])
    # in place, and without slots; the step gives what a sequence of one row gives
    here, again = state.clone(), torch.empty_like(out)
    m.Step(gt, x, here, here, again, kind, d_slots=slots.cuda())
    assert torch.equal(here, nxt) and torch.equal(again, out)
    m.Step(gt, x, here, here, again, kind)
    y, hT = torch.empty(n, 1, c, dtype=x.dtype, device="cuda"), torch.empty(n, c, device="cuda")
    m.Forward(None, gt.unsqueeze(1), x.unsqueeze(1), y, kind, nxt[:n].contiguous(), hT)
    assert torch.equal(y[:, 0], again) and torch.equal(hT, here[:n])


def test_strides_past_32_bits(lcpp):
    """Rows 2^24 elements apart: the last of 200 lies past 2^31 elements."""
    log("recurrence, rows 2^24 apart")
    t, c, far = 200, 64, 1 << 24
    base = torch.empty((t - 1) * far + c, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((1, t, c), (0, far, 1))
    x.copy_(torch.randn(1, t, c, generator=gen(4)))
    gt = gates(gen(5), "sigmoid", (1, t, c), "bfloat16")
    tight, y = torch.empty(1, t, c, dtype=x.dtype, device="cuda"), torch.empty(1, t, c, dtype=x.dtype, device="cuda")
    m = lcpp.DeviceGatedRecurrence()
    m.Forward(temp_for(lcpp, 1, t, c), gt, x.contiguous(), tight, "sigmoid")
    m.Forward(temp_for(lcpp, 1, t, c), gt, x, y, "sigmoid")
    assert torch.equal(y, tight)


def test_withheld_tile_is_reported(lcpp):
    """A tile that does not publish makes the waits behind it give up: the call drains and the status word says so."""
    L = lcpp.lib()
    n, t, c = 1, 1000, 64
    g = gen(1)
    gt, x = gates(g, "sigmoid", (n, t, c), "float32"), ref.rows(g, (n, t, c), "float32")
    y, saved = torch.empty_like(x), saved_for(lcpp, n, t, c)
    temp = temp_for(lcpp, n, t, c)
    stream = torch.cuda.current_stream().cuda_stream
    m = lcpp.DeviceGatedRecurrence()

    def status():
        return L.lcpp_temp_status(temp.data_ptr(), temp.numel(), stream)

    try:
        for run in (lambda: m.Forward(temp, gt, x, y, "sigmoid", d_checkpoints=saved),
                    lambda: m.Backward(temp, gt, x, saved, x, torch.empty_like(x), torch.empty_like(x), "sigmoid")):
            log("recurrence with a withheld tile")
            L.lcpp_test_set_lookback_fault(2, 64)
            run()
            assert status() == -5
            L.lcpp_test_set_lookback_fault(0xFFFFFFFF, 0)
            run()
            assert status() == 0
    finally:
        L.lcpp_test_set_lookback_fault(0xFFFFFFFF, 0)


def test_refusals(lcpp):
    m = lcpp.DeviceGatedRecurrence()
    x = torch.zeros(2, 300, 32, device="cuda")
    y, s = torch.zeros_like(x), torch.zeros(2, 32, device="cuda")
    t = temp_for(lcpp, 2, 300, 32)
    with pytest.raises(ValueError):
        m.Forward(t, x, x, y, "relu")
    with pytest.raises(TypeError):
        m.Forward(t, x, x, y.half(), "decay")
    with pytest.raises(TypeError):
        m.Forward(t, x.int(), x.int(), y.int(), "decay")
    with pytest.raises(TypeError):
        m.Forward(t, x, x, y, "decay", s.half())
    with pytest.raises(ValueError):
        m.Forward(t, x[:, :299], x, y, "decay")
    with pytest.raises(ValueError):
        m.Forward(t, x, x, y, "decay", s[:1])
    with pytest.raises(ValueError):
        m.Forward(t, x, x, y[:1].expand(2, 300, 32), "decay")
    with pytest.raises(ValueError):
        m.Forward(t, x[0], x[0], y[0], "decay")
    with pytest.raises(ValueError):
        m.Forward(t, x[0], x[0], y[0], "decay", d_begin_offsets=torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        m.Forward(t, x, x, y, "decay", d_checkpoints=torch.zeros(2, 1, 32, device="cuda"))
    with pytest.raises(lcpp.LcppError) as e:
        m.Forward(t[:256], x, x, y, "decay")
    assert e.value.status == -2
    with pytest.raises(lcpp.LcppError):
        m.Forward(t[1:], x, x, y, "decay")
    with pytest.raises(lcpp.LcppError):
        m.Backward(t, x, x, None, x, y, y.clone(), "decay")
    with pytest.raises(ValueError):
        m.Step(x[0], x[0], s, s, y[0], "decay")  # fewer states than sequences
    with pytest.raises(TypeError):
        m.Step(x[0, :2], x[0, :2], s, s, y[0, :2], "decay", d_slots=torch.zeros(2, device="cuda"))
    m.Forward(None, x[:, :0], x[:, :0], y[:, :0], "decay", s, s.clone())
