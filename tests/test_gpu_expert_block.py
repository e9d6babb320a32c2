"""The RMS norm, router, token sort and experts' products together: the example model, graphs, streams, threads, workspaces
that hold something, rows that lie far apart."""
import importlib.util
import os
import threading

import pytest
import torch

from conftest import ROOT, log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(gpu):
    spec = importlib.util.spec_from_file_location("expert_block", os.path.join(ROOT, "examples", "expert_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.fixture(scope="module")
def lcpp(gpu):
    import lc_parallel_primitive_amd as m

    return m


def test_it_trains(example):
    log("example: training")
    losses = example.train(example.Model(), steps=3)
    assert len(losses) == 3 and all(v == v and abs(v) != float("inf") for v in losses)


def plain(model, tokens, chosen, matrices=None):
    """The model's logits in float64 by torch's own operations, with these choices of experts."""
    params = {k: v.detach().double().cpu().requires_grad_() for k, v in model.named_parameters()}

    def norm(h, i):
        return h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * params[f"norm.{i}"]

    h = params["embed"][tokens]
    for i in range(model.layers):
        n = norm(h, i)
        up, down = matrices[i] if matrices else (params[f"up.{i}"], params[f"down.{i}"])
        at = chosen[i].long().cpu()
        weights = torch.softmax((n @ params[f"router.{i}"].t()).gather(1, at), 1)
        out = []
        for t in range(n.shape[0]):
            row = 0
            for j in range(model.choices):
                gate, upper = (up[at[t, j]] @ n[t]).chunk(2)
                row = row + weights[t, j] * (down[at[t, j]] @ (torch.nn.functional.silu(gate) * upper))
            out.append(row)
        h = h + torch.stack(out)
    return norm(h, model.layers) @ params["head"].t(), params


def test_gradients_of_the_whole_model(example):
    """Every parameter's gradient against autograd in float64, in float32.  A sum of n terms is off by at most n 2^-24 of
    its terms' sizes, which are some sqrt(n) times the sum; the longest way to a gradient passes twelve sums of at most
    96 terms (the forward pass and back): 12 * 96 * 10 * 2^-24 = 7e-4, taken as 1e-3."""
    log("example: gradients")
    model = example.Model(vocab=16, width=96, hidden=40, experts=5, choices=2, dtype=torch.float32)
    g = torch.Generator()
    g.manual_seed(3)
    tokens, targets = torch.randint(0, 16, (70,), generator=g), torch.randint(0, 16, (70,), generator=g)
    got = model(tokens.cuda())
    torch.nn.functional.cross_entropy(got, targets.cuda()).backward()
    logits, params = plain(model, tokens, model.chosen)
    torch.nn.functional.cross_entropy(logits, targets).backward()
    assert float((got.detach().double().cpu() - logits.detach()).norm() / logits.detach().norm()) < 1e-3
    for k, v in model.named_parameters():
        want = params[k].grad
        off = float((v.grad.double().cpu() - want).norm() / want.norm())
        assert off < 1e-3, (k, off)


def test_serving_in_eight_bits(example):
    """Against float64 with the same matrices of 8 bits: the rows' roundings are at most 2^-4 of each value and one does
    not know of another, so a product's results are off by no more than 2^-4 of their norm; the activation passes on
    those of its two factors (each of a slope of at most 1.1) and its own: 3.2 * 2^-4 of a block's result, which is less
    than the residual it is added to; two blocks."""
    log("example: 8 bits")
    model = example.Model(dtype=torch.float32)
    tokens = torch.arange(40) % 64
    eight = model.in_eight_bits()
    got = model.serve(tokens.cuda(), eight)

    def wide(values, scales):
        s = scales.repeat_interleave(128, 1)[:, :values.shape[1]].repeat_interleave(128, 2)[:, :, :values.shape[2]]
        return (values.float() * s).double().cpu()

    with torch.no_grad():
        logits, _ = plain(model, tokens, model.chosen, [(wide(*u), wide(*d)) for u, d in eight])
    assert float((got.double().cpu() - logits).norm() / logits.norm()) < 2 * 3.2 * 2.0**-4


def _call_set(lcpp, seed, dtype=torch.bfloat16, tokens=3001, k=2, cols=136, hidden=72, experts=7):
    """One of each call on buffers of its own: (run(stream), outputs, inputs)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    pairs = tokens * k
    x, r, dy = (rand(tokens, cols).to(dtype) for _ in range(3))
    logits, w = rand(tokens, experts).to(dtype), rand(cols)
    m = (rand(experts, hidden, cols) * 0.1).to(dtype)
    m8 = m.float().to(torch.float8_e4m3fn)
    ms = torch.ones(experts, 1, 2, device="cuda")
    down = (rand(experts, cols, hidden) * 0.1).to(dtype)
    zeros = lambda *s, t=dtype: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    f, i32 = torch.float32, torch.int32
    s, y, out, dn, ds, dr = (zeros(tokens, cols) for _ in range(6))
    q, qs, rstd = zeros(tokens, cols, t=torch.float8_e4m3fn), zeros(tokens, 2, t=f), zeros(tokens, t=f)
    ids, pos, weights, dw = zeros(tokens, k, t=i32), zeros(tokens, k, t=i32), zeros(tokens, k, t=f), zeros(tokens, k, t=f)
    off, src = zeros(experts + 1, t=i32), zeros(pairs, t=i32)
    rows, res, dres, drows = (zeros(pairs, cols) for _ in range(4))
    rows8, scales8 = zeros(pairs, cols, t=torch.float8_e4m3fn), zeros(pairs, 2, t=f)
    mid, mid8, dmid = (zeros(pairs, hidden) for _ in range(3))
    dm, ddown, dnw, dl = zeros(experts, hidden, cols, t=f), torch.zeros_like(down), zeros(cols, t=f), torch.zeros_like(logits)
    norm, router, order, product = lcpp.DeviceRMSNorm(), lcpp.DeviceExpertRouter(), lcpp.DeviceTokenSort(), lcpp.DeviceExpertProduct()
    tn = torch.empty(norm.GetBackwardTempStorageBytes(dtype, tokens, cols), dtype=torch.uint8, device="cuda")
    ts = torch.empty(order.GetTempStorageBytes(tokens, k, experts), dtype=torch.uint8, device="cuda")
    assert ts.numel() > 0

    def run(stream=None):
        norm.AddForward(x, r, s, y, w, 1e-6, rstd, q, qs, stream=stream)
        router.Forward(logits, ids, weights, stream=stream)
        order.Sort(ts, ids, experts, pos, off, src, stream=stream)
        order.Dispatch(y, pos, rows, stream=stream)
        order.Dispatch(q, pos, rows8, stream=stream)
        order.Dispatch(qs, pos, scales8, stream=stream)
        product.Forward(rows, m, off, mid, stream=stream)
        product.Forward(rows8, m8, off, mid8, scales8, ms, stream=stream)
        product.Forward(mid, down, off, res, stream=stream)
        order.Combine(res, pos, weights, out, s, stream=stream)
        order.CombineBackward(dy, res, pos, weights, dres, dw, stream=stream)
        product.Backward(dres, mid, down, off, dmid, ddown, stream=stream)
        product.Backward(dmid, rows, m, off, drows, dm, stream=stream)
        order.DispatchBackward(drows, pos, dn, stream=stream)
        router.Backward(logits, ids, dw, dl, stream=stream)
        norm.Backward(tn, dn, s, w, rstd, ds, dnw, dy, stream=stream)

    outputs = (s, y, out, dn, ds, q, qs, rstd, ids, pos, weights, dw, off, src, rows, res, dres, drows, rows8, scales8, mid, mid8,
               dmid, dm, ddown, dnw, dl)
    return run, outputs, (x, r, dy, logits)


def _same(a, b):
    return torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


def _clear(outputs):
    for o in outputs:
        (o.view(torch.uint8) if o.element_size() == 1 else o).zero_()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_in_a_graph(lcpp, dtype):
    """A captured run replayed with new inputs, and so other rows for each expert, against the eager calls."""
    run, outputs, inputs = _call_set(lcpp, 5, dtype)
    run()
    torch.cuda.synchronize()
    log("expert block: capture")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run()
    torch.cuda.current_stream().wait_stream(side)
    seen = []
    for i in range(4):
        for v in inputs:
            v.copy_(torch.randn(v.shape, device="cuda"))
        # (the later replays leave an expert without rows)
        inputs[3][:, 3].fill_(-1e9 if i > 1 else 0.5)
        _clear(outputs)
        torch.cuda.synchronize()
        log(f"expert block: replay {i}")
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outputs]
        _clear(outputs)
        run()
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(got, outputs)):
            assert _same(a, b), n
        seen.append(got[12].tolist())
    assert seen[0] != seen[1] and seen[2][3] == seen[2][4] < seen[2][7]


def test_streams_and_threads(lcpp):
    """Four host threads on streams of their own give what one stream gives."""
    sets = [_call_set(lcpp, 20 + i) for i in range(4)]
    want = []
    for run, outputs, _ in sets:
        run()
        torch.cuda.synchronize()
        want.append([o.clone() for o in outputs])
        _clear(outputs)
    torch.cuda.synchronize()
    log("expert block: four threads")
    streams = [torch.cuda.Stream() for _ in sets]
    errors = []

    def work(i):
        try:
            for _ in range(10):
                sets[i][0](streams[i])
            streams[i].synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    for (run, outputs, _), expect in zip(sets, want):
        for n, (a, b) in enumerate(zip(outputs, expect)):
            assert _same(a, b), n


@pytest.mark.parametrize("tokens", [0, 1, 700, 5000])
def test_workspaces_that_hold_something(lcpp, tokens):
    """A status word of an earlier call is not reported as this one's, and what a workspace holds changes nothing."""
    log(f"expert block: stale workspaces, {tokens} tokens")
    debug = torch.cuda.current_stream()
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    ids = torch.randint(-1, 9, (tokens, 2), generator=g, device="cuda", dtype=torch.int32)
    results = []
    for fill in (0, 255):
        order, norm = lcpp.DeviceTokenSort().create(debug_stream=debug), lcpp.DeviceRMSNorm().create(debug_stream=debug)
        temp = torch.full((1 << 20,), fill, dtype=torch.uint8, device="cuda")
        pos, off = torch.zeros_like(ids), torch.zeros(10, dtype=torch.int32, device="cuda")
        order.Sort(temp, ids, 9, pos, off)
        assert int(temp[:4].view(torch.int32)[0]) == 0
        x = torch.ones(tokens, 50, device="cuda")
        w, dx, dw = torch.ones(50, device="cuda"), torch.zeros_like(x), torch.full((50,), 7.0, device="cuda")
        temp = torch.full((1 << 20,), fill, dtype=torch.uint8, device="cuda")
        norm.Backward(temp, x, x, w, torch.ones(tokens, device="cuda"), dx, dw)
        assert int(temp[:4].view(torch.int32)[0]) == 0
        results.append((pos, off, dx, dw))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert float(results[0][3][0]) == tokens


def test_rows_far_apart(lcpp):
    """Rows 2^27 + 8 elements apart: offsets of rows and matrices pass 32 bits, in bytes and in elements."""
    log("expert block: rows far apart")
    n, cols, far = 40, 72, (1 << 27) + 8
    store = torch.empty(n * far, dtype=torch.bfloat16, device="cuda")
    target = torch.empty(n * far, dtype=torch.bfloat16, device="cuda")
    x, y = store.as_strided((n, cols), (far, 1)), target.as_strided((n, cols), (far, 1))
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    near = torch.randn(n, cols, generator=g, device="cuda").bfloat16()
    x.copy_(near)
    norm, order, product = lcpp.DeviceRMSNorm(), lcpp.DeviceTokenSort(), lcpp.DeviceExpertProduct()
    # norm and its gradient
    want, rstd = torch.empty_like(near), torch.empty(n, device="cuda")
    norm.Forward(near, want, None, 1e-6, rstd)
    norm.Forward(x, y)
    assert torch.equal(y, want)
    dx = torch.empty_like(near)
    norm.Backward(None, near, near, None, rstd, dx)
    norm.Backward(None, x, x, None, rstd, y)
    assert torch.equal(y, dx)
    # copies and sums
    pos = torch.randperm(n, generator=g, device="cuda").to(torch.int32).view(n // 2, 2)
    weights = torch.rand(n // 2, 2, generator=g, device="cuda")
    rows = torch.empty_like(near)
    order.Dispatch(near[: n // 2], pos, rows)
    order.Dispatch(x[: n // 2], pos, y)
    assert torch.equal(y, rows)
    total = torch.empty_like(near[: n // 2])
    order.Combine(near, pos, weights, total)
    order.Combine(x, pos, weights, y[: n // 2])
    assert torch.equal(y[: n // 2], total)
    # products: rows, then matrices, far apart
    off = torch.tensor([0, 7, 7, n], dtype=torch.int32, device="cuda")
    m = torch.randn(3, cols, cols, generator=g, device="cuda").bfloat16()
    out, dx, dm = torch.empty_like(near), torch.empty_like(near), torch.empty_like(m)
    product.Forward(near, m, off, out)
    product.Forward(x, m, off, y)
    assert torch.equal(y, out)
    product.Backward(out, near, m, off, dx, dm)
    y.copy_(out)
    far_dm = torch.empty_like(m)
    third = torch.empty(n * far, dtype=torch.bfloat16, device="cuda").as_strided((n, cols), (far, 1))
    product.Backward(y, x, m, off, third, far_dm)
    assert torch.equal(third, dx) and torch.equal(far_dm, dm)
    for strides in ((far, cols, 1), (cols, far, 1)):
        count = 3 if strides[0] == far else 1
        wide = store.as_strided((count, 36, cols), strides)
        wide.copy_(m[:count, :36])
        offsets = off if count == 3 else torch.tensor([0, n], dtype=torch.int32, device="cuda")
        a, b = torch.empty(n, 36, device="cuda", dtype=near.dtype), torch.empty(n, 36, device="cuda", dtype=near.dtype)
        product.Forward(near, m[:count, :36].contiguous(), offsets, a)
        product.Forward(near, wide, offsets, b)
        assert torch.equal(a, b)
        c, d = torch.empty_like(near), torch.empty_like(near)
        dm1, dm2 = torch.empty(count, 36, cols, device="cuda", dtype=near.dtype), target.as_strided((count, 36, cols), strides)
        product.Backward(a, near, m[:count, :36].contiguous(), offsets, c, dm1)
        product.Backward(a, near, wide, offsets, d, dm2)
        assert torch.equal(c, d) and torch.equal(dm1, dm2)
