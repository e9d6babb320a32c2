"""The example model: layer norm, recurrence and dropout together, trained and decoded; graphs, streams and threads."""
import importlib.util
import os
import threading

import pytest
import torch

from conftest import ROOT, log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(gpu):
    spec = importlib.util.spec_from_file_location("recurrent_block", os.path.join(ROOT, "examples", "recurrent_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_it_learns_and_decodes(example):
    log("example: training")
    model = example.Model()
    losses = example.train(model, steps=60)
    # guessing costs log 32 = 3.47; the next token is certain from the third on
    assert losses[0] > 3.0 and sum(losses[-5:]) / 5 < 0.7, (losses[0], losses[-5:])
    log("example: decoding")
    # activations are rounded to bfloat16 (2^-8) at ten places of either way, in the products in another order
    assert example.decoding_error(model) < 10 * 2.0**-8


def plain(model, tokens, spans):
    """The model's logits in float64 by torch's own operations, dropout off, and the loss's gradients by autograd."""
    params = {k: v.detach().double().cpu().requires_grad_() for k, v in model.named_parameters()}

    def norm(h, i):
        c = h - h.mean(1, keepdim=True)
        return c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * params[f"norm_w.{i}"] + params[f"norm_b.{i}"]

    h = params["embed"][tokens]
    for i in range(model.layers):
        gate, value = (norm(h, i) @ params[f"mix_in.{i}"]).split(model.width, 1)
        rows = []
        for b, e in spans:
            s = torch.zeros(model.width, dtype=torch.float64)
            for t in range(b, e):
                a = torch.sigmoid(gate[t])
                s = a * s + (1 - a) * value[t]
                rows.append(s)
        h = h + torch.stack(rows) @ params[f"mix_out.{i}"]
    return norm(h, model.layers) @ params["head"], params


def test_gradients_of_the_whole_model(example):
    """Every parameter's gradient through both blocks, against autograd in float64.  The activations are bfloat16: each
    rounding is 2^-8 of a value, independent of the others, and some thirty of them lie on the longest way to a
    gradient, so the gradients' vectors are within 2^-8 sqrt(30) = 2.1 %, doubled for the few that add up."""
    log("example: gradients")
    model = example.Model(vocab=16, width=64, p=0.0)
    lengths = [5, 1, 30, 150]
    g = torch.Generator()
    g.manual_seed(3)
    tokens, targets, begin, end, longest = example.batch(g, lengths, 16)
    loss = torch.nn.functional.cross_entropy(model(tokens, begin, end, longest), targets)
    loss.backward()
    logits, params = plain(model, tokens.cpu(), list(zip(begin.tolist(), end.tolist())))
    torch.nn.functional.cross_entropy(logits, targets.cpu()).backward()
    for k, v in model.named_parameters():
        want = params[k].grad
        off = float((v.grad.double().cpu() - want).norm() / want.norm())
        assert off < 0.043, (k, off)


def _call_set(lcpp, seed):
    """One of each call on buffers of its own: (run(stream), outputs)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, t, c = 3, 300, 200
    x, r, gate = (torch.randn(n * t, c, generator=g, device="cuda").bfloat16() for _ in range(3))
    w, b = torch.rand(c, generator=g, device="cuda"), torch.rand(c, generator=g, device="cuda")
    s, y, m, dg, dm, dx, dres, d = (torch.zeros_like(x) for _ in range(8))
    mean, rstd = torch.zeros(n * t, device="cuda"), torch.zeros(n * t, device="cuda")
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    counter = torch.zeros(1, dtype=torch.int64, device="cuda")
    norm, mix, drop = lcpp.DeviceLayerNorm(), lcpp.DeviceGatedRecurrence(), lcpp.DeviceDropout()
    tn = torch.empty(lcpp.DeviceLayerNorm.GetBackwardTempStorageBytes(x.dtype, n * t, c), dtype=torch.uint8, device="cuda")
    tm = torch.empty(lcpp.DeviceGatedRecurrence.GetTempStorageBytes(n, t, c), dtype=torch.uint8, device="cuda")
    saved = torch.empty(n, lcpp.DeviceGatedRecurrence.GetCheckpointRows(t), c, device="cuda")
    shape = (n, t, c)

    def run(stream=None):
        norm.AddForward(x, r, s, y, w, b, 1e-5, mean, rstd, p=0.2, seed=seed, d_offset=counter, stream=stream)
        mix.Forward(tm, gate.view(shape), y.view(shape), m.view(shape), "sigmoid", d_checkpoints=saved, stream=stream)
        drop.Forward(m, d, 0.3, seed, 7, d_offset=counter, stream=stream)
        mix.Backward(tm, gate.view(shape), y.view(shape), saved, d.view(shape), dg.view(shape), dm.view(shape), "sigmoid",
                     stream=stream)
        norm.AddBackward(tn, dm, d, s, w, mean, rstd, dres, dx, dw, db, p=0.2, seed=seed, d_offset=counter, stream=stream)

    return run, (s, y, m, d, dg, dm, dres, dx, dw, db), counter, (x, r, gate)


def test_captured_in_a_graph(gpu):
    """A captured step replayed with new inputs and an advanced counter, against the eager calls."""
    import lc_parallel_primitive_amd as lcpp

    run, outputs, counter, inputs = _call_set(lcpp, 5)
    run()  # caches what the library asks the device
    torch.cuda.synchronize()
    log("recurrent block: capture")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run()
    torch.cuda.current_stream().wait_stream(side)
    seen = []
    for i in range(4):
        counter.fill_(i)
        for v in inputs:
            v.copy_(torch.randn(v.shape, device="cuda"))
        torch.cuda.synchronize()
        log(f"recurrent block: replay {i}")
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outputs]
        for o in outputs:
            o.zero_()
        run()
        torch.cuda.synchronize()
        for a, b in zip(got, outputs):
            assert torch.equal(a, b)
        seen.append((got[3] == 0).clone())
    # the counter changed the mask
    assert not torch.equal(seen[0], seen[1])


def test_streams_and_threads(gpu):
    """Four host threads on streams of their own give what one stream gives."""
    import lc_parallel_primitive_amd as lcpp

    sets = [_call_set(lcpp, 20 + i) for i in range(4)]
    want = []
    for run, outputs, _, _ in sets:
        run()
        torch.cuda.synchronize()
        want.append([o.clone() for o in outputs])
        for o in outputs:
            o.zero_()
    torch.cuda.synchronize()
    log("recurrent block: four threads")
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
    for (run, outputs, _, _), expect in zip(sets, want):
        for a, b in zip(outputs, expect):
            assert torch.equal(a, b)


def test_debug_stream_reads_the_status(gpu):
    import lc_parallel_primitive_amd as lcpp

    log("recurrent block: debug stream")
    x = torch.randn(2, 400, 70, device="cuda")
    temp = torch.full((lcpp.DeviceGatedRecurrence.GetTempStorageBytes(2, 400, 70),), 255, dtype=torch.uint8, device="cuda")
    m = lcpp.DeviceGatedRecurrence().create(debug_stream=torch.cuda.current_stream())
    y = torch.empty_like(x)
    m.Forward(temp, x, x, y, "sigmoid")
    n = lcpp.DeviceLayerNorm().create(debug_stream=torch.cuda.current_stream())
    rows = x.view(-1, 70)
    stat = torch.ones(800, device="cuda")
    w = torch.ones(70, device="cuda")
    tb = torch.full((lcpp.DeviceLayerNorm.GetBackwardTempStorageBytes(x.dtype, 800, 70),), 255, dtype=torch.uint8, device="cuda")
    n.Backward(tb, rows, rows, w, stat, stat, torch.empty_like(rows), w.clone(), w.clone())
    L = lcpp.lib()
    try:
        L.lcpp_test_set_lookback_fault(1, 64)
        with pytest.raises(lcpp.LcppError) as e:
            m.Forward(temp, x, x, y, "sigmoid")
        assert e.value.status == -5
    finally:
        L.lcpp_test_set_lookback_fault(0xFFFFFFFF, 0)
