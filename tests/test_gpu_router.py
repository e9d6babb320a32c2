"""The expert router against its definition: choices exactly, weights and gradients in 64 bits."""
import numpy as np
import pytest
import torch

import block_ref as ref
import expert_ref as eref
from conftest import log

pytestmark = pytest.mark.gpu


def run(lcpp, logits, k, bias=None, grad=None, **how):
    t = logits.shape[0]
    ids, w = torch.empty(t, k, dtype=torch.int32, device="cuda"), torch.empty(t, k, device="cuda")
    r = lcpp.DeviceExpertRouter()
    r.Forward(logits, ids, w, d_bias=bias, **how)
    if grad is None:
        return ids, w
    dl = torch.empty_like(logits)
    r.Backward(logits, ids, grad, dl, **how)
    return ids, w, dl


def logits_of(seed, tokens, experts, dtype, kind="plain", pad=0):
    g = torch.Generator()
    g.manual_seed(seed)
    l = ref.rows(g, (tokens, experts), dtype, pad, scale=2.0)
    if kind == "masked":
        l.masked_fill_((torch.rand(tokens, experts, generator=g) < 0.6).cuda(), float("-inf"))
        l[tokens // 2] = float("-inf")
    elif kind == "ties":
        l.copy_((torch.randint(0, 4, (tokens, experts), generator=g) - 1.5))
        l[:, ::3] = 0.0
        l[:, 1::3] = -0.0
    elif kind == "lowest":
        l.masked_fill_((torch.rand(tokens, experts, generator=g) < 0.9).cuda(), torch.finfo(l.dtype).min)
    return l


SIZES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (9, 8, 2), (17, 9, 9), (33, 64, 6), (31, 127, 8), (48, 128, 8), (50, 129, 4), (20, 255, 20),
         (70, 256, 8), (13, 257, 33), (40, 384, 6), (9, 512, 10), (7, 513, 64), (11, 1000, 16), (5, 1024, 64), (1000, 60, 4)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("kind", ["plain", "masked", "ties", "lowest"])
@pytest.mark.parametrize("tokens,experts,k", SIZES)
def test_router(gpu, tokens, experts, k, kind, dtype):
    import lc_parallel_primitive_amd as lcpp

    log(f"router {tokens} x {experts} top {k} {kind} {dtype}")
    l = logits_of(tokens + experts, tokens, experts, dtype, kind, pad=experts % 3)
    host = ref.host(l).numpy()
    g = torch.Generator()
    g.manual_seed(k)
    bias = torch.randn(experts, generator=g) * 0.5
    grad = torch.randn(tokens, k, generator=g)
    for score, normalize, scale, b in (("softmax", True, 1.0, None), ("softmax", False, 2.5, bias), ("sigmoid", True, 2.5, bias),
                                       ("sigmoid", False, 1.0, None)):
        if kind == "lowest" and score == "sigmoid" and normalize:
            continue  # (a row of the lowest values alone has the sum 0 in 64 bits too)
        how = dict(score=score, normalize=normalize, scale=scale)
        ids, w, dl = run(lcpp, l, k, None if b is None else b.cuda(), grad.cuda(), **how)
        want = eref.chosen(host, None if b is None else b.numpy(), k)
        np.testing.assert_array_equal(ids.cpu().numpy(), want)
        size = host[np.isfinite(host) & (np.abs(host) < 1e4)]
        near = np.where(np.abs(host) < 1e4, host, np.where(host < 0, -np.inf, host))  # (the lowest values' shares are 0)
        share, p, rel = eref.shares(near if score == "softmax" else host, want, score, normalize)
        if kind == "lowest":
            rel = eref.U32 * (300 + 30 * float(np.abs(size).max() if size.size else 0))
            if score == "softmax" and normalize:
                # rows whose chosen are all the lowest value share evenly
                even = (np.take_along_axis(host, np.maximum(want, 0), 1) < -1e4).all(1)
                share[torch.from_numpy(even)] = 1.0 / k
            if score == "softmax" and not normalize and (np.abs(host) > 1e4).all(1).any():
                continue
        ref.check(w, scale * share, scale * share * rel, "float32", f"weights {how}")
        if kind == "lowest":
            continue
        d, bound = eref.router_grad(host, want, share, p, grad.double(), score, normalize, scale, rel)
        ref.check(dl, d, bound, dtype, f"gradient {how}")


def test_gradient_by_differences(gpu):
    import lc_parallel_primitive_amd as lcpp

    l = logits_of(5, 3, 20, "float32")
    g = torch.Generator()
    g.manual_seed(1)
    grad = torch.randn(3, 4, generator=g)
    host, h = ref.host(l), 1e-6
    for score in ("softmax", "sigmoid"):
        for normalize in (False, True):
            ids, _, dl = run(lcpp, l, 4, None, grad.cuda(), score=score, normalize=normalize)
            f = lambda x: float((eref.shares(x, ids.cpu().long(), score, normalize)[0] * grad).sum())  # noqa: E731
            for i, j in ((0, int(ids[0, 0])), (1, int(ids[1, 3])), (2, 7), (2, 0)):
                e = torch.zeros_like(host)
                e[i, j] = h
                # (1e-16 / h of the values, h^2 of a third derivative of about 1)
                assert abs((f(host + e) - f(host - e)) / (2 * h) - float(dl[i, j])) < 1e-6, (score, normalize, i, j)


def test_values_that_are_not_finite(gpu):
    import lc_parallel_primitive_amd as lcpp

    l = torch.zeros(4, 70, device="cuda")
    l[0, 50] = float("nan")
    l[1, 60] = float("inf")
    l[2] = float("-inf")
    l[3, 5:] = float("-inf")
    bias = torch.zeros(70, device="cuda")
    bias[2] = float("-inf")
    for score, normalize in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        ids, w, dl = run(lcpp, l, 6, bias, torch.ones(4, 6, device="cuda"), score=score, normalize=normalize)
        assert ids[0].tolist()[0] == 50 and torch.isnan(w[0, 0])
        assert ids[1].tolist()[0] == 60
        assert ids[2].tolist() == [-1] * 6 and torch.all(w[2] == 0) and torch.all(dl[2] == 0)
        assert ids[3].tolist() == [0, 1, 3, 4, -1, -1] and torch.all(w[3, 4:] == 0) and torch.all(torch.isfinite(w[3]))
        assert torch.all(torch.isfinite(dl[3]))


def test_extreme_sigmoid(gpu):
    """Scores that all round to 0 or to 1 still share as their ratios say."""
    import lc_parallel_primitive_amd as lcpp

    l = torch.tensor([[-200.0, -201.0, -300.0], [60.0, 50.0, 40.0]], device="cuda")
    _, w = run(lcpp, l, 2, score="sigmoid")
    e = float(np.exp(-1.0))
    assert torch.allclose(w.cpu(), torch.tensor([[1 / (1 + e), e / (1 + e)], [0.5, 0.5]]), rtol=3e-5)


def test_gradient_in_place_and_foreign_experts(gpu):
    import lc_parallel_primitive_amd as lcpp

    r = lcpp.DeviceExpertRouter()
    for experts, normalize in ((60, True), (300, False)):
        l = logits_of(9, 50, experts, "bfloat16")
        ids, w, dl = run(lcpp, l, 5, None, torch.ones(50, 5, device="cuda").cumsum(1), normalize=normalize)
        over = l.clone()
        r.Backward(over, ids, torch.ones(50, 5, device="cuda").cumsum(1), over, normalize=normalize)
        assert torch.equal(over, dl)
        # experts that are none have no gradient
        bad = ids.clone()
        bad[:, 1], bad[:, 3] = experts, -7
        keep = ids.clone()
        keep[:, 1] = keep[:, 3] = -1
        outs = []
        for which in (bad, keep):
            outs.append(torch.empty_like(l))
            r.Backward(l, which, torch.ones(50, 5, device="cuda"), outs[-1], normalize=normalize)
        assert torch.equal(*outs)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_gradient_of_an_expert_named_twice(gpu, score, normalize):
    """Choices that were not made by the forward call may name an expert twice: it has the sum, as autograd in float64
    says.  Logits of at most 2: a share is off by some 200 roundings of 2^-24, a gradient by four times as many and 80
    more, of terms that are at most twice the largest gradient of a weight: 2 * 880 * 2^-24 = 1.05e-4 of it."""
    log(f"router: an expert twice, {score} {normalize}")
    import lc_parallel_primitive_amd as m

    g = torch.Generator()
    g.manual_seed(9)
    rows, experts, k = 33, 70, 20
    logits = torch.rand(rows, experts, generator=g) * 4 - 2
    ids = torch.randint(0, experts, (rows, k), generator=g, dtype=torch.int32)
    ids[:, 1] = ids[:, 0]
    ids[:, 19] = ids[:, 2]
    dw = torch.randn(rows, k, generator=g)
    wide = logits.double().requires_grad_()
    share = torch.sigmoid(wide) if score == "sigmoid" else torch.softmax(wide, 1)
    w = share.gather(1, ids.long())
    if normalize:
        w = w / w.sum(1, keepdim=True)
    (w * dw.double() * 1.5).sum().backward()
    got = torch.empty(rows, experts, device="cuda")
    m.DeviceExpertRouter().Backward(logits.cuda(), ids.cuda(), dw.cuda(), got, score, normalize, 1.5)
    again = torch.empty_like(got)
    m.DeviceExpertRouter().Backward(logits.cuda(), ids.cuda(), dw.cuda(), again, score, normalize, 1.5)
    assert float((got.double().cpu() - wide.grad).abs().max()) <= 1.5 * 1.05e-4 * float(dw.abs().max())
    assert torch.equal(got, again)
