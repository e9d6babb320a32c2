"""The router with more tokens than one launch has threads for.  Each row of logits begins one value behind the one before, so
the logits take the memory of their number of tokens."""
import pytest
import torch

from conftest import log

pytestmark = pytest.mark.gpu
PIECE = 1 << 24


def pieces(n):
    return ((a, min(n, a + PIECE)) for a in range(0, n, PIECE))


def test_two_experts(gpu):
    """2^28 + 5 tokens, 16 lanes each: 2^32 threads and a few."""
    import lc_parallel_primitive_amd as lcpp

    n = 2**28 + 5
    log(f"router {n} x 2, 1 chosen")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    b = torch.empty(n + 1, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    logits = b.as_strided((n, 2), (1, 1))
    experts = torch.full((n, 1), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((n, 1), -7.0, device="cuda")
    router = lcpp.DeviceExpertRouter()
    router.Forward(logits, experts, weights, normalize=False)
    dw = torch.empty(n, 1, device="cuda").normal_(generator=g)
    grad = torch.full((n, 2), -7.0, dtype=torch.bfloat16, device="cuda")
    router.Backward(logits, experts, dw, grad, normalize=False)
    for a, z in pieces(n):
        l = logits[a:z].double()
        want = (l[:, 1] > l[:, 0]).int()
        assert torch.equal(experts[a:z, 0], want), f"experts of {a} .. {z}"
        p = torch.softmax(l, 1)
        best = p.amax(1)
        # an exponential is off by (8 + 2 |x|) 2^-24, the logits' difference below 20; a sum, a division and a product follow
        rel = (2 * (8 + 2 * 20) + 8) * 2.0**-24
        assert bool(((weights[a:z, 0].double() - best).abs() <= rel * best).all()), f"weights of {a} .. {z}"
        d = best * (1 - best) * dw[a:z, 0].double()
        want = torch.where(torch.arange(2, device="cuda") == want[:, None], d[:, None], -d[:, None])
        # (1 - p is a difference of numbers near 1: off by rel of 1; and one rounding to the type)
        off = (grad[a:z].double() - want).abs() - (2.0**-8 * want.abs() * 1.01 + 4 * rel * (best * dw[a:z, 0].abs())[:, None] + 1e-37)
        assert float(off.max()) <= 0, f"gradients of {a} .. {z}"


@pytest.mark.parametrize("experts,n,score", [(300, 2**26 + 3, "softmax"), (130, 2**27 + 9, "sigmoid")])
def test_wide_rows(gpu, experts, n, score):
    """Rows of 64 and of 32 lanes: the first, the last and those around every power of two."""
    import lc_parallel_primitive_amd as lcpp

    log(f"router {n} x {experts}, 2 chosen")
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    b = torch.empty(n + experts, device="cuda").uniform_(generator=g)
    logits = b.as_strided((n, experts), (1, 1))
    ids = torch.full((n, 2), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((n, 2), -7.0, device="cuda")
    lcpp.DeviceExpertRouter().Forward(logits, ids, weights, score)
    assert bool(((ids >= 0) & (ids < experts)).all()) and bool(((weights > 0) & (weights < 1)).all())
    edges = {0, n} | {1 << i for i in range(12, 28)} | {3 << i for i in range(20, 26)} | {n // 2}
    for edge in sorted(e for e in edges if e <= n):
        a, z = max(0, edge - 500), min(n, edge + 500)
        rows = logits[a:z].contiguous().cpu()
        want = rows.sort(dim=1, descending=True, stable=True).indices[:, :2]
        assert torch.equal(ids[a:z].cpu().long(), want), f"experts around {edge}"
        l = rows.double().gather(1, want)
        w = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l) / torch.sigmoid(l).sum(1, keepdim=True)
        # (logits of 0 to 1: some exponentials and logarithms of (8 + 2) 2^-24 each)
        assert float((weights[a:z].cpu().double() - w).abs().max()) <= 100 * 2.0**-24, f"weights around {edge}"
