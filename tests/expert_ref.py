"""The RMS norm, the expert router, the tokens' sort and the experts' products from their definitions, in 64 bits on the
CPU, with bounds of what 32-bit arithmetic may be off by (U32 and the like as in block_ref)."""
import numpy as np
import torch

from block_ref import U32

# A row's sum: at most 32 elements in a thread (40 in rows of 40000 columns), 10 steps over lanes and waves, the division.
CHAIN = 64
# One rounding to 8 bits, relative, and half the step of subnormal values.
U8 = {torch.float8_e4m3fn: (2.0**-4, 2.0**-10), torch.float8_e5m2: (2.0**-3, 2.0**-17)}
QMAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


# ---------------------------------------------------------------------- RMS norm
def rms(s, w, eps):
    """(y, rstd, y's relative error, rstd's): every square is positive, so their sum's roundings are relative to it; half
    of that, the root and the division reach rstd, two products follow."""
    ms = (s * s).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(ms + eps)
    rel = U32 * (0.5 * (CHAIN + 4) + 4)
    return s * rstd * w, rstd, rel + 3 * U32, rel


def rms_grad(s, w, rstd, dy, dsum):
    """(ds, dw) and their bounds, from rstd as it is given."""
    u, v = s * rstd, dy * w
    mean = (v * u).mean(1, keepdim=True)
    size = (v * u).abs().mean(1, keepdim=True)
    ds = rstd * (v - u * mean)
    bound = U32 * rstd * (4 * v.abs() + (CHAIN + 10) * u.abs() * size)
    if dsum is not None:
        ds = ds + dsum
        bound = bound + U32 * (ds.abs() + dsum.abs())
    # (a sum of n terms in any order: none of them passes more than n additions)
    dw, bw = (dy * u).sum(0), U32 * (s.shape[0] + 6) * (dy * u).abs().sum(0)
    return ds, dw, bound, bw


def quantised(y, rel, group, qdtype):
    """(scales, their relative error, y of each group) where all of y is finite."""
    rows, cols = y.shape
    g = group or cols
    parts = -(-cols // g)
    wide = torch.zeros(rows, parts * g, dtype=torch.float64)
    wide[:, :cols] = y
    amax = wide.view(rows, parts, g).abs().amax(2).clamp(min=2.0**-100)
    return amax / QMAX[qdtype], rel + 2 * U32


def check_quantised(q, scales, y, rel, group, what):
    """q is y / scale rounded to its type, with the scale as it was given; both are off by their own roundings."""
    want, rel_scale = quantised(y, rel, group, q.dtype)
    got = scales.double().cpu()
    assert got.shape == want.shape, what
    off = ((got - want).abs() - rel_scale * want * 1.0001).max() if want.numel() else 0.0
    assert float(off) <= 0, f"{what}: scales {float(off):.3e} past the bound"
    g = group or y.shape[1]
    each = got.repeat_interleave(g, 1)[:, :y.shape[1]]
    v = y / each
    u, half = U8[q.dtype]
    # (before its rounding the quotient is off by y's error and three roundings)
    near = v.abs() * (rel + 3 * U32)
    tol = torch.clamp(u * (v.abs() + near), min=half) + near
    off = ((q.to(torch.float32).double().cpu() - v).abs() - tol * 1.0001).max() if v.numel() else 0.0
    assert float(off) <= 0, f"{what}: values {float(off):.3e} past the bound"


# ---------------------------------------------------------------------- router
def chosen(logits, bias, k):
    """The experts of each row: falling keys of one rounding, ties to the lowest index, -1 where the rest is -infinity."""
    l32 = logits.astype(np.float32)
    key = l32 + bias.astype(np.float32) if bias is not None else l32
    rank = np.where(np.isnan(key), np.inf, key.astype(np.float64))
    # NaN before infinity: sorted by (not NaN, -key)
    order = np.argsort(-rank, axis=1, kind="stable")
    for r in np.nonzero(np.isnan(key).any(1))[0]:
        order[r] = np.lexsort((np.arange(key.shape[1]), -rank[r], ~np.isnan(key[r])))
    ids = order[:, :k].astype(np.int64)
    none = (np.take_along_axis(l32, ids, 1) == -np.inf) | (np.take_along_axis(key, ids, 1) == -np.inf)
    # (those that are never chosen come last whatever their logit)
    for r in np.nonzero(none.any(1))[0]:
        good = [e for e in order[r] if not (l32[r, e] == -np.inf or key[r, e] == -np.inf)][:k]
        ids[r] = good + [-1] * (k - len(good))
    return ids


def shares(logits, ids, score, normalize):
    """(shares of the chosen, of all experts, relative error): an exponential of x is off by (8 + 2 |x|) roundings."""
    l = torch.as_tensor(logits, dtype=torch.float64)
    at = torch.as_tensor(ids)
    has = at >= 0
    if score == "sigmoid":
        t = -torch.log1p(torch.exp(-l))
        p = torch.exp(t)
    else:
        p = torch.softmax(l, 1)
        p = torch.where(torch.isnan(p), torch.zeros_like(p), p)
    w = torch.where(has, p.gather(1, at.clamp(min=0)), torch.zeros(()).double())
    if normalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, w)
    finite = l[torch.isfinite(l)]
    size = float(finite.abs().max()) if finite.numel() else 0.0
    exp_ = U32 * (8 + 2 * 2 * size)  # (differences reach twice the size)
    rel = 2 * (exp_ + 2 * U32 * (8 + 2 * size) + U32 * (6 * size + 6)) + 75 * U32
    return w, p, rel


def router_grad(logits, ids, w, p, g, score, normalize, scale, rel):
    """(dl, its bound): each of its factors is off by rel or so of its size, the sum over the choices by 64 roundings."""
    at, has = torch.as_tensor(ids), torch.as_tensor(ids) >= 0
    g = torch.where(has, g, torch.zeros_like(g))
    m, size = (g * w).sum(1, keepdim=True), (g * w).abs().sum(1, keepdim=True)
    l = torch.as_tensor(logits, dtype=torch.float64)
    place = lambda v: torch.zeros_like(l).scatter_add(1, at.clamp(min=0), torch.where(has, v, torch.zeros_like(v)))  # noqa: E731
    if normalize:
        d, b = place(scale * w * (g - m)), place(scale * w * (g.abs() + size))
    elif score == "sigmoid":
        d, b = place(scale * w * g), place(scale * w * g.abs())
    else:
        d = place(scale * w * g) - scale * p * m
        b = place(scale * w * g.abs()) + scale * p * size
    if score == "sigmoid":
        slope = 1 / (1 + torch.exp(l))
        d, b = d * slope, b * slope
    return d, b.abs() * (4 * rel + 80 * U32)


# ---------------------------------------------------------------------- sort
def sorted_pairs(ids, experts):
    """(positions, offsets, sources) of the pairs, in numpy."""
    flat = ids.reshape(-1).astype(np.int64)
    good = (flat >= 0) & (flat < experts)
    key = np.where(good, flat, experts)
    order = np.argsort(key, kind="stable")
    n = int(good.sum())
    positions = np.full(flat.size, -1, dtype=np.int32)
    positions[order[:n]] = np.arange(n, dtype=np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[good], minlength=experts))]).astype(np.int32)
    return positions.reshape(ids.shape), offsets, order[:n].astype(np.int32)
