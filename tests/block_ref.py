"""Layer norm, dropout and the gated recurrence from their definitions, in 64 bits on the CPU, with bounds of what
32-bit arithmetic may be off by.

U[t] is the relative error of one rounding to type t.  Every bound is a count of 32-bit roundings times the size of
what they round, plus one rounding of the result to its type; `tiny` covers float16's subnormal steps."""
import numpy as np
import torch

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = {"float32": 2.0**-24, "bfloat16": 2.0**-8, "float16": 2.0**-11}
U32 = 2.0**-24


def tiny(dtype):
    return {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0**-25}[dtype]


def check(got, want, bound, dtype, what):
    """|got - want| <= one rounding of the result to dtype + bound, and the same values that are not finite."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: non-finite values differ"
    tol = U[dtype] * want.abs() * (1 + 1e-6) + bound * (1 + U[dtype]) + tiny(dtype)
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} past the bound"


def rows(g, shape, dtype, pad=0, shift=0.0, scale=1.0, offset=0, device="cuda"):
    """Normal values of `shape` in a larger buffer: rows `pad` elements apart, beginning at element `offset`."""
    n = int(np.prod(shape[:-1])) * (shape[-1] + pad)
    flat = torch.zeros(n + offset, dtype=TYPES[dtype], device=device)[offset:]
    view = flat.view(*shape[:-1], shape[-1] + pad)[..., :shape[-1]]
    view.copy_((torch.randn(shape, generator=g, dtype=torch.float64) * scale + shift).to(TYPES[dtype]))
    return view


def host(t):
    return t.detach().double().cpu()


# ---------------------------------------------------------------------- dropout
def philox_bits(nrows, ncols, seed, offset):
    """The 16 random bits of each element, in Python's own integers (one row of blocks at a time)."""
    out = np.empty((nrows, -(-ncols // 8) * 8), dtype=np.int64)
    for r in range(nrows):
        for b in range(-(-ncols // 8)):
            c = [b, r, offset & 0xFFFFFFFF, offset >> 32]
            k = [seed & 0xFFFFFFFF, seed >> 32]
            for _ in range(7):
                p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
                c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
                k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
            for i in range(8):
                out[r, b * 8 + i] = (c[i // 2] >> (16 * (i % 2))) & 0xFFFF
    return torch.from_numpy(out[:, :ncols])


def dropped(x, p, seed, offset):
    """(x where it is kept, scaled, else 0; the kept places)"""
    cut = int(p * 65536 + 0.5)
    keep = philox_bits(*x.shape, seed, offset) >= cut
    scale = 65536 / (65536 - cut) if cut < 65536 else 0.0
    return torch.where(keep, x * scale, torch.zeros_like(x)), keep


# ---------------------------------------------------------------------- layer norm
# The longest chain of a row's sum: 32 elements in a thread (40 in rows of up to 40000 columns), 10 steps over lanes and
# waves, then the division: under 64 roundings.  The mean is off by that many of the mean magnitude, the centred value
# by one more of |s|, rstd by half of the squares' error and a few of its own, and three roundings follow.
CHAIN = 64


def norm(s, w, b, eps):
    n = s.shape[1]
    mean = s.mean(1, keepdim=True)
    var = ((s - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    y = (s - mean) * rstd * w + b
    mag = s.abs().mean(1, keepdim=True)
    e_mean = U32 * (CHAIN * mag + mean.abs())
    e_centred = e_mean + U32 * (s.abs() + mean.abs())
    # var: its sum's own roundings, and each square's through its centred value
    e_var = U32 * (CHAIN + 4) * var + 2 * (e_centred * (s - mean).abs()).mean(1, keepdim=True) + (e_centred**2).mean(1, keepdim=True)
    rel_rstd = 0.5 * e_var / (var + eps) + 6 * U32
    bound = w.abs() * rstd * (e_centred + (s - mean).abs() * (rel_rstd + 3 * U32)) * 1.01 + 2 * U32 * (y.abs() + b.abs())
    return y, mean, rstd, bound, e_mean, rel_rstd * rstd * 1.01


def norm_grad(s, w, mean, rstd, dy, rounds):
    """(ds, dw, db) and their bounds, from statistics as they are given (32-bit values); `rounds`: the roundings of a
    column's sum over rows."""
    u = (s - mean) * rstd
    size = (s.abs() + mean.abs()) * rstd  # what u's own roundings are relative to
    v = dy * w
    av, avu = v.mean(1, keepdim=True), (v * u).mean(1, keepdim=True)
    ds = rstd * (v - av - u * avu)
    avu_size = (v.abs() * size).mean(1, keepdim=True)
    bound = U32 * rstd * (4 * v.abs() + (CHAIN + 4) * v.abs().mean(1, keepdim=True) + (CHAIN + 10) * size * avu_size)
    dw, db = (dy * u).sum(0), dy.sum(0)
    bw, bb = U32 * (rounds + 4) * (dy.abs() * size).sum(0), U32 * rounds * dy.abs().sum(0)
    return ds, dw, db, bound, bw, bb


# ---------------------------------------------------------------------- recurrence
def gate_values(kind, g):
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    return (torch.exp(g) if kind == "log" else g), torch.ones_like(g)


def gate_error(kind, g):
    """The relative error of a and of 1 - a: the exponential's argument is rounded once (|g| roundings of the result)
    and the exponential, the sum, the reciprocal and the product take a few each."""
    return U32 * (8 + 2 * g.abs()) if kind != "decay" else torch.zeros_like(g)


def recurrence(kind, g, x, h0):
    """One sequence: g, x (rows, channels).  Returns h of every row, a, 1 - a (or 1), and h's bounds: each step adds the
    roundings of its gate, its products and sums, and what was wrong before it is carried on by |a|; composing tiles
    takes at most three roundings more a step."""
    a, share = gate_values(kind, g)
    e = gate_error(kind, g)
    b = share * x
    h, err = h0.clone(), torch.zeros_like(h0)
    hs, errs = torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[0]):
        err = a[t].abs() * err + (6 * U32 + e[t]) * ((a[t] * h).abs() + b[t].abs() + a[t].abs() * err)
        h = a[t] * h + b[t]
        hs[t], errs[t] = h, err
    return hs, a, share, errs


def recurrence_grad(kind, g, x, h0, hs, errs, a, share, dy, dhT):
    """(dg, dx, dh0) and their bounds."""
    e = gate_error(kind, g)
    back, err = dhT.clone(), torch.zeros_like(dhT)
    dh, dh_err = torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[0] - 1, -1, -1):
        err = err + 6 * U32 * (dy[t].abs() + back.abs() + err)
        back = back + dy[t]
        dh[t], dh_err[t] = back, err
        err = a[t].abs() * err + (6 * U32 + e[t]) * (a[t] * back).abs()
        back = back * a[t]
    before = torch.cat([h0[None], hs[:-1]]) if x.shape[0] else hs
    before_err = torch.cat([torch.zeros_like(h0)[None], errs[:-1]]) if x.shape[0] else errs
    if kind == "sigmoid":
        f = (a * share).abs()
        diff = before - x
        dg = dh * diff * a * share
        bg = f * (dh_err * diff.abs() + (dh.abs() + dh_err) * (before_err + U32 * (before.abs() + x.abs()))) \
            + (6 * U32 + 2 * e) * dg.abs() * 2
        dx, bx = dh * share, share * dh_err + (2 * U32 + e) * (dh * share).abs() * 2
    else:
        f = a.abs() if kind == "log" else torch.ones_like(a)
        dg = dh * before * (a if kind == "log" else 1)
        bg = f * (dh_err * before.abs() + (dh.abs() + dh_err) * before_err) + (4 * U32 + e) * dg.abs() * 2
        dx, bx = dh, dh_err
    return dg, dx, back, bg, bx, err
