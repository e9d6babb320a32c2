"""What the operators of a recurrent language model's block are timed on.

A pre-normalised residual block of such a model is layer norm, a gated linear
recurrence over time and dropout; a case is one of these in one direction, at
sizes that training, prefill or decoding give it.

    layer norm    y = (s - mean) / sqrt(var + eps) * w + b over each row, where s
                  is the input or, with "add", residual + dropout(input); the sum
                  s is stored in the inputs' type and it is the stored s that is
                  normalised.
    dropout       x / (1 - p) where the element's 16 random bits are at least
                  65536 p, else 0.  The bits come from Philox 4x32 with 7 rounds
                  (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
                  as 1, 2, 3", 2011): the counter (column / 8, row, offset, offset
                  >> 32) under the 64-bit seed gives 128 bits, 16 for each of eight
                  columns, so no mask is kept for the backward pass.
    recurrence    h_t = a_t h_{t-1} + b_t per channel, with (a, b) from the gate g
                  and the input x: "decay" (g, x), "log" (exp(g), x), "sigmoid"
                  (sigmoid(g), sigmoid(-g) x).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_SIZE = {"bfloat16": 2, "float16": 2, "float32": 4}
EPS = 1e-5


def listed():
    return [
        # Decoding: the norm of a few sequences' single tokens, where one launch is all there is.
        {"name": "norm_forward_16x1024_bf16", "op": "norm", "pass": "forward", "add": False, "dtype": "bfloat16",
         "weights": "bfloat16", "rows": 16, "cols": 1024, "pad": 0, "p": 0.0},
        # Prefill of a table of odd width in single precision.
        {"name": "norm_forward_4099x1000_f32", "op": "norm", "pass": "forward", "add": False, "dtype": "float32",
         "weights": "float32", "rows": 4099, "cols": 1000, "pad": 0, "p": 0.0},
        # Training in half precision where neither the width nor the row stride fits a vector.
        {"name": "norm_train_1777x5001_f16", "op": "norm", "pass": "train", "add": False, "dtype": "float16",
         "weights": "float16", "rows": 1777, "cols": 5001, "pad": 6, "p": 0.0},
        # Training: a batch of long sequences, bfloat16 activations with single-precision weights.
        {"name": "norm_train_16384x4096_bf16", "op": "norm", "pass": "train", "add": False, "dtype": "bfloat16",
         "weights": "float32", "rows": 16384, "cols": 4096, "pad": 0, "p": 0.0},
        # Training: the block's end, residual + dropout(x), and the next block's norm of it.
        {"name": "norm_train_add_16384x2048_bf16", "op": "norm", "pass": "train", "add": True, "dtype": "bfloat16",
         "weights": "float32", "rows": 16384, "cols": 2048, "pad": 0, "p": 0.1},
        # Dropout of a small classifier's features.
        {"name": "dropout_100x1000_f32", "op": "dropout", "add": False, "dtype": "float32", "rows": 100,
         "cols": 1000, "pad": 0, "p": 0.5},
        # Dropout on the residual path of a large batch.
        {"name": "dropout_add_16384x8192_bf16", "op": "dropout", "add": True, "dtype": "bfloat16", "rows": 16384,
         "cols": 8192, "pad": 0, "p": 0.1},
        # Decoding: one token for each of 64 sequences, whose states lie in a pool of slots.
        {"name": "recurrence_step_64x2048_bf16", "op": "recurrence", "pass": "step", "gate": "sigmoid",
         "dtype": "bfloat16", "sequences": 64, "length": 1, "channels": 2048, "packed": False, "pad": 0},
        # Prefill of a few short prompts of odd length, gate and input being halves of one projection.
        {"name": "recurrence_forward_3x777x1000_f32", "op": "recurrence", "pass": "forward", "gate": "decay",
         "dtype": "float32", "sequences": 3, "length": 777, "channels": 1000, "packed": False, "pad": 1000},
        # Prefill of one long document.
        {"name": "recurrence_forward_1x65536x2048_bf16", "op": "recurrence", "pass": "forward", "gate": "sigmoid",
         "dtype": "bfloat16", "sequences": 1, "length": 65536, "channels": 2048, "packed": False, "pad": 0},
        # Training on a batch of sequences.
        {"name": "recurrence_train_8x4096x2048_bf16", "op": "recurrence", "pass": "train", "gate": "sigmoid",
         "dtype": "bfloat16", "sequences": 8, "length": 4096, "channels": 2048, "packed": False, "pad": 0},
        # Training on documents of all lengths packed one behind the other, some of them empty.
        {"name": "recurrence_train_packed_24x16391x1536_bf16", "op": "recurrence", "pass": "train", "gate": "log",
         "dtype": "bfloat16", "sequences": 24, "length": 16391, "channels": 1536, "packed": True, "pad": 0},
    ]


def _log_size(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n | 1 if rng.random() < 0.4 else n))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "recurrence", "recurrence", "recurrence"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    pad = rng.choice([0, 0, 0, 1, 8, 64])
    p = rng.choice([0.0, 0.05, 0.1, 0.1, 0.2, 0.5])
    if op in ("norm", "dropout"):
        cols = _log_size(rng, 64, 20000)
        rows = _log_size(rng, 1, max(1, min(30000, (1 << 25) // cols)))
        if op == "dropout":
            return {"op": op, "add": rng.random() < 0.5, "dtype": dtype, "rows": rows, "cols": cols, "pad": pad, "p": p}
        add = rng.random() < 0.5
        return {"op": op, "pass": rng.choice(["forward", "train", "train"]), "add": add, "dtype": dtype,
                "weights": rng.choice([dtype, "float32"]), "rows": rows, "cols": cols, "pad": pad, "p": p if add else 0.0}
    gate = rng.choice(["decay", "log", "sigmoid", "sigmoid"])
    channels = _log_size(rng, 32, 6000)
    way = rng.choice(["step", "forward", "train", "train"])
    if way == "step":
        return {"op": op, "pass": way, "gate": gate, "dtype": dtype, "sequences": _log_size(rng, 1, 512), "length": 1,
                "channels": channels, "packed": False, "pad": pad}
    packed = rng.random() < 0.3
    most = (1 << 25) // channels  # rows of all sequences together
    if packed:
        length = _log_size(rng, 1, max(1, min(most, 40000)))
        return {"op": op, "pass": way, "gate": gate, "dtype": dtype, "sequences": _log_size(rng, 1, 48),
                "length": length, "channels": channels, "packed": True, "pad": pad}
    length = _log_size(rng, 1, max(1, min(most, 40000)))
    return {"op": op, "pass": way, "gate": gate, "dtype": dtype,
            "sequences": _log_size(rng, 1, max(1, min(64, most // length))), "length": length, "channels": channels,
            "packed": False, "pad": pad}


# ---------------------------------------------------------------------- inputs
def _rows(g, shape, dtype, pad, scale=1.0, shift=0.0):
    """Normal values in rows that lie `pad` elements further apart than they are long."""
    wide = torch.empty(*shape[:-1], shape[-1] + pad, dtype=_TYPES[dtype], device="cuda")
    view = wide[..., :shape[-1]]
    view.copy_(torch.randn(shape, generator=g, device="cuda") * scale + shift)
    return view


def _empty(shape, dtype, pad=0):
    return torch.empty(*shape[:-1], shape[-1] + pad, dtype=_TYPES[dtype], device="cuda")[..., :shape[-1]]


def _lengths(case, seed):
    """The packed sequences' lengths: a random cut of all rows, and one empty sequence where there are two."""
    rng = np.random.default_rng([seed, case["sequences"]])
    s, rows = case["sequences"], case["length"]
    if s < 2:
        return np.array([rows])
    cuts = np.sort(rng.integers(0, rows + 1, size=s - 2))
    lens = np.diff(np.concatenate([[0], cuts, [rows]]))
    return np.insert(lens, int(rng.integers(0, s)), 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"case": case, "seed": 0x9E3779B97F4A7C15 ^ (seed * 0xD1342543DE82EF95 & (1 << 62) - 1), "offset": seed % 1000}
    dt = case["dtype"]
    if case["op"] in ("norm", "dropout"):
        shape, pad = (case["rows"], case["cols"]), case["pad"]
        st["x"] = _rows(g, shape, dt, pad, 1.0, 0.25)
        st["y"] = _empty(shape, dt, pad)
        if case["add"]:
            st["residual"] = _rows(g, shape, dt, pad, 2.0, -0.5)
        if case["op"] == "dropout":
            return st
        wt = case["weights"]
        st["w"] = _rows(g, (case["cols"],), wt, 0, 0.2, 1.0)
        st["b"] = _rows(g, (case["cols"],), wt, 0, 0.1, 0.0)
        if case["add"]:
            st["s"] = _empty(shape, dt, pad)
        if case["pass"] == "train":
            st["mean"], st["rstd"] = (torch.empty(case["rows"], device="cuda") for _ in range(2))
            st["dy"] = _rows(g, shape, dt, pad, 1e-2)
            st["dx"] = _empty(shape, dt, pad)
            st["dw"], st["db"] = (torch.empty(case["cols"], dtype=_TYPES[wt], device="cuda") for _ in range(2))
            if case["add"]:
                st["ds"] = _rows(g, shape, dt, pad, 1e-2)  # the gradient that reaches s along the residual path
                st["dres"] = _empty(shape, dt, pad)
        return st
    s, t, c, pad = case["sequences"], case["length"], case["channels"], case["pad"]
    shape = (s, c) if case["pass"] == "step" else (t, c) if case["packed"] else (s, t, c)
    # gates whose memory is some steps to some thousand steps long
    if case["gate"] == "sigmoid":
        st["g"] = _rows(g, shape, dt, pad, 1.5, 2.0)
    else:
        memory = torch.exp(torch.rand(shape, generator=g, device="cuda") * 6.0)
        st["g"] = _empty(shape, dt, pad)
        st["g"].copy_(-1.0 / memory if case["gate"] == "log" else torch.exp(-1.0 / memory))
    st["x"] = _rows(g, shape, dt, pad)
    st["y"] = _empty(shape, dt, pad)
    if case["pass"] == "step":
        slots = s + s // 2 + 1
        st["state"] = torch.randn(slots, c, generator=g, device="cuda")
        st["next"] = st["state"].clone()
        st["slots"] = torch.randperm(slots, generator=g, device="cuda")[:s].to(torch.int32)
        return st
    st["h0"] = torch.randn(s, c, generator=g, device="cuda")
    st["hT"] = torch.empty(s, c, device="cuda")
    if case["packed"]:
        lens = _lengths(case, seed)
        end = np.cumsum(lens)
        st["begin"] = torch.from_numpy((end - lens).astype(np.int32)).cuda().view(torch.uint32)
        st["end"] = torch.from_numpy(end.astype(np.int32)).cuda().view(torch.uint32)
        st["longest"] = int(lens.max())
    if case["pass"] == "train":
        st["dy"] = _rows(g, shape, dt, pad, 1e-2)
        st["dhT"] = torch.randn(s, c, generator=g, device="cuda") * 1e-2
        st["dg"], st["dx"] = _empty(shape, dt, pad), _empty(shape, dt, pad)
        st["dh0"] = torch.empty(s, c, device="cuda")
    return st


# ---------------------------------------------------------------------- the framework's calls
def _run_own(st):
    import lc_parallel_primitive_amd as lcpp

    case = st["case"]
    if "module" not in st:  # the module and the workspaces that a program keeps between its calls
        st["module"] = {"norm": lcpp.DeviceLayerNorm, "dropout": lcpp.DeviceDropout,
                        "recurrence": lcpp.DeviceGatedRecurrence}[case["op"]]()
        tb = 0
        if case["op"] == "norm" and case["pass"] == "train":
            tb = lcpp.DeviceLayerNorm.GetBackwardTempStorageBytes(st["x"].dtype, case["rows"], case["cols"])
        elif case["op"] == "recurrence" and case["pass"] != "step":
            longest = st.get("longest", case["length"])
            tb = lcpp.DeviceGatedRecurrence.GetTempStorageBytes(case["sequences"], longest, case["channels"])
            rows = lcpp.DeviceGatedRecurrence.GetCheckpointRows(longest)
            st["saved"] = (torch.empty(case["sequences"], rows, case["channels"], device="cuda")
                           if case["pass"] == "train" else None)
        st["temp"] = torch.empty(tb, dtype=torch.uint8, device="cuda") if tb else None
    m, temp = st["module"], st["temp"]
    if case["op"] == "dropout":
        m.Forward(st["x"], st["y"], case["p"], st["seed"], st["offset"], d_residual=st.get("residual"))
        return {"y": st["y"]}
    if case["op"] == "norm":
        mean, rstd = st.get("mean"), st.get("rstd")
        train = case["pass"] == "train"
        if case["add"]:
            m.AddForward(st["x"], st["residual"], st["s"], st["y"], st["w"], st["b"], EPS, mean, rstd, p=case["p"],
                         seed=st["seed"], offset=st["offset"])
            if train:
                m.AddBackward(temp, st["dy"], st["ds"], st["s"], st["w"], mean, rstd, st["dres"], st["dx"], st["dw"],
                              st["db"], p=case["p"], seed=st["seed"], offset=st["offset"])
        else:
            m.Forward(st["x"], st["y"], st["w"], st["b"], EPS, mean, rstd)
            if train:
                m.Backward(temp, st["dy"], st["x"], st["w"], mean, rstd, st["dx"], st["dw"], st["db"])
        return {k: st[k] for k in ("y", "s", "mean", "rstd", "dx", "dres", "dw", "db") if k in st}
    if case["pass"] == "step":
        m.Step(st["g"], st["x"], st["state"], st["next"], st["y"], case["gate"], d_slots=st["slots"])
        return {"y": st["y"], "state": st["next"]}
    where = {}
    if case["packed"]:
        where = {"d_begin_offsets": st["begin"], "d_end_offsets": st["end"], "max_length": st["longest"]}
    m.Forward(temp, st["g"], st["x"], st["y"], case["gate"], d_initial=st["h0"], d_final=st["hT"],
              d_checkpoints=st["saved"], **where)
    if case["pass"] == "train":
        m.Backward(temp, st["g"], st["x"], st["saved"], st["dy"], st["dg"], st["dx"], case["gate"],
                   d_grad_final=st["dhT"], d_grad_initial=st["dh0"], **where)
    return {k: st[k] for k in ("y", "hT", "dg", "dx", "dh0") if k in st}


# ---------------------------------------------------------------------- the plain forms
def _bits(rows, cols, seed, offset):
    """16 random bits for each element, by Philox 4x32-7 in 64-bit integers."""
    low = 0xFFFFFFFF
    c0 = torch.arange(-(-cols // 8), dtype=torch.int64, device="cuda")[None, :].expand(rows, -1)
    c1 = torch.arange(rows, dtype=torch.int64, device="cuda")[:, None].expand_as(c0)
    c2, c3 = torch.full_like(c0, offset & low), torch.full_like(c0, offset >> 32)
    k0, k1 = seed & low, seed >> 32

    def turn(c, r):
        if r == 7:
            return c
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # the wrapped 64-bit products; their upper halves by shifts
        a, b = (k0 + r * 0x9E3779B9) & low, (k1 + r * 0xBB67AE85) & low
        return turn((((q >> 32) & low) ^ c[1] ^ a, q & low, ((p >> 32) & low) ^ c[3] ^ b, p & low), r + 1)

    words = torch.stack(turn((c0, c1, c2, c3), 0), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, -1)[:, :cols]


def _keep(p, shape, seed, offset):
    """(the kept elements, what they are multiplied by)"""
    cut = int(p * 65536 + 0.5)
    return _bits(*shape, seed, offset) >= cut, 65536.0 / (65536 - cut)


def _plain_norm(st):
    case, dt = st["case"], st["x"].dtype
    w, b = st["w"].float(), st["b"].float()
    out = {}
    if case["add"]:
        x = st["x"].float()
        if case["p"]:
            keep, scale = _keep(case["p"], x.shape, st["seed"], st["offset"])
            x = torch.where(keep, x * scale, 0.0)
        s = out["s"] = (st["residual"].float() + x).to(dt)
    else:
        s = st["x"]
    s = s.float()
    mean = s.mean(1)
    centred = s - mean[:, None]
    rstd = torch.rsqrt((centred * centred).mean(1) + EPS)
    unit = centred * rstd[:, None]
    out["y"] = (unit * w + b).to(dt)
    if case["pass"] == "forward":
        return out
    out["mean"], out["rstd"] = mean, rstd
    dy = st["dy"].float()
    out["dw"], out["db"] = (dy * unit).sum(0).to(st["w"].dtype), dy.sum(0).to(st["w"].dtype)
    dw = dy * w
    ds = rstd[:, None] * (dw - dw.mean(1, keepdim=True) - unit * (dw * unit).mean(1, keepdim=True))
    if case["add"]:
        ds = ds + st["ds"].float()
        out["dres"] = ds.to(dt)
        if case["p"]:
            ds = torch.where(keep, ds * scale, 0.0)
    out["dx"] = ds.to(dt)
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, h before the first being 0: the pairs' recurrence, then the even places."""
    n = a.shape[1]
    if n == 1:
        return b
    even = n - n % 2
    a0, a1, b0, b1 = a[:, 0:even:2], a[:, 1:even:2], b[:, 0:even:2], b[:, 1:even:2]
    odd = _scan(a0 * a1, a1 * b0 + b1)
    h = torch.empty_like(b)
    h[:, 1::2] = odd
    h[:, 0] = b[:, 0]
    h[:, 2::2] = a[:, 2::2] * odd[:, :a[:, 2::2].shape[1]] + b[:, 2::2]
    return h


def _plain_recurrence(st):
    case, dt = st["case"], st["x"].dtype
    g, x = st["g"].float(), st["x"].float()
    if case["gate"] == "sigmoid":
        a, share = torch.sigmoid(g), torch.sigmoid(-g)
    else:
        a, share = (torch.exp(g) if case["gate"] == "log" else g), None
    b = x if share is None else share * x
    if case["pass"] == "step":
        at = st["slots"].long()
        h = a * st["state"][at] + b
        return {"y": h.to(dt), "state": st["state"].index_copy(0, at, h)}
    h0 = st["h0"]
    if case["packed"]:  # one chain that the rows at which a sequence begins cut
        a, b, g, x = a[None], b[None], g[None], x[None]
        share = share[None] if share is not None else None
        first, last = st["begin"].view(torch.int32).long(), st["end"].view(torch.int32).long() - 1
        some = last >= first
        first, last = (first[some],), (last[some],)
        row = lambda i: (torch.zeros_like(i[0]), i[0])  # noqa: E731
        first, last = row(first), row(last)
    else:
        s = torch.arange(a.shape[0], device="cuda")
        first, last = (s, torch.zeros_like(s)), (s, torch.full_like(s, a.shape[1] - 1))
        some = torch.ones_like(s, dtype=torch.bool)
    chain = a.clone()
    chain[first] = 0.0
    start = b.clone()
    start[first] = a[first] * h0[some] + b[first]
    h = _scan(chain, start)
    final = h0.clone()
    final[some] = h[last]
    whole = (lambda v: v[0]) if case["packed"] else (lambda v: v)
    out = {"y": whole(h).to(dt), "hT": final}
    if case["pass"] == "forward":
        return out
    before = torch.empty_like(h)
    before[:, 1:] = h[:, :-1]
    before[first] = h0[some]
    dy = st["dy"].float()
    dy = (dy[None] if case["packed"] else dy).clone()
    dy[last] += st["dhT"][some]
    chain.copy_(a)
    chain[last] = 0.0
    # e_t = a_t dh_t is what reaches h_{t-1}
    e = _scan(chain.flip(1), (a * dy).flip(1)).flip(1)
    after = torch.zeros_like(e)
    after[:, :-1] = e[:, 1:]
    after[last] = 0.0
    dh = dy + after
    dh0 = st["dhT"].clone()
    dh0[some] = e[first]
    if case["gate"] == "sigmoid":
        dg, dx = dh * (before - x) * a * share, dh * share
    else:
        dg, dx = dh * before * (a if case["gate"] == "log" else 1.0), dh
    return out | {"dg": whole(dg).to(dt), "dx": whole(dx).to(dt), "dh0": dh0}


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "norm":
        return _plain_norm(state)
    if case["op"] == "recurrence":
        return _plain_recurrence(state)
    x = state["x"].float()
    if case["p"]:
        keep, scale = _keep(case["p"], x.shape, state["seed"], state["offset"])
        x = torch.where(keep, x * scale, 0.0)
    if case["add"]:
        x = x + state["residual"].float()
    return {"y": x.to(state["x"].dtype)}


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * e * (3 if case["add"] else 2), "flops": n * (2 if case["add"] else 1)}
    if case["op"] == "norm":
        n, train = case["rows"] * case["cols"], case["pass"] == "train"
        # forward: x (and the residual), y (and the sum); backward: dy and the normalised rows again (and the
        # residual path's gradient), dx (and the residual's gradient)
        tensors = (4 if case["add"] else 2) + ((5 if case["add"] else 3) if train else 0)
        per_col = _SIZE[case["weights"]] * (5 if train else 2)
        per_row = 16 if train else 0
        return {"bytes": n * e * tensors + case["cols"] * per_col + case["rows"] * per_row,
                "flops": n * (22 if train else 8)}
    c, s = case["channels"], case["sequences"]
    if case["pass"] == "step":
        return {"bytes": s * (c * (3 * e + 8) + 4), "flops": s * c * 8}
    n = case["length"] * c * (1 if case["packed"] else s)
    train = case["pass"] == "train"
    return {"bytes": n * e * (8 if train else 3) + s * c * 4 * (4 if train else 2), "flops": n * (22 if train else 8)}


# ---------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    n, p = case.get("cols"), case.get("p", 0.0)
    limit = math.floor(p * 65536 + 0.5)

    def drawn(first, last):
        """The 16-bit numbers of some rows, from the generator's definition in numpy's unsigned integers."""
        u, low, half = np.uint64, np.uint64(0xFFFFFFFF), np.uint64(32)
        block, row = np.meshgrid(np.arange(-(-n // 8), dtype=u), np.arange(first, last, dtype=u))
        x, y = [block, row], [st["offset"] & 0xFFFFFFFF, st["offset"] >> 32]
        c = x + [np.full_like(block, v) for v in y]
        key = [st["seed"] & 0xFFFFFFFF, st["seed"] >> 32]
        for _ in range(7):
            m0, m1 = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
            c = [(m1 >> half) ^ c[1] ^ u(key[0]), m1 & low, (m0 >> half) ^ c[3] ^ u(key[1]), m0 & low]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return np.stack(c, -1).astype("<u4").view("<u2").reshape(last - first, -1)[:, :n]

    if limit:
        step = max(1, (1 << 22) // n)
        kept = torch.empty(case["rows"], n, dtype=torch.bool, device="cuda")
        for r in range(0, case["rows"], step):
            most = min(r + step, case["rows"])
            kept[r:most] = torch.from_numpy(drawn(r, most) >= limit).cuda()

    def dropped(v):
        return torch.where(kept, v / (1.0 - limit / 65536.0), torch.zeros_like(v)) if limit else v

    if case["op"] == "dropout":
        v = dropped(st["x"].double())
        return {"y": v + st["residual"].double() if case["add"] else v}

    if case["op"] == "norm":
        out, rows = {}, st["x"].double()
        if case["add"]:
            rows = out["s"] = st["residual"].double() + dropped(rows)
            rows = rows.float().to(st["x"].dtype).double()  # the stored sum is what is normalised
        mu = rows.sum(1, keepdim=True) / n
        sd = torch.sqrt(((rows - mu) ** 2).sum(1, keepdim=True) / n + EPS)
        z, w = (rows - mu) / sd, st["w"].double()
        out["y"] = z * w + st["b"].double()
        if case["pass"] == "forward":
            return out
        dy = st["dy"].double()
        out |= {"mean": mu[:, 0], "rstd": 1.0 / sd[:, 0], "dw": torch.sum(dy * z, 0), "db": torch.sum(dy, 0)}
        dz = dy * w
        d = (dz - dz.sum(1, keepdim=True) / n - z * torch.sum(dz * z, 1, keepdim=True) / n) / sd
        if case["add"]:
            d = out["dres"] = d + st["ds"].double()
        return out | {"dx": dropped(d)}

    gate, x, kind = st["g"].double(), st["x"].double(), case["gate"]
    if kind == "sigmoid":
        decay, drive = 1.0 / (1.0 + torch.exp(-gate)), x / (1.0 + torch.exp(gate))
    else:
        decay, drive = (gate if kind == "decay" else torch.exp(gate)), x
    if case["pass"] == "step":
        states, y = st["state"].double(), torch.empty_like(drive)
        for i, slot in enumerate(st["slots"].tolist()):
            y[i] = states[slot] = decay[i] * states[slot] + drive[i]
        return {"y": y, "state": states}
    if case["packed"]:
        ends = st["end"].view(torch.int32).tolist()
        chains = [(b, e, i) for i, (b, e) in enumerate(zip(st["begin"].view(torch.int32).tolist(), ends))]
        decay, drive, gate, x = decay[None], drive[None], gate[None], x[None]
        dy = st["dy"].double()[None] if "dy" in st else None
    else:
        chains = [(0, case["length"], slice(None))]
        dy = st["dy"].double() if "dy" in st else None
    states, finals = torch.empty_like(x), torch.empty_like(st["hT"], dtype=torch.float64)
    for first, end, s in chains:
        h = st["h0"][s].double()
        for t in range(first, end):
            h = decay[:, t] * h + drive[:, t]
            states[:, t] = h
        finals[s] = h
    whole = (lambda v: v[0]) if case["packed"] else (lambda v: v)
    out = {"y": whole(states), "hT": finals}
    if case["pass"] == "forward":
        return out
    earlier, back, dh0 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(finals)
    for first, end, s in chains:
        v = st["dhT"][s].double()
        for t in range(end - 1, first - 1, -1):
            v = v + dy[:, t]
            back[:, t] = v
            v = v * decay[:, t]
        dh0[s] = v
        if end > first:
            earlier[:, first] = st["h0"][s].double()
            earlier[:, first + 1:end] = states[:, first:end - 1]
    if kind == "sigmoid":
        shut = 1.0 / (1.0 + torch.exp(gate))
        dg, dx = back * (earlier - x) * decay * shut, back * shut
    else:
        dg, dx = back * earlier * (decay if kind == "log" else 1.0), back
    return out | {"dg": whole(dg), "dx": whole(dx), "dh0": dh0}
