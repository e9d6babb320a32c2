"""What the operators of a sparse feed-forward half of a language model's block are timed on.

Such a half normalises its input, lets a router choose some experts for every token, sorts the tokens by expert,
multiplies each expert's rows by its own weights and adds the results up again, token by token.  A case is one of these
steps in one direction, at sizes that training, prefill or decoding give it.

    norm      y = s rstd w over each row, rstd = 1 / sqrt(mean(s^2) + eps), where s is the input or, with "add",
              residual + input, stored in the inputs' type and normalised as it is stored.  "quant": y in 8-bit floating
              point instead, in groups of columns with a scale each, max(|y|, 2^-100) / (the format's largest value).
    router    the k experts whose logit (plus, with "bias", a number for each expert that has no part in the weights)
              is largest, ties to the lowest index, none whose logit is -infinity (-1 and weight 0 in their place), and
              their weights: softmax over all experts or sigmoid, "normalize"d to the sum 1 over the chosen ones or not.
    sort      the (token, choice) pairs in the order of their experts, stable: each pair's row there, where each
              expert's rows begin, and each row's pair.  Pairs of no expert (-1) have no row.
    dispatch  the way there: each token's row copied (with "weights" times the choice's weight) to the rows of its pairs;
              its gradient.
    product   each expert's rows, which lie one behind the other, times the transpose of its (outputs, inputs) matrix;
              the gradients of rows and matrices.  In 8-bit floating point with a scale for each row's 128 inputs and
              for each matrix's 128 outputs x 128 inputs.
    combine   the way back: the weighted sum of each token's rows, and what it adds to ("add"); its gradient.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32,
          "float8_e4m3fn": torch.float8_e4m3fn, "float8_e5m2": torch.float8_e5m2}
_SIZE = {"bfloat16": 2, "float16": 2, "float32": 4, "float8_e4m3fn": 1, "float8_e5m2": 1}
_LARGEST = {"float8_e4m3fn": 448.0, "float8_e5m2": 57344.0}
EPS = 1e-6


def listed():
    return [
        # Prefill: the residual's sum and rows in 8 bits with a scale for each 128 columns.
        {"name": "norm_add_quant_32768x2048_bf16", "op": "norm", "pass": "forward", "add": True, "dtype": "bfloat16",
         "weights": "bfloat16", "quant": "float8_e4m3fn", "group": 128, "rows": 32768, "cols": 2048, "pad": 0},
        # Training: the residual's sum, its norm and their gradients, single-precision weights.
        {"name": "norm_train_add_16384x4096_bf16", "op": "norm", "pass": "train", "add": True, "dtype": "bfloat16",
         "weights": "float32", "quant": "", "group": 0, "rows": 16384, "cols": 4096, "pad": 0},
        # Decoding: 8 of 128 experts for each of some tokens.
        {"name": "router_forward_48x128_top8_bf16", "op": "router", "pass": "forward", "score": "softmax",
         "normalize": True, "bias": False, "masked": False, "dtype": "bfloat16", "tokens": 48, "experts": 128,
         "choices": 8, "pad": 0},
        # Training with sigmoid scores and a bias that balances the experts' loads.
        {"name": "router_train_32768x256_top8_f32", "op": "router", "pass": "train", "score": "sigmoid",
         "normalize": True, "bias": True, "masked": False, "dtype": "float32", "tokens": 32768, "experts": 256,
         "choices": 8, "pad": 0},
        # Decoding: the order of some tokens' pairs.
        {"name": "sort_48x8_of_128", "op": "sort", "tokens": 48, "choices": 8, "experts": 128, "dropped": 0.0},
        # Training: a batch's pairs, some of them dropped.
        {"name": "sort_32768x8_of_256", "op": "sort", "tokens": 32768, "choices": 8, "experts": 256, "dropped": 0.02},
        # Training: the copies and the sums of their gradients.
        {"name": "dispatch_train_8192x4x2048_bf16", "op": "dispatch", "pass": "train", "weights": False,
         "dtype": "bfloat16", "tokens": 8192, "choices": 4, "experts": 64, "cols": 2048, "pad": 0, "dropped": 0.02},
        # Decoding: a few rows for each of many experts, whose weights are all there is to read.
        {"name": "product_forward_384_of_128_2048x1024_bf16", "op": "product", "pass": "forward", "dtype": "bfloat16",
         "tokens": 48, "choices": 8, "experts": 128, "outputs": 2048, "inputs": 1024, "pad": 0, "dropped": 0.0},
        # Training: the products of a batch and both their gradients.
        {"name": "product_train_32768_of_16_2816x2048_bf16", "op": "product", "pass": "train", "dtype": "bfloat16",
         "tokens": 8192, "choices": 4, "experts": 16, "outputs": 2816, "inputs": 2048, "pad": 0, "dropped": 0.0},
        # Prefill in 8 bits.
        {"name": "product_forward_16384_of_32_4096x2048_e4m3", "op": "product", "pass": "forward", "dtype": "float8_e4m3fn",
         "tokens": 4096, "choices": 4, "experts": 32, "outputs": 4096, "inputs": 2048, "pad": 0, "dropped": 0.0},
        # Decoding: the experts' results added to the residual.
        {"name": "combine_37x8x2048_f16", "op": "combine", "pass": "forward", "add": True, "dtype": "float16",
         "tokens": 37, "choices": 8, "experts": 128, "cols": 2048, "pad": 0, "dropped": 0.0},
        # Training: a large batch.
        {"name": "combine_train_16384x4x4096_bf16", "op": "combine", "pass": "train", "add": False, "dtype": "bfloat16",
         "tokens": 16384, "choices": 4, "experts": 128, "cols": 4096, "pad": 0, "dropped": 0.0},
    ]


def _log_size(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n | 1 if rng.random() < 0.4 else n))


def draw(rng):
    op = rng.choice(["norm", "norm", "router", "sort", "dispatch", "product", "product", "combine"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    pad = rng.choice([0, 0, 0, 1, 8, 64])
    if op == "norm":
        cols = _log_size(rng, 64, 16000)
        rows = _log_size(rng, 1, max(1, min(32768, (1 << 26) // cols)))
        quant = rng.choice(["", "", "float8_e4m3fn", "float8_e4m3fn", "float8_e5m2"])
        return {"op": op, "pass": "forward" if quant else rng.choice(["forward", "train", "train"]),
                "add": rng.random() < 0.6, "dtype": dtype, "weights": rng.choice([dtype, "float32"]), "quant": quant,
                "group": rng.choice([0, 32, 64, 128, 128, 256, 512]) if quant else 0, "rows": rows, "cols": cols,
                "pad": pad}
    choices = rng.choice([1, 2, 2, 3, 4, 6, 8, 8, 10, 16])
    experts = _log_size(rng, max(8, choices), 512)
    if op == "router":
        return {"op": op, "pass": rng.choice(["forward", "train"]), "score": rng.choice(["softmax", "sigmoid"]),
                "normalize": rng.random() < 0.6, "bias": rng.random() < 0.4, "masked": rng.random() < 0.25,
                "dtype": dtype, "tokens": _log_size(rng, 1, 32768), "experts": experts, "choices": choices, "pad": pad}
    dropped = rng.choice([0.0, 0.0, 0.02, 0.3])
    if op == "sort":
        return {"op": op, "tokens": _log_size(rng, 1, 32768), "choices": choices, "experts": experts, "dropped": dropped}
    if op == "product":
        experts = _log_size(rng, max(4, choices), 128)
        outputs, inputs = _log_size(rng, 48, 2816), _log_size(rng, 48, 2816)
        experts = max(choices, min(experts, (1 << 28) // (outputs * inputs)))
        most = (1 << (34 if dtype == "float32" else 37)) // (outputs * inputs * choices)
        way = rng.choice(["forward", "train"])
        if way == "forward" and rng.random() < 0.5:
            dtype = "float8_e4m3fn"
        return {"op": op, "pass": way, "dtype": dtype, "tokens": _log_size(rng, 1, max(1, min(8192, most))),
                "choices": choices, "experts": experts, "outputs": outputs, "inputs": inputs, "pad": pad,
                "dropped": dropped}
    cols = _log_size(rng, 64, 8192)
    most = (1 << (27 if dtype == "float32" else 28)) // (cols * choices)
    case = {"op": op, "pass": rng.choice(["forward", "train", "train"]), "dtype": dtype,
            "tokens": _log_size(rng, 1, max(1, min(16384, most))), "choices": choices, "experts": experts, "cols": cols,
            "pad": pad, "dropped": dropped}
    if op == "combine":
        return case | {"add": rng.random() < 0.5}
    if case["pass"] == "forward" and rng.random() < 0.4:
        return case | {"dtype": "float8_e4m3fn", "weights": False}
    return case | {"weights": rng.random() < 0.3}


# ---------------------------------------------------------------------- inputs
def _empty(shape, dtype, pad=0):
    return torch.empty(*shape[:-1], shape[-1] + pad, dtype=_TYPES[dtype], device="cuda")[..., :shape[-1]]


def _rows(g, shape, dtype, pad, scale=1.0, shift=0.0):
    """Normal values in rows that lie `pad` elements further apart than they are long."""
    view = _empty(shape, dtype, pad)
    view.copy_(torch.randn(shape, generator=g, device="cuda") * scale + shift)
    return view


def _zeros(shape, dtype, pad=0):
    wide = torch.zeros(*shape[:-1], (shape[-1] + pad) * _SIZE[dtype], dtype=torch.uint8, device="cuda")
    return wide.view(_TYPES[dtype])[..., :shape[-1]]


def _choices(g, case):
    """Different experts for each token, some of them much liked, and -1 for the dropped pairs."""
    t, k, e = case["tokens"], case["choices"], case["experts"]
    liking = torch.randn(e, generator=g, device="cuda")
    drawn = torch.rand(t, e, generator=g, device="cuda").clamp_(min=1e-12).log_().neg_().log_().neg_()
    ids = (drawn + liking).topk(k, 1).indices.to(torch.int32)
    return torch.where(torch.rand(t, k, generator=g, device="cuda") < case["dropped"], -1, ids).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st, dt, pad = {"case": case}, case.get("dtype"), case.get("pad", 0)
    if case["op"] == "norm":
        shape = (case["rows"], case["cols"])
        st["x"] = _rows(g, shape, dt, pad, 1.0, 0.1)
        st["w"] = _rows(g, (case["cols"],), case["weights"], 0, 0.2, 1.0)
        if case["add"]:
            st["residual"], st["s"] = _rows(g, shape, dt, pad, 2.0), _empty(shape, dt, pad)
        if case["quant"]:
            st["q"] = _empty(shape, case["quant"], pad)
            st["scales"] = torch.empty(case["rows"], -(-case["cols"] // (case["group"] or case["cols"])), device="cuda")
        else:
            st["y"] = _empty(shape, dt, pad)
        if case["pass"] == "train":
            st["rstd"] = torch.empty(case["rows"], device="cuda")
            st["dy"], st["dx"] = _rows(g, shape, dt, pad, 1e-2), _empty(shape, dt, pad)
            st["dw"] = _empty((case["cols"],), case["weights"])
            if case["add"]:
                st["ds"] = _rows(g, shape, dt, pad, 1e-2)  # what reaches s along the residual path
        return st
    t, k = case["tokens"], case["choices"]
    if case["op"] == "router":
        e = case["experts"]
        st["logits"] = _rows(g, (t, e), dt, pad, 1.5)
        if case["masked"]:
            st["logits"].masked_fill_(torch.rand(t, e, generator=g, device="cuda") < 0.5, -math.inf)
            st["logits"][t // 2] = -math.inf
        if case["bias"]:
            st["bias"] = torch.randn(e, generator=g, device="cuda") * 0.2
        st["experts"] = torch.empty(t, k, dtype=torch.int32, device="cuda")
        st["weights"] = torch.empty(t, k, device="cuda")
        if case["pass"] == "train":
            st["dweights"], st["dlogits"] = torch.randn(t, k, generator=g, device="cuda"), _empty((t, e), dt, pad)
        return st
    ids = _choices(g, case)
    if case["op"] == "sort":
        st["ids"], st["positions"] = ids, torch.empty_like(ids)
        st["offsets"] = torch.empty(case["experts"] + 1, dtype=torch.int32, device="cuda")
        st["sources"] = torch.full((t * k,), -1, dtype=torch.int32, device="cuda")
        return st
    # the places come from the ids: the largest id's pairs last, the dropped ones nowhere
    flat = ids.flatten()
    order = torch.where(flat < 0, case["experts"], flat).sort(stable=True).indices
    places = torch.empty_like(order).scatter_(0, order, torch.arange(t * k, device="cuda"))
    st["positions"] = torch.where(flat < 0, -1, places).to(torch.int32).view(t, k)
    if case["op"] == "product":
        e, n, m = case["experts"], case["outputs"], case["inputs"]
        counts = torch.bincount(flat[flat >= 0], minlength=e)
        st["offsets"] = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
        st["offsets"][1:] = counts.cumsum(0)
        st["longest"] = int(counts.max())  # (of the experts' rows, for the plain form's padding)
        if case["dtype"] == "float8_e4m3fn":
            parts = -(-m // 128)
            x = torch.randn(t * k, parts * 128, generator=g, device="cuda")
            x[:, m:] = 0.0
            st["x_scales"] = x.view(t * k, parts, 128).abs().amax(2) / 448.0
            st["x"], st["y"] = _empty((t * k, m), dt, pad), _zeros((t * k, n), "bfloat16", pad)
            st["x"].copy_((x.view(t * k, parts, 128) / st["x_scales"][:, :, None]).view(t * k, -1)[:, :m])
            st["w"] = _empty((e, n, m), dt)
            st["w"].copy_((torch.randn(e, n, m, generator=g, device="cuda") * 100.0).clamp_(-448.0, 448.0))
            st["w_scales"] = (torch.rand(e, -(-n // 128), parts, generator=g, device="cuda") + 0.5) * (0.01 * m**-0.5)
            return st
        st["x"], st["y"] = _rows(g, (t * k, m), dt, pad), _zeros((t * k, n), dt, pad)
        st["w"] = _rows(g, (e, n, m), dt, 0, m**-0.5)
        if case["pass"] == "train":
            st["dy"], st["dx"] = _rows(g, (t * k, n), dt, pad), _zeros((t * k, m), dt, pad)
            st["dw"] = _empty((e, n, m), dt)
        return st
    few, many = (t, case["cols"]), (t * k, case["cols"])
    w = torch.rand(t, k, generator=g, device="cuda") + 0.05
    w = w / w.sum(1, keepdim=True)
    if case["op"] == "dispatch":
        st["x"], st["y"] = _rows(g, few, dt, pad), _zeros(many, dt, pad)
        st["w"] = w if case["weights"] else None
        if case["pass"] == "train":
            st["dy"], st["dx"] = _rows(g, many, dt, pad, 1e-2), _empty(few, dt, pad)
            st["dw"] = torch.empty(t, k, device="cuda") if case["weights"] else None
        return st
    st["x"], st["y"], st["w"] = _rows(g, many, dt, pad), _empty(few, dt, pad), w
    st["residual"] = _rows(g, few, dt, pad) if case["add"] else None
    if case["pass"] == "train":
        st["dy"], st["dx"], st["dw"] = _rows(g, few, dt, pad, 1e-2), _zeros(many, dt, pad), torch.empty(t, k, device="cuda")
    return st


# ---------------------------------------------------------------------- the framework's calls
def _run_own(st):
    import lc_parallel_primitive_amd as lcpp

    case, op = st["case"], st["case"]["op"]
    train = case.get("pass") == "train"
    if "module" not in st:  # the module and the workspace that a program keeps between its calls
        st["module"] = {"norm": lcpp.DeviceRMSNorm, "router": lcpp.DeviceExpertRouter,
                        "product": lcpp.DeviceExpertProduct}.get(op, lcpp.DeviceTokenSort)()
        tb = 0
        if op == "norm" and train:
            tb = lcpp.DeviceRMSNorm.GetBackwardTempStorageBytes(st["x"].dtype, case["rows"], case["cols"])
        elif op == "sort":
            tb = lcpp.DeviceTokenSort.GetTempStorageBytes(case["tokens"], case["choices"], case["experts"])
        st["temp"] = torch.empty(tb, dtype=torch.uint8, device="cuda") if tb else None
    m = st["module"]
    if op == "product":
        m.Forward(st["x"], st["w"], st["offsets"], st["y"], st.get("x_scales"), st.get("w_scales"))
        if train:
            m.Backward(st["dy"], st["x"], st["w"], st["offsets"], st["dx"], st["dw"])
        return {k: st[k] for k in ("y", "dx", "dw") if k in st}
    if op == "norm":
        quant = {"d_quant": st["q"], "d_scales": st["scales"], "group": case["group"]} if case["quant"] else {}
        y, rstd = st.get("y"), st.get("rstd")
        if case["add"]:
            m.AddForward(st["x"], st["residual"], st["s"], y, st["w"], EPS, rstd, **quant)
        else:
            m.Forward(st["x"], y, st["w"], EPS, rstd, **quant)
        if train:
            m.Backward(st["temp"], st["dy"], st["s" if case["add"] else "x"], st["w"], rstd, st["dx"], st["dw"],
                       d_grad_sum=st.get("ds"))
        return {k: st[k] for k in ("y", "s", "q", "scales", "rstd", "dx", "dw") if k in st}
    if op == "router":
        how = {"score": case["score"], "normalize": case["normalize"]}
        m.Forward(st["logits"], st["experts"], st["weights"], d_bias=st.get("bias"), **how)
        if train:
            m.Backward(st["logits"], st["experts"], st["dweights"], st["dlogits"], **how)
        return {k: st[k] for k in ("experts", "weights", "dlogits") if k in st}
    if op == "sort":
        m.Sort(st["temp"], st["ids"], case["experts"], st["positions"], st["offsets"], st["sources"])
        return {k: st[k] for k in ("positions", "offsets", "sources")}
    if op == "dispatch":
        m.Dispatch(st["x"], st["positions"], st["y"], st["w"])
        if train:
            m.DispatchBackward(st["dy"], st["positions"], st["dx"], st["w"], st["x"] if case["weights"] else None, st["dw"])
    else:
        m.Combine(st["x"], st["positions"], st["w"], st["y"], st["residual"])
        if train:
            m.CombineBackward(st["dy"], st["x"], st["positions"], st["w"], st["dx"], st["dw"])
    return {k: st[k] for k in ("y", "dx", "dw") if st.get(k) is not None}


# ---------------------------------------------------------------------- the plain forms
def _plain_norm(st):
    case, dt = st["case"], st["x"].dtype
    out, s, w = {}, st["x"], st["w"].float()
    if case["add"]:
        s = out["s"] = (st["residual"].float() + s.float()).to(dt)
    s = s.float()
    rstd = torch.rsqrt((s * s).mean(1) + EPS)
    y = s * rstd[:, None] * w
    if case["quant"]:
        rows, cols = y.shape
        group = case["group"] or cols
        parts = -(-cols // group)
        wide = torch.zeros(rows, parts * group, device="cuda")
        wide[:, :cols] = y
        wide = wide.view(rows, parts, group)
        out["scales"] = wide.abs().amax(2).clamp(min=2.0**-100) / _LARGEST[case["quant"]]
        out["q"] = (wide / out["scales"][:, :, None]).to(_TYPES[case["quant"]]).view(rows, -1)[:, :cols]
        return out
    out["y"] = y.to(dt)
    if case["pass"] == "forward":
        return out
    dy = st["dy"].float()
    v = dy * w
    ds = rstd[:, None] * (v - s * (rstd * rstd * (v * s).mean(1))[:, None])
    if case["add"]:
        ds = ds + st["ds"].float()
    return out | {"rstd": rstd, "dx": ds.to(dt), "dw": (dy * s * rstd[:, None]).sum(0).to(st["w"].dtype)}


def _plain_router(st):
    case = st["case"]
    logits = st["logits"].float()
    key = logits + st["bias"] if case["bias"] else logits
    at = key.sort(dim=1, descending=True, stable=True).indices[:, :case["choices"]]
    there = logits.gather(1, at) > -math.inf
    out = {"experts": torch.where(there, at, -1).to(torch.int32)}
    if case["score"] == "sigmoid":
        share = torch.sigmoid(logits)
        slope = torch.sigmoid(-logits)
    else:
        share = torch.exp(logits - logits.amax(1, keepdim=True).clamp(min=-1e30))
        share = share / share.sum(1, keepdim=True).clamp(min=1e-30)
    w = torch.where(there, share.gather(1, at), 0.0)
    if case["normalize"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-30)
    out["weights"] = w
    if case["pass"] == "forward":
        return out
    dw = torch.where(there, st["dweights"], 0.0)
    mean = (dw * w).sum(1, keepdim=True)
    d = torch.zeros_like(logits).scatter(1, at, w * (dw - mean) if case["normalize"] else w * dw)
    if case["score"] == "sigmoid":
        d = d * slope
    elif not case["normalize"]:
        d = d - share * mean
    return out | {"dlogits": d.to(st["logits"].dtype)}


def _plain_sort(st):
    ids, e = st["ids"].flatten(), st["case"]["experts"]
    n = ids.numel()
    key = torch.where(ids < 0, e, ids)
    ordered, order = key.sort(stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(e + 1, dtype=torch.int32, device="cuda"))
    rank = torch.empty_like(order).scatter_(0, order, torch.arange(n, device="cuda"))
    return {"positions": torch.where(ids < 0, -1, rank).to(torch.int32).view_as(st["ids"]),
            "offsets": offsets.to(torch.int32), "sources": torch.where(ordered < e, order, -1).to(torch.int32)}


def _spread(st, rows, weights, like):
    """Each token's row, times its weights, at the rows of its pairs; zeros elsewhere."""
    at = st["positions"].flatten().long()
    some = at >= 0
    k = st["positions"].shape[1]
    out = torch.zeros(like.shape, dtype=like.dtype, device="cuda")
    if weights is None:
        picked = rows[:, None].expand(-1, k, -1).flatten(0, 1)
    else:
        picked = (rows.float()[:, None] * weights[:, :, None]).to(like.dtype).flatten(0, 1)
    if like.element_size() == 1:
        out.view(torch.uint8)[at[some]] = picked.contiguous().view(torch.uint8)[some]
    else:
        out[at[some]] = picked[some]
    return out


def _pairs(st, rows):
    """The rows of each token's pairs, (tokens, choices, columns), zeros where a pair has none."""
    at = st["positions"].long()
    return torch.where((at >= 0)[:, :, None], rows.float()[at.clamp(min=0)], 0.0)


def _plain_dispatch(st):
    out = {"y": _spread(st, st["x"], st["w"], st["y"])}
    if st["case"]["pass"] == "forward":
        return out
    parts = _pairs(st, st["dy"])
    if st["w"] is not None:
        out["dw"] = (parts * st["x"].float()[:, None]).sum(2)
        parts = parts * st["w"][:, :, None]
    return out | {"dx": parts.sum(1).to(st["x"].dtype)}


def _plain_combine(st):
    parts = _pairs(st, st["x"])
    y = (parts * st["w"][:, :, None]).sum(1)
    if st["residual"] is not None:
        y = y + st["residual"].float()
    out = {"y": y.to(st["x"].dtype)}
    if st["case"]["pass"] == "forward":
        return out
    dy = st["dy"].float()
    return out | {"dw": (parts * dy[:, None]).sum(2), "dx": _spread(st, st["dy"], st["w"], st["x"])}


def _plain_product(st):
    case, dt = st["case"], st["y"].dtype
    e, many = case["experts"], st["x"].shape[0]
    row = torch.arange(many, device="cuda")
    offsets = st["offsets"].long()
    expert = torch.searchsorted(offsets, row, right=True) - 1
    some = expert < e
    expert = expert.clamp(max=e - 1)
    place = torch.where(some, expert * st["longest"] + row - offsets[expert], e * st["longest"])

    def padded(rows):
        """Each expert's rows as a matrix of its own, zeros behind them."""
        wide = torch.zeros(e * st["longest"] + 1, rows.shape[1], device="cuda")
        return wide.index_copy_(0, place[some], rows.float()[some])[:-1].view(e, st["longest"], -1)

    def rows_of(wide):
        flat = torch.cat([wide.flatten(0, 1), torch.zeros(1, wide.shape[2], device="cuda")])
        return flat[place].to(dt)

    x, w = st["x"].float(), st["w"].float()
    if "x_scales" in st:
        part = torch.arange(case["inputs"], device="cuda") // 128
        x = x * st["x_scales"][:, part]
        w = w * st["w_scales"][:, torch.arange(case["outputs"], device="cuda") // 128][:, :, part]
    x = padded(x)
    out = {"y": rows_of(torch.bmm(x, w.transpose(1, 2).contiguous()))}
    if case["pass"] == "forward":
        return out
    dy = padded(st["dy"])
    return out | {"dx": rows_of(torch.bmm(dy, w)), "dw": torch.bmm(dy.transpose(1, 2).contiguous(), x).to(dt)}


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "router": _plain_router, "sort": _plain_sort, "dispatch": _plain_dispatch,
            "product": _plain_product, "combine": _plain_combine}[state["case"]["op"]](state)


def work(case):
    e = _SIZE.get(case.get("dtype"), 4)
    train = case.get("pass") == "train"
    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        n = r * c
        # forward: x (and the residual), y (and the sum); backward: dy and the normalised rows again (and the residual
        # path's gradient), dx
        tensors = (3 if case["add"] else 1) + (0 if case["quant"] else 1) + ((4 if case["add"] else 3) if train else 0)
        extra = n + 4 * r * -(-c // (case["group"] or c)) if case["quant"] else 0
        return {"bytes": n * e * tensors + extra + c * _SIZE[case["weights"]] * (3 if train else 1) + r * (8 if train else 0),
                "flops": n * (16 if train else 7 if case["quant"] else 5)}
    t, k = case["tokens"], case["choices"]
    if case["op"] == "router":
        n = t * case["experts"]
        return {"bytes": n * e * (3 if train else 1) + t * k * (16 if train else 8), "flops": n * (10 if train else 5)}
    if case["op"] == "sort":
        return {"bytes": t * k * 12 + case["experts"] * 4, "flops": t * k}
    pairs = t * k * (1.0 - case["dropped"])
    if case["op"] == "product":
        n, m = case["outputs"], case["inputs"]
        # (no more experts are read than there are pairs)
        weights = n * m * (min(case["experts"], pairs) + (case["experts"] if train else 0))
        out = e
        if case["dtype"] == "float8_e4m3fn":
            out, weights = 2, weights * (1.0 + 4 / 128**2)
        return {"bytes": pairs * (out * n + e * m) * (2 if train else 1) + e * weights,
                "flops": 2 * pairs * n * m * (3 if train else 1)}
    c = case["cols"]
    if case["op"] == "dispatch":
        rows, dots = (t + pairs) * (2 if train else 1), train and case["weights"]
        small = t * k * (4 + (4 if case["weights"] else 0)) * (2 if train else 1) + (t * k * 4 if dots else 0)
        return {"bytes": (rows + (t if dots else 0)) * c * e + small,
                "flops": pairs * c * ((2 if train else 1) if not case["weights"] else (5 if train else 1))}
    # backward: the token's gradient and the pairs' rows again, the pairs' gradients
    rows = t + pairs + (t if case["add"] else 0) + ((t + 2 * pairs) if train else 0)
    return {"bytes": rows * c * e + t * k * (8 if not train else 20), "flops": pairs * c * (5 if train else 2)}


# ---------------------------------------------------------------------- the definitions in 64 bits
def _to_8_bits(v, name):
    """Values rounded to the nearest of a format with so many bits of fraction and so low a normal exponent, ties to even."""
    bits, lowest = (3, -6) if name == "float8_e4m3fn" else (2, -14)
    exponent = torch.frexp(v).exponent.double() - 1
    step = torch.exp2(torch.clamp(exponent, min=float(lowest)) - bits)
    return torch.round(v / step) * step


def exact(case, seed):
    if case["op"] == "sort":
        return None
    st = prepare(case, seed)
    if case["op"] == "norm":
        out, rows, cols = {}, st["x"].double(), case["cols"]
        if case["add"]:
            out["s"] = rows + st["residual"].double()
            rows = out["s"].float().to(st["x"].dtype).double()  # the stored sum is what is normalised
        size = torch.sqrt(torch.sum(rows**2, 1, keepdim=True) / cols + EPS)
        u, w = rows / size, st["w"].double()
        y = u * w
        if case["quant"]:
            cuts = torch.split(y, case["group"] or cols, dim=1)
            scales = [torch.clamp(c.abs().max(1, keepdim=True).values, min=2.0**-100) / _LARGEST[case["quant"]] for c in cuts]
            q = [_to_8_bits(c / s, case["quant"]) for c, s in zip(cuts, scales)]
            return out | {"scales": torch.cat(scales, 1), "q": torch.cat(q, 1)}
        out["y"] = y
        if case["pass"] == "train":
            dy = st["dy"].double()
            du = dy * w
            dx = (du - u * torch.sum(du * u, 1, keepdim=True) / cols) / size
            out |= {"rstd": 1.0 / size[:, 0], "dw": torch.sum(dy * u, 0), "dx": dx + st["ds"].double() if case["add"] else dx}
        return out
    t, k = case["tokens"], case["choices"]
    if case["op"] == "router":
        logits = st["logits"].double()
        key = (st["logits"].float() + st["bias"] if case["bias"] else st["logits"].float()).cpu().numpy()
        # sorted by (falling key, index): numpy's stable order of the negated keys
        best = torch.from_numpy(np.argsort(-key, axis=1, kind="stable")[:, :k].copy()).cuda()
        chosen = torch.zeros_like(logits, dtype=torch.bool).scatter_(1, best, True) & ~torch.isinf(logits)
        if case["score"] == "sigmoid":
            p = 1.0 / (1.0 + torch.exp(-logits))
        else:
            p = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
            p = torch.where(torch.isnan(p), 0.0, p)
        full = torch.where(chosen, p, 0.0)
        total = full.sum(1, keepdim=True)
        if case["normalize"]:
            full = torch.where(total > 0, full / total, 0.0)
        out = {"experts": None, "weights": full.gather(1, best)}
        if case["pass"] == "train":
            grad = torch.zeros_like(logits).scatter_(1, best, st["dweights"].double())
            grad = torch.where(chosen, grad, 0.0)
            if case["normalize"]:  # through the division by the sum
                grad = torch.where(chosen & (total > 0), (grad - torch.sum(grad * full, 1, keepdim=True)) / total, 0.0)
            if case["score"] == "sigmoid":
                out["dlogits"] = grad * p * (1.0 - p)
            else:
                out["dlogits"] = p * (grad - torch.sum(grad * p, 1, keepdim=True))
        return out
    if case["op"] == "product":
        names = ("y", "dx", "dw") if case["pass"] == "train" else ("y",)
        out = {name: torch.zeros(st[name].shape, dtype=torch.float64, device="cuda") for name in names}
        edges = st["offsets"].tolist()
        for i, (first, end) in enumerate(zip(edges, edges[1:])):
            rows, matrix = st["x"][first:end].double(), st["w"][i].double()
            if "x_scales" in st:
                scale = st["w_scales"][i].double().repeat_interleave(128, 0)[:case["outputs"]]
                matrix = matrix * scale.repeat_interleave(128, 1)[:, :case["inputs"]]
                rows = rows * st["x_scales"][first:end].double().repeat_interleave(128, 1)[:, :case["inputs"]]
            out["y"][first:end] = torch.mm(rows, matrix.t().contiguous())
            if case["pass"] == "train":
                back = st["dy"][first:end].double()
                out["dx"][first:end], out["dw"][i] = torch.mm(back, matrix), torch.mm(back.t().contiguous(), rows)
        return out
    at = st["positions"].long()
    token, choice = torch.nonzero(at >= 0, as_tuple=True)
    row = at[token, choice]
    source = torch.full((t * k,), -1, dtype=torch.int64, device="cuda")
    source[row] = token * k + choice
    used = source >= 0
    pair_w = None if st["w"] is None else st["w"].double().flatten()

    def spread(rows):
        """What each row of the experts' order is given, column block by column block."""
        out = rows[(source.clamp(min=0) // k)].double()
        if pair_w is not None:
            out *= pair_w[source.clamp(min=0)][:, None]
        out[~used] = 0.0
        return out

    def gathered(rows, weighted=True):
        out = torch.zeros(t, case["cols"], dtype=torch.float64, device="cuda")
        for j in range(k):
            some = at[:, j] >= 0
            v = rows[at[some, j]].double()
            out[some] += v * st["w"][some, j].double()[:, None] if weighted and pair_w is not None else v
        return out

    def dots(few, many):
        out = torch.zeros(t, k, dtype=torch.float64, device="cuda")
        for j in range(k):
            some = at[:, j] >= 0
            out[some, j] = torch.sum(few[some].double() * many[at[some, j]].double(), 1)
        return out

    if case["op"] == "dispatch":
        rows = st["x"].float() if st["x"].element_size() == 1 else st["x"]
        out = {"y": spread(rows)}
        if case["pass"] == "train":
            out["dx"] = gathered(st["dy"])
            if pair_w is not None:
                out["dw"] = dots(st["x"], st["dy"])
        return out
    y = gathered(st["x"])
    out = {"y": y + st["residual"].double() if case["add"] else y}
    if case["pass"] == "train":
        out |= {"dx": spread(st["dy"]), "dw": dots(st["dy"], st["x"])}
    return out
