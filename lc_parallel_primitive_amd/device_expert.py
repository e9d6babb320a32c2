"""The sparse feed-forward half of a language model's block: the router that chooses experts for every token, the
tokens sorted by expert and back, and the experts' products, forward and backward.

The reference has none of them; they follow its manner as the classes of device_block.py do.  A pair is a token's
choice of an expert: choice j of token t is pair t * choices + j.  Offsets, positions and experts are 32-bit integers
on the GPU, and no call waits for them.

    router, order, product, norm = DeviceExpertRouter(), DeviceTokenSort(), DeviceExpertProduct(), DeviceRMSNorm()
    norm.AddForward(d_in, d_residual, d_residual_out, d_normed, weight)
    router.Forward(d_normed @ gate, d_experts, d_weights)
    order.Sort(temp, d_experts, num_experts, d_positions, d_offsets)
    order.Dispatch(d_normed, d_positions, d_rows)
    product.Forward(d_rows, d_matrices, d_offsets, d_results)
    order.Combine(d_results, d_positions, d_weights, d_out, d_residual_out)
"""
from __future__ import annotations

from ._capi import LCPP_FLOAT8_E4M3, LCPP_FLOAT16, LCPP_FLOAT32, LCPP_SCORES, _float_codes, float_code, lib, quant_code
from .device import _ptr, _query, _stream
from .device_block import _BlockModule, _float_vector, _like, _like_out, _matrix, _off_gpu, _temp, _unlike


def _indices(t, n: int, what: str):
    """The address of a contiguous tensor of at least n 32-bit integers, or None."""
    if t is None:
        return None
    if t.element_size() != 4 or t.is_floating_point():
        raise TypeError(f"{what}: must be 32-bit integers, got {t.dtype}")
    if t.numel() < n:
        raise ValueError(f"{what}: holds {t.numel()} values, need {n}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")
    if not t.is_cuda:
        _off_gpu(t, what)
    return t.data_ptr()


def _pairs(t, what: str):
    """(tokens, choices) of a tensor of shape (tokens, choices)."""
    if t.dim() != 2:
        raise ValueError(f"{what}: shape (tokens, choices), got {tuple(t.shape)}")
    return t.shape


def _rows(t, rows, cols: int, dtype, what: str, output: bool = False):
    """(address, row stride) of a matrix of this type and so many columns, and rows (None: any)."""
    if t.dim() != 2 or t.shape[1] != cols or (rows is not None and t.shape[0] != rows) or t.dtype != dtype:
        _unlike(t, (t.shape[0] if rows is None and t.dim() else rows, cols), dtype, what)
    return t.data_ptr(), (_like_out if output else _like)(t, t.shape, dtype, what)


class DeviceExpertRouter(_BlockModule):
    """The `choices` best experts of each row of logits and their weights.

    The largest keys win, a key being the logit plus d_bias of its expert (which has no part in the weights), ties going
    to the lowest index and a NaN before all others.  An expert whose logit or key is -infinity is never chosen: where
    too few are left, the expert is -1 and its weight 0.  Weights are `scale` times

        "softmax"   exp(l) / sum of exp(l)         over the row, or with normalize over the chosen ones
        "sigmoid"   1 / (1 + exp(-l))              with normalize divided by the sum over the chosen ones

    Up to 1024 experts and 64 choices."""

    @staticmethod
    def _score(score):
        code = LCPP_SCORES.get(score)
        if code is None:
            raise ValueError(f"unsupported score {score!r}: one of {', '.join(LCPP_SCORES)}")
        return code

    def _sizes(self, d_logits, d_experts, what: str):
        if d_logits.dim() != 2:
            raise ValueError(f"d_logits: shape (tokens, experts), got {tuple(d_logits.shape)}")
        code = float_code(d_logits.dtype)
        _, tokens, experts, stride = _matrix(d_logits, "d_logits")
        rows, choices = _pairs(d_experts, "d_experts")
        if rows != tokens:
            raise ValueError(f"d_experts: {rows} rows for {tokens} tokens")
        return code, tokens, experts, choices, stride

    def Forward(self, d_logits, d_experts, d_weights, score: str = "softmax", normalize: bool = True, scale: float = 1.0,
                d_bias=None, stream=None):
        """d_logits: shape (tokens, experts); d_experts (int32), d_weights (float32): shape (tokens, choices)."""
        code, tokens, experts, choices, stride = self._sizes(d_logits, d_experts, "d_experts")
        self._call("lcpp_router_forward", None, _stream(stream), code, self._score(score), int(normalize), scale,
                   d_logits.data_ptr(), stride, _float_vector(d_bias, experts, "d_bias"),
                   _indices(d_experts, tokens * choices, "d_experts"),
                   _float_vector(d_weights, tokens * choices, "d_weights"), tokens, experts, choices)

    def Backward(self, d_logits, d_experts, d_grad_weights, d_grad_logits, score: str = "softmax", normalize: bool = True,
                 scale: float = 1.0, stream=None):
        """The gradient of Forward's d_logits (d_bias has none), with the forward call's d_experts."""
        code, tokens, experts, choices, stride = self._sizes(d_logits, d_experts, "d_experts")
        self._call("lcpp_router_backward", None, _stream(stream), code, self._score(score), int(normalize), scale,
                   d_logits.data_ptr(), stride, _indices(d_experts, tokens * choices, "d_experts"),
                   _float_vector(d_grad_weights, tokens * choices, "d_grad_weights"), d_grad_logits.data_ptr(),
                   _like_out(d_grad_logits, d_logits.shape, d_logits.dtype, "d_grad_logits"), tokens, experts, choices)


class DeviceTokenSort(_BlockModule):
    """Tokens in the order of the experts that were chosen for them, and back.

    Sort gives each pair a row: the pairs of expert 0 first, then those of expert 1, each expert's in their own order.
    Dispatch copies each token's row to its pairs' rows, Combine adds each token's rows up again, with its weights.
    Pairs whose expert is not in 0 .. experts - 1 have the position -1 and count nothing.  Sums are made in the order of
    the choices in 32 bits: the same bits at every call."""

    @staticmethod
    def GetTempStorageBytes(tokens: int, choices: int, experts: int) -> int:
        return _query(lib().lcpp_token_sort_temp_bytes, tokens, choices, experts)

    def Sort(self, temp_storage, d_experts, experts: int, d_positions, d_offsets, d_sources=None, stream=None):
        """d_experts, d_positions: int32 of shape (tokens, choices); d_offsets: int32, where each expert's rows begin and,
        behind the last, the number of all (experts + 1 values); d_sources: int32, each row's pair (those behind the
        last row are left alone), or None."""
        tokens, choices = _pairs(d_experts, "d_experts")
        n = tokens * choices
        if d_positions.shape != d_experts.shape:
            raise ValueError(f"d_positions: shape {tuple(d_positions.shape)}, expected {tuple(d_experts.shape)}")
        self._call("lcpp_token_sort", temp_storage, _stream(stream), *_temp(temp_storage),
                   _indices(d_experts, n, "d_experts"), tokens, choices, experts, _indices(d_positions, n, "d_positions"),
                   _indices(d_offsets, experts + 1, "d_offsets"), _indices(d_sources, n, "d_sources"))

    def _spread(self, d_in, d_positions, d_weights, out, other, dots, rows, stream):
        tokens, choices = _pairs(d_positions, "d_positions")
        _, held, cols, si = _matrix(d_in, "d_in")
        if held != tokens:
            raise ValueError(f"{held} rows for {tokens} tokens")
        n = tokens * choices
        dtype = d_in.dtype
        code = float_code(dtype) if d_weights is not None or dots is not None else _row_code(dtype)
        self._call("lcpp_token_spread", None, _stream(stream), code, d_in.data_ptr(), si,
                   _indices(d_positions, n, "d_positions"), _float_vector(d_weights, n, "d_weights"), *out, *other,
                   _float_vector(dots, n, "d_grad_weights"), rows, tokens, choices, cols)

    def _sum(self, d_in, d_positions, d_weights, residual, d_out, other, dots, stream):
        tokens, choices = _pairs(d_positions, "d_positions")
        dtype = d_out.dtype
        code = float_code(dtype)
        cols = d_out.shape[-1]
        n = tokens * choices
        self._call("lcpp_token_sum", None, _stream(stream), code, *_rows(d_in, None, cols, dtype, "d_in"), d_in.shape[0],
                   _indices(d_positions, n, "d_positions"), _float_vector(d_weights, n, "d_weights"), *residual,
                   *_rows(d_out, tokens, cols, dtype, "d_out", True), *other, _float_vector(dots, n, "d_grad_weights"),
                   tokens, choices, cols)

    def Dispatch(self, d_in, d_positions, d_out, d_weights=None, stream=None):
        """d_out[d_positions[t, j]] = d_in[t], with d_weights (float32, of the pairs) times d_weights[t, j].  Without them
        any type of 1, 2 or 4 bytes is copied (rows in 8 bits, their scales).  Rows of d_out that no pair has are left
        alone."""
        self._spread(d_in, d_positions, d_weights, _rows(d_out, None, d_in.shape[-1], d_in.dtype, "d_out", True),
                     (None, 0), None, d_out.shape[0], stream)

    def DispatchBackward(self, d_grad_out, d_positions, d_grad_in, d_weights=None, d_in=None, d_grad_weights=None,
                         stream=None):
        """The gradient of Dispatch's d_in, and with d_in that of d_weights (None if not wanted)."""
        other = (None, 0)
        if d_grad_weights is not None:
            if d_in is None:
                raise ValueError("d_grad_weights needs d_in")
            other = _rows(d_in, d_grad_in.shape[0], d_grad_in.shape[-1], d_grad_in.dtype, "d_in")
        self._sum(d_grad_out, d_positions, d_weights, (None, 0), d_grad_in, other, d_grad_weights, stream)

    def Combine(self, d_in, d_positions, d_weights, d_out, d_residual=None, stream=None):
        """d_out[t] = [d_residual[t] +] the sum over j of d_weights[t, j] (None: 1) times d_in[d_positions[t, j]].  d_out may
        be d_residual."""
        residual = (None, 0)
        if d_residual is not None:
            residual = _rows(d_residual, d_out.shape[0], d_out.shape[-1], d_out.dtype, "d_residual")
        self._sum(d_in, d_positions, d_weights, residual, d_out, (None, 0), None, stream)

    def CombineBackward(self, d_grad_out, d_in, d_positions, d_weights, d_grad_in, d_grad_weights=None, stream=None):
        """The gradients of Combine's d_in (None if not wanted; rows that no pair has are left alone) and d_weights (None
        if not wanted); d_residual's is d_grad_out itself."""
        cols, dtype = d_grad_out.shape[-1], d_grad_out.dtype
        if d_grad_in is None and d_grad_weights is None:
            return
        out, other, rows = (None, 0), (None, 0), None
        if d_grad_in is not None:
            out, rows = _rows(d_grad_in, None, cols, dtype, "d_grad_in", True), d_grad_in.shape[0]
        if d_grad_weights is not None:
            other, rows = _rows(d_in, rows, cols, dtype, "d_in"), d_in.shape[0]
        self._spread(d_grad_out, d_positions, d_weights, out, other, d_grad_weights, rows, stream)


def _matrices(t, what: str, output: bool = False):
    """(experts, outputs, inputs, address, row stride, stride from one matrix to the next) of matrices."""
    if t.dim() != 3:
        raise ValueError(f"{what}: shape (experts, outputs, inputs), got {tuple(t.shape)}")
    (experts, outputs, inputs), (se, so, si) = t.shape, t.stride()
    if si != 1 and inputs > 1:
        raise ValueError(f"{what}: the values of a matrix's row must be adjacent, got strides {(se, so, si)}")
    if output and ((so < inputs and outputs > 1) or (experts > 1 and se < (outputs - 1) * so + inputs
                                                     and (se < inputs or so < (experts - 1) * se + inputs))):
        # (one behind the other, or side by side in the rows of one another)
        raise ValueError(f"{what}: the matrices of an output must not overlap, got strides {(se, so, si)}")
    if not t.is_cuda:
        _off_gpu(t, what)
    return experts, outputs, inputs, t.data_ptr(), so, se


class DeviceExpertProduct(_BlockModule):
    """Each expert's rows, which lie one behind the other as DeviceTokenSort puts them, times its matrix: d_out[r] =
    d_weight[e] d_in[r], e being the expert whose rows d_offsets[e] .. d_offsets[e + 1] hold r.  Matrices are of shape
    (experts, outputs, inputs); sums are made in 32 bits on the matrix cores and rounded once.  One expert with the
    offsets (0, rows) is a plain product."""

    def Forward(self, d_in, d_weight, d_offsets, d_out, d_in_scales=None, d_weight_scales=None, stream=None):
        """d_in: (rows, inputs); d_out: (rows, outputs); d_offsets: int32, experts + 1 values.  Rows past the last offset
        are left alone.  In 8 bits (float8_e4m3fn) d_in_scales, float32 of shape (rows, ceil(inputs / 128)) and any
        strides, and d_weight_scales, (experts, ceil(outputs / 128), ceil(inputs / 128)), multiply the values of 128 inputs
        each; d_out is then of any of the three types.  There the matrix cores add products in eights, cut 13 bits below
        the largest of the eight.  Up to 1024 experts."""
        experts, outputs, inputs, weight, so, se = _matrices(d_weight, "d_weight")
        dtype = d_in.dtype
        out_code = _float_codes.get(d_out.dtype) or float_code(d_out.dtype)
        code = _float_codes.get(dtype)
        rows = d_in.shape[0]
        scales, weight_scales = (None, 0, 0), None
        if code is None:
            code = quant_code(dtype)
            groups = -(-inputs // 128)
            if d_in_scales is None or d_weight_scales is None:
                raise ValueError("products in 8 bits need d_in_scales and d_weight_scales")
            if tuple(d_in_scales.shape) != (rows, groups):
                raise ValueError(f"d_in_scales: shape {tuple(d_in_scales.shape)}, expected {(rows, groups)}")
            if float_code(d_in_scales.dtype) != 2:
                raise TypeError(f"d_in_scales: must be float32, got {d_in_scales.dtype}")
            if not d_in_scales.is_cuda:
                _off_gpu(d_in_scales, "d_in_scales")
            scales = d_in_scales.data_ptr(), *d_in_scales.stride()
            shape = experts, -(-outputs // 128), groups
            if tuple(d_weight_scales.shape) != shape:
                raise ValueError(f"d_weight_scales: shape {tuple(d_weight_scales.shape)}, expected {shape}")
            weight_scales = _float_vector(d_weight_scales, d_weight_scales.numel(), "d_weight_scales")
        elif d_in_scales is not None or d_weight_scales is not None:
            raise ValueError("scales go with products in 8 bits")
        elif d_out.dtype != dtype:
            raise TypeError(f"d_out: dtype {d_out.dtype}, expected {dtype}")
        if d_weight.dtype != dtype:
            raise TypeError(f"d_weight: dtype {d_weight.dtype}, expected {dtype}")
        self._call("lcpp_expert_product", None, _stream(stream), code, *_rows(d_in, None, inputs, dtype, "d_in"), weight, so, se,
                   _indices(d_offsets, experts + 1, "d_offsets"), out_code,
                   *_rows(d_out, rows, outputs, d_out.dtype, "d_out", True), *scales, weight_scales, rows, experts, outputs,
                   inputs)

    def Backward(self, d_grad_out, d_in, d_weight, d_offsets, d_grad_in=None, d_grad_weight=None, stream=None):
        """The gradients of Forward's d_in and d_weight (each None if not wanted; the latter of d_weight's type or float32,
        0 for experts without rows).  d_in is needed for d_grad_weight, d_weight's values for d_grad_in.  Rows past the
        last offset are left alone."""
        experts, outputs, inputs, weight, so, se = _matrices(d_weight, "d_weight")
        dtype = d_grad_out.dtype
        code = _float_codes.get(dtype) or float_code(dtype)
        if d_weight.dtype != dtype:
            raise TypeError(f"d_weight: dtype {d_weight.dtype}, expected {dtype}")
        rows = d_grad_out.shape[0]
        grad_out = _rows(d_grad_out, None, outputs, dtype, "d_grad_out")
        grad_in, x, grad_weight, weight_code = (None, 0), (None, 0), (None, 0, 0), code
        if d_grad_in is not None:
            grad_in = _rows(d_grad_in, rows, inputs, dtype, "d_grad_in", True)
        if d_grad_weight is not None:
            x = _rows(d_in, rows, inputs, dtype, "d_in")
            if d_grad_weight.shape != d_weight.shape:
                _unlike(d_grad_weight, d_weight.shape, dtype, "d_grad_weight")
            weight_code = _float_codes.get(d_grad_weight.dtype) or float_code(d_grad_weight.dtype)
            if weight_code != code and weight_code != 2:
                raise TypeError("d_grad_weight must have d_weight's dtype or float32")
            grad_weight = _matrices(d_grad_weight, "d_grad_weight", True)[3:]
        self._call("lcpp_expert_product_backward", None, _stream(stream), code, *grad_out, *x, weight, so, se,
                   _indices(d_offsets, experts + 1, "d_offsets"), *grad_in, weight_code, *grad_weight, rows, experts, outputs,
                   inputs)


_COPIED = {1: LCPP_FLOAT8_E4M3, 2: LCPP_FLOAT16, 4: LCPP_FLOAT32}


def _row_code(dtype) -> int:
    """An lcpp_dtype of as many bytes as the elements of rows that are copied."""
    code = _COPIED.get(dtype.itemsize)
    if code is None:
        raise TypeError(f"unsupported dtype {dtype}: rows that are copied have elements of 1, 2 or 4 bytes")
    return code
