"""The operators of a recurrent language model's residual block: layer norm,
dropout and the gated linear recurrence, forward and backward.

The reference has none of them; they follow its manner here as the classes of
device.py do: caller-owned outputs and temp storage, an asynchronous call on a
stream (default: torch's current stream), sizes and types checked before any
launch (TypeError, ValueError), errors of the library raised as LcppError.

Activations and their gradients are float32, bfloat16 or float16; weights are
of the same type or float32; statistics and recurrent states are float32.
Everything is computed in 32 bits and rounded once when it is stored.  Sizes
are those of the tensors.  Rows need unit stride along their last dimension
and may lie any distance apart.

    norm, mix, drop = DeviceLayerNorm(), DeviceGatedRecurrence(), DeviceDropout()
    norm.AddForward(d_mixed, d_residual, d_residual_out, d_normed, weight, bias, 1e-5, mean, rstd, p=0.1, seed=7)
    mix.Forward(temp, d_gate, d_value, d_mixed, "sigmoid", d_checkpoints=saved)
"""
from __future__ import annotations

import ctypes

from ._capi import LCPP_GATES, check, float_code, lib
from .device import _Module, _nbytes, _ptr, _query, _stream


def _matrix(t, what: str):
    """(rows, columns, row stride) of a tensor whose last dimension has unit stride."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        if shape[1] > 1 and stride[1] != 1:
            raise ValueError(f"{what}: the columns of a row must be adjacent, got strides {stride}")
        return shape[0], shape[1], stride[0]
    if len(shape) == 0 or not t.is_contiguous():
        raise ValueError(f"{what}: must be two-dimensional or contiguous, got shape {tuple(shape)}, strides {stride}")
    cols = shape[-1]
    return t.numel() // cols if cols else 0, cols, cols


def _like(t, ref, what: str):
    """The row stride of a tensor that must have the shape and type of `ref`."""
    if t.shape != ref.shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {tuple(ref.shape)}")
    if t.dtype != ref.dtype:
        raise TypeError(f"{what}: dtype {t.dtype}, expected {ref.dtype}")
    return _matrix(t, what)[2]


def _own_rows(t, rows: int, cols: int, stride: int, what: str):
    if rows > 1 and stride < cols:
        raise ValueError(f"{what}: the rows of an output must not overlap")


def _vector(t, n: int, what: str, dtype_of=None):
    """A contiguous tensor of at least n values, or None."""
    if t is None:
        return None
    if t.numel() < n:
        raise ValueError(f"{what}: holds {t.numel()} values, need {n}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")
    if dtype_of is not None and t.dtype != dtype_of.dtype:
        raise TypeError(f"{what}: dtype {t.dtype}, expected {dtype_of.dtype}")
    return t.data_ptr()


def _float_vector(t, n: int, what: str):
    p = _vector(t, n, what)
    if p is not None and float_code(t.dtype) != 2:
        raise TypeError(f"{what}: must be float32, got {t.dtype}")
    return p


def _weight_code(code: int, *weights):
    """The lcpp_dtype of the weights that are given: the activations' or float32."""
    wt = None
    for w in weights:
        if w is not None:
            c = float_code(w.dtype)
            if wt is not None and c != wt:
                raise TypeError("weight, bias and their gradients must have one dtype")
            wt = c
    if wt is None:
        return code
    if wt != code and wt != 2:
        raise TypeError("weights must have the activations' dtype or float32")
    return wt


def _counter(t, what: str):
    if t is None:
        return None
    if t.numel() < 1 or t.element_size() != 8:
        raise ValueError(f"{what}: must hold a 64-bit integer")
    return t.data_ptr()


_U64 = (1 << 64) - 1


class DeviceLayerNorm(_Module):
    """y = (s - mean) / sqrt(var + eps) * weight + bias over the rows of s."""

    @staticmethod
    def GetBackwardTempStorageBytes(dtype, rows: int, cols: int) -> int:
        return _query(lib().lcpp_layer_norm_backward_temp_bytes, float_code(dtype), rows, cols)

    def Forward(self, d_in, d_out, d_weight=None, d_bias=None, eps: float = 1e-5, d_mean=None, d_rstd=None, stream=None):
        """d_out = the layer norm of d_in; d_mean, d_rstd: float32 row statistics for Backward, or None."""
        code = float_code(d_in.dtype)
        rows, cols, si = _matrix(d_in, "d_in")
        so = _like(d_out, d_in, "d_out")
        _own_rows(d_out, rows, cols, so, "d_out")
        self._check(lib().lcpp_layer_norm_forward(
            code, _weight_code(code, d_weight, d_bias), d_in.data_ptr(), si, _vector(d_weight, cols, "d_weight"),
            _vector(d_bias, cols, "d_bias"), eps, d_out.data_ptr(), so, _float_vector(d_mean, rows, "d_mean"),
            _float_vector(d_rstd, rows, "d_rstd"), rows, cols, _stream(stream)),
            "lcpp_layer_norm_forward", None, stream)

    def AddForward(self, d_in, d_residual, d_sum, d_out, d_weight=None, d_bias=None, eps: float = 1e-5, d_mean=None,
                   d_rstd=None, p: float = 0.0, seed: int = 0, offset: int = 0, d_offset=None, stream=None):
        """d_sum = d_residual + dropout(d_in), d_out = the layer norm of d_sum as it is stored.  p, seed, offset,
        d_offset as DeviceDropout.Forward."""
        code = float_code(d_in.dtype)
        rows, cols, si = _matrix(d_in, "d_in")
        sr, ss, so = _like(d_residual, d_in, "d_residual"), _like(d_sum, d_in, "d_sum"), _like(d_out, d_in, "d_out")
        _own_rows(d_sum, rows, cols, ss, "d_sum")
        _own_rows(d_out, rows, cols, so, "d_out")
        self._check(lib().lcpp_layer_norm_add_forward(
            code, _weight_code(code, d_weight, d_bias), d_in.data_ptr(), si, d_residual.data_ptr(), sr, p, seed & _U64,
            offset & _U64, _counter(d_offset, "d_offset"), _vector(d_weight, cols, "d_weight"),
            _vector(d_bias, cols, "d_bias"), eps, d_sum.data_ptr(), ss, d_out.data_ptr(), so,
            _float_vector(d_mean, rows, "d_mean"), _float_vector(d_rstd, rows, "d_rstd"), rows, cols, _stream(stream)),
            "lcpp_layer_norm_add_forward", None, stream)

    def Backward(self, temp_storage, d_grad_out, d_in, d_weight, d_mean, d_rstd, d_grad_in, d_grad_weight=None,
                 d_grad_bias=None, stream=None):
        """The gradients of Forward's d_in, d_weight and d_bias (the latter two None if not wanted)."""
        code = float_code(d_in.dtype)
        rows, cols, si = _matrix(d_in, "d_in")
        sg, so = _like(d_grad_out, d_in, "d_grad_out"), _like(d_grad_in, d_in, "d_grad_in")
        _own_rows(d_grad_in, rows, cols, so, "d_grad_in")
        self._check(lib().lcpp_layer_norm_backward(
            code, _weight_code(code, d_weight, d_grad_weight, d_grad_bias), _ptr(temp_storage), _nbytes(temp_storage),
            d_grad_out.data_ptr(), sg, d_in.data_ptr(), si, _vector(d_weight, cols, "d_weight"),
            _float_vector(d_mean, rows, "d_mean"), _float_vector(d_rstd, rows, "d_rstd"), d_grad_in.data_ptr(), so,
            _vector(d_grad_weight, cols, "d_grad_weight"), _vector(d_grad_bias, cols, "d_grad_bias"), rows, cols,
            _stream(stream)), "lcpp_layer_norm_backward", temp_storage, stream)

    def AddBackward(self, temp_storage, d_grad_out, d_grad_sum, d_sum, d_weight, d_mean, d_rstd, d_grad_residual,
                    d_grad_in, d_grad_weight=None, d_grad_bias=None, p: float = 0.0, seed: int = 0, offset: int = 0,
                    d_offset=None, stream=None):
        """The gradients of AddForward.  d_grad_sum: what reaches d_sum along the residual path (None: nothing).
        d_grad_residual = d_sum's whole gradient, d_grad_in = its dropout with the forward call's random bits; either
        is None if not wanted."""
        code = float_code(d_sum.dtype)
        rows, cols, ss = _matrix(d_sum, "d_sum")
        sg = _like(d_grad_out, d_sum, "d_grad_out")
        sx, sr, si = (0 if t is None else _like(t, d_sum, nm) for t, nm in (
            (d_grad_sum, "d_grad_sum"), (d_grad_residual, "d_grad_residual"), (d_grad_in, "d_grad_in")))
        if d_grad_residual is not None:
            _own_rows(d_grad_residual, rows, cols, sr, "d_grad_residual")
        if d_grad_in is not None:
            _own_rows(d_grad_in, rows, cols, si, "d_grad_in")
        self._check(lib().lcpp_layer_norm_add_backward(
            code, _weight_code(code, d_weight, d_grad_weight, d_grad_bias), _ptr(temp_storage), _nbytes(temp_storage),
            d_grad_out.data_ptr(), sg, _ptr(d_grad_sum), sx, d_sum.data_ptr(), ss, _vector(d_weight, cols, "d_weight"),
            _float_vector(d_mean, rows, "d_mean"), _float_vector(d_rstd, rows, "d_rstd"), p, seed & _U64, offset & _U64,
            _counter(d_offset, "d_offset"), _ptr(d_grad_residual), sr, _ptr(d_grad_in), si,
            _vector(d_grad_weight, cols, "d_grad_weight"), _vector(d_grad_bias, cols, "d_grad_bias"), rows, cols,
            _stream(stream)), "lcpp_layer_norm_add_backward", temp_storage, stream)


class DeviceDropout(_Module):
    """Dropout whose mask is computed from (seed, offset, row, column) wherever it is needed, and never stored."""

    def Forward(self, d_in, d_out, p: float, seed: int, offset: int = 0, d_residual=None, d_offset=None, stream=None):
        """d_out = (kept ? d_in / (1 - p) : 0) [+ d_residual].  p is met to 2^-17.  offset tells the calls of one seed
        apart (a layer's number, a step's); d_offset, a device tensor of one 64-bit integer, is added to it when the
        kernel runs, so a captured graph's replays can differ."""
        code = float_code(d_in.dtype)
        rows, cols, si = _matrix(d_in, "d_in")
        so = _like(d_out, d_in, "d_out")
        _own_rows(d_out, rows, cols, so, "d_out")
        sr = 0 if d_residual is None else _like(d_residual, d_in, "d_residual")
        self._check(lib().lcpp_dropout(code, d_in.data_ptr(), si, _ptr(d_residual), sr, d_out.data_ptr(), so, rows, cols, p,
                                       seed & _U64, offset & _U64, _counter(d_offset, "d_offset"), _stream(stream)),
                    "lcpp_dropout", None, stream)

    def Backward(self, d_grad_out, d_grad_in, p: float, seed: int, offset: int = 0, d_offset=None, stream=None):
        """The gradient of Forward's d_in, with the forward call's p, seed and offset (d_residual's is d_grad_out itself)."""
        self.Forward(d_grad_out, d_grad_in, p, seed, offset, None, d_offset, stream)


def _sequence_strides(t, ref, what: str, packed: bool, output: bool = False):
    """(row stride, sequence stride) of (sequences, rows, channels), or with offsets (rows, channels)."""
    if t.shape != ref.shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {tuple(ref.shape)}")
    if t.dtype != ref.dtype:
        raise TypeError(f"{what}: dtype {t.dtype}, expected {ref.dtype}")
    stride, shape = t.stride(), t.shape
    if shape[-1] > 1 and stride[-1] != 1:
        raise ValueError(f"{what}: the channels of a row must be adjacent, got strides {stride}")
    if output:
        # no two rows may share memory: in the order of their strides, each dimension steps over the one below it
        span = shape[-1]
        for n, st in sorted(((n, st) for n, st in zip(shape[:-1], stride[:-1]) if n > 1), key=lambda d: d[1]):
            if st < span:
                raise ValueError(f"{what}: the rows of an output must not overlap, got strides {stride}")
            span = st * n
    return (stride[0], 0) if packed else (stride[1], stride[0])


class DeviceGatedRecurrence(_Module):
    """h_t = a_t h_{t-1} + b_t per channel, with a and b from a gate g and an input x:

        "decay"    a = g, b = x
        "log"      a = exp(g), b = x
        "sigmoid"  a = sigmoid(g), b = (1 - a) x

    Sequences are tensors of shape (sequences, length, channels), or, packed one behind the other, (rows, channels)
    with 32-bit begin and end offsets of each sequence and `max_length`, the longest one's length (a longer one is cut
    there).  States are float32 of shape (sequences, channels)."""

    @staticmethod
    def GetTempStorageBytes(sequences: int, max_length: int, channels: int) -> int:
        return _query(lib().lcpp_recurrence_temp_bytes, sequences, max_length, channels)

    @staticmethod
    def GetCheckpointRows(max_length: int) -> int:
        """d_checkpoints has shape (sequences, this, channels), float32."""
        out = ctypes.c_uint64()
        check(lib().lcpp_recurrence_checkpoint_rows(max_length, ctypes.byref(out)), "lcpp_recurrence_checkpoint_rows")
        return out.value

    def _sizes(self, d_gate, d_in, gate, d_begin_offsets, d_end_offsets, max_length):
        if gate not in LCPP_GATES:
            raise ValueError(f"unsupported gate {gate!r}: one of {', '.join(LCPP_GATES)}")
        packed = d_begin_offsets is not None
        if packed != (d_end_offsets is not None):
            raise ValueError("begin and end offsets go together")
        if d_in.dim() != (2 if packed else 3):
            raise ValueError("d_in: shape (sequences, length, channels), or with offsets (rows, channels)")
        if packed:
            if d_begin_offsets.element_size() != 4 or d_end_offsets.element_size() != 4:
                raise TypeError("offsets must be 32-bit")
            if max_length is None:
                raise ValueError("offsets need max_length")
            sequences, (rows, channels) = d_begin_offsets.numel(), d_in.shape
            if d_end_offsets.numel() != sequences or not (d_begin_offsets.is_contiguous() and d_end_offsets.is_contiguous()):
                raise ValueError("begin and end offsets must be contiguous and of one length")
        else:
            if max_length is not None:
                raise ValueError("max_length goes with offsets")
            sequences, max_length, channels = d_in.shape
            rows = 0
        return packed, (sequences, max_length, channels, _ptr(d_begin_offsets), _ptr(d_end_offsets), rows)

    def Forward(self, temp_storage, d_gate, d_in, d_out, gate: str, d_initial=None, d_final=None, d_checkpoints=None,
                d_begin_offsets=None, d_end_offsets=None, max_length=None, stream=None):
        """d_out = h for every row.  d_initial: the states before the first rows (None: 0); d_final: those after the
        last; d_checkpoints: what Backward needs."""
        code = float_code(d_in.dtype)
        packed, sizes = self._sizes(d_gate, d_in, gate, d_begin_offsets, d_end_offsets, max_length)
        states = sizes[0] * sizes[2]
        g = _sequence_strides(d_gate, d_in, "d_gate", packed)
        x = _sequence_strides(d_in, d_in, "d_in", packed)
        y = _sequence_strides(d_out, d_in, "d_out", packed, True)
        saved = None
        if d_checkpoints is not None:
            saved = _float_vector(d_checkpoints, states * self.GetCheckpointRows(sizes[1]), "d_checkpoints")
        self._check(lib().lcpp_recurrence_forward(
            code, LCPP_GATES[gate], _ptr(temp_storage), _nbytes(temp_storage), d_gate.data_ptr(), *g, d_in.data_ptr(), *x,
            d_out.data_ptr(), *y, _float_vector(d_initial, states, "d_initial"), _float_vector(d_final, states, "d_final"),
            saved, *sizes, _stream(stream)), "lcpp_recurrence_forward", temp_storage, stream)

    def Backward(self, temp_storage, d_gate, d_in, d_checkpoints, d_grad_out, d_grad_gate, d_grad_in, gate: str,
                 d_grad_final=None, d_grad_initial=None, d_begin_offsets=None, d_end_offsets=None, max_length=None,
                 stream=None):
        """The gradients of Forward's d_gate, d_in and d_initial from those of d_out and d_final (None: 0)."""
        code = float_code(d_in.dtype)
        packed, sizes = self._sizes(d_gate, d_in, gate, d_begin_offsets, d_end_offsets, max_length)
        states = sizes[0] * sizes[2]
        g = _sequence_strides(d_gate, d_in, "d_gate", packed)
        x = _sequence_strides(d_in, d_in, "d_in", packed)
        dy = _sequence_strides(d_grad_out, d_in, "d_grad_out", packed)
        dg = _sequence_strides(d_grad_gate, d_in, "d_grad_gate", packed, True)
        dx = _sequence_strides(d_grad_in, d_in, "d_grad_in", packed, True)
        self._check(lib().lcpp_recurrence_backward(
            code, LCPP_GATES[gate], _ptr(temp_storage), _nbytes(temp_storage), d_gate.data_ptr(), *g, d_in.data_ptr(), *x,
            _float_vector(d_checkpoints, states * self.GetCheckpointRows(sizes[1]), "d_checkpoints"), d_grad_out.data_ptr(),
            *dy, d_grad_gate.data_ptr(), *dg, d_grad_in.data_ptr(), *dx,
            _float_vector(d_grad_final, states, "d_grad_final"), _float_vector(d_grad_initial, states, "d_grad_initial"),
            *sizes, _stream(stream)), "lcpp_recurrence_backward", temp_storage, stream)

    def Step(self, d_gate, d_in, d_state_in, d_state_out, d_out, gate: str, d_slots=None, stream=None):
        """One token for each of some sequences: d_gate, d_in and d_out of shape (sequences, channels).  The states are
        float32 of shape (slots, channels); d_state_out may be d_state_in.  d_slots: int32, the row of each sequence's
        state, all different; -1 marks padding (out is 0, no state changes).  None: row s for sequence s."""
        if gate not in LCPP_GATES:
            raise ValueError(f"unsupported gate {gate!r}: one of {', '.join(LCPP_GATES)}")
        code = float_code(d_in.dtype)
        if d_in.dim() != 2:
            raise ValueError("d_in: shape (sequences, channels)")
        rows, cols, sx = _matrix(d_in, "d_in")
        sg, so = _like(d_gate, d_in, "d_gate"), _like(d_out, d_in, "d_out")
        _own_rows(d_out, rows, cols, so, "d_out")
        if d_state_in.shape != d_state_out.shape or d_state_in.dim() != 2 or d_state_in.shape[1] != cols:
            raise ValueError(f"states: shapes {tuple(d_state_in.shape)} and {tuple(d_state_out.shape)}, expected (slots, {cols})")
        slots = d_state_in.shape[0]
        if d_slots is not None:
            if d_slots.element_size() != 4 or d_slots.is_floating_point():
                raise TypeError("d_slots: must be int32")
            _vector(d_slots, rows, "d_slots")
        elif slots < rows:
            raise ValueError(f"states: {slots} rows for {rows} sequences")
        self._check(lib().lcpp_recurrence_step(
            code, LCPP_GATES[gate], d_gate.data_ptr(), sg, d_in.data_ptr(), sx, _float_vector(d_state_in, 0, "d_state_in"),
            _float_vector(d_state_out, 0, "d_state_out"), _ptr(d_slots), slots, d_out.data_ptr(), so, rows, cols,
            _stream(stream)), "lcpp_recurrence_step", None, stream)
