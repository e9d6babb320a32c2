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
and may lie any distance apart.  A tensor that is not on the GPU is refused
(ValueError): its address would fault there.

    norm, mix, drop = DeviceLayerNorm(), DeviceGatedRecurrence(), DeviceDropout()
    norm.AddForward(d_mixed, d_residual, d_residual_out, d_normed, weight, bias, 1e-5, mean, rstd, p=0.1, seed=7)
    mix.Forward(temp, d_gate, d_value, d_mixed, "sigmoid", d_checkpoints=saved)
"""
from __future__ import annotations

import ctypes
import functools

from ._capi import LCPP_GATES, _float_codes, check, float_code, lib
from .device import _Module, _ptr, _query, _stream


# What a call does before its launch is most of a small call's time (device.py),
# so a tensor's shape and strides are asked for once, refusals are worded in
# functions of their own, and the common layouts are checked first.


def _off_gpu(t, what: str):
    raise ValueError(f"{what}: must be on the GPU, got a tensor on {t.device}")


def _matrix(t, what: str):
    """(shape, rows, columns, row stride) of a tensor whose last dimension has unit stride."""
    if not t.is_cuda:
        _off_gpu(t, what)
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        if stride[1] == 1 or shape[1] <= 1:
            return shape, shape[0], shape[1], stride[0]
        raise ValueError(f"{what}: the columns of a row must be adjacent, got strides {stride}")
    if len(shape) == 0 or not t.is_contiguous():
        raise ValueError(f"{what}: must be two-dimensional or contiguous, got shape {tuple(shape)}, strides {stride}")
    cols = shape[-1]
    return shape, t.numel() // cols if cols else 0, cols, cols


def _unlike(t, shape, dtype, what: str):
    if t.shape != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    raise TypeError(f"{what}: dtype {t.dtype}, expected {dtype}")


def _like(t, shape, dtype, what: str):
    """The row stride of a tensor that must have this shape and type."""
    if t.shape != shape or t.dtype != dtype:
        _unlike(t, shape, dtype, what)
    if not t.is_cuda:
        _off_gpu(t, what)
    stride = t.stride()
    if len(stride) == 2 and (stride[1] == 1 or shape[1] <= 1):
        return stride[0]
    return _matrix(t, what)[3]


def _like_out(t, shape, dtype, what: str):
    """The same for an output, whose rows must not overlap."""
    if t.shape != shape or t.dtype != dtype:
        _unlike(t, shape, dtype, what)
    if not t.is_cuda:
        _off_gpu(t, what)
    stride = t.stride()
    if len(stride) != 2 or (stride[1] != 1 and shape[1] > 1):
        return _matrix(t, what)[3]
    if stride[0] < shape[1] and shape[0] > 1:
        raise ValueError(f"{what}: the rows of an output must not overlap")
    return stride[0]


def _in_out(x, y, in_name: str = "d_in", out_name: str = "d_out"):
    """(shape, dtype, lcpp_dtype, rows, columns, row strides) of an input and an output of its shape and type."""
    shape, dtype, sx, sy = x.shape, x.dtype, x.stride(), y.stride()
    code = _float_codes.get(dtype)
    if (code and y.shape == shape and len(sx) == 2 and sx[1] == sy[1] == 1 and y.dtype == dtype and sy[0] >= shape[1]
            and x.is_cuda and y.is_cuda):
        return shape, dtype, code, shape[0], shape[1], sx[0], sy[0]
    code = float_code(dtype)
    _, rows, cols, si = _matrix(x, in_name)
    return shape, dtype, code, rows, cols, si, _like_out(y, shape, dtype, out_name)


def _vector(t, n: int, what: str):
    """The address of a contiguous tensor of at least n values, or None."""
    if t is None:
        return None
    if t.numel() >= n and t.is_contiguous() and t.is_cuda:
        return t.data_ptr()
    if t.numel() < n:
        raise ValueError(f"{what}: holds {t.numel()} values, need {n}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")
    _off_gpu(t, what)


def _temp(t):
    """(address, bytes) of the temp storage, or (None, 0)."""
    if t is None:
        return None, 0
    if not t.is_cuda:
        _off_gpu(t, "temp_storage")
    return t.data_ptr(), t.nbytes


def _float_vector(t, n: int, what: str):
    if t is None:
        return None
    if _float_codes.get(t.dtype) != 2 and float_code(t.dtype) != 2:
        raise TypeError(f"{what}: must be float32, got {t.dtype}")
    if t.numel() >= n and t.is_contiguous() and t.is_cuda:
        return t.data_ptr()
    return _vector(t, n, what)


def _weight_code(code: int, weight, *others):
    """The lcpp_dtype of the weights that are given: the activations' or float32."""
    dtype = None if weight is None else weight.dtype
    for w in others:
        if w is not None:
            if dtype is None:
                dtype = w.dtype
            elif w.dtype != dtype:
                raise TypeError("weight, bias and their gradients must have one dtype")
    if dtype is None:
        return code
    wt = _float_codes.get(dtype) or float_code(dtype)
    if wt != code and wt != 2:
        raise TypeError("weights must have the activations' dtype or float32")
    return wt


def _counter(t, what: str):
    if t is None:
        return None
    if t.numel() < 1 or t.element_size() != 8 or t.is_floating_point() or t.is_complex():
        raise ValueError(f"{what}: must hold a 64-bit integer")
    if not t.is_cuda:
        _off_gpu(t, what)
    return t.data_ptr()


_entries: dict = {}


def _entry(name: str):
    f = _entries[name] = getattr(lib(), name)
    return f


class _BlockModule(_Module):
    def _call(self, name: str, temp, stream, *args):
        status = (_entries.get(name) or _entry(name))(*args, stream)
        if status or self._debug:
            self._check(status, name, temp, stream)


class DeviceLayerNorm(_BlockModule):
    """y = (s - mean) / sqrt(var + eps) * weight + bias over the rows of s."""

    @staticmethod
    def GetBackwardTempStorageBytes(dtype, rows: int, cols: int) -> int:
        return _query(lib().lcpp_layer_norm_backward_temp_bytes, float_code(dtype), rows, cols)

    def Forward(self, d_in, d_out, d_weight=None, d_bias=None, eps: float = 1e-5, d_mean=None, d_rstd=None, stream=None):
        """d_out = the layer norm of d_in; d_mean, d_rstd: float32 row statistics for Backward, or None."""
        _, _, code, rows, cols, si, so = _in_out(d_in, d_out)
        self._call("lcpp_layer_norm_forward", None, _stream(stream), code, _weight_code(code, d_weight, d_bias),
                   d_in.data_ptr(), si, _vector(d_weight, cols, "d_weight"), _vector(d_bias, cols, "d_bias"), eps,
                   d_out.data_ptr(), so, _float_vector(d_mean, rows, "d_mean"), _float_vector(d_rstd, rows, "d_rstd"), rows,
                   cols)

    def AddForward(self, d_in, d_residual, d_sum, d_out, d_weight=None, d_bias=None, eps: float = 1e-5, d_mean=None,
                   d_rstd=None, p: float = 0.0, seed: int = 0, offset: int = 0, d_offset=None, stream=None):
        """d_sum = d_residual + dropout(d_in), d_out = the layer norm of d_sum as it is stored; d_sum may be d_residual
        or d_in, but not d_out.  p, seed, offset, d_offset as DeviceDropout.Forward."""
        dtype = d_in.dtype
        code = float_code(dtype)
        shape, rows, cols, si = _matrix(d_in, "d_in")
        sr = _like(d_residual, shape, dtype, "d_residual")
        ss, so = _like_out(d_sum, shape, dtype, "d_sum"), _like_out(d_out, shape, dtype, "d_out")
        self._call("lcpp_layer_norm_add_forward", None, _stream(stream), code, _weight_code(code, d_weight, d_bias),
                   d_in.data_ptr(), si, d_residual.data_ptr(), sr, p, seed, offset,
                   _counter(d_offset, "d_offset"), _vector(d_weight, cols, "d_weight"), _vector(d_bias, cols, "d_bias"), eps,
                   d_sum.data_ptr(), ss, d_out.data_ptr(), so, _float_vector(d_mean, rows, "d_mean"),
                   _float_vector(d_rstd, rows, "d_rstd"), rows, cols)

    def Backward(self, temp_storage, d_grad_out, d_in, d_weight, d_mean, d_rstd, d_grad_in, d_grad_weight=None,
                 d_grad_bias=None, stream=None):
        """The gradients of Forward's d_in, d_weight and d_bias (the latter two None if not wanted)."""
        shape, dtype, code, rows, cols, si, so = _in_out(d_in, d_grad_in, "d_in", "d_grad_in")
        sg = _like(d_grad_out, shape, dtype, "d_grad_out")
        # (a call of nothing may launch nothing and leave the status word)
        self._call("lcpp_layer_norm_backward", temp_storage if rows and cols else None, _stream(stream), code,
                   _weight_code(code, d_weight, d_grad_weight, d_grad_bias), *_temp(temp_storage),
                   d_grad_out.data_ptr(), sg, d_in.data_ptr(), si, _vector(d_weight, cols, "d_weight"),
                   _float_vector(d_mean, rows, "d_mean"), _float_vector(d_rstd, rows, "d_rstd"), d_grad_in.data_ptr(), so,
                   _vector(d_grad_weight, cols, "d_grad_weight"), _vector(d_grad_bias, cols, "d_grad_bias"), rows, cols)

    def AddBackward(self, temp_storage, d_grad_out, d_grad_sum, d_sum, d_weight, d_mean, d_rstd, d_grad_residual,
                    d_grad_in, d_grad_weight=None, d_grad_bias=None, p: float = 0.0, seed: int = 0, offset: int = 0,
                    d_offset=None, stream=None):
        """The gradients of AddForward.  d_grad_sum: what reaches d_sum along the residual path (None: nothing).
        d_grad_residual = d_sum's whole gradient, d_grad_in = its dropout with the forward call's random bits; either
        is None if not wanted."""
        dtype = d_sum.dtype
        code = float_code(dtype)
        shape, rows, cols, ss = _matrix(d_sum, "d_sum")
        sg = _like(d_grad_out, shape, dtype, "d_grad_out")
        sx = 0 if d_grad_sum is None else _like(d_grad_sum, shape, dtype, "d_grad_sum")
        sr = 0 if d_grad_residual is None else _like_out(d_grad_residual, shape, dtype, "d_grad_residual")
        si = 0 if d_grad_in is None else _like_out(d_grad_in, shape, dtype, "d_grad_in")
        # (a call of nothing may launch nothing and leave the status word)
        self._call("lcpp_layer_norm_add_backward", temp_storage if rows and cols else None, _stream(stream), code,
                   _weight_code(code, d_weight, d_grad_weight, d_grad_bias), *_temp(temp_storage),
                   d_grad_out.data_ptr(), sg, _ptr(d_grad_sum), sx, d_sum.data_ptr(), ss,
                   _vector(d_weight, cols, "d_weight"), _float_vector(d_mean, rows, "d_mean"),
                   _float_vector(d_rstd, rows, "d_rstd"), p, seed, offset, _counter(d_offset, "d_offset"),
                   _ptr(d_grad_residual), sr, _ptr(d_grad_in), si, _vector(d_grad_weight, cols, "d_grad_weight"),
                   _vector(d_grad_bias, cols, "d_grad_bias"), rows, cols)


class DeviceDropout(_BlockModule):
    """Dropout whose mask is computed from (seed, offset, row, column) wherever it is needed, and never stored."""

    def Forward(self, d_in, d_out, p: float, seed: int, offset: int = 0, d_residual=None, d_offset=None, stream=None):
        """d_out = (kept ? d_in / (1 - p) : 0) [+ d_residual].  p is met to 2^-17.  offset tells the calls of one seed
        apart (a layer's number, a step's); d_offset, a device tensor of one 64-bit integer, is added to it when the
        kernel runs, so a captured graph's replays can differ."""
        shape, dtype, code, rows, cols, si, so = _in_out(d_in, d_out)
        sr = 0 if d_residual is None else _like(d_residual, shape, dtype, "d_residual")
        self._call("lcpp_dropout", None, _stream(stream), code, d_in.data_ptr(), si, _ptr(d_residual), sr,
                   d_out.data_ptr(), so, rows, cols, p, seed, offset, _counter(d_offset, "d_offset"))

    def Backward(self, d_grad_out, d_grad_in, p: float, seed: int, offset: int = 0, d_offset=None, stream=None):
        """The gradient of Forward's d_in, with the forward call's p, seed and offset (d_residual's is d_grad_out itself)."""
        self.Forward(d_grad_out, d_grad_in, p, seed, offset, None, d_offset, stream)


def _sequence_strides(t, shape, dtype, what: str, output: bool = False):
    """(address, row stride, sequence stride) of a tensor of shape (sequences, rows, channels), or with offsets (rows,
    channels)."""
    if t.shape != shape or t.dtype != dtype:
        _unlike(t, shape, dtype, what)
    return _strides(t, shape, what, output)


def _strides(t, shape, what: str, output: bool = False):
    """The same of a tensor that is known to have this shape."""
    if not t.is_cuda:
        _off_gpu(t, what)
    stride = t.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{what}: the channels of a row must be adjacent, got strides {stride}")
    if output and not (stride[-2] >= shape[-1] and (len(shape) == 2 or stride[0] >= stride[1] * shape[1])):
        # no two rows may share memory: in the order of their strides, each dimension steps over the one below it
        span = shape[-1]
        for n, st in sorted(((n, st) for n, st in zip(shape[:-1], stride[:-1]) if n > 1), key=lambda d: d[1]):
            if st < span:
                raise ValueError(f"{what}: the rows of an output must not overlap, got strides {stride}")
            span = st * n
    return (t.data_ptr(), stride[0], 0) if len(shape) == 2 else (t.data_ptr(), stride[1], stride[0])


@functools.lru_cache(maxsize=1024)
def _checkpoint_rows(max_length: int) -> int:
    out = ctypes.c_uint64()
    check(lib().lcpp_recurrence_checkpoint_rows(max_length, ctypes.byref(out)), "lcpp_recurrence_checkpoint_rows")
    return out.value


@functools.lru_cache(maxsize=1024)
def _packed_checkpoint_rows(sequences: int, max_length: int, rows: int) -> int:
    out = ctypes.c_uint64()
    check(lib().lcpp_recurrence_packed_checkpoint_rows(sequences, max_length, rows, ctypes.byref(out)),
          "lcpp_recurrence_packed_checkpoint_rows")
    return out.value


def _checkpoints(t, sizes):
    """The address of the checkpoints of a call of these sizes (DeviceGatedRecurrence._sizes), or None."""
    if t is None:
        return None
    n, max_length, channels, begin, _, rows = sizes
    held = n * _checkpoint_rows(max_length) if begin is None else _packed_checkpoint_rows(n, max_length, rows)
    return _float_vector(t, held * channels, "d_checkpoints")


class DeviceGatedRecurrence(_BlockModule):
    """h_t = a_t h_{t-1} + b_t per channel, with a and b from a gate g and an input x:

        "decay"    a = g, b = x
        "log"      a = exp(g), b = x
        "sigmoid"  a = sigmoid(g), b = (1 - a) x

    Sequences are tensors of shape (sequences, length, channels), or, packed one behind the other, (rows, channels)
    with 32-bit begin and end offsets of each sequence and `max_length`, the longest one's length (a longer one is cut
    there).  States are float32 of shape (sequences, channels)."""

    @staticmethod
    def GetTempStorageBytes(sequences: int, max_length: int, channels: int, rows: int | None = None) -> int:
        """For sequences of max_length each; with `rows`, for packed ones of that many rows in all, which need far less
        where their lengths differ."""
        if rows is None:
            return _query(lib().lcpp_recurrence_temp_bytes, sequences, max_length, channels)
        return _query(lib().lcpp_recurrence_packed_temp_bytes, sequences, max_length, channels, rows)

    @staticmethod
    def GetCheckpointRows(max_length: int) -> int:
        """d_checkpoints has shape (sequences, this, channels), float32."""
        return _checkpoint_rows(max_length)

    @staticmethod
    def GetPackedCheckpointRows(sequences: int, max_length: int, rows: int) -> int:
        """With offsets, d_checkpoints of shape (this, channels) is enough."""
        return _packed_checkpoint_rows(sequences, max_length, rows)

    @staticmethod
    def _gate(gate):
        code = LCPP_GATES.get(gate)
        if code is None:
            raise ValueError(f"unsupported gate {gate!r}: one of {', '.join(LCPP_GATES)}")
        return code

    @staticmethod
    def _sizes(shape, begin, end, max_length):
        """The last arguments of the C calls: sequences, max_length, channels, begin, end, rows."""
        if (begin is None) != (end is None):
            raise ValueError("begin and end offsets go together")
        if begin is None:
            if len(shape) != 3:
                raise ValueError("d_in: shape (sequences, length, channels), or with offsets (rows, channels)")
            if max_length is not None:
                raise ValueError("max_length goes with offsets")
            return (*shape, None, None, 0)
        if len(shape) != 2:
            raise ValueError("d_in: shape (sequences, length, channels), or with offsets (rows, channels)")
        if begin.element_size() != 4 or end.element_size() != 4 or begin.is_floating_point() or end.is_floating_point():
            raise TypeError("offsets must be 32-bit integers")
        if max_length is None:
            raise ValueError("offsets need max_length")
        if begin.numel() != end.numel() or not (begin.is_contiguous() and end.is_contiguous()):
            raise ValueError("begin and end offsets must be contiguous and of one length")
        if not (begin.is_cuda and end.is_cuda):
            _off_gpu(end if begin.is_cuda else begin, "offsets")
        return begin.numel(), max_length, shape[1], begin.data_ptr(), end.data_ptr(), shape[0]

    def Forward(self, temp_storage, d_gate, d_in, d_out, gate: str, d_initial=None, d_final=None, d_checkpoints=None,
                d_begin_offsets=None, d_end_offsets=None, max_length=None, stream=None):
        """d_out = h for every row.  d_initial: the states before the first rows (None: 0); d_final: those after the
        last; d_checkpoints: what Backward needs."""
        shape, dtype, kind = d_in.shape, d_in.dtype, self._gate(gate)
        sizes = self._sizes(shape, d_begin_offsets, d_end_offsets, max_length)
        states = sizes[0] * sizes[2]
        # (a call without states launches nothing and leaves the status word)
        self._call("lcpp_recurrence_forward", temp_storage if states else None, _stream(stream), float_code(dtype), kind,
                   *_temp(temp_storage), *_sequence_strides(d_gate, shape, dtype, "d_gate"),
                   *_strides(d_in, shape, "d_in"), *_sequence_strides(d_out, shape, dtype, "d_out", True),
                   _float_vector(d_initial, states, "d_initial"), _float_vector(d_final, states, "d_final"),
                   _checkpoints(d_checkpoints, sizes), *sizes)

    def Backward(self, temp_storage, d_gate, d_in, d_checkpoints, d_grad_out, d_grad_gate, d_grad_in, gate: str,
                 d_grad_final=None, d_grad_initial=None, d_begin_offsets=None, d_end_offsets=None, max_length=None,
                 stream=None):
        """The gradients of Forward's d_gate, d_in and d_initial from those of d_out and d_final (None: 0)."""
        shape, dtype, kind = d_in.shape, d_in.dtype, self._gate(gate)
        sizes = self._sizes(shape, d_begin_offsets, d_end_offsets, max_length)
        states = sizes[0] * sizes[2]
        # (a call without states launches nothing and leaves the status word)
        self._call("lcpp_recurrence_backward", temp_storage if states else None, _stream(stream), float_code(dtype), kind,
                   *_temp(temp_storage), *_sequence_strides(d_gate, shape, dtype, "d_gate"),
                   *_strides(d_in, shape, "d_in"),
                   _checkpoints(d_checkpoints, sizes),
                   *_sequence_strides(d_grad_out, shape, dtype, "d_grad_out"),
                   *_sequence_strides(d_grad_gate, shape, dtype, "d_grad_gate", True),
                   *_sequence_strides(d_grad_in, shape, dtype, "d_grad_in", True),
                   _float_vector(d_grad_final, states, "d_grad_final"),
                   _float_vector(d_grad_initial, states, "d_grad_initial"), *sizes)

    def Step(self, d_gate, d_in, d_state_in, d_state_out, d_out, gate: str, d_slots=None, stream=None):
        """One token for each of some sequences: d_gate, d_in and d_out of shape (sequences, channels).  The states are
        float32 of shape (slots, channels); d_state_out may be d_state_in.  d_slots: int32, the row of each sequence's
        state, all different; -1 marks padding (out is 0, no state changes).  None: row s for sequence s."""
        shape, dtype, code, rows, cols, sx, so = _in_out(d_in, d_out)
        if len(shape) != 2:
            raise ValueError("d_in: shape (sequences, channels)")
        sg = _like(d_gate, shape, dtype, "d_gate")
        pool = d_state_in.shape
        if len(pool) != 2 or pool[1] != cols or (d_state_out is not d_state_in and d_state_out.shape != pool):
            raise ValueError(f"states: shapes {tuple(pool)} and {tuple(d_state_out.shape)}, expected (slots, {cols})")
        slots = pool[0]
        state = _float_vector(d_state_in, 0, "d_state_in")
        if d_slots is not None:
            if d_slots.element_size() != 4 or d_slots.is_floating_point():
                raise TypeError("d_slots: must be int32")
        elif slots < rows:
            raise ValueError(f"states: {slots} rows for {rows} sequences")
        self._call("lcpp_recurrence_step", None, _stream(stream), code, self._gate(gate), d_gate.data_ptr(), sg,
                   d_in.data_ptr(), sx, state,
                   state if d_state_out is d_state_in else _float_vector(d_state_out, 0, "d_state_out"),
                   _vector(d_slots, rows, "d_slots"), slots, d_out.data_ptr(), so, rows, cols)
