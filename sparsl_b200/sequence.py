"""The sequence operators of :class:`~sparsl_b200.backend.Device`: the short causal
convolution, the selective state space scan and layer norm (``sparsl_dev_*_device``
in include/sparsl_cuda.h, which states their formulas).

Arrays are device arrays of the device's GPU: torch tensors, or objects with a
tensor's ``data_ptr()``, ``shape`` (a tuple), ``stride()``, ``dtype``,
``is_contiguous()``, ``numel()`` and ``element_size()``.  Token arrays are
[tokens, channels] with the channels next to each other; rows may be strided, so
column ranges of a wider array serve as they are.  Every call only enqueues its
work: on ``stream`` (a cudaStream_t, 0 the legacy default stream, or a torch
stream), or, with None, on the device's own, which does not wait for torch's.
Outputs are the caller's arrays; an output must not overlap an input.
"""
from __future__ import annotations

import struct

from . import _lib

_CODES = {}  # dtype -> sparsl dtype code, for those seen
_KINDS = {0: "float32", 1: "float16", 2: "bfloat16", 10: "int32", 11: "uint8"}
_CALLS = {}  # the library's entries, for those called
_NONE = (0, 0)  # no rows


def _code(t, name: str) -> int:
    dt = t.dtype
    c = _CODES.get(dt)
    if c is None:
        c = {"float32": 0, "float16": 1, "bfloat16": 2, "int32": 10, "uint32": 10, "uint8": 11,
             "bool": 11}.get(str(dt).rsplit(".", 1)[-1], -1)
        _CODES[dt] = c
    if c < 0:
        raise TypeError(f"`{name}` has an unsupported dtype: {dt}")
    return c


def _token_code(x) -> int:
    c = _code(x, "x")
    if c > 2:
        raise TypeError("`x` must be float32, float16 or bfloat16")
    return c


def _length(what: str, got, expected):
    from .backend import OpError

    return OpError("Length", f"`{what}` must have shape {list(expected)}, got {list(got)}", what=what,
                   expected=tuple(expected), got=tuple(got))


def _rows(t, name: str, shape, dtype):
    """A token array as (address, row stride in elements)."""
    if t.shape != shape:
        raise _length(name, t.shape, shape)
    if t.dtype != dtype:
        raise TypeError(f"`{name}` must be {dtype}, got {t.dtype}")
    st = t.stride()
    if st[1] != 1 and shape[1] > 1:
        raise TypeError(f"`{name}` must have its channels next to each other")
    return t.data_ptr(), st[0] if shape[0] > 1 else shape[1]


def _runs(t, name: str, tokens: int, groups: int, states: int, dtype):
    """A [tokens, states] or [tokens, groups, states] array as (address, row stride, group stride)."""
    shape = t.shape
    if shape != (tokens, groups, states) and not (groups == 1 and shape == (tokens, states)):
        raise _length(name, shape, (tokens, groups, states))
    if t.dtype != dtype:
        raise TypeError(f"`{name}` must be {dtype}, got {t.dtype}")
    st = t.stride()
    if st[-1] != 1 and states > 1:
        raise TypeError(f"`{name}` must have its states next to each other")
    group = st[1] if len(shape) == 3 and groups > 1 else states
    return t.data_ptr(), st[0] if tokens > 1 else (groups - 1) * group + states, group


def _flat(t, name: str, shape, code: int) -> int:
    """The address of a contiguous array; 0 for None."""
    if t is None:
        return 0
    if t.shape != shape:
        raise _length(name, t.shape, shape)
    if _code(t, name) != code:
        raise TypeError(f"`{name}` must be {_KINDS[code]}, got {t.dtype}")
    if not t.is_contiguous():
        raise TypeError(f"`{name}` must be contiguous")
    return t.data_ptr()


def _params(weight, bias, token_code: int) -> int:
    """Parameters are float32 or of the tokens' type, alike: the dtype code of both."""
    code = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        c = _code(t, name)
        if c not in (0, token_code) or (code is not None and c != code):
            raise TypeError(f"`{name}` must be float32 or have the tokens' dtype, like the other parameters")
        code = c
    return 0 if code is None else code


def _seqs(tokens: int, seq_ptr, n_seq, slots, resume, n_slots: int):
    """The fields of ``sparsl_seqs``."""
    ptr = 0
    if seq_ptr is not None:
        n = seq_ptr.shape[0] - 1
        if n < 0 or (n_seq is not None and n_seq != n):
            raise _length("seq_ptr", seq_ptr.shape, ((n_seq if n_seq is not None else 0) + 1,))
        ptr = _flat(seq_ptr, "seq_ptr", (n + 1,), 10)
    else:
        n = 1 if n_seq is None else int(n_seq)
        if n < 0:
            raise ValueError("`n_seq` must not be negative")
    return (tokens, n, ptr, _flat(slots, "slots", (n,), 10), _flat(resume, "resume", (n,), 11), n_slots)


def _states(arrays, tail, code: int):
    """State arrays [rows, *tail], all with as many rows: (rows, their addresses)."""
    out, rows = [], None
    for name, t in arrays:
        if t is None:
            out.append(0)
            continue
        n = t.shape[0] if len(t.shape) else 0
        if rows is not None and n != rows:
            raise _length(name, t.shape, (rows, *tail))
        rows = n
        out.append(_flat(t, name, (n, *tail), code))
    return rows or 0, out


def _scratch(t):
    """(address, bytes) of a workspace."""
    if t is None:
        return _NONE
    if hasattr(t, "is_contiguous") and not t.is_contiguous():
        raise TypeError("a workspace must be contiguous")
    return t.data_ptr(), t.numel() * t.element_size()


def _stream(stream):
    """A cudaStream_t for the C ABI: a stream's handle or a torch stream's, where 0 is
    CUDA's legacy default stream (NULL would be the device's own there); None is the
    device's own stream."""
    if stream is None:
        return None
    return (stream if isinstance(stream, int) else stream.cuda_stream) or 1  # cudaStreamLegacy


# The argument blocks of include/sparsl_cuda.h, packed in one go (filling
# ctypes structures field by field took longer than the launch).
_CONV = struct.Struct("=6Q3i2I4x4Q4Q4Q2Q2Q2Q")
_SCAN = struct.Struct("=6Q2i4I12Q2Q7Q12Q2Q5Q2Q")
_NORM = struct.Struct("=2Q2i4Q4QfI4Q2Q2Q")


class SequenceOps:
    """Mixed into ``Device``."""

    def _run_sequence(self, fn: str, args: bytes, operation: str, stream):
        call = _CALLS.get(fn)
        if call is None:
            call = _CALLS[fn] = getattr(_lib.load(), fn)
        rc = call(self._h, args, _stream(stream))
        if rc:
            from .backend import _check

            _check(rc, operation)

    # ---- the short causal convolution ----
    @staticmethod
    def _conv_head(x, weight, bias, silu):
        tokens, channels = x.shape
        if len(weight.shape) != 2 or weight.shape[0] != channels:
            raise _length("weight", weight.shape, (channels, "width"))
        width = weight.shape[1]
        code = _token_code(x)
        pc = _params(weight, bias, code)
        head = (code, 1 if pc == 0 else 0, 1 if silu else 0, channels, width)
        params = (_flat(weight, "weight", (channels, width), pc), _flat(bias, "bias", (channels,), pc))
        return tokens, channels, width, code, head, _rows(x, "x", (tokens, channels), x.dtype), params

    def causal_conv_device(self, x, weight, y, *, bias=None, silu: bool = False, seq_ptr=None, n_seq=None, state=None,
                           final_state=None, slots=None, resume=None, stream=None) -> None:
        """y[t, c] = bias[c] + sum_k weight[c, k] x[t - (width - 1) + k, c] within each
        sequence, times its own sigmoid with ``silu``.

        ``x``, ``y``: [tokens, channels]; ``weight``: [channels, width], width
        2 to 4.  The sequences lie one after another: sequence i holds the
        tokens ``seq_ptr[i]`` to ``seq_ptr[i + 1]`` (int32, on the device), or
        ``n_seq`` (default 1) equal ones.  ``state`` / ``final_state``:
        [rows, width - 1, channels] of x's dtype, the inputs before the next
        token; sequence i uses row ``slots[i]`` (int32; a negative one: none)
        or row i, starting from zero without ``state`` or where ``resume[i]``
        is 0.  ``final_state`` may be ``state`` itself."""
        tokens, channels, width, code, head, xr, params = self._conv_head(x, weight, bias, silu)
        yr = _rows(y, "y", (tokens, channels), x.dtype)
        rows, (st, fin) = _states((("state", state), ("final_state", final_state)), (width - 1, channels), code)
        args = _CONV.pack(*_seqs(tokens, seq_ptr, n_seq, slots, resume, rows), *head, *xr, *yr, *params, st, fin,
                          0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        self._run_sequence("sparsl_dev_causal_conv_device", args, "causal_conv", stream)

    @staticmethod
    def causal_conv_backward_workspace(tokens: int, channels: int, width: int) -> int:
        """Bytes of workspace for :meth:`causal_conv_backward_device`."""
        return _lib.load().sparsl_causal_conv_backward_workspace(tokens, channels, width)

    def causal_conv_backward_device(self, dy, x, weight, dx, dweight, workspace, *, bias=None, dbias=None,
                                    silu: bool = False, seq_ptr=None, n_seq=None, state=None, dstate=None,
                                    dfinal_state=None, stream=None) -> None:
        """Gradients of :meth:`causal_conv_device` on the same inputs: ``dx`` like x,
        ``dweight`` [channels, width] and ``dbias`` [channels] in float32,
        overwritten.  Row i of the state arrays is sequence i's; ``dstate``
        receives the gradient of ``state``, ``dfinal_state`` holds that of the
        final state."""
        tokens, channels, width, code, head, xr, params = self._conv_head(x, weight, bias, silu)
        shape = (tokens, channels)
        dyr, dxr = _rows(dy, "dy", shape, x.dtype), _rows(dx, "dx", shape, x.dtype)
        rows, (st, ds, df) = _states((("state", state), ("dstate", dstate), ("dfinal_state", dfinal_state)),
                                     (width - 1, channels), code)
        args = _CONV.pack(*_seqs(tokens, seq_ptr, n_seq, None, None, rows), *head, *xr, 0, 0, *params, st, 0, *dyr, *dxr,
                          _flat(dweight, "dweight", (channels, width), 0), _flat(dbias, "dbias", (channels,), 0), ds, df,
                          *_scratch(workspace))
        self._run_sequence("sparsl_dev_causal_conv_backward_device", args, "causal_conv_backward", stream)

    def causal_conv_step_device(self, x, weight, y, state, *, bias=None, silu: bool = False, slots=None,
                                stream=None) -> None:
        """One token of each sequence: ``x``, ``y`` [sequences, channels]; ``state``
        [rows, width - 1, channels] is updated in place.  Where ``slots[i]`` is
        negative, row i of y stays as it was."""
        tokens, channels, width, code, head, xr, params = self._conv_head(x, weight, bias, silu)
        yr = _rows(y, "y", (tokens, channels), x.dtype)
        rows, (st,) = _states((("state", state),), (width - 1, channels), code)
        args = _CONV.pack(*_seqs(tokens, None, tokens, slots, None, rows), *head, *xr, *yr, *params, 0, st,
                          0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        self._run_sequence("sparsl_dev_causal_conv_step_device", args, "causal_conv_step", stream)

    # ---- the selective scan ----
    @staticmethod
    def _scan_head(x, dt, a, b, c, d, z, dt_bias, softplus):
        tokens, channels = x.shape
        if len(a.shape) != 2 or a.shape[0] != channels:
            raise _length("a", a.shape, (channels, "states"))
        states = a.shape[1]
        groups = b.shape[1] if len(b.shape) == 3 else 1
        code = _token_code(x)
        kind, shape = x.dtype, (tokens, channels)
        br, cr = _runs(b, "b", tokens, groups, states, kind), _runs(c, "c", tokens, groups, states, kind)
        sizes = (code, 1 if softplus else 0, channels, states, groups, 0)
        rows = (*_rows(x, "x", shape, kind), *_rows(dt, "dt", shape, kind),
                *(_NONE if z is None else _rows(z, "z", shape, kind)), br[0], br[1], cr[0], cr[1])
        params = (br[2], cr[2], _flat(a, "a", (channels, states), 0), _flat(d, "d", (channels,), 0),
                  _flat(dt_bias, "dt_bias", (channels,), 0))
        return tokens, channels, states, groups, sizes, rows, params

    @staticmethod
    def selective_scan_workspace(tokens: int, channels: int, states: int, n_seq: int = 1, groups: int = 1) -> int:
        """Bytes of workspace for :meth:`selective_scan_device` (0: none is needed)."""
        return _lib.load().sparsl_selective_scan_workspace(tokens, channels, states, n_seq, groups)

    @staticmethod
    def selective_scan_checkpoints(tokens: int, channels: int, states: int) -> int:
        """Bytes that a forward call keeps for its backward call."""
        return _lib.load().sparsl_selective_scan_checkpoints(tokens, channels, states)

    @staticmethod
    def selective_scan_backward_workspace(tokens: int, channels: int, states: int, n_seq: int = 1, groups: int = 1) -> int:
        """Bytes of workspace for :meth:`selective_scan_backward_device`."""
        return _lib.load().sparsl_selective_scan_backward_workspace(tokens, channels, states, n_seq, groups)

    def selective_scan_device(self, x, dt, a, b, c, y, workspace=None, *, d=None, z=None, dt_bias=None,
                              softplus: bool = False, seq_ptr=None, n_seq=None, state=None, final_state=None, slots=None,
                              resume=None, checkpoints=None, stream=None) -> None:
        """h[c, n] <- exp(s a[c, n]) h[c, n] + s b[n] x with s = dt + dt_bias (through
        log(1 + e^s) with ``softplus``), y = sum_n c[n] h[c, n] + d x, times
        z sigmoid(z) with ``z``; token by token within each sequence.

        ``x``, ``dt``, ``z``, ``y``: [tokens, channels]; ``a``: [channels,
        states], states 1 to 64; ``b``, ``c``: [tokens, states], or [tokens,
        groups, states] where channels / groups neighbouring channels share a
        run; ``a``, ``d``, ``dt_bias`` are float32.  Sequences, slots and
        resume as in :meth:`causal_conv_device`; ``state`` / ``final_state``:
        [rows, channels, states] float32.  ``checkpoints`` keeps what
        :meth:`selective_scan_backward_device` needs."""
        tokens, channels, states, groups, sizes, rows, params = self._scan_head(x, dt, a, b, c, d, z, dt_bias, softplus)
        n, (st, fin) = _states((("state", state), ("final_state", final_state)), (channels, states), 0)
        args = _SCAN.pack(*_seqs(tokens, seq_ptr, n_seq, slots, resume, n), *sizes, *rows,
                          *_rows(y, "y", (tokens, channels), x.dtype), *params, st, fin, *_scratch(checkpoints),
                          0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, *_scratch(workspace))
        self._run_sequence("sparsl_dev_selective_scan_device", args, "selective_scan", stream)

    def selective_scan_backward_device(self, dy, x, dt, a, b, c, checkpoints, dx, ddt, da, db, dc, workspace, *, d=None,
                                       dd=None, z=None, dz=None, dt_bias=None, ddt_bias=None, softplus: bool = False,
                                       seq_ptr=None, n_seq=None, state=None, dstate=None, dfinal_state=None,
                                       stream=None) -> None:
        """Gradients of :meth:`selective_scan_device` on the same inputs, with the
        ``checkpoints`` it wrote: ``dx``, ``ddt``, ``dz`` like x, ``db``,
        ``dc`` like b and c, ``da``, ``dd``, ``ddt_bias`` float32, all
        overwritten.  ``dz`` goes with ``z``.  Row i of the state arrays is
        sequence i's; ``dstate`` receives the gradient of ``state``,
        ``dfinal_state`` holds that of the final state."""
        tokens, channels, states, groups, sizes, rows, params = self._scan_head(x, dt, a, b, c, d, z, dt_bias, softplus)
        shape, kind = (tokens, channels), x.dtype
        if (z is None) != (dz is None):
            raise TypeError("`dz` goes with `z`")
        dbr, dcr = _runs(db, "db", tokens, groups, states, kind), _runs(dc, "dc", tokens, groups, states, kind)
        n, (st, ds, df) = _states((("state", state), ("dstate", dstate), ("dfinal_state", dfinal_state)),
                                  (channels, states), 0)
        args = _SCAN.pack(*_seqs(tokens, seq_ptr, n_seq, None, None, n), *sizes, *rows, 0, 0, *params, st, 0,
                          *_scratch(checkpoints), *_rows(dy, "dy", shape, kind), *_rows(dx, "dx", shape, kind),
                          *_rows(ddt, "ddt", shape, kind), *(_NONE if dz is None else _rows(dz, "dz", shape, kind)),
                          dbr[0], dbr[1], dcr[0], dcr[1], dbr[2], dcr[2], _flat(da, "da", (channels, states), 0),
                          _flat(dd, "dd", (channels,), 0), _flat(ddt_bias, "ddt_bias", (channels,), 0), ds, df,
                          *_scratch(workspace))
        self._run_sequence("sparsl_dev_selective_scan_backward_device", args, "selective_scan_backward", stream)

    def selective_scan_step_device(self, x, dt, a, b, c, y, state, *, d=None, z=None, dt_bias=None,
                                   softplus: bool = False, slots=None, stream=None) -> None:
        """One token of each sequence: the token arrays have a row per sequence;
        ``state`` [rows, channels, states] is updated in place.  Where
        ``slots[i]`` is negative, row i of y stays as it was."""
        tokens, channels, states, groups, sizes, rows, params = self._scan_head(x, dt, a, b, c, d, z, dt_bias, softplus)
        n, (st,) = _states((("state", state),), (channels, states), 0)
        args = _SCAN.pack(*_seqs(tokens, None, tokens, slots, None, n), *sizes, *rows,
                          *_rows(y, "y", (tokens, channels), x.dtype), *params, 0, st,
                          0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        self._run_sequence("sparsl_dev_selective_scan_step_device", args, "selective_scan_step", stream)

    # ---- layer norm ----
    def layer_norm_device(self, x, y, *, weight=None, bias=None, eps: float = 1e-5, mean=None, rstd=None,
                          stream=None) -> None:
        """y = (x - mean) rstd weight + bias over each row of ``x`` [rows, channels];
        ``mean`` and ``rstd`` [rows] float32 keep what
        :meth:`layer_norm_backward_device` needs."""
        rows, channels = shape = x.shape
        code = _token_code(x)
        pc = _params(weight, bias, code)
        args = _NORM.pack(rows, channels, code, 1 if pc == 0 else 0, *_rows(x, "x", shape, x.dtype),
                          *_rows(y, "y", shape, x.dtype), _flat(weight, "weight", (channels,), pc),
                          _flat(bias, "bias", (channels,), pc), _flat(mean, "mean", (rows,), 0),
                          _flat(rstd, "rstd", (rows,), 0), eps, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        self._run_sequence("sparsl_dev_layer_norm_device", args, "layer_norm", stream)

    @staticmethod
    def layer_norm_backward_workspace(rows: int, channels: int) -> int:
        """Bytes of workspace for :meth:`layer_norm_backward_device`."""
        return _lib.load().sparsl_layer_norm_backward_workspace(rows, channels)

    def layer_norm_backward_device(self, dy, x, mean, rstd, dx, workspace, *, weight=None, dweight=None, dbias=None,
                                   stream=None) -> None:
        """Gradients of :meth:`layer_norm_device`: ``dx`` like x, ``dweight`` and
        ``dbias`` [channels] float32, overwritten."""
        rows, channels = shape = x.shape
        code = _token_code(x)
        pc = _params(weight, None, code)
        args = _NORM.pack(rows, channels, code, 1 if pc == 0 else 0, *_rows(x, "x", shape, x.dtype), 0, 0,
                          _flat(weight, "weight", (channels,), pc), 0, _flat(mean, "mean", (rows,), 0),
                          _flat(rstd, "rstd", (rows,), 0), 0.0, 0, *_rows(dy, "dy", shape, x.dtype),
                          *_rows(dx, "dx", shape, x.dtype), _flat(dweight, "dweight", (channels,), 0),
                          _flat(dbias, "dbias", (channels,), 0), *_scratch(workspace))
        self._run_sequence("sparsl_dev_layer_norm_backward_device", args, "layer_norm_backward", stream)
