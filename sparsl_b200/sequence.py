"""The sequence operators of :class:`~sparsl_b200.backend.Device`: the short causal
convolution, the selective state space scan and layer norm (``sparsl_dev_*_device``
in include/sparsl_cuda.h, which states their formulas).

Arrays are device arrays of the device's GPU: torch tensors, or objects with
``data_ptr()``, ``shape``, ``stride()`` and ``dtype``.  Token arrays are
[tokens, channels] with the channels next to each other; rows may be strided, so
column ranges of a wider array serve as they are.  Every call only enqueues its
work: on ``stream`` (a cudaStream_t or a torch stream), or on the device's own.
Outputs are the caller's arrays; an output must not overlap an input.
"""
from __future__ import annotations

from ctypes import byref

from . import _lib

_CODES = {}  # dtype -> sparsl dtype code, for those seen


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


def _want(t, name: str, code: int, kind: str):
    if _code(t, name) != code:
        raise TypeError(f"`{name}` must be {kind}, got {t.dtype}")


_KINDS = {0: "float32", 1: "float16", 2: "bfloat16", 10: "int32", 11: "uint8"}


def _length(what: str, got, expected):
    from .backend import OpError

    return OpError("Length", f"`{what}` must have shape {list(expected)}, got {list(got)}", what=what,
                   expected=tuple(expected), got=tuple(got))


def _fill_rows(to, t, name: str, shape, code: int):
    """A token array into a ``sparsl_rows``."""
    if tuple(t.shape) != shape:
        raise _length(name, t.shape, shape)
    _want(t, name, code, _KINDS[code])
    st = t.stride()
    if st[1] != 1 and shape[1] > 1:
        raise TypeError(f"`{name}` must have its channels next to each other")
    to.p = t.data_ptr()
    to.stride = st[0] if shape[0] > 1 else shape[1]


def _fill_runs(to, t, name: str, tokens: int, groups: int, states: int, code: int) -> int:
    """A [tokens, states] or [tokens, groups, states] array; returns the group stride."""
    shape = tuple(t.shape)
    if shape != (tokens, groups, states) and not (groups == 1 and shape == (tokens, states)):
        raise _length(name, shape, (tokens, groups, states))
    _want(t, name, code, _KINDS[code])
    st = t.stride()
    if st[-1] != 1 and states > 1:
        raise TypeError(f"`{name}` must have its states next to each other")
    group = st[1] if len(shape) == 3 and groups > 1 else states
    to.p = t.data_ptr()
    to.stride = st[0] if tokens > 1 else (groups - 1) * group + states
    return group


def _flat(t, name: str, shape, code: int):
    """The address of a contiguous array."""
    if tuple(t.shape) != shape:
        raise _length(name, t.shape, shape)
    _want(t, name, code, _KINDS[code])
    if not t.is_contiguous():
        raise TypeError(f"`{name}` must be contiguous")
    return t.data_ptr()


def _params(named, shapes, token_code: int) -> int:
    """Parameters are float32 or of the tokens' type, all alike: 1 for float32."""
    f32 = None
    for (name, t), shape in zip(named, shapes):
        if t is None:
            continue
        c = _code(t, name)
        if c not in (0, token_code) or (f32 is not None and f32 != (c == 0)):
            raise TypeError(f"`{name}` must be float32 or have the tokens' dtype, like the other parameters")
        f32 = c == 0
    return 1 if f32 or f32 is None else 0


def _fill_seqs(s, tokens: int, seq_ptr, n_seq, slots=None, resume=None):
    s.tokens = tokens
    if seq_ptr is not None:
        n = seq_ptr.shape[0] - 1
        if n < 0 or (n_seq is not None and n_seq != n):
            raise _length("seq_ptr", seq_ptr.shape, ((n_seq if n_seq is not None else 0) + 1,))
        s.seq_ptr = _flat(seq_ptr, "seq_ptr", (n + 1,), 10)
    else:
        n = 1 if n_seq is None else int(n_seq)
        if n < 0:
            raise ValueError("`n_seq` must not be negative")
    s.n_seq = n
    if slots is not None:
        s.slots = _flat(slots, "slots", (n,), 10)
    if resume is not None:
        s.resume = _flat(resume, "resume", (n,), 11)
    return n


def _fill_states(s, arrays, tail, code: int):
    """State arrays [rows, *tail], all with as many rows; their addresses by name."""
    out, rows = [], None
    for name, t in arrays:
        if t is None:
            out.append(None)
            continue
        n = t.shape[0] if len(t.shape) else 0
        if rows is not None and n != rows:
            raise _length(name, t.shape, (rows, *tail))
        rows = n
        out.append(_flat(t, name, (n, *tail), code))
    s.n_slots = rows or 0
    return out


def _scratch(t):
    """(address, bytes) of a workspace."""
    if t is None:
        return None, 0
    if hasattr(t, "is_contiguous") and not t.is_contiguous():
        raise TypeError("a workspace must be contiguous")
    return t.data_ptr(), t.numel() * t.element_size()


def _stream(stream):
    """A cudaStream_t for the C ABI.  A torch stream's handle, where 0 means CUDA's
    legacy default stream; None is the device's own stream."""
    if stream is None or isinstance(stream, int):
        return stream
    return stream.cuda_stream or 1  # cudaStreamLegacy


class SequenceOps:
    """Mixed into ``Device``."""

    def _run_sequence(self, fn: str, args, operation: str, stream):
        rc = getattr(_lib.load(), fn)(self._h, byref(args), _stream(stream))
        if rc:
            from .backend import _check

            _check(rc, operation)

    # ---- the short causal convolution ----
    def _conv_args(self, x, weight, bias, silu):
        tokens, channels = x.shape
        if len(weight.shape) != 2 or weight.shape[0] != channels:
            raise _length("weight", weight.shape, (channels, "width"))
        width = weight.shape[1]
        a = _lib.ConvArgs()
        code = _code(x, "x")
        if code > 2:
            raise TypeError("`x` must be float32, float16 or bfloat16")
        a.dtype, a.silu, a.channels, a.width = code, int(bool(silu)), channels, width
        a.params_f32 = _params((("weight", weight), ("bias", bias)), ((channels, width), (channels,)), code)
        _fill_rows(a.x, x, "x", (tokens, channels), code)
        pc = 0 if a.params_f32 else code
        a.weight = _flat(weight, "weight", (channels, width), pc)
        if bias is not None:
            a.bias = _flat(bias, "bias", (channels,), pc)
        return a, tokens, channels, width, code

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
        a, tokens, channels, width, code = self._conv_args(x, weight, bias, silu)
        _fill_rows(a.y, y, "y", (tokens, channels), code)
        _fill_seqs(a.seqs, tokens, seq_ptr, n_seq, slots, resume)
        a.state, a.final_state = _fill_states(a.seqs, (("state", state), ("final_state", final_state)),
                                              (width - 1, channels), code)
        self._run_sequence("sparsl_dev_causal_conv_device", a, "causal_conv", stream)

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
        a, tokens, channels, width, code = self._conv_args(x, weight, bias, silu)
        _fill_rows(a.dy, dy, "dy", (tokens, channels), code)
        _fill_rows(a.dx, dx, "dx", (tokens, channels), code)
        a.dweight = _flat(dweight, "dweight", (channels, width), 0)
        if dbias is not None:
            a.dbias = _flat(dbias, "dbias", (channels,), 0)
        _fill_seqs(a.seqs, tokens, seq_ptr, n_seq)
        a.state, a.dstate, a.dfinal_state = _fill_states(
            a.seqs, (("state", state), ("dstate", dstate), ("dfinal_state", dfinal_state)), (width - 1, channels), code)
        a.workspace, a.workspace_bytes = _scratch(workspace)
        self._run_sequence("sparsl_dev_causal_conv_backward_device", a, "causal_conv_backward", stream)

    def causal_conv_step_device(self, x, weight, y, state, *, bias=None, silu: bool = False, slots=None,
                                stream=None) -> None:
        """One token of each sequence: ``x``, ``y`` [sequences, channels]; ``state``
        [rows, width - 1, channels] is updated in place.  Where ``slots[i]`` is
        negative, row i of y stays as it was."""
        a, tokens, channels, width, code = self._conv_args(x, weight, bias, silu)
        _fill_rows(a.y, y, "y", (tokens, channels), code)
        _fill_seqs(a.seqs, tokens, None, tokens, slots)
        (a.final_state,) = _fill_states(a.seqs, (("state", state),), (width - 1, channels), code)
        self._run_sequence("sparsl_dev_causal_conv_step_device", a, "causal_conv_step", stream)

    # ---- the selective scan ----
    def _scan_args(self, x, dt, a, b, c, d, z, dt_bias, softplus):
        tokens, channels = x.shape
        if len(a.shape) != 2 or a.shape[0] != channels:
            raise _length("a", a.shape, (channels, "states"))
        states = a.shape[1]
        groups = b.shape[1] if len(b.shape) == 3 else 1
        code = _code(x, "x")
        if code > 2:
            raise TypeError("`x` must be float32, float16 or bfloat16")
        k = _lib.ScanArgs()
        k.dtype, k.softplus, k.channels, k.states, k.groups = code, int(bool(softplus)), channels, states, groups
        shape = (tokens, channels)
        _fill_rows(k.x, x, "x", shape, code)
        _fill_rows(k.dt, dt, "dt", shape, code)
        if z is not None:
            _fill_rows(k.z, z, "z", shape, code)
        k.b_group = _fill_runs(k.b, b, "b", tokens, groups, states, code)
        k.c_group = _fill_runs(k.c, c, "c", tokens, groups, states, code)
        k.a = _flat(a, "a", (channels, states), 0)
        if d is not None:
            k.d = _flat(d, "d", (channels,), 0)
        if dt_bias is not None:
            k.dt_bias = _flat(dt_bias, "dt_bias", (channels,), 0)
        return k, tokens, channels, states, groups, code

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
        k, tokens, channels, states, groups, code = self._scan_args(x, dt, a, b, c, d, z, dt_bias, softplus)
        _fill_rows(k.y, y, "y", (tokens, channels), code)
        _fill_seqs(k.seqs, tokens, seq_ptr, n_seq, slots, resume)
        k.state, k.final_state = _fill_states(k.seqs, (("state", state), ("final_state", final_state)),
                                              (channels, states), 0)
        if checkpoints is not None:
            k.checkpoints, k.checkpoint_bytes = _scratch(checkpoints)
        k.workspace, k.workspace_bytes = _scratch(workspace)
        self._run_sequence("sparsl_dev_selective_scan_device", k, "selective_scan", stream)

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
        k, tokens, channels, states, groups, code = self._scan_args(x, dt, a, b, c, d, z, dt_bias, softplus)
        shape = (tokens, channels)
        _fill_rows(k.dy, dy, "dy", shape, code)
        _fill_rows(k.dx, dx, "dx", shape, code)
        _fill_rows(k.ddt, ddt, "ddt", shape, code)
        if (z is None) != (dz is None):
            raise TypeError("`dz` goes with `z`")
        if dz is not None:
            _fill_rows(k.dz, dz, "dz", shape, code)
        k.db_group = _fill_runs(k.db, db, "db", tokens, groups, states, code)
        k.dc_group = _fill_runs(k.dc, dc, "dc", tokens, groups, states, code)
        k.da = _flat(da, "da", (channels, states), 0)
        if dd is not None:
            k.dd = _flat(dd, "dd", (channels,), 0)
        if ddt_bias is not None:
            k.ddt_bias = _flat(ddt_bias, "ddt_bias", (channels,), 0)
        _fill_seqs(k.seqs, tokens, seq_ptr, n_seq)
        k.state, k.dstate, k.dfinal_state = _fill_states(
            k.seqs, (("state", state), ("dstate", dstate), ("dfinal_state", dfinal_state)), (channels, states), 0)
        k.checkpoints, k.checkpoint_bytes = _scratch(checkpoints)
        k.workspace, k.workspace_bytes = _scratch(workspace)
        self._run_sequence("sparsl_dev_selective_scan_backward_device", k, "selective_scan_backward", stream)

    def selective_scan_step_device(self, x, dt, a, b, c, y, state, *, d=None, z=None, dt_bias=None,
                                   softplus: bool = False, slots=None, stream=None) -> None:
        """One token of each sequence: the token arrays have a row per sequence;
        ``state`` [rows, channels, states] is updated in place.  Where
        ``slots[i]`` is negative, row i of y stays as it was."""
        k, tokens, channels, states, groups, code = self._scan_args(x, dt, a, b, c, d, z, dt_bias, softplus)
        _fill_rows(k.y, y, "y", (tokens, channels), code)
        _fill_seqs(k.seqs, tokens, None, tokens, slots)
        (k.final_state,) = _fill_states(k.seqs, (("state", state),), (channels, states), 0)
        self._run_sequence("sparsl_dev_selective_scan_step_device", k, "selective_scan_step", stream)

    # ---- layer norm ----
    def _norm_args(self, x, weight, bias):
        rows, channels = x.shape
        code = _code(x, "x")
        if code > 2:
            raise TypeError("`x` must be float32, float16 or bfloat16")
        a = _lib.NormArgs()
        a.rows, a.channels, a.dtype = rows, channels, code
        a.params_f32 = _params((("weight", weight), ("bias", bias)), ((channels,), (channels,)), code)
        pc = 0 if a.params_f32 else code
        _fill_rows(a.x, x, "x", (rows, channels), code)
        if weight is not None:
            a.weight = _flat(weight, "weight", (channels,), pc)
        if bias is not None:
            a.bias = _flat(bias, "bias", (channels,), pc)
        return a, rows, channels, code

    def layer_norm_device(self, x, y, *, weight=None, bias=None, eps: float = 1e-5, mean=None, rstd=None,
                          stream=None) -> None:
        """y = (x - mean) rstd weight + bias over each row of ``x`` [rows, channels];
        ``mean`` and ``rstd`` [rows] float32 keep what
        :meth:`layer_norm_backward_device` needs."""
        a, rows, channels, code = self._norm_args(x, weight, bias)
        _fill_rows(a.y, y, "y", (rows, channels), code)
        a.eps = eps
        if mean is not None:
            a.mean = _flat(mean, "mean", (rows,), 0)
        if rstd is not None:
            a.rstd = _flat(rstd, "rstd", (rows,), 0)
        self._run_sequence("sparsl_dev_layer_norm_device", a, "layer_norm", stream)

    @staticmethod
    def layer_norm_backward_workspace(rows: int, channels: int) -> int:
        """Bytes of workspace for :meth:`layer_norm_backward_device`."""
        return _lib.load().sparsl_layer_norm_backward_workspace(rows, channels)

    def layer_norm_backward_device(self, dy, x, mean, rstd, dx, workspace, *, weight=None, dweight=None, dbias=None,
                                   stream=None) -> None:
        """Gradients of :meth:`layer_norm_device`: ``dx`` like x, ``dweight`` and
        ``dbias`` [channels] float32, overwritten."""
        a, rows, channels, code = self._norm_args(x, weight, None)
        _fill_rows(a.dy, dy, "dy", (rows, channels), code)
        _fill_rows(a.dx, dx, "dx", (rows, channels), code)
        a.mean = _flat(mean, "mean", (rows,), 0)
        a.rstd = _flat(rstd, "rstd", (rows,), 0)
        if dweight is not None:
            a.dweight = _flat(dweight, "dweight", (channels,), 0)
        if dbias is not None:
            a.dbias = _flat(dbias, "dbias", (channels,), 0)
        a.workspace, a.workspace_bytes = _scratch(workspace)
        self._run_sequence("sparsl_dev_layer_norm_backward_device", a, "layer_norm_backward", stream)
